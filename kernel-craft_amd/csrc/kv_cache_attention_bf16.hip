// kv_cache_attention_bf16.hip -- the matrix-core kernel of kv_attention_mfma.hpp for bf16 queries.
#include "kv_attention_mfma.hpp"

void kc::kv::launch_mfma_bf16(const Attention& p, bool fp8, dim3 grid, hipStream_t stream) {
    if (fp8) launch<true, true, 16>(p, grid, stream);
    else launch<true, false, 32>(p, grid, stream);
}
