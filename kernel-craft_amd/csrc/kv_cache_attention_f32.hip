// kv_cache_attention_f32.hip -- the matrix-core kernel of kv_attention_mfma.hpp for fp32 queries.
#include "kv_attention_mfma.hpp"

void kc::kv::launch_mfma_f32(const Attention& p, bool fp8, dim3 grid, hipStream_t stream) {
    if (fp8) launch<false, true, 16>(p, grid, stream);
    else launch<false, false, 32>(p, grid, stream);
}
