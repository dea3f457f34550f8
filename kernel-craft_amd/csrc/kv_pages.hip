// kv_pages.hip -- pages of the paged key/value cache for the requests of a step on
// gfx950: block tables, positions and slots from request lengths, and the pages of
// finished sequences back onto the stack of free ones.
//
// With l = length, n = new tokens, P = page size, e = rows of the packed batch up to and
// with the request:
//   held   = ceil(l / P),  fits = l + n <= max_pages P and e <= total_new
//   ask    = fits ? ceil((l + n) / P) - held : 0
//   served = fits and (ask == 0 or sum of ask up to and with the request <= free)
// and page held + j of a request is free_pages[free - 1 - (asks before it) - j].
//
// Bound by latency: a few bytes per request and 12 per token.  One launch: every
// workgroup scans all requests by itself (three block scans, 8 bytes a request from the
// cache), so that none waits for another, and takes as many rows of the batch as it has
// threads.  256 requests of a token each 5.0 us, 40 chunks of 16000 tokens together 5.3;
// releasing half of 64 or of 1000 requests 3.5 and 5.1, where an empty launch takes 1.5.
#include <algorithm>

#include "kc_common.hpp"

namespace {

using kc::kWave;

// Threads of a workgroup: 256 where that is one request each, else 1024 (a scan over 16
// waves and 1024 LDS entries: 1.3 us more for 256 requests).
constexpr int kFew = 256, kMany = 1024;

constexpr int kMaxRequests = 1 << 20;  // every workgroup goes over all of them

struct Pages {
    int32_t* table;
    int32_t* stack;
    const int32_t* count;
    int64_t max_pages, capacity;  // of a table row, of the stack
    int page, seqs;
    int32_t *lens_out, *count_out;
    const int32_t* lens;
};

// Sum of v over the threads before this one; `total` over all.  `part` is LDS of a sum per wave.
template <int kThreads>
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* part, int64_t& total) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    int64_t up = v;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
        const int64_t below = __shfl_up(up, off, kWave);
        if (lane >= off) up += below;
    }
    __syncthreads();  // the sums of the last scan have been read
    if (lane == kWave - 1) part[wave] = up;
    __syncthreads();
    int64_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kThreads / kWave; ++w) {
        if (w < wave) before += part[w];
        total += part[w];
    }
    return before + up - v;
}

// The last thread whose first item is at most `at` (starts ascend from 0).
template <int kThreads>
__device__ __forceinline__ int last_at_most(const int64_t* starts, int64_t at) {
    int lo = 0;
#pragma unroll
    for (int step = kThreads / 2; step > 0; step >>= 1)
        if (starts[lo + step] <= at) lo += step;
    return lo;
}

__device__ __forceinline__ int32_t saturate(int64_t v) {
    return static_cast<int32_t>(v < INT32_MAX ? v : INT32_MAX);
}

// Pages of `tokens` < 2^32, by a division in 32 bits.
__device__ __forceinline__ int64_t pages_of(int64_t tokens, int page) {
    const uint32_t t = static_cast<uint32_t>(tokens), n = static_cast<uint32_t>(page), q = t / n;
    return int64_t{q} + (q * n != t);
}

// What a request asks for: its length, new tokens, whether it fits and its pages.
struct Request {
    int64_t len, fresh, held, ask;
    bool fits;
};

__device__ __forceinline__ Request request(const Pages& p, const int32_t* fresh, int64_t rows, int b, int64_t before) {
    Request r;
    r.len = max(p.lens[b], 0);
    r.fresh = max(fresh[b], 0);
    const int64_t after = r.len + r.fresh, room = p.max_pages * p.page;
    r.held = pages_of(r.len, p.page);
    r.fits = after <= room && after <= INT32_MAX && before + r.fresh <= rows;
    r.ask = r.fits ? pages_of(after, p.page) - r.held : 0;
    return r;
}

template <int kThreads>
__global__ __launch_bounds__(kThreads) void extend_kernel(const Pages p, const int32_t* __restrict__ fresh,
                                                          int64_t rows, int32_t* cu_new, int32_t* cu_after,
                                                          int32_t* positions, int64_t* slots) {
    __shared__ int64_t part[kThreads / kWave], first_row[kThreads], first_ask[kThreads];
    __shared__ unsigned long long used;
    const int tid = threadIdx.x, each = (p.seqs + kThreads - 1) / kThreads;
    const int b0 = min(tid * each, p.seqs), b1 = min(b0 + each, p.seqs);
    const int64_t free = min(static_cast<int64_t>(max(p.count[0], 0)), p.capacity);
    if (tid == 0) used = 0;

    int64_t sum = 0, total_rows, total;
    for (int b = b0; b < b1; ++b) sum += max(fresh[b], 0);
    const int64_t row0 = block_scan<kThreads>(sum, part, total_rows);
    sum = 0;
    for (int64_t b = b0, at = row0; b < b1; ++b) {
        const Request r = request(p, fresh, rows, b, at);
        at += r.fresh;
        sum += r.ask;
    }
    const int64_t ask0 = block_scan<kThreads>(sum, part, total);
    first_row[tid] = row0;
    first_ask[tid] = ask0;
    if (blockIdx.x == 0) {  // what there is one of for each request
        int64_t after = 0;
        auto walk = [&](auto&& each_request) {
            int64_t at = row0, ask = ask0;
            for (int b = b0; b < b1; ++b) {
                const Request r = request(p, fresh, rows, b, at);
                const bool served = r.fits && (r.ask == 0 || ask + r.ask <= free);
                each_request(b, at, served ? r.len + r.fresh : r.len, served && r.ask > 0 ? ask + r.ask : 0);
                at += r.fresh;
                ask += r.ask;
            }
        };
        int64_t most = 0;
        walk([&](int, int64_t, int64_t len, int64_t upto) {
            after += len;
            most = max(most, upto);
        });
        int64_t cu = block_scan<kThreads>(after, part, total);
        if (most > 0) atomicMax(&used, static_cast<unsigned long long>(most));
        walk([&](int b, int64_t at, int64_t len, int64_t) {
            p.lens_out[b] = static_cast<int32_t>(len);
            cu_new[b] = saturate(at);
            cu_after[b] = saturate(cu);
            cu += len;
        });
        if (tid == 0) {
            cu_new[p.seqs] = saturate(total_rows);
            cu_after[p.seqs] = saturate(total);
        }
    }
    __syncthreads();
    if (blockIdx.x == 0 && tid == 0) p.count_out[0] = static_cast<int32_t>(free - static_cast<int64_t>(used));

    const int64_t row = static_cast<int64_t>(blockIdx.x) * kThreads + tid;
    if (row >= rows) return;
    int32_t pos = -1;
    int64_t slot = -1;
    if (row < total_rows) {
        const int t = last_at_most<kThreads>(first_row, row);
        int64_t at = first_row[t], ask = first_ask[t];
        int b = t * each;
        Request r = request(p, fresh, rows, b, at);
        while (row >= at + r.fresh) {  // the thread's other requests: rows < total_rows ends it
            at += r.fresh;
            ask += r.ask;
            r = request(p, fresh, rows, ++b, at);
        }
        if (r.fits && (r.ask == 0 || ask + r.ask <= free)) {
            pos = static_cast<int32_t>(r.len + (row - at));
            const int64_t column = pos / p.page;
            const int off = pos - static_cast<int>(column) * p.page;
            int32_t* entry = p.table + b * p.max_pages + column;
            int32_t page;
            if (column < r.held) {
                page = *entry;
            } else {
                page = p.stack[free - 1 - ask - (column - r.held)];
                if (off == 0) *entry = page;  // a new page begins with a new token
            }
            slot = page < 0 ? -1 : static_cast<int64_t>(page) * p.page + off;
        }
    }
    positions[row] = pos;
    slots[row] = slot;
}

template <int kThreads>
__global__ __launch_bounds__(kThreads) void release_kernel(const Pages p, const uint8_t* __restrict__ finished) {
    __shared__ int64_t part[kThreads / kWave], first[kThreads];
    const int tid = threadIdx.x, each = (p.seqs + kThreads - 1) / kThreads;
    const int b0 = min(tid * each, p.seqs), b1 = min(b0 + each, p.seqs);
    const int64_t free = min(static_cast<int64_t>(max(p.count[0], 0)), p.capacity);
    auto pages = [&](int b) {
        return finished[b] ? min(pages_of(max(p.lens[b], 0), p.page), p.max_pages) : int64_t{0};
    };
    int64_t sum = 0, total;
    for (int b = b0; b < b1; ++b) sum += pages(b);
    first[tid] = block_scan<kThreads>(sum, part, total);
    const int64_t back = min(total, p.capacity - free);
    if (blockIdx.x == 0) {
        for (int b = b0; b < b1; ++b) p.lens_out[b] = finished[b] ? 0 : max(p.lens[b], 0);
        if (tid == 0) p.count_out[0] = static_cast<int32_t>(free + back);
    }
    __syncthreads();
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + tid; i < back;
         i += static_cast<int64_t>(gridDim.x) * kThreads) {
        const int t = last_at_most<kThreads>(first, i);
        int64_t at = first[t];
        int b = t * each;
        for (int64_t n = pages(b); i >= at + n; n = pages(++b)) at += n;
        p.stack[free + i] = p.table[b * p.max_pages + (i - at)];
    }
}

int check(const char* fn, const kc_kv_pages* pages, const int32_t* lens, const int32_t* lens_out,
          const int32_t* count_out) {
    if (!pages) return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: null pages", fn);
    if (pages->seqs < 0 || pages->max_pages < 0 || pages->num_pages < 0 || pages->page_size <= 0)
        return kc::set_error(KC_ERR_INVALID_ARGUMENT,
                             "%s: bad shape seqs=%d max_pages=%lld num_pages=%lld page_size=%d", fn, pages->seqs,
                             (long long)pages->max_pages, (long long)pages->num_pages, pages->page_size);
    if (pages->max_pages > INT32_MAX || pages->num_pages > INT32_MAX || pages->seqs > kMaxRequests)
        return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: seqs=%d max_pages=%lld num_pages=%lld too large", fn,
                             pages->seqs, (long long)pages->max_pages, (long long)pages->num_pages);
    const bool table = pages->seqs > 0 && pages->max_pages > 0;
    if (!pages->free_count || !count_out || (table && !pages->block_table) ||
        (pages->num_pages > 0 && !pages->free_pages) || (pages->seqs > 0 && (!lens || !lens_out)))
        return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: null device pointer", fn);
    return KC_SUCCESS;
}

Pages args(const kc_kv_pages* pages, const int32_t* lens, int32_t* lens_out, int32_t* count_out) {
    return Pages{pages->block_table, pages->free_pages, pages->free_count, pages->max_pages, pages->num_pages,
                 pages->page_size,   pages->seqs,       lens_out,          count_out,        lens};
}

}  // namespace

extern "C" int kc_kv_cache_extend(const kc_kv_pages* pages, const int32_t* d_seq_lens, const int32_t* d_new_lens,
                                  int64_t total_new, int32_t* d_seq_lens_out, int32_t* d_free_count_out,
                                  int32_t* d_cu_new, int32_t* d_cu_seqlens, int32_t* d_positions, int64_t* d_slots,
                                  kc_stream_t stream) {
    const char* fn = "kc_kv_cache_extend";
    const int st = check(fn, pages, d_seq_lens, d_seq_lens_out, d_free_count_out);
    if (st != KC_SUCCESS) return st;
    if (total_new < 0 || total_new > INT32_MAX)
        return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: total_new=%lld", fn, (long long)total_new);
    if (!d_cu_new || !d_cu_seqlens || (pages->seqs > 0 && !d_new_lens) ||
        (total_new > 0 && (!d_positions || !d_slots)))
        return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: null device pointer", fn);
    const Pages p = args(pages, d_seq_lens, d_seq_lens_out, d_free_count_out);
    const bool few = pages->seqs <= kFew;
    const int threads = few ? kFew : kMany;
    const unsigned grid = static_cast<unsigned>(std::max<int64_t>(1, (total_new + threads - 1) / threads));
    if (few)
        extend_kernel<kFew><<<grid, kFew, 0, stream>>>(p, d_new_lens, total_new, d_cu_new, d_cu_seqlens, d_positions,
                                                       d_slots);
    else
        extend_kernel<kMany><<<grid, kMany, 0, stream>>>(p, d_new_lens, total_new, d_cu_new, d_cu_seqlens, d_positions,
                                                         d_slots);
    return kc::check_launch(fn);
}

extern "C" int kc_kv_cache_release(const kc_kv_pages* pages, const uint8_t* d_finished, const int32_t* d_seq_lens,
                                   int32_t* d_seq_lens_out, int32_t* d_free_count_out, kc_stream_t stream) {
    const char* fn = "kc_kv_cache_release";
    const int st = check(fn, pages, d_seq_lens, d_seq_lens_out, d_free_count_out);
    if (st != KC_SUCCESS) return st;
    if (pages->seqs > 0 && !d_finished)
        return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: null device pointer", fn);
    const Pages p = args(pages, d_seq_lens, d_seq_lens_out, d_free_count_out);
    const bool few = pages->seqs <= kFew;
    const int threads = few ? kFew : kMany;
    // A thread for each entry of the block table, as far as 256 workgroups go.
    const int64_t most = std::min<int64_t>(pages->seqs * pages->max_pages, pages->num_pages);
    const unsigned grid = static_cast<unsigned>(std::clamp<int64_t>((most + threads - 1) / threads, 1, 256));
    if (few) release_kernel<kFew><<<grid, kFew, 0, stream>>>(p, d_finished);
    else release_kernel<kMany><<<grid, kMany, 0, stream>>>(p, d_finished);
    return kc::check_launch(fn);
}
