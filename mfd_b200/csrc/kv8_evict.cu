// kv8_evict.cu -- drop the pages of least attention mass from every request that is over its budget of pages.
//
// The pages that stay are the first `sink`, the last `recent` and, of the others (the middle), the keep - sink -
// recent of largest mass, equal masses by lower index; table and mass are compacted in order and the dropped pages
// listed.  Whole pages leave with their scales, so no code is rounded again and no byte of the cache moves.
//
// Bound: latency (12 bytes in and 12 out per page).  One CTA per request: the threshold (the smallest kept mass) by
// radix selection on the masses' order-preserving 32-bit keys, most significant byte first, its 256 counters in shared
// memory; then one pass of block scans, in which every page's place follows from the number of middle pages before it
// that are above the threshold and that are at it (of those at it the first few stay).
//
// Measured: a table of 1024 pages 6.3 us, 128 tables of 4095 pages 12.4 us.
#include "kv8.cuh"

namespace mfd {
namespace kv8 {

constexpr int kEvictThreads = 1024;
constexpr int kHeldKeys = 32768;  // keys kept in shared memory (a longer table re-reads its masses)

struct EvictParams {
    const int32_t* table;
    const float* mass;
    const int32_t* lens;
    int max_pages, page, page_shift, keep, sink, recent;
    int32_t* table_out;
    float* mass_out;
    int32_t* new_lens;
    int32_t* freed;
    int32_t* freed_counts;
};

// order of the masses as unsigned integers; NaN below everything
__device__ __forceinline__ uint32_t mass_key(float v) { return v == v ? ord_f32(v) : 0u; }

__global__ void __launch_bounds__(kEvictThreads) kv8_evict_kernel(const EvictParams p) {
    extern __shared__ uint32_t held[];
    __shared__ int hist[256];
    __shared__ int warp_sum[2][32];
    __shared__ uint32_t s_prefix;
    __shared__ int s_need;
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t row = (int64_t)b * p.max_pages;
    const int cap = p.max_pages << p.page_shift;
    const int len = min(max(__ldg(p.lens + b), 0), cap);
    const int pages = (len + p.page - 1) >> p.page_shift;
    const int32_t* table = p.table + row;
    const float* mass = p.mass + row;
    int32_t* table_out = p.table_out + row;
    float* mass_out = p.mass_out + row;
    int32_t* freed = p.freed + row;

    if (pages <= p.keep) {
        for (int i = tid; i < p.max_pages; i += kEvictThreads) {
            table_out[i] = i < pages ? __ldg(table + i) : -1;
            mass_out[i] = i < pages ? __ldg(mass + i) : 0.f;
            freed[i] = -1;
        }
        if (tid == 0) {
            p.new_lens[b] = len;
            p.freed_counts[b] = 0;
        }
        return;
    }
    // the middle pages [m0, m1) compete for `want` places
    const int m0 = p.sink, m1 = pages - p.recent, want = p.keep - p.sink - p.recent;
    const bool in_smem = m1 - m0 <= kHeldKeys;
    auto key = [&](int i) { return in_smem ? held[i - m0] : mass_key(__ldg(mass + i)); };
    if (in_smem)
        for (int i = m0 + tid; i < m1; i += kEvictThreads) held[i - m0] = mass_key(__ldg(mass + i));
    if (tid == 0) s_prefix = 0u, s_need = want;
    uint32_t threshold = 0xffffffffu;  // want = 0: nothing is above it, and of those at it none stays
    int at_threshold = 0;              // how many keys equal to the threshold stay
    if (want > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            const uint32_t prefix = s_prefix;
            const uint32_t above = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
            for (int i = m0 + tid; i < m1; i += kEvictThreads) {
                const uint32_t k = key(i);
                if ((k & above) == prefix) atomicAdd(&hist[(k >> shift) & 255u], 1);
            }
            __syncthreads();
            if (warp == 0) {  // the byte in which the `need`-th largest key lies: lane l holds bins 255 - 8 l downwards
                const int need = s_need;
                int h[8], sum = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) sum += h[j] = hist[255 - 8 * lane - j];
                int before = sum;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const int o = __shfl_up_sync(MFD_FULL_MASK, before, d);
                    if (lane >= d) before += o;
                }
                before -= sum;  // keys in higher bins than this lane's
                if (before < need && need <= before + sum) {
                    int left = need - before, j = 0;
#pragma unroll
                    for (int u = 0; u < 7; ++u)
                        if (j == u && left > h[u]) left -= h[u], j = u + 1;
                    s_prefix = prefix | ((uint32_t)(255 - 8 * lane - j) << shift);
                    s_need = left;
                }
            }
            __syncthreads();
        }
        threshold = s_prefix;
        at_threshold = s_need;
    }
    __syncthreads();
    // places: `run_hi` middle pages above the threshold and `run_eq` at it precede the tile
    int run_hi = 0, run_eq = 0;
    for (int t0 = 0; t0 < pages; t0 += kEvictThreads) {
        const int i = t0 + tid;
        const bool inside = i < pages, middle = i >= m0 && i < m1;
        const uint32_t k = middle ? key(i) : 0u;
        const bool hi = middle && k > threshold, eq = middle && want > 0 && k == threshold;
        const uint32_t bh = __ballot_sync(MFD_FULL_MASK, hi), be = __ballot_sync(MFD_FULL_MASK, eq);
        const uint32_t below = (1u << lane) - 1u;
        if (lane == 0) warp_sum[0][warp] = __popc(bh), warp_sum[1][warp] = __popc(be);
        __syncthreads();
        const int wh = warp_sum[0][lane], we = warp_sum[1][lane];
        const int ph = run_hi + __reduce_add_sync(MFD_FULL_MASK, lane < warp ? wh : 0) + __popc(bh & below);
        const int pe = run_eq + __reduce_add_sync(MFD_FULL_MASK, lane < warp ? we : 0) + __popc(be & below);
        run_hi += __reduce_add_sync(MFD_FULL_MASK, wh);
        run_eq += __reduce_add_sync(MFD_FULL_MASK, we);
        __syncthreads();
        if (inside) {
            const int fixed = min(i, m0) + max(i - m1, 0);  // sink and recent pages before i
            const int to = fixed + ph + min(pe, at_threshold);
            const bool stays = !middle || hi || (eq && pe < at_threshold);
            const int32_t id = __ldg(table + i);
            if (stays) {
                table_out[to] = id;
                mass_out[to] = __ldg(mass + i);
            } else {
                freed[i - to] = id;
            }
        }
    }
    const int gone = pages - p.keep;
    for (int i = p.keep + tid; i < p.max_pages; i += kEvictThreads) {
        table_out[i] = -1;
        mass_out[i] = 0.f;
    }
    for (int i = gone + tid; i < p.max_pages; i += kEvictThreads) freed[i] = -1;
    if (tid == 0) {
        p.new_lens[b] = len - (gone << p.page_shift);
        p.freed_counts[b] = gone;
    }
}

}  // namespace kv8
}  // namespace mfd

using namespace mfd;

extern "C" int mfd_kv8_evict(const int32_t* page_table, const float* mass, const int32_t* seq_lens, int64_t bs,
                             int64_t max_pages, int64_t page_size, int64_t keep_pages, int64_t sink_pages,
                             int64_t recent_pages, int32_t* table_out, float* mass_out, int32_t* new_lens,
                             int32_t* freed, int32_t* freed_counts, void* stream) {
    const char* who = "mfd_kv8_evict";
    if (bs > 0 && (!page_table || !mass || !seq_lens || !table_out || !mass_out || !new_lens || !freed || !freed_counts ||
                   table_out == page_table || mass_out == mass || freed == page_table)) {
        set_error("%s: null or overlapping pointers", who);
        return MFD_ERR_INVALID;
    }
    if (bs < 0 || max_pages <= 0 || sink_pages < 0 || recent_pages < 1 || sink_pages > keep_pages ||
        recent_pages > keep_pages - sink_pages) {
        set_error("%s: invalid sizes (keep %lld pages, sink %lld, recent %lld)", who, (long long)keep_pages,
                  (long long)sink_pages, (long long)recent_pages);
        return MFD_ERR_INVALID;
    }
    if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128) {
        set_error("%s: page size %lld is not 16, 32, 64 or 128", who, (long long)page_size);
        return MFD_ERR_UNSUPPORTED;
    }
    if (max_pages > (int64_t)0x3fffffff / page_size) {
        set_error("%s: more than 2^30 tokens a request", who);
        return MFD_ERR_UNSUPPORTED;
    }
    if (bs == 0) return MFD_OK;
    kv8::EvictParams p;
    p.table = page_table;
    p.mass = mass;
    p.lens = seq_lens;
    p.max_pages = (int)max_pages;
    p.page = (int)page_size;
    p.page_shift = __builtin_ctz((unsigned)page_size);
    // a budget above the table's width is one that no request exceeds
    p.keep = (int)(keep_pages < max_pages ? keep_pages : max_pages);
    p.sink = (int)(sink_pages < p.keep ? sink_pages : p.keep);
    p.recent = (int)(recent_pages < p.keep ? recent_pages : p.keep);
    p.table_out = table_out;
    p.mass_out = mass_out;
    p.new_lens = new_lens;
    p.freed = freed;
    p.freed_counts = freed_counts;
    const int held = 4 * (int)(max_pages < kv8::kHeldKeys ? max_pages : kv8::kHeldKeys);
    static bool opted[64];
    cudaError_t e = kv8::opt_in_smem((const void*)kv8::kv8_evict_kernel, 4 * kv8::kHeldKeys, opted);
    if (e != cudaSuccess) {
        set_error("%s: %s", who, cudaGetErrorString(e));
        return MFD_ERR_CUDA;
    }
    kv8::kv8_evict_kernel<<<(unsigned)bs, kv8::kEvictThreads, held, (cudaStream_t)stream>>>(p);
    MFD_CHECK_LAUNCH(who);
    return MFD_OK;
}
