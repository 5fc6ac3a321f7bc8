// kv8_weights.cu -- the attention weight every cached page received from the accepted query rows.
//
//   out[b, p] = decay mass[b, p] + sum_{heads, listed nodes i, tokens j of page p} exp(q_i . k_j scale - lse_i)
//
// The log-sum-exps are those of the attention that ran before, so one pass over K gives the final probabilities: no
// maximum, no second product.  Scores are formed as in the attention (codes exact in float16, query rows divided by a
// power of two, float32 sums); every weight and sum is float32.
//
// Bound: K's bytes (128 codes a token and KV head), next the tensor instructions (2 * 128 flop per listed row and
// token) and the shared-memory reads of the query operands.  A warp takes 32 tokens of one KV head, their codes in
// registers as operands, and runs all listed rows past them, 16 at a time from shared memory; twice the tokens a warp
// halve those reads, and 64 tokens do not fit the registers of two CTAs an SM.
//
// Split: the 32-token tasks of all (request, KV head) units are laid end to end and cut into equal ranges, one per CTA,
// so ragged lengths balance.  Each 16 tokens' sum goes to the workspace; the CTA that finishes a request last adds
// them up per page, in a fixed order over tokens and heads (no float atomics).
#include "kv8.cuh"

namespace mfd {
namespace kv8 {

constexpr int kWWarps = 8;
constexpr int kWThreads = 32 * kWWarps;
constexpr int kWTiles = 8;      // 16-row tiles staged at a time
constexpr int kWCtasPerSm = 2;

struct WeightParams {
    Cache c;
    const __nv_bfloat16* q;
    int64_t sq_b, sq_n, sq_h;
    const float* lse;
    const int64_t* path;
    int64_t path_stride;
    int rows;
    const int32_t* counts;
    int bs, n, H, G;
    float scale_log2, decay;
    const float* mass;
    float* out;
    int64_t mass_stride;
    float* part;  // [bs, groups, Hkv]
    int groups_max;
    unsigned int* tickets;
};

template <bool FP8>
__global__ void __launch_bounds__(kWThreads, kWCtasPerSm) kv8_weights_kernel(const WeightParams p) {
    __shared__ uint4 s_q[kWTiles][8][32];           // query operands: tile, 16-column step, lane
    __shared__ float s_rf[kWTiles * 16], s_lse[kWTiles * 16];
    __shared__ int s_last;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int Hkv = p.c.Hkv;
    auto tasks_of = [&](int len) { return max(1, (len + 31) / 32); };
    const Lengths lens(p.c, p.bs);
    const int total = lens.sum(tasks_of) * Hkv;
    int per = quotient(total + gridDim.x - 1, gridDim.x);
    if (per < kWWarps) per = kWWarps;
    int pos = (int)min((int64_t)blockIdx.x * per, (int64_t)total);
    const int end = (int)min((int64_t)total, (int64_t)pos + per);

    while (pos < end) {
        int before, len;
        const int b = lens.find(pos, Hkv, tasks_of, before, len);
        if (b < 0) return;
        const int tasks = tasks_of(len);
        const int off = pos - before;
        const int hk = quotient(off, tasks), t0 = off - hk * tasks;
        const int t1 = min(tasks, t0 + (end - pos));
        const int listed = listed_rows(p.path, p.path_stride, p.rows, p.counts, p.n, b);
        const int nrows = listed * p.G;
        float* part = p.part + (int64_t)b * p.groups_max * Hkv + hk;

        // one pass in all but extreme cases: 128 rows are staged at a time
        for (int r0 = 0; r0 == 0 || r0 < nrows; r0 += kWTiles * 16) {
            const int tiles = min(kWTiles, (nrows - r0 + 15) / 16);
            __syncthreads();
            if (warp < tiles) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int r = r0 + warp * 16 + g + 8 * h;
                    const bool live = r < nrows;
                    const int i = live ? r / p.G : 0;
                    const int64_t node = live && p.path ? __ldg((const long long*)p.path + (int64_t)b * p.path_stride + i) : i;
                    const int head = hk * p.G + (live ? r % p.G : 0);
                    const __nv_bfloat16* row = p.q + (int64_t)b * p.sq_b + node * p.sq_n + (int64_t)head * p.sq_h;
                    uint4 x[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        x[u] = make_uint4(0u, 0u, 0u, 0u);
                        if (live) x[u] = __ldg(reinterpret_cast<const uint4*>(row + 16 * t + 8 * (u & 1) + 64 * (u >> 1)));
                    }
                    float mx = 0.f;
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const uint32_t w[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float2 f = bf2(w[j]);
                            mx = fmaxf(mx, fmaxf(fabsf(f.x), fabsf(f.y)));
                        }
                    }
                    mx = quad_max(mx);
                    float down, up;
                    row_power(mx, down, up);
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const uint32_t w[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const float2 f0 = bf2(w[2 * j]), f1 = bf2(w[2 * j + 1]);
                            const int ks = 4 * (u >> 1) + 2 * (u & 1) + j;
                            uint32_t* dst = reinterpret_cast<uint32_t*>(&s_q[warp][ks][lane]);
                            dst[h] = pack_half2(f0.x * down, f0.y * down);       // operand registers: rows g, g + 8 at
                            dst[2 + h] = pack_half2(f1.x * down, f1.y * down);   // columns k, then both at k + 8
                        }
                    }
                    if (t == 0) {
                        const float ls = live ? __ldg(p.lse + ((int64_t)b * p.n + node) * p.H + head) : -INFINITY;
                        s_rf[warp * 16 + g + 8 * h] = live ? up * p.scale_log2 : 0.f;
                        // a row that saw nothing, or padding, weighs nothing
                        s_lse[warp * 16 + g + 8 * h] = ls == -INFINITY ? -INFINITY : -ls * kLog2e;
                    }
                }
            }
            __syncthreads();
            for (int task = t0 + warp; task < t1; task += kWWarps) {
                uint32_t kb[4][8][2];  // 8-token tiles: operands of the 8 steps
                float sk[2];
                uint4 raw[4][2];
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const int key0 = task * 32 + 16 * q;
                    const int id = key0 < len ? page_id(p.c, b, key0 >> p.c.page_shift) : 0;
                    sk[q] = key0 < len ? __ldg(p.c.k_scale + (int64_t)id * Hkv + hk) : 0.f;
                    const uint8_t* src = p.c.k + (int64_t)id * p.c.sc_p + (int64_t)hk * p.c.sc_h +
                                         (int64_t)((key0 & (p.c.page - 1)) + g) * p.c.sc_t + 16 * t;
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            raw[2 * q + kt][i] = make_uint4(0u, 0u, 0u, 0u);
                            if (key0 < len) raw[2 * q + kt][i] = ldg_stream_u4(src + (int64_t)(8 * kt) * p.c.sc_t + 64 * i);
                        }
                }
#pragma unroll
                for (int kt = 0; kt < 4; ++kt) {
                    const uint32_t w[8] = {raw[kt][0].x, raw[kt][0].y, raw[kt][0].z, raw[kt][0].w,
                                           raw[kt][1].x, raw[kt][1].y, raw[kt][1].z, raw[kt][1].w};
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks) halves<FP8>(w[ks], kb[kt][ks][0], kb[kt][ks][1]);
                }
                float sum[2] = {0.f, 0.f};
                const int key = task * 32 + 2 * t;  // this lane's tokens: key, key + 1 of every 8-token tile
                for (int tl = 0; tl < tiles; ++tl) {
                    float acc[4][4];
#pragma unroll
                    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[kt][e] = 0.f;
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks) {
                        const uint4 a = s_q[tl][ks][lane];
#pragma unroll
                        for (int kt = 0; kt < 4; ++kt) mma_f16(acc[kt], a.x, a.y, a.z, a.w, kb[kt][ks][0], kb[kt][ks][1]);
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float rf = s_rf[tl * 16 + g + 8 * h], nl = s_lse[tl * 16 + g + 8 * h];
#pragma unroll
                        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const float w = fast_exp2(fmaf(acc[kt][2 * h + e], rf * sk[kt >> 1], nl));
                                sum[kt >> 1] += key + 8 * kt + e < len ? w : 0.f;
                            }
                    }
                }
#pragma unroll
                for (int q = 0; q < 2; ++q) {
#pragma unroll
                    for (int d = 16; d; d >>= 1) sum[q] += __shfl_xor_sync(MFD_FULL_MASK, sum[q], d);
                    if (lane == 0 && task * 32 + 16 * q < len) {
                        float* dst = part + (int64_t)(2 * task + q) * Hkv;
                        *dst = r0 == 0 ? sum[q] : *dst + sum[q];
                    }
                }
            }
        }
        pos += t1 - t0;
        // ---- the request's last CTA adds up its pages
        if (pos >= end || pos >= before + tasks * Hkv) {
            const int pieces = quotient(before + tasks * Hkv - 1, per) - quotient(before, per) + 1;
            __threadfence();
            __syncthreads();
            if (tid == 0) s_last = pieces == 1 || atomicAdd(p.tickets + b, 1u) == (unsigned)(pieces - 1);
            __syncthreads();
            if (s_last) {
                __threadfence();
                const int pages = (len + p.c.page - 1) >> p.c.page_shift, groups = (len + 15) / 16;
                const int gpp = p.c.page / 16;
                const float* src = p.part + (int64_t)b * p.groups_max * Hkv;
                for (int i = tid; i < p.c.max_pages; i += kWThreads) {
                    float v = 0.f;
                    if (i < pages) {
                        const int n0 = i * gpp * Hkv, n1 = min((i + 1) * gpp, groups) * Hkv;
#pragma unroll 8
                        for (int e = n0; e < n1; ++e) v += __ldcg(src + e);
                        v = fmaf(p.mass[(int64_t)b * p.mass_stride + i], p.decay, v);  // (out may be mass)
                    }
                    p.out[(int64_t)b * p.mass_stride + i] = v;
                }
                if (tid == 0 && pieces > 1) p.tickets[b] = 0u;
            }
        }
    }
}

}  // namespace kv8
}  // namespace mfd

using namespace mfd;

extern "C" size_t mfd_kv8_page_weights_workspace(int64_t bs, int64_t max_pages, int64_t page_size,
                                                 int64_t num_kv_heads) {
    if (bs < 0 || max_pages <= 0 || page_size < 16 || num_kv_heads <= 0) return 0;
    return 256 + (size_t)bs * (size_t)max_pages * (size_t)(page_size / 16) * (size_t)num_kv_heads * sizeof(float);
}

extern "C" int mfd_kv8_page_weights(const void* q, int64_t sq_b, int64_t sq_n, int64_t sq_h, const float* lse,
                                    const void* k_cache, int64_t sc_p, int64_t sc_h, int64_t sc_t, int code_dtype,
                                    const float* k_scale, int64_t num_pages, int64_t page_size,
                                    const int32_t* page_table, int64_t table_stride, int64_t max_pages,
                                    const int32_t* seq_lens, const int64_t* path, int64_t path_stride, int64_t rows,
                                    const int32_t* counts, int64_t bs, int64_t n, int64_t num_heads,
                                    int64_t num_kv_heads, int64_t head_dim, float scale, float decay,
                                    const float* mass, float* out, int64_t mass_stride, void* workspace,
                                    size_t workspace_bytes, unsigned int* tickets, int64_t tickets_len, void* stream) {
    const char* who = "mfd_kv8_page_weights";
    int st;
    if (!kv8::check_cache(who, k_cache, k_cache, sc_p, sc_h, sc_t, code_dtype, num_pages, page_size, page_table,
                          max_pages, seq_lens, bs, num_kv_heads, head_dim, &st))
        return st;
    if (!q || !lse || !k_scale || !mass || !out || !workspace || !tickets) {
        set_error("%s: null pointer", who);
        return MFD_ERR_INVALID;
    }
    if (n <= 0 || num_heads <= 0 || num_heads % num_kv_heads || rows < 0 || (!path && rows > n) ||
        mass_stride < max_pages) {
        set_error("%s: invalid sizes (n %lld, rows %lld, %lld query heads over %lld KV heads)", who, (long long)n,
                  (long long)rows, (long long)num_heads, (long long)num_kv_heads);
        return MFD_ERR_INVALID;
    }
    if (n > 0x3fffff || rows > 0x3fffff || num_heads > 16384 || (num_heads / num_kv_heads) * rows > 0x3fffffff) {
        set_error("%s: too many rows", who);
        return MFD_ERR_UNSUPPORTED;
    }
    if (sq_b % 8 || sq_n % 8 || sq_h % 8 || (uintptr_t)q % 16) {
        set_error("%s: query rows need strides that are multiples of 8 elements and a 16-byte aligned base", who);
        return MFD_ERR_INVALID;
    }
    if (workspace_bytes < mfd_kv8_page_weights_workspace(bs, max_pages, page_size, num_kv_heads) || tickets_len < bs) {
        set_error("%s: workspace or tickets too small", who);
        return MFD_ERR_INVALID;
    }
    if (!kv8::work_fits(bs, num_kv_heads, max_pages, page_size, 32)) {
        set_error("%s: the requests' capacity is beyond this build's limits", who);
        return MFD_ERR_UNSUPPORTED;
    }
    if (bs == 0) return MFD_OK;
    kv8::WeightParams p;
    p.c.k = p.c.v = (const uint8_t*)k_cache;
    p.c.sc_p = sc_p, p.c.sc_h = sc_h, p.c.sc_t = sc_t;
    p.c.k_scale = p.c.v_scale = k_scale;
    p.c.num_pages = num_pages;
    p.c.page = (int)page_size, p.c.page_shift = __builtin_ctz((unsigned)page_size);
    p.c.table = page_table, p.c.table_stride = table_stride, p.c.max_pages = (int)max_pages;
    p.c.lens = seq_lens;
    p.c.Hkv = (int)num_kv_heads;
    p.q = (const __nv_bfloat16*)q, p.sq_b = sq_b, p.sq_n = sq_n, p.sq_h = sq_h;
    p.lse = lse;
    p.path = path, p.path_stride = path_stride, p.rows = (int)rows, p.counts = counts;
    p.bs = (int)bs, p.n = (int)n, p.H = (int)num_heads, p.G = (int)(num_heads / num_kv_heads);
    p.scale_log2 = scale * kLog2e, p.decay = decay;
    p.mass = mass, p.out = out, p.mass_stride = mass_stride;
    const int64_t base = ((uintptr_t)workspace + 255) / 256 * 256 - (uintptr_t)workspace;
    p.part = (float*)((char*)workspace + base);
    p.groups_max = (int)(max_pages * (page_size / 16));
    p.tickets = tickets;
    const int grid = kv8::sm_count() * kv8::kWCtasPerSm;
    if (code_dtype == MFD_E4M3) kv8::kv8_weights_kernel<true><<<grid, kv8::kWThreads, 0, (cudaStream_t)stream>>>(p);
    else kv8::kv8_weights_kernel<false><<<grid, kv8::kWThreads, 0, (cudaStream_t)stream>>>(p);
    MFD_CHECK_LAUNCH(who);
    return MFD_OK;
}
