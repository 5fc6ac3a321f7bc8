// kv8_weights.cu -- the attention weight every cached page received from the accepted query rows.
//
//   out[b, p] = decay mass[b, p] + sum_{heads, listed nodes i, tokens j of page p} exp(q_i . k_j scale - lse_i)
//
// The log-sum-exps are those of the attention that ran before, so one pass over K gives the final probabilities: no
// maximum, no second product.  Scores are formed as in the attention (codes exact in float16, query rows divided by a
// power of two, float32 sums); every weight and sum is float32.
//
// Bound: K's bytes (128 codes a token and KV head); next, instructions: the scores' products of 2 * 128 flop and an
// exponential per listed row and token.  As in kv8_attention_rows.cu the 16 tokens are the wide operand of the tensor
// instruction and 8 query rows the narrow one, and every warp copies its own codes asynchronously into a ring of its own
// (two stages of 32 tokens).  It turns 32 tokens' codes into operands once and runs all listed rows past them, 16 at a time
// from shared memory: 32 tokens rather than 16 halve those reads, and two row tiles side by side give four independent
// chains of products.
//
// Split: the tiles of all (request, KV head) units are laid end to end by their cost (tokens, and rows that pass them) and
// cut into equal ranges, one per CTA, so ragged lengths and counts balance.  Each 16 tokens' sum goes to the workspace; the
// CTA that finishes a request last adds them up per page, in a fixed order over tokens and heads (no float atomics).
//
// Measured (H 32 over 8 KV heads, paths of 17 of 65 nodes: 68 rows a KV head): one request of 4096 tokens 14.4 us, where
// launch, prologue and the last CTA's sum are nearly all; 32 requests of 1K - 8K tokens 64 us, 2.2 TB/s of codes.  There one
// listed row takes 43 of the 64 us of 68 rows (32 requests of 4096 tokens): the rest is the products at the legacy tensor
// rate.  The same on tcgen05 (keys as rows of a 128-wide product, codes to bf16 tiles by warps of their own) ran 69 us
// with two CTAs an SM and 81 with one: turning the codes into operand tiles took what the products gave.
#include "kv8.cuh"

namespace mfd {
namespace kv8 {

constexpr int kWWarps = 8;
constexpr int kWThreads = 32 * kWWarps;
constexpr int kWTile = 32 * kWWarps;     // tokens the warps take side by side
constexpr int kWStages = 2;
constexpr int kWStageBytes = 32 * kD;    // of a warp
constexpr int kWRingBytes = kWWarps * kWStages * kWStageBytes;
constexpr int kWRowTiles = 16;  // 8-row tiles staged at a time
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
__global__ void __launch_bounds__(kWThreads, kWCtasPerSm)
    kv8_weights_kernel(const WeightParams p) {
    extern __shared__ __align__(128) unsigned char ring[];
    auto s_q = reinterpret_cast<uint2(*)[8][32]>(ring + kWRingBytes);  // query operands: tile, step, lane
    __shared__ __align__(16) float2 s_row[kWRowTiles][8];  // score factor and -log2(e) * log-sum-exp of a row
    __shared__ int s_last;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int Hkv = p.c.Hkv;
    // a tile's cost: about four row tiles' for its codes, and one for every 8 rows that pass them
    auto tiles_of = [&](int len) { return max(1, (len + kWTile - 1) / kWTile); };
    auto weight_of = [&](int b) {
        const int rows = p.counts ? min(max(__ldg(p.counts + b), 0), p.rows) : p.rows;
        return 4 + min((rows * p.G + 7) >> 3, 60);
    };
    auto cost_of = [&](int len, int b) { return tiles_of(len) * weight_of(b); };
    const Lengths lens(p.c, p.bs);
    const int total = lens.sum(cost_of) * Hkv;
    const int per = max(1, quotient(total + gridDim.x - 1, gridDim.x));
    int pos = (int)min((int64_t)blockIdx.x * per, (int64_t)total);
    const int end = (int)min((int64_t)total, (int64_t)pos + per);

    while (pos < end) {
        int before, len;
        const int b = lens.find(pos, Hkv, cost_of, before, len);
        if (b < 0) return;
        // of the unit (b, hk) the tiles whose cost begins in [pos, end)
        const int tiles = tiles_of(len), weight = weight_of(b), unit = tiles * weight;
        const int off = pos - before;
        const int hk = quotient(off, unit), u0 = off - hk * unit, u1 = min(unit, u0 + (end - pos));
        const int t0 = quotient(u0 + weight - 1, weight), t1 = quotient(u1 + weight - 1, weight);
        const int listed = listed_rows(p.path, p.path_stride, p.rows, p.counts, p.n, b);
        const int nrows = listed * p.G;
        float* part = p.part + (int64_t)b * p.groups_max * Hkv + hk;

        // ---- this warp's copies: lane l takes chunk l % 8 of rows l / 8 + 4 i; the page ids are read a tile ahead
        unsigned char* mine = ring + warp * (kWStages * kWStageBytes);
        const int64_t lane_off = (int64_t)hk * p.c.sc_h + (int64_t)(lane >> 3) * p.c.sc_t + (lane & 7) * 16;
        auto key_of = [&](int tile, int q) { return tile * kWTile + 32 * warp + 16 * q; };
        auto id_of = [&](int tile, int q) {
            return tile < t1 && key_of(tile, q) < len ? page_id(p.c, b, key_of(tile, q) >> p.c.page_shift) : -1;
        };
        auto fetch = [&](int tile, const int (&id)[2]) {
            unsigned char* dst = mine + (tile - t0) % kWStages * kWStageBytes;
            float2 sc = make_float2(0.f, 0.f);
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                if (id[q] < 0) continue;
                const uint8_t* src = p.c.k + (int64_t)id[q] * p.c.sc_p + (int64_t)(key_of(tile, q) & (p.c.page - 1)) * p.c.sc_t + lane_off;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    copy16(dst + chunk_at(16 * q + 4 * i + (lane >> 3), lane & 7), src + (int64_t)(4 * i) * p.c.sc_t);
                (q ? sc.y : sc.x) = __ldg(p.c.k_scale + (int64_t)id[q] * Hkv + hk);
            }
            copies_commit();
            return sc;
        };

        // one pass in all but extreme cases: 128 rows are staged at a time
#pragma unroll 1
        for (int r0 = 0; t0 < t1 && (r0 == 0 || r0 < nrows); r0 += kWRowTiles * 8) {
            const int row_tiles = min(kWRowTiles, (nrows - r0 + 7) / 8);
            int id[2] = {id_of(t0, 0), id_of(t0, 1)};
            float2 sc0 = fetch(t0, id);
            id[0] = id_of(t0 + 1, 0), id[1] = id_of(t0 + 1, 1);
            // ---- the listed rows as operands: row g of tile w for warp w
#pragma unroll 1
            for (int rt = warp; rt < row_tiles; rt += kWWarps) {
                const int r = r0 + rt * 8 + g;
                const bool live = r < nrows;
                const int i = live ? quotient(r, p.G) : 0;
                const int64_t node = live && p.path ? __ldg((const long long*)p.path + (int64_t)b * p.path_stride + i) : i;
                const int head = hk * p.G + (live ? r - i * p.G : 0);
                const uint4* row = reinterpret_cast<const uint4*>(p.q + (int64_t)b * p.sq_b + node * p.sq_n +
                                                                  (int64_t)head * p.sq_h + 32 * t);
                uint4 x[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    x[u] = make_uint4(0u, 0u, 0u, 0u);
                    if (live) x[u] = __ldg(row + u);
                }
                const float ls = live ? __ldg(p.lse + ((int64_t)b * p.n + node) * p.H + head) : -INFINITY;
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
                        s_q[rt][2 * u + j][lane] =
                            make_uint2(pack_half2(f0.x * down, f0.y * down), pack_half2(f1.x * down, f1.y * down));
                    }
                }
                // a row that saw nothing, or padding, weighs nothing
                if (t == 0)
                    s_row[rt][g] = make_float2(live ? up * p.scale_log2 : 0.f, ls == -INFINITY ? -INFINITY : -ls * kLog2e);
            }
            __syncthreads();
#pragma unroll 1
            for (int tile = t0; tile < t1; ++tile) {
                __syncwarp();  // (every lane has read the stage that the copies below overwrite)
                const float2 sc1 = fetch(tile + 1, id);
                id[0] = id_of(tile + 2, 0), id[1] = id_of(tile + 2, 1);
                copies_wait<1>();
                __syncwarp();
                const int key0 = key_of(tile, 0);
                if (key0 >= len) break;
                const unsigned char* kt = mine + (tile - t0) % kWStages * kWStageBytes;
                uint4 raw[2][2][2];  // of 16 tokens each: token g, g + 8; chunks 2 t, 2 t + 1
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            raw[q][h][i] = *reinterpret_cast<const uint4*>(kt + chunk_at(16 * q + 8 * h + g, 2 * t + i));
                const float sk[2] = {sc0.x, sc0.y};
                sc0 = sc1;
                uint32_t a[2][8][4];
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t w[8] = {raw[q][h][0].x, raw[q][h][0].y, raw[q][h][0].z, raw[q][h][0].w,
                                               raw[q][h][1].x, raw[q][h][1].y, raw[q][h][1].z, raw[q][h][1].w};
#pragma unroll
                        for (int ks = 0; ks < 8; ++ks) halves<FP8>(w[ks], a[q][ks][h], a[q][ks][2 + h]);
                    }
                float sum[2] = {0.f, 0.f};
                const bool tail = key0 + 32 > len;
#pragma unroll 1
                for (int rt = 0; rt < row_tiles; rt += 2) {
                    float acc[2][2][4];  // row tile, 16 tokens
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int q = 0; q < 2; ++q)
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[u][q][e] = 0.f;
                    const bool two = rt + 1 < row_tiles;
                    if (two) {
#pragma unroll
                        for (int ks = 0; ks < 8; ++ks)
#pragma unroll
                            for (int u = 0; u < 2; ++u) {
                                const uint2 x = s_q[rt + u][ks][lane];
#pragma unroll
                                for (int q = 0; q < 2; ++q)
                                    mma_f16(acc[u][q], a[q][ks][0], a[q][ks][1], a[q][ks][2], a[q][ks][3], x.x, x.y);
                            }
                    } else {
#pragma unroll
                        for (int ks = 0; ks < 8; ++ks) {
                            const uint2 x = s_q[rt][ks][lane];
#pragma unroll
                            for (int q = 0; q < 2; ++q)
                                mma_f16(acc[0][q], a[q][ks][0], a[q][ks][1], a[q][ks][2], a[q][ks][3], x.x, x.y);
                        }
                    }
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        if (u == 1 && !two) break;
                        const float4 f = *reinterpret_cast<const float4*>(&s_row[rt + u][2 * t]);  // rows 2 t and 2 t + 1
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            const float fx = f.x * sk[q], fz = f.z * sk[q];
                            float w[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                w[e] = fast_exp2(fmaf(acc[u][q][e], (e & 1) ? fz : fx, (e & 1) ? f.w : f.y));
                            if (tail) {
                                if (key0 + 16 * q + g >= len) w[0] = w[1] = 0.f;
                                if (key0 + 16 * q + g + 8 >= len) w[2] = w[3] = 0.f;
                            }
                            sum[q] += (w[0] + w[1]) + (w[2] + w[3]);
                        }
                    }
                }
#pragma unroll
                for (int q = 0; q < 2; ++q) {
#pragma unroll 1
                    for (int d = 16; d; d >>= 1) sum[q] += __shfl_xor_sync(MFD_FULL_MASK, sum[q], d);
                    if (lane == 0 && key0 + 16 * q < len) {
                        float* dst = part + (int64_t)((key0 >> 4) + q) * Hkv;
                        *dst = r0 == 0 ? sum[q] : *dst + sum[q];
                    }
                }
            }
            copies_wait<0>();
            __syncthreads();  // the staged rows are done with
        }
        pos += u1 - u0;
        // ---- the request's last CTA adds up its pages
        if (pos >= end || pos >= before + unit * Hkv) {
            const int pieces = quotient(before + unit * Hkv - 1, per) - quotient(before, per) + 1;
            __threadfence();
            __syncthreads();
            if (tid == 0) s_last = pieces == 1 || atomicAdd(p.tickets + b, 1u) == (unsigned)(pieces - 1);
            __syncthreads();
            if (s_last) {
                __threadfence();
                const int pages = (len + p.c.page - 1) >> p.c.page_shift, groups = (len + 15) / 16;
                const int gpp = p.c.page / 16;
                const float* src = p.part + (int64_t)b * p.groups_max * Hkv;
                const bool wide = (gpp * Hkv) % 4 == 0;
                for (int i = tid; i < p.c.max_pages; i += kWThreads) {
                    float v = 0.f;
                    if (i < pages) {
                        int e = i * gpp * Hkv;
                        const int stop = min((i + 1) * gpp, groups) * Hkv;
                        if (wide) {  // (the page's sums are contiguous: one latency for 32 of them)
#pragma unroll 8
                            for (; e + 4 <= stop; e += 4) {
                                const float4 x = __ldcg(reinterpret_cast<const float4*>(src + e));
                                v += (x.x + x.y) + (x.z + x.w);
                            }
                        }
#pragma unroll 8
                        for (; e < stop; ++e) v += __ldcg(src + e);
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
    if ((bs > 0 && (!q || !lse || !mass || !out)) || !k_scale || !workspace || !tickets) {
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
    if (!kv8::work_fits(bs, num_kv_heads * 64, max_pages, page_size, 256)) {
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
    constexpr int kSmem = kv8::kWRingBytes + kv8::kWRowTiles * 8 * 32 * 8;
    static bool opted[2][64];
    const bool fp8 = code_dtype == MFD_E4M3;
    const void* kernel = fp8 ? (const void*)kv8::kv8_weights_kernel<true> : (const void*)kv8::kv8_weights_kernel<false>;
    cudaError_t e = kv8::opt_in_smem(kernel, kSmem, opted[fp8]);
    if (e != cudaSuccess) {
        set_error("%s: %s", who, cudaGetErrorString(e));
        return MFD_ERR_CUDA;
    }
    if (fp8) kv8::kv8_weights_kernel<true><<<grid, kv8::kWThreads, kSmem, (cudaStream_t)stream>>>(p);
    else kv8::kv8_weights_kernel<false><<<grid, kv8::kWThreads, kSmem, (cudaStream_t)stream>>>(p);
    MFD_CHECK_LAUNCH(who);
    return MFD_OK;
}
