// kv8_attention_rows.cu -- attention of a few query rows over the 8-bit paged cache: the decode step and short drafts.
//
// The mathematics, for a row with query q over keys j (page P(j), codes a_j and c_j, scales sk and sv):
//   score  s_j = sk (q . a_j) scale log2(e),      w_j = s_j + log2(sv),      m = max_j w_j
//   O = sum_j 2^(w_j - m) c_j,   l = sum_j 2^(w_j - m) / sv,                 out = O / l,  lse = ln2 (m + log2 l)
// so the value scale rides in the exponent and no code is multiplied by its scale.  The scores are products of float16
// operands (codes and the query row divided by a power of two are exact there), for the nodes' own keys of bf16
// operands.  The weights meet the values in bf16 as hi + lo, two tensor instructions: one bf16 weight (8 bits) would
// err by as much as the output's own rounding, and float16 (11 bits) loses a small weight beside a large one in a
// column where the large one's code is 0; hi + lo keeps 16 bits over the whole float32 range.  All sums and statistics
// are float32.
//
// Bound: bytes (256 codes a token and KV head for 4 G n multiply-adds each).  So the codes go from memory straight to
// registers, 16 bytes a lane, in a layout in which they are the operands: the d index of the first product is permuted
// (lane quad t holds d = 16 t .. 16 t + 15 of either half row, the query alike), and the value rows of two keys are
// interleaved byte by byte before they become float16 pairs.  No shared memory is touched in the loop.
//   scores   m16n8k16: A = query rows (16), B = 8 keys; lane (g, t) loads 32 bytes of key g's row
//   values   m16n8k16: A = weights (16 rows x 16 keys, the score registers), B = 16 keys x 8 columns; lane (g, t) loads
//            columns 16 g .. 16 g + 15 of keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9, so column tile j is d = 16 g + j
// A warp takes 16 keys at a time (one page has all 16: one scale), its 8 loads in flight together; 16 warps an SM
// hold 64 KB in flight.  The 8 warps of a CTA take every eighth group of 16 keys with their own (m, l, O) and merge in
// shared memory at the end of the piece.
//
// Split: the groups of all (request, KV head, 16 rows) units are laid end to end and cut into equal pieces, one per
// CTA (two CTAs an SM), so ragged lengths balance and one long request fills the GPU; the lengths are read on the
// device.  A unit cut into pieces is merged by the CTA that finishes last (its partial (m, l, O) in the workspace, a
// ticket per unit; the pieces are added in their order, so the result does not depend on who merges).
#include "kv8_attention.cuh"
#include "tcgen05.cuh"

namespace mfd {
namespace kv8 {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kTBlock = 36, kRowStride = 4 * kTBlock;  // floats: a lane quad's 32 columns, padded against bank conflicts
constexpr int kSlot = 16 * (kD + 2);                   // floats of a partial: m[16], l[16], O[16][128]
constexpr int kCtasPerSm = 2;

__device__ __forceinline__ bool not_finite_pair(uint32_t w) {  // a bf16 pair holds an infinity or a NaN
    return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}

// TALL: 16 rows a unit, else at most 8 (rows 8 .. 15 of every product are zero and cost no registers)
template <bool FP8, bool TALL>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) kv8_rows_kernel(const AttnParams p) {
    constexpr int kHalves = TALL ? 2 : 1;  // row halves (g and g + 8) a lane holds
    constexpr int kRows = 8 * kHalves;
    extern __shared__ __align__(16) float smem[];  // [kWarps][kRows][kRowStride]; merge weights
    __shared__ float s_m[kWarps][kRows], s_l[kWarps][kRows];
    __shared__ uint32_t s_q[8][32][2 * kHalves];  // query operands of the 8 16-column steps, the same for every warp
    __shared__ int s_last;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int nrows = p.rows - p.row0;
    const int RB = (nrows + 15) / 16;

    // ---- this CTA's share of the work, in groups of 16 keys (cached tokens, then own keys)
    auto groups_of = [&](int len) { return max(1, (len + 15) / 16 + (p.nn + 15) / 16); };  // (one, to write zeros)
    const Lengths lens(p.c, p.bs);
    const Cut cut = make_cut(lens, groups_of, p.c.Hkv * RB, gridDim.x, kWarps);
    int64_t pos, end;
    cut_range(cut, blockIdx.x, pos, end);

    Piece pc;
    while (next_piece(lens, groups_of, cut, blockIdx.x, pos, end, pc)) {
        const int hk = pc.u / RB, rb = pc.u % RB, len = pc.len;
        const int gp = (len + 15) / 16;  // groups of cached tokens; own keys follow
        const int base = p.row0 + rb * 16;

        // ---- the query rows as float16 operands, divided by a power of two
        float rf[kHalves];            // score factor of the row: the power of two, the scale and log2(e)
        int node[kHalves];
        const __nv_bfloat16* qrow[kHalves];
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
            const int r = base + g + 8 * h;
            const bool live = r < p.rows;
            node[h] = live ? r / p.G : -1;
            qrow[h] = p.q + (int64_t)pc.b * p.sq_b + (int64_t)(live ? r / p.G : 0) * p.sq_n +
                      (int64_t)(hk * p.G + (live ? r % p.G : 0)) * p.sq_h;
            uint4 x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // columns 16 t + 8 (i & 1) + 64 (i >> 1) ..
                x[i] = make_uint4(0u, 0u, 0u, 0u);
                if (live) x[i] = __ldg(reinterpret_cast<const uint4*>(qrow[h] + 16 * t + 8 * (i & 1) + 64 * (i >> 1)));
            }
            float mx = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 f = bf2(w[j]);
                    mx = fmaxf(mx, fmaxf(fabsf(f.x), fabsf(f.y)));
                }
            }
            mx = quad_max(mx);
            float down, up;
            row_power(mx, down, up);
            rf[h] = up * p.scale_log2;
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // 8 columns: words 2 (i & 1), 2 (i & 1) + 1 of half i >> 1
                const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float2 f0 = bf2(w[2 * j]), f1 = bf2(w[2 * j + 1]);
                    const int ks = 4 * (i >> 1) + 2 * (i & 1) + j;
                    if (warp == 0) {  // rows g, g + 8 at columns k, then both at k + 8
                        s_q[ks][lane][h] = pack_half2(f0.x * down, f0.y * down);
                        s_q[ks][lane][kHalves + h] = pack_half2(f1.x * down, f1.y * down);
                    }
                }
            }
        }
        __syncthreads();

        float o[16][2 * kHalves];
        float m[kHalves], l[kHalves];
#pragma unroll
        for (int j = 0; j < 16; ++j)
#pragma unroll
            for (int e = 0; e < 2 * kHalves; ++e) o[j][e] = 0.f;
#pragma unroll
        for (int h = 0; h < kHalves; ++h) m[h] = -INFINITY, l[h] = 0.f;

        // the softmax step of a group: raw scores sc[key tile][row half x 2] already scaled into w (log2), -inf where
        // masked; returns the weights, rescales O
        auto step = [&](float (&w)[2][2 * kHalves], float inv_sv) {
            float mx[kHalves];
            bool grow = false;
#pragma unroll
            for (int h = 0; h < kHalves; ++h) {
                mx[h] = quad_max(fmaxf(fmaxf(w[0][2 * h], w[0][2 * h + 1]), fmaxf(w[1][2 * h], w[1][2 * h + 1])));
                // a maximum that grows by less than 2^8 is left: a rescale of O costs more than the range
                grow |= mx[h] > m[h] + 8.f || (m[h] == -INFINITY && mx[h] > -INFINITY);
            }
            if (__any_sync(MFD_FULL_MASK, grow)) {
#pragma unroll
                for (int h = 0; h < kHalves; ++h) {
                    const float mn = fmaxf(m[h], mx[h]);
                    const float a = m[h] == -INFINITY ? 0.f : fast_exp2(m[h] - mn);
                    m[h] = mn;
                    l[h] *= a;
#pragma unroll
                    for (int j = 0; j < 16; ++j) o[j][2 * h] *= a, o[j][2 * h + 1] *= a;
                }
            }
#pragma unroll
            for (int h = 0; h < kHalves; ++h) {
                const float mr = m[h] == -INFINITY ? 0.f : m[h];
                float sum = 0.f;
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) sum += w[kt][2 * h + e] = fast_exp2(w[kt][2 * h + e] - mr);
                l[h] = fmaf(sum, inv_sv, l[h]);
            }
        };

        // O's column tile += weights (hi + lo) x 16 keys of it
        auto values = [&](float (&oj)[2 * kHalves], const uint32_t (&hi)[2][kHalves], const uint32_t (&lo)[2][kHalves],
                          uint32_t b0, uint32_t b1) {
            float d[4] = {oj[0], oj[1], TALL ? oj[2 * kHalves - 2] : 0.f, TALL ? oj[2 * kHalves - 1] : 0.f};
            mma_bf16(d, hi[0][0], TALL ? hi[0][kHalves - 1] : 0u, hi[1][0], TALL ? hi[1][kHalves - 1] : 0u, b0, b1);
            mma_bf16(d, lo[0][0], TALL ? lo[0][kHalves - 1] : 0u, lo[1][0], TALL ? lo[1][kHalves - 1] : 0u, b0, b1);
            oj[0] = d[0], oj[1] = d[1];
            if (TALL) oj[2 * kHalves - 2] = d[2], oj[2 * kHalves - 1] = d[3];
        };

        // ---- cached tokens
        const uint8_t* kbase = p.c.k + (int64_t)hk * p.c.sc_h + (int64_t)g * p.c.sc_t + 16 * t;
        const uint8_t* vbase = p.c.v + (int64_t)hk * p.c.sc_h + (int64_t)(2 * t) * p.c.sc_t + 16 * g;
        const int slot_mask = p.c.page - 1;
        int gi = pc.g0 + warp;
        int id_next = gi < min(pc.g1, gp) ? page_id(p.c, pc.b, (gi * 16) >> p.c.page_shift) : 0;
        for (; gi < min(pc.g1, gp); gi += kWarps) {
            const int key0 = gi * 16;
            const int id = id_next;
            const int64_t off = (int64_t)id * p.c.sc_p + (int64_t)(key0 & slot_mask) * p.c.sc_t;
            uint4 kw[2][2], vw[4];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    kw[kt][i] = ldg_stream_u4(kbase + off + (int64_t)(8 * kt) * p.c.sc_t + 64 * i);
#pragma unroll
            for (int i = 0; i < 4; ++i)  // keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9
                vw[i] = ldg_stream_u4(vbase + off + (int64_t)((i & 1) + 8 * (i >> 1)) * p.c.sc_t);
            const float sk = __ldg(p.c.k_scale + (int64_t)id * p.c.Hkv + hk);
            const float sv = fmaxf(__ldg(p.c.v_scale + (int64_t)id * p.c.Hkv + hk), kScaleFloor);
            if (gi + kWarps < min(pc.g1, gp)) id_next = page_id(p.c, pc.b, ((gi + kWarps) * 16) >> p.c.page_shift);

            float acc[2][4];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[kt][e] = 0.f;
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) {
                uint32_t a[4] = {0u, 0u, 0u, 0u};
                if (TALL) {
                    const uint4 x = *reinterpret_cast<const uint4*>(s_q[ks][lane]);
                    a[0] = x.x, a[1] = x.y, a[2] = x.z, a[3] = x.w;
                } else {
                    const uint2 x = *reinterpret_cast<const uint2*>(s_q[ks][lane]);
                    a[0] = x.x, a[2] = x.y;
                }
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) {
                    const uint4 r = kw[kt][ks >> 2];
                    const uint32_t w = (ks & 3) == 0 ? r.x : (ks & 3) == 1 ? r.y : (ks & 3) == 2 ? r.z : r.w;
                    uint32_t b0, b1;
                    halves<FP8>(w, b0, b1);
                    mma_f16(acc[kt], a[0], a[1], a[2], a[3], b0, b1);
                }
            }
            const float lsv = __log2f(sv);
            float w[2][2 * kHalves];
            const bool tail = key0 + 16 > len;
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int h = 0; h < kHalves; ++h)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        w[kt][2 * h + e] = fmaf(acc[kt][2 * h + e], sk * rf[h], lsv);
                        if (tail && key0 + 8 * kt + 2 * t + e >= len) w[kt][2 * h + e] = -INFINITY;
                    }
            if (tail) {  // slots past the length hold any bits (an e4m3 NaN too): their weight is 0, their codes too
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (key0 + 2 * t + (i & 1) + 8 * (i >> 1) >= len) vw[i] = make_uint4(0u, 0u, 0u, 0u);
            }
            step(w, __frcp_rn(sv));
            uint32_t hi[2][kHalves], lo[2][kHalves];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int h = 0; h < kHalves; ++h) split_bf16(pk2(w[kt][2 * h], w[kt][2 * h + 1]), hi[kt][h], lo[kt][h]);
            const uint32_t v0[4] = {vw[0].x, vw[0].y, vw[0].z, vw[0].w}, v1[4] = {vw[1].x, vw[1].y, vw[1].z, vw[1].w};
            const uint32_t v2[4] = {vw[2].x, vw[2].y, vw[2].z, vw[2].w}, v3[4] = {vw[3].x, vw[3].y, vw[3].z, vw[3].w};
#pragma unroll
            for (int j4 = 0; j4 < 4; ++j4) {  // columns 16 g + 4 j4 .. + 3
                uint32_t b0[4], b1[4];
                bfloats<FP8>(__byte_perm(v0[j4], v1[j4], 0x5140), b0[0], b0[1]);
                bfloats<FP8>(__byte_perm(v0[j4], v1[j4], 0x7362), b0[2], b0[3]);
                bfloats<FP8>(__byte_perm(v2[j4], v3[j4], 0x5140), b1[0], b1[1]);
                bfloats<FP8>(__byte_perm(v2[j4], v3[j4], 0x7362), b1[2], b1[3]);
#pragma unroll
                for (int u = 0; u < 4; ++u) values(o[4 * j4 + u], hi, lo, b0[u], b1[u]);
            }
        }

        // ---- the nodes' own keys, in bf16
        const int g_own = min(pc.g1, gp + (p.nn + 15) / 16);
        for (; gi < g_own; gi += kWarps) {
            const int j0 = (gi - gp) * 16;
            const __nv_bfloat16* kn = p.kn + (int64_t)pc.b * p.sn_b + (int64_t)hk * p.sn_h;
            const __nv_bfloat16* vn = p.vn + (int64_t)pc.b * p.sn_b + (int64_t)hk * p.sn_h;
            float acc[2][4];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[kt][e] = 0.f;
                const int key = min(j0 + 8 * kt + g, p.nn - 1);  // past the end: the last key again, masked below
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int col = 16 * t + 8 * (i & 1) + 64 * (i >> 1);
                    const uint4 kx = __ldg(reinterpret_cast<const uint4*>(kn + (int64_t)key * p.sn_n + col));
                    const uint4 q0 = __ldg(reinterpret_cast<const uint4*>(qrow[0] + col));
                    uint4 q1 = make_uint4(0u, 0u, 0u, 0u);
                    if (TALL) q1 = __ldg(reinterpret_cast<const uint4*>(qrow[kHalves - 1] + col));
                    mma_bf16(acc[kt], q0.x, q1.x, q0.y, q1.y, kx.x, kx.y);
                    mma_bf16(acc[kt], q0.z, q1.z, q0.w, q1.w, kx.z, kx.w);
                }
            }
            uint32_t see[kHalves];  // bit i: this lane's row sees own key j0 + i
            float w[2][2 * kHalves];
#pragma unroll
            for (int h = 0; h < kHalves; ++h) {
                see[h] = node[h] >= 0 ? (uint32_t)(visible_word(p, pc.b, node[h], j0 >> 6) >> (j0 & 63)) & 0xffffu : 0u;
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        w[kt][2 * h + e] = (see[h] >> (8 * kt + 2 * t + e)) & 1u ? acc[kt][2 * h + e] * p.scale_log2
                                                                                : -INFINITY;
            }
            step(w, 1.f);
            uint32_t hi[2][kHalves], lo[2][kHalves];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int h = 0; h < kHalves; ++h) split_bf16(pk2(w[kt][2 * h], w[kt][2 * h + 1]), hi[kt][h], lo[kt][h]);
            bool odd = false;  // a non-finite value among this group's
#pragma unroll
            for (int half = 0; half < 2; ++half) {  // columns 16 g + 8 half .. + 7
                uint32_t x[4][4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = min(j0 + 2 * t + (i & 1) + 8 * (i >> 1), p.nn - 1);
                    const uint4 vx = __ldg(reinterpret_cast<const uint4*>(vn + (int64_t)key * p.sn_n + 16 * g + 8 * half));
                    x[i][0] = vx.x, x[i][1] = vx.y, x[i][2] = vx.z, x[i][3] = vx.w;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        odd |= not_finite_pair(x[i][c]);
                        // 0 times an infinity is not 0: such a value leaves the product and is added below
                        if ((x[i][c] & 0x7f80u) == 0x7f80u) x[i][c] &= 0xffff0000u;
                        if ((x[i][c] & 0x7f800000u) == 0x7f800000u) x[i][c] &= 0xffffu;
                    }
                }
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int j = 8 * half + 2 * c + e;
                        const uint32_t sel = e ? 0x7632 : 0x5410;
                        values(o[j], hi, lo, __byte_perm(x[0][c], x[1][c], sel), __byte_perm(x[2][c], x[3][c], sel));
                    }
            }
            if (__any_sync(MFD_FULL_MASK, odd)) {
                // rare: add the infinities and NaNs to the rows that see their key (a weight is above 0, so their
                // size does not matter): O[row][d] of this lane are d = 32 t + j and 32 t + 16 + j
                for (int i = 0; i < min(16, p.nn - j0); ++i) {
                    const __nv_bfloat16* vrow = vn + (int64_t)(j0 + i) * p.sn_n + 32 * t;
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const float y0 = __bfloat162float(vrow[j]), y1 = __bfloat162float(vrow[16 + j]);
#pragma unroll
                        for (int h = 0; h < kHalves; ++h) {
                            if (!((see[h] >> i) & 1u)) continue;
                            if (!(fabsf(y0) < INFINITY)) o[j][2 * h] += y0;
                            if (!(fabsf(y1) < INFINITY)) o[j][2 * h + 1] += y1;
                        }
                    }
                }
            }
        }

        // ---- the warps of the piece merge
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
            l[h] = quad_sum(l[h]);
            if (t == 0) s_m[warp][g + 8 * h] = m[h], s_l[warp][g + 8 * h] = l[h];
        }
        __syncthreads();
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
            float mm = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, s_m[w][g + 8 * h]);
            const float a = m[h] == -INFINITY ? 0.f : fast_exp2(m[h] - mm);
            float* row = smem + (warp * kRows + g + 8 * h) * kRowStride + t * kTBlock;
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int j = 0; j < 16; j += 4)
                    *reinterpret_cast<float4*>(row + 16 * e + j) =
                        make_float4(o[j][2 * h + e] * a, o[j + 1][2 * h + e] * a, o[j + 2][2 * h + e] * a,
                                    o[j + 3][2 * h + e] * a);
        }
        __syncthreads();
        const int live_rows = min(16, p.rows - base);
        const bool whole = pc.pieces == 1;
        float* slot = p.part + (int64_t)pc.slot * kSlot;
        auto store = [&](int r, int col, float4 v, float mm, float ll) {  // columns col .. col + 3 of row r, and lse
            const float inv = ll > 0.f ? 1.f / ll : (ll == 0.f ? 0.f : ll);
            const int row = base + r, nd = row / p.G, hd = hk * p.G + row % p.G;
            *reinterpret_cast<uint2*>(p.out + (int64_t)pc.b * p.so_b + (int64_t)nd * p.so_n + (int64_t)hd * p.so_h + col) =
                make_uint2(pack_bf16(v.x * inv, v.y * inv), pack_bf16(v.z * inv, v.w * inv));
            if (p.lse && col == 0)
                p.lse[((int64_t)pc.b * p.n + nd) * p.H + hd] = ll == 0.f ? -INFINITY : 0.6931471805599453f * (mm + log2f(ll));
        };
        for (int e = tid; e < live_rows * 32; e += kThreads) {
            const int r = e >> 5, c4 = e & 31;
            float mm = -INFINITY, ll = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, s_m[w][r]);
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float mw = s_m[w][r];
                ll += s_l[w][r] * (mw == -INFINITY ? 0.f : fast_exp2(mw - mm));  // (a NaN sum stays one)
                const float4 x = *reinterpret_cast<const float4*>(smem + (w * kRows + r) * kRowStride + (c4 >> 3) * kTBlock +
                                                                  (c4 & 7) * 4);
                v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
            }
            if (whole) {
                store(r, 4 * c4, v, mm, ll);
            } else {
                if (c4 == 0) slot[r] = mm, slot[16 + r] = ll;
                *reinterpret_cast<float4*>(slot + 32 + r * kD + 4 * c4) = v;
            }
        }
        if (!whole) {
            // ---- the unit's last CTA merges its pieces, in their order
            __threadfence();
            __syncthreads();
            unsigned int* ticket = p.tickets + (int64_t)pc.b * cut.per_req + pc.u;
            if (tid == 0) s_last = atomicAdd(ticket, 1u) == (unsigned)(pc.pieces - 1);
            __syncthreads();
            if (s_last) {
                __threadfence();
                auto record = [&](int i) { return p.part + slot_of(pc, i) * kSlot; };
                float* wgt = smem;  // [pieces][16] weights in turn, the rows' (m, l) in s_m[0], s_l[0]
                constexpr int kBatch = 512;
                float4 v[2];
                v[0] = v[1] = make_float4(0.f, 0.f, 0.f, 0.f);
                for (int r = warp; r < live_rows; r += kWarps) {
                    float mm = -INFINITY;
                    for (int i = lane; i < pc.pieces; i += 32) mm = fmaxf(mm, __ldcg(record(i) + r));
                    mm = warp_max_f32(mm);
                    float ll = 0.f;
                    for (int i = lane; i < pc.pieces; i += 32) {
                        const float mi = __ldcg(record(i) + r);
                        const float a = mi == -INFINITY ? 0.f : fast_exp2(mi - mm);
                        if (i < kBatch) wgt[i * 16 + r] = a;
                        ll += a * __ldcg(record(i) + 16 + r);
                    }
#pragma unroll
                    for (int d = 16; d; d >>= 1) ll += __shfl_xor_sync(MFD_FULL_MASK, ll, d);
                    if (lane == 0) s_m[0][r] = mm, s_l[0][r] = ll;
                }
                __syncthreads();
#pragma unroll
                for (int u = 0; u < kRows * 32 / kThreads; ++u) {
                    const int e = tid + u * kThreads;
                    const int r = e >> 5, c4 = e & 31;
                    if (r < live_rows) {
#pragma unroll 4
                        for (int i = 0; i < pc.pieces; ++i) {
                            const float* sl = record(i);
                            float a;
                            if (i < kBatch) {
                                a = wgt[i * 16 + r];
                            } else {
                                const float mi = __ldcg(sl + r);
                                a = mi == -INFINITY ? 0.f : fast_exp2(mi - s_m[0][r]);
                            }
                            const float4 x = __ldcg(reinterpret_cast<const float4*>(sl + 32 + r * kD + 4 * c4));
                            v[u].x = fmaf(a, x.x, v[u].x), v[u].y = fmaf(a, x.y, v[u].y);
                            v[u].z = fmaf(a, x.z, v[u].z), v[u].w = fmaf(a, x.w, v[u].w);
                        }
                        store(r, 4 * c4, v[u], s_m[0][r], s_l[0][r]);
                    }
                }
                if (tid == 0) *ticket = 0u;
            }
        }
        __syncthreads();  // smem, s_m and s_l are free for the next piece
    }
}

int64_t rows_tickets(int64_t bs, int64_t hkv, int64_t rows) { return bs * hkv * ((rows + 15) / 16); }
size_t rows_workspace(int sms) { return (size_t)sms * kCtasPerSm * 2 * kSlot * sizeof(float); }

template <bool FP8, bool TALL>
static int launch_one(const AttnParams& p, int sms, cudaStream_t stream) {
    constexpr int kSmem = kWarps * (TALL ? 16 : 8) * kRowStride * 4;
    static_assert(kSmem >= 512 * 16 * 4, "the merge weights fit");
    static bool opted[64];
    cudaError_t e = opt_in_smem((const void*)kv8_rows_kernel<FP8, TALL>, kSmem, opted);
    if (e != cudaSuccess) {
        set_error("mfd_kv8_attention: %s", cudaGetErrorString(e));
        return MFD_ERR_CUDA;
    }
    kv8_rows_kernel<FP8, TALL><<<sms * kCtasPerSm, kThreads, kSmem, stream>>>(p);
    MFD_CHECK_LAUNCH("mfd_kv8_attention");
    return MFD_OK;
}

int launch_rows(const AttnParams& p, int sms, cudaStream_t stream) {
    const bool tall = p.rows - p.row0 > 8;
    if (p.fp8) return tall ? launch_one<true, true>(p, sms, stream) : launch_one<true, false>(p, sms, stream);
    return tall ? launch_one<false, true>(p, sms, stream) : launch_one<false, false>(p, sms, stream);
}

}  // namespace kv8
}  // namespace mfd
