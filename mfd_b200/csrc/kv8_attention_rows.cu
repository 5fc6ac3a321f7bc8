// kv8_attention_rows.cu -- attention of a few query rows over the 8-bit paged cache: the decode step and short drafts.
//
// The mathematics, for a row with query q over keys j (page P(j), codes a_j and c_j, scales sk and sv):
//   score  s_j = sk (q . a_j) scale log2(e),      w_j = s_j + log2(sv),      m = max_j w_j - 12
//   O = sum_j 2^(w_j - m) c_j,   l = sum_j 2^(w_j - m - u) / sv,             out = O 2^-u / l,  lse = ln2 (m + u + log2 l)
// so the value scale rides in the exponent and no code is multiplied by its scale.  1 / sv goes from 2^-121 (the largest
// bf16 values) to 2^100 (a page of zeros), the weights to 2^15: with u = 18 no sum of 2^30 of them leaves float32, and one
// key of the largest values is still 22 bits.  The products have float16 operands
// and float32 sums: codes are exact there, and so is the query row divided by a power of two.  The weights go in as
// float16 hi + lo, two tensor instructions, lifted to at most 2^15: 22 bits of a weight, down to 2^-37 of the row's
// largest.  (One float16 or bf16 weight would err by a good part of the output's own rounding.)  The nodes' own bf16
// keys and values are few: float32 products on the CUDA cores, of the keys a row sees, joined at the piece's merge.  All
// sums and statistics are float32.
//
// Bound: bytes (256 codes a token and KV head for 4 G n multiply-adds each); next, instructions: turning the codes into
// operands.  The codes are the wide operand of the tensor instruction and the query rows, which are few, the narrow one,
// in a layout in which a lane's operand registers are its bytes in order:
//   scores   m16n8k16: A = 16 keys, B = 8 query rows; the d index is permuted (lane (g, t) holds d = 32 t .. 32 t + 31 of
//            keys g and g + 8, the query alike)
//   values   m16n8k16: A = 16 columns of the values x 16 keys, B = the weights (the scores' registers transposed by
//            movmatrix); lane (g, t) holds d = 16 g .. 16 g + 15 of keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9 and interleaves
//            the bytes of two keys before they become float16 pairs; column tile j is d = 16 g + 2 j and the next
// A warp takes every eighth group of 16 keys (one page has all 16: one scale), with its own (m, l, O), and copies its codes
// itself, asynchronously, two groups ahead into a ring of its own in shared memory (8 warps x 3 x 4 KB, two CTAs an SM:
// 128 KB in flight; loads straight to registers kept too few bytes in flight).  Nothing in the loop waits for another
// warp.  TMA copies of whole pages ran no faster, and encoding their two tensor maps cost every call 4 us on the host.
// The warps merge in shared memory at the end of the piece.
//
// Split: the tiles of all (request, KV head, 16 rows) units are laid end to end and cut into equal pieces, one per CTA, so
// ragged lengths balance and one long request fills the GPU; the lengths are read on the device.  The nodes' own keys
// belong to a unit's last piece.  A unit cut into pieces is merged by the CTA that finishes last (its partial (m, l, O) in
// the workspace, a ticket per unit; the pieces are added in their order, so the result does not depend on who merges).
// It reads all pieces of its rows together: one after another they took 8 us of the 21 of a request of 4096 tokens (now
// 12.5).
//
// Measured (H 32 over 8 KV heads, one node): a request of 1000 tokens 10 us, launch and latency; 131072 tokens 62 us, 4.3 TB/s;
// 64 requests of 1K - 8K tokens 126 us, 5.1 TB/s of codes, 0.79 of a copy's bandwidth.
#include "kv8_attention.cuh"
#include "tcgen05.cuh"

namespace mfd {
namespace kv8 {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kTile = 16 * kWarps;       // keys the warps take side by side
constexpr int kStages = 3;
constexpr int kStageBytes = 2 * 16 * kD;  // of a warp: 16 rows of K, then of V
constexpr int kRingBytes = kWarps * kStages * kStageBytes;
// floats: a lane's 16 columns, padded so that the 8 lanes of a store hit different banks
constexpr int kDBlock = 20, kRowStride = 8 * kDBlock + 4;
constexpr int kSlot = 16 * (kD + 2);  // floats of a partial: m[16], l[16], O[16][128]
constexpr int kCtasPerSm = 2;
constexpr int kMaxPieces = 512;   // of a unit: at most one a CTA
// What a unit's start and merge, and its own keys, take in tiles (below).  Without them the CTAs that get several short
// requests end last: 64 requests of 1K - 8K tokens 139 us, with them 126; the 4 rows over the pairs of 32 trees of 65 nodes 103
// and 77.
constexpr int kUnitTiles = 4, kOwnTiles = 6;
constexpr float kLift = 12.f;  // the largest weights are 2^12, and up to 2^15 before the reference moves
constexpr float kLazy = 3.f;
constexpr float kUnit = 3.814697265625e-06f, kUnitLog2 = 18.f;  // 2^-u and u
constexpr int kMaxOwn = kRowsMaxOwn;  // own keys a request

// NT: 8-row tiles a unit
template <bool FP8, int NT>
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
    kv8_rows_kernel(const AttnParams p) {
    constexpr int kRows = 8 * NT;
    // the warps' rings; at a piece's end [kWarps][kRows][kRowStride] floats, then the merge weights
    extern __shared__ __align__(128) unsigned char ring[];
    float* smem = reinterpret_cast<float*>(ring);
    __shared__ float s_own[kRows][kMaxOwn];     // scores (log2) of the own keys a row sees, then their weights
    __shared__ uint8_t s_key[kRows][kMaxOwn];   // which keys they are
    __shared__ int s_seen[kRows];               // how many
    __shared__ float s_m[kWarps][kRows], s_l[kWarps][kRows], s_mm[kRows], s_ll[kRows];
    __shared__ uint2 s_q[NT][8][32];  // query operands, the same for every warp (in registers they would spill)
    __shared__ int s_last;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int nrows = p.rows - p.row0;
    const int RB = (nrows + 15) / 16;
    // ---- this CTA's share of the work, in tiles
    // (at least one, for the own keys or to write zeros; of many units, which share CTAs, each counts kUnitTiles more for
    // its start and merge and kOwnTiles for its own keys)
    const int more = p.bs * p.c.Hkv * RB > (int)gridDim.x / 2 ? kUnitTiles + max(0, min(p.nn - 1, kOwnTiles)) : 0;
    auto tiles_of = [&](int len) { return max(1, (len + kTile - 1) / kTile) + more; };
    const Lengths lens(p.c, p.bs);
    const Cut cut = make_cut(lens, tiles_of, p.c.Hkv * RB, gridDim.x);
    int pos, end;
    cut_range(cut, blockIdx.x, pos, end);

    Piece pc;
    while (next_piece(lens, tiles_of, cut, blockIdx.x, pos, end, pc)) {
        const int hk = pc.u / RB, rb = pc.u % RB, len = pc.len;
        const int base = p.row0 + rb * 16;

        // ---- this warp's copies: lane l takes chunk l % 8 of rows l / 8 + 4 i; the page id is read a tile ahead, the scales
        // with the copies, two tiles before they are used
        unsigned char* mine = ring + warp * (kStages * kStageBytes);
        const int64_t lane_off = (int64_t)hk * p.c.sc_h + (int64_t)(lane >> 3) * p.c.sc_t + (lane & 7) * 16;
        auto key_of = [&](int tile) { return tile * kTile + 16 * warp; };
        auto inside = [&](int tile) { return tile < pc.g1 && key_of(tile) < len; };
        auto id_of = [&](int tile) { return inside(tile) ? page_id(p.c, pc.b, key_of(tile) >> p.c.page_shift) : 0; };
        float2 sc0 = make_float2(0.f, 1.f), sc1 = sc0, sc2 = sc0;  // scales of this tile and of the next two
        auto fetch = [&](int tile, int id) {
            float2 sc = make_float2(0.f, 1.f);
            if (inside(tile)) {
                const int64_t off = (int64_t)id * p.c.sc_p + (int64_t)(key_of(tile) & (p.c.page - 1)) * p.c.sc_t + lane_off;
                unsigned char* dst = mine + (tile - pc.g0) % kStages * kStageBytes;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = (lane >> 3) + 4 * i;
                    copy16(dst + chunk_at(r, lane & 7), p.c.k + off + (int64_t)(4 * i) * p.c.sc_t);
                    copy16(dst + 16 * kD + chunk_at(r, lane & 7), p.c.v + off + (int64_t)(4 * i) * p.c.sc_t);
                }
                sc = make_float2(__ldg(p.c.k_scale + (int64_t)id * p.c.Hkv + hk), __ldg(p.c.v_scale + (int64_t)id * p.c.Hkv + hk));
            }
            copies_commit();
            return sc;
        };
        int id = id_of(pc.g0), id_next = id_of(pc.g0 + 1);
        sc0 = fetch(pc.g0, id);
        id = id_of(pc.g0 + 2);
        sc1 = fetch(pc.g0 + 1, id_next);

        // ---- query row g (+ 8 nt) as float16 operands, divided by a power of two; the lane's softmax rows are 2 t, 2 t + 1
        float rf[NT][2];  // score factor of rows 2 t and 2 t + 1: the power of two, the scale and log2(e)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int r = base + 8 * n + g;
            const bool live = r < p.rows;
            const int nd = live ? r / p.G : 0, hd = hk * p.G + (live ? r - nd * p.G : 0);
            const __nv_bfloat16* qrow = p.q + (int64_t)pc.b * p.sq_b + (int64_t)nd * p.sq_n + (int64_t)hd * p.sq_h;
            uint4 x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // columns 32 t + 8 i ..
                x[i] = make_uint4(0u, 0u, 0u, 0u);
                if (live) x[i] = __ldg(reinterpret_cast<const uint4*>(qrow + 32 * t + 8 * i));
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
#pragma unroll
            for (int e = 0; e < 2; ++e) rf[n][e] = __shfl_sync(MFD_FULL_MASK, up, 4 * (2 * t + e)) * p.scale_log2;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float2 f0 = bf2(w[2 * j]), f1 = bf2(w[2 * j + 1]);
                    const int ks = 2 * i + j;
                    if (warp == 0)
                        s_q[n][ks][lane] = make_uint2(pack_half2(f0.x * down, f0.y * down), pack_half2(f1.x * down, f1.y * down));
                }
            }
        }

        __syncthreads();

        // O of rows 2 t, 2 t + 1 (+ 8 n): o[n][j] = d 16 g + 2 j (both rows), then the next d (both rows)
        float o[NT][8][4];
        float m[NT][2], l[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[n][j][e] = 0.f;
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
        }

        // the softmax step of a group: w (log2; -inf where masked) of key g (row 2 t, 2 t + 1), then key g + 8, becomes
        // the weights; O is rescaled when a row's reference moves
        auto step = [&](float (&w)[NT][4], float inv_sv) {
            bool grow = false;
            float mx[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    mx[n][e] = column_max(fmaxf(w[n][e], w[n][2 + e])) - kLift;
                    grow |= mx[n][e] > m[n][e] + kLazy || (m[n][e] == -INFINITY && mx[n][e] > -INFINITY);
                }
            if (__any_sync(MFD_FULL_MASK, grow)) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float mn = fmaxf(m[n][e], mx[n][e]);
                        const float a = m[n][e] == -INFINITY ? 0.f : fast_exp2(m[n][e] - mn);
                        m[n][e] = mn;
                        l[n][e] *= a;
#pragma unroll
                        for (int j = 0; j < 8; ++j) o[n][j][e] *= a, o[n][j][2 + e] *= a;
                    }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float mr = m[n][e] == -INFINITY ? 0.f : m[n][e];
                    w[n][e] = fast_exp2(w[n][e] - mr);
                    w[n][2 + e] = fast_exp2(w[n][2 + e] - mr);
                    l[n][e] = fmaf((w[n][e] + w[n][2 + e]) * kUnit, inv_sv, l[n][e]);
                }
        };

        // ---- scores of the nodes' own keys, while the first tiles are on their way: few products, on the CUDA cores (a
        // second set of tensor instructions for them cost more in instruction fetches than in arithmetic).  A warp takes a
        // row, lists the keys it sees (of a tree's nodes a row sees its ancestors) and gives each eight lanes, 16 columns a
        // lane.  The weights meet the values in the merge below.
        const int live_rows = min(16, p.rows - base);
        const int own = pc.g1 == pc.of ? p.nn : 0;  // of a unit's last piece
        auto own_words = [&](int r) {  // lane w: word w of what the row sees
            return lane < kMaxOwn / 64 ? visible_word(p, pc.b, quotient(base + r, p.G), lane) : 0ull;
        };
#pragma unroll 1
        for (int r = warp; r < kRows; r += kWarps) {
            int seen = 0;
            if (r < live_rows && own > 0) {
                const int nd = quotient(base + r, p.G), hd = hk * p.G + base + r - nd * p.G;
                const int c = lane & 7;
                const uint4* qp = reinterpret_cast<const uint4*>(p.q + (int64_t)pc.b * p.sq_b + (int64_t)nd * p.sq_n +
                                                                 (int64_t)hd * p.sq_h + 16 * c);
                const uint4 q0 = __ldg(qp), q1 = __ldg(qp + 1);
                const uint64_t word = own_words(r);
#pragma unroll 1
                for (int j0 = 0; j0 < own; j0 += 32) {
                    const uint64_t v = __shfl_sync(MFD_FULL_MASK, word, j0 >> 6);
                    const bool sees = (v >> ((j0 & 63) + lane)) & 1ull;
                    const uint32_t m = __ballot_sync(MFD_FULL_MASK, sees);
                    if (sees) s_key[r][seen + __popc(m & ((1u << lane) - 1u))] = (uint8_t)(j0 + lane);
                    seen += __popc(m);
                }
                __syncwarp();
                const __nv_bfloat16* kn = p.kn + (int64_t)pc.b * p.sn_b + (int64_t)hk * p.sn_h + 16 * c;
                const __nv_bfloat16* vn = p.vn + (int64_t)pc.b * p.sn_b + (int64_t)hk * p.sn_h + 16 * c;
#pragma unroll 1
                for (int k0 = 0; k0 < seen; k0 += 16) {  // sixteen keys' loads in flight: their latency is the cost
                    uint4 y[4][2];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int64_t off = (int64_t)s_key[r][min(k0 + 4 * i + (lane >> 3), seen - 1)] * p.sn_n;
                        const uint4* kp = reinterpret_cast<const uint4*>(kn + off);
                        y[i][0] = __ldg(kp), y[i][1] = __ldg(kp + 1);
                        asm volatile("prefetch.global.L2 [%0];" ::"l"(vn + off));  // for the merge
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int k = k0 + 4 * i + (lane >> 3);
                        const uint32_t u[8] = {q0.x, q0.y, q0.z, q0.w, q1.x, q1.y, q1.z, q1.w};
                        const uint32_t v[8] = {y[i][0].x, y[i][0].y, y[i][0].z, y[i][0].w,
                                               y[i][1].x, y[i][1].y, y[i][1].z, y[i][1].w};
                        float dot = 0.f;
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float2 f = bf2(u[j]), h = bf2(v[j]);
                            dot = fmaf(f.x, h.x, fmaf(f.y, h.y, dot));
                        }
#pragma unroll
                        for (int d = 1; d < 8; d <<= 1) dot += __shfl_xor_sync(MFD_FULL_MASK, dot, d);
                        if (c == 0 && k < seen) s_own[r][k] = dot * p.scale_log2;
                        if (k0 + 4 * i + 4 >= seen) break;  // (uniform)
                    }
                }
            }
            if (lane == 0) s_seen[r] = seen;
        }

        // ---- cached tokens
#pragma unroll 1
        for (int tile = pc.g0; tile < pc.g1; ++tile) {
            __syncwarp();  // (every lane has read the stage that the copies below overwrite)
            sc2 = fetch(tile + 2, id);
            id = id_of(tile + 3);
            copies_wait<2>();
            __syncwarp();
            const int key0 = key_of(tile);
            if (key0 >= len) break;
            const bool tail = key0 + 16 > len;
            const unsigned char* kt = mine + (tile - pc.g0) % kStages * kStageBytes;
            uint4 kw[2][2], vw[4];  // K: key g, g + 8; chunk 2 t, 2 t + 1.  V: keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    kw[h][i] = *reinterpret_cast<const uint4*>(kt + chunk_at(g + 8 * h, 2 * t + i));
            const float sv = fmaxf(sc0.y, kScaleFloor), lsv = __log2f(sv), skc = sc0.x;
            sc0 = sc1, sc1 = sc2;
            float acc[NT][4], acc2[NT][4];  // two chains: the instruction's latency is several times its issue
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[n][e] = acc2[n][e] = 0.f;
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) {
                const uint4 x = kw[0][ks >> 2], y = kw[1][ks >> 2];
                const uint32_t wx = (ks & 3) == 0 ? x.x : (ks & 3) == 1 ? x.y : (ks & 3) == 2 ? x.z : x.w;
                const uint32_t wy = (ks & 3) == 0 ? y.x : (ks & 3) == 1 ? y.y : (ks & 3) == 2 ? y.z : y.w;
                uint32_t a0, a1, a2, a3;
                halves<FP8>(wx, a0, a2);
                halves<FP8>(wy, a1, a3);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const uint2 q = s_q[n][ks][lane];
                    mma_f16((ks & 1) ? acc2[n] : acc[n], a0, a1, a2, a3, q.x, q.y);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                vw[i] = *reinterpret_cast<const uint4*>(kt + 16 * kD + chunk_at(2 * t + (i & 1) + 8 * (i >> 1), g));
            float w[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) w[n][e] = fmaf(acc[n][e] + acc2[n][e], skc * rf[n][e & 1], lsv);
            if (tail) {  // slots past the length hold any bits (an e4m3 NaN too): their weight is 0, their codes too
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (key0 + g + 8 * (e >> 1) >= len) w[n][e] = -INFINITY;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (key0 + 2 * t + (i & 1) + 8 * (i >> 1) >= len) vw[i] = make_uint4(0u, 0u, 0u, 0u);
            }
            step(w, __frcp_rn(sv));
            uint32_t hi[NT][2], lo[NT][2];  // keys 0 .. 7 and 8 .. 15: B operands
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    split_half(w[n][2 * h], w[n][2 * h + 1], hi[n][h], lo[n][h]);
                    hi[n][h] = transpose8(hi[n][h]);
                    lo[n][h] = transpose8(lo[n][h]);
                }
            const uint32_t v0[4] = {vw[0].x, vw[0].y, vw[0].z, vw[0].w}, v1[4] = {vw[1].x, vw[1].y, vw[1].z, vw[1].w};
            const uint32_t v2[4] = {vw[2].x, vw[2].y, vw[2].z, vw[2].w}, v3[4] = {vw[3].x, vw[3].y, vw[3].z, vw[3].w};
#pragma unroll
            for (int j2 = 0; j2 < 4; ++j2) {  // d = 16 g + 4 j2 .. + 3: two column tiles
                uint32_t a[4], c[4];           // keys 2 t, 2 t + 1, then 2 t + 8, 2 t + 9, of the four d
                halves<FP8>(__byte_perm(v0[j2], v1[j2], 0x5140), a[0], a[1]);
                halves<FP8>(__byte_perm(v2[j2], v3[j2], 0x5140), c[0], c[1]);
                halves<FP8>(__byte_perm(v0[j2], v1[j2], 0x7362), a[2], a[3]);
                halves<FP8>(__byte_perm(v2[j2], v3[j2], 0x7362), c[2], c[3]);
#pragma unroll
                for (int part = 0; part < 2; ++part)
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int n = 0; n < NT; ++n)
                            mma_f16(o[n][2 * j2 + u], a[2 * u], a[2 * u + 1], c[2 * u], c[2 * u + 1],
                                    part ? lo[n][0] : hi[n][0], part ? lo[n][1] : hi[n][1]);
            }
        }

        copies_wait<0>();
        // ---- the warps of the piece merge: O as it is in shared memory, their weights per row beside it
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = 8 * n + 2 * t + e;
                l[n][e] = column_sum(l[n][e]);
                if (g == 0) s_m[warp][r] = m[n][e], s_l[warp][r] = l[n][e];
            }
        __syncthreads();  // (and every warp is past the ring)
#pragma unroll 1
        for (int r = warp; r < kRows; r += kWarps) {  // a warp a row: the warps' (m, l), then the own keys
            float mm = lane < kWarps ? s_m[lane][r] : -INFINITY;
            const int seen = s_seen[r];
            for (int j = lane; j < seen; j += 32) mm = fmaxf(mm, s_own[r][j]);
            mm = warp_max_f32(mm);
            float ll = 0.f;
            if (lane < kWarps) {
                const float a = s_m[lane][r] == -INFINITY ? 0.f : fast_exp2(s_m[lane][r] - mm);
                ll = s_l[lane][r] * a;  // (a NaN sum stays one)
                s_m[lane][r] = a;
            }
            for (int j = lane; j < seen; j += 32) {
                const float a = s_own[r][j] == -INFINITY ? 0.f : fast_exp2(s_own[r][j] - mm);
                ll = fmaf(a, kUnit, ll);
                s_own[r][j] = a;
            }
#pragma unroll 1
            for (int d = 16; d; d >>= 1) ll += __shfl_xor_sync(MFD_FULL_MASK, ll, d);
            if (lane == 0) s_mm[r] = mm, s_ll[r] = ll;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float* row = smem + (warp * kRows + 8 * n + 2 * t + e) * kRowStride + g * kDBlock;
#pragma unroll
                for (int j = 0; j < 8; j += 2)
                    *reinterpret_cast<float4*>(row + 2 * j) = make_float4(o[n][j][e], o[n][j][2 + e], o[n][j + 1][e],
                                                                          o[n][j + 1][2 + e]);
            }
        __syncthreads();
        const bool whole = pc.pieces == 1;
        float* slot = p.part + (int64_t)pc.slot * kSlot;
        auto store = [&](int r, int col, float4 v, float mm, float ll) {  // columns col .. col + 3 of row r, and lse
            const float inv = ll > 0.f ? kUnit / ll : (ll == 0.f ? 0.f : ll);
            const int row = base + r, nd = row / p.G, hd = hk * p.G + row % p.G;
            *reinterpret_cast<uint2*>(p.out + (int64_t)pc.b * p.so_b + (int64_t)nd * p.so_n + (int64_t)hd * p.so_h + col) =
                make_uint2(pack_bf16(v.x * inv, v.y * inv), pack_bf16(v.z * inv, v.w * inv));
            if (p.lse && col == 0)
                p.lse[((int64_t)pc.b * p.n + nd) * p.H + hd] = ll == 0.f ? -INFINITY : 0.6931471805599453f * (mm + (kUnitLog2 + log2f(ll)));
        };
#pragma unroll 1
        for (int e = tid; e < live_rows * 32; e += kThreads) {
            const int r = e >> 5, c4 = e & 31;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
            for (int w = 0; w < kWarps; ++w) {
                const float a = s_m[w][r];
                const float4 x = *reinterpret_cast<const float4*>(smem + (w * kRows + r) * kRowStride + (c4 >> 2) * kDBlock +
                                                                  (c4 & 3) * 4);
                v.x = fmaf(a, x.x, v.x), v.y = fmaf(a, x.y, v.y), v.z = fmaf(a, x.z, v.z), v.w = fmaf(a, x.w, v.w);
            }
            const __nv_bfloat16* vn = p.vn + (int64_t)pc.b * p.sn_b + (int64_t)hk * p.sn_h + 4 * c4;
            const int seen = s_seen[r];
#pragma unroll 1
            for (int j0 = 0; j0 < seen; j0 += 16) {
                uint2 y[16];
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    y[j] = __ldg(reinterpret_cast<const uint2*>(vn + (int64_t)s_key[r][min(j0 + j, seen - 1)] * p.sn_n));
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    if (j0 + j >= seen) break;
                    const float a = s_own[r][j0 + j];
                    const float2 f = bf2(y[j].x), h = bf2(y[j].y);
                    v.x = fmaf(a, f.x, v.x), v.y = fmaf(a, f.y, v.y), v.z = fmaf(a, h.x, v.z), v.w = fmaf(a, h.y, v.w);
                }
            }
            if (whole) {
                store(r, 4 * c4, v, s_mm[r], s_ll[r]);
            } else {
                if (c4 == 0) slot[r] = s_mm[r], slot[16 + r] = s_ll[r];
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
                auto record = [&](int i) { return p.part + (int64_t)slot_of(pc, i) * kSlot; };
                float* wgt = smem;  // [pieces][16]: the pieces' m, then their weights
                float* sum = smem + kMaxPieces * 16;  // and l
                const int held = pc.pieces * 16;
#pragma unroll 2
                for (int e = tid; e < held; e += kThreads) {
                    const float* rec = record(e >> 4) + (e & 15);
                    wgt[e] = __ldcg(rec), sum[e] = __ldcg(rec + 16);  // (rows that are not live: never used)
                }
                __syncthreads();
#pragma unroll 1
                for (int r = warp; r < live_rows; r += kWarps) {
                    float mm = -INFINITY, ll = 0.f;
                    for (int i = lane; i < pc.pieces; i += 32) mm = fmaxf(mm, wgt[i * 16 + r]);
                    mm = warp_max_f32(mm);
                    for (int i = lane; i < pc.pieces; i += 32) {
                        const float mi = wgt[i * 16 + r], a = mi == -INFINITY ? 0.f : fast_exp2(mi - mm);
                        wgt[i * 16 + r] = a;
                        ll += a * sum[i * 16 + r];
                    }
#pragma unroll
                    for (int d = 16; d; d >>= 1) ll += __shfl_xor_sync(MFD_FULL_MASK, ll, d);
                    if (lane == 0) s_mm[r] = mm, s_ll[r] = ll;
                }
                __syncwarp();
                // (a warp's rows are the same here: warp, and warp + 8)
                if (warp < live_rows) {
                    float4 v[NT];
                    int row[NT];
#pragma unroll
                    for (int u = 0; u < NT; ++u) {
                        v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                        row[u] = min(warp + u * kWarps, live_rows - 1);
                    }
#pragma unroll 8
                    for (int i = 0; i < pc.pieces; ++i) {
                        const float* rec = record(i) + 32 + 4 * lane;
#pragma unroll
                        for (int u = 0; u < NT; ++u) {
                            const float a = wgt[i * 16 + row[u]];
                            const float4 x = __ldcg(reinterpret_cast<const float4*>(rec + row[u] * kD));
                            v[u].x = fmaf(a, x.x, v[u].x), v[u].y = fmaf(a, x.y, v[u].y);
                            v[u].z = fmaf(a, x.z, v[u].z), v[u].w = fmaf(a, x.w, v[u].w);
                        }
                    }
#pragma unroll
                    for (int u = 0; u < NT; ++u) {
                        const int r = warp + u * kWarps;
                        if (r < live_rows) store(r, 4 * lane, v[u], s_mm[r], s_ll[r]);
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

template <bool FP8, int NT>
static int launch_one(const AttnParams& p, int sms, cudaStream_t stream) {
    static_assert(kWarps * 8 * NT * kRowStride * 4 <= kRingBytes && kMaxPieces * 2 * 16 * 4 <= kRingBytes, "the merge fits the ring");
    static bool opted[64];
    cudaError_t e = opt_in_smem((const void*)kv8_rows_kernel<FP8, NT>, kRingBytes, opted);
    if (e != cudaSuccess) {
        set_error("mfd_kv8_attention: %s", cudaGetErrorString(e));
        return MFD_ERR_CUDA;
    }
    const int ctas = sms * kCtasPerSm < kMaxPieces ? sms * kCtasPerSm : kMaxPieces;
    kv8_rows_kernel<FP8, NT><<<ctas, kThreads, kRingBytes, stream>>>(p);
    MFD_CHECK_LAUNCH("mfd_kv8_attention");
    return MFD_OK;
}

int launch_rows(const AttnParams& p, int sms, cudaStream_t stream) {
    const bool tall = p.rows - p.row0 > 8;
    if (p.fp8) return tall ? launch_one<true, 2>(p, sms, stream) : launch_one<true, 1>(p, sms, stream);
    return tall ? launch_one<false, 2>(p, sms, stream) : launch_one<false, 1>(p, sms, stream);
}

}  // namespace kv8
}  // namespace mfd
