// kv8_attention_tc.cu -- attention of many query rows (trees, long drafts) over the 8-bit paged cache on the
// 5th-generation tensor cores (tcgen05 + TMEM).
//
// The mathematics is that of kv8_attention_rows.cu, with every operand in bf16 (the codes, the queries and the nodes'
// own keys and values are exact there; the weights go in as hi + lo, 16 bits of each):
//   S = Q K8^T,  w = sk scale log2(e) S + log2(sv),  P = 2^(w - m) = P_hi + P_lo,  O = P_hi V8 + P_lo V8,
//   l = sum P 2^-u / sv,  out = O 2^-u / l.
//
// Rows r = node * G + g of a (request, KV head) in tiles of 128 (one row per TMEM lane).  Two softmax groups of four
// warps, each with its own S buffer and O accumulator in TMEM, so one group's softmax runs while the other's products
// do:
//   PAIR   a CTA takes two row tiles; each key tile, converted once, feeds 256 rows (group t = row tile t)
//   single a CTA takes one row tile; group t takes every other key tile and the two (m, l, O) merge at the end
// In both, step s is group s & 1; the products run PV(s), S(s + 2) in order.
//
// Warp roles (512 threads, one CTA an SM; the softmax warps take registers from the others: 256 x 152 + 256 x 104 = 512 x
// 128, what the CTA was launched with):
//   warps 0-7    softmax, thread = row, 32 scores at a time from TMEM
//   warps 8-13   converters: raw codes -> bf16 tiles in the 128-byte-swizzled operand layout; the nodes' own keys are
//                copied there (past the end of a request: zeros, whatever the page holds)
//   warp 14      producer: page ids and scales, one TMA load per page and tensor into the raw ring (no multicast)
//   warp 15      MMA issuer
// Shared memory: Q (32 KB a row tile), two K and two V tiles of 32 KB, raw codes 32 KB a stage (K's and V's halves filled
// and freed on their own).  With a second raw stage in the second K tile's place 32 trees of 65 nodes take 401 us, this
// way 388: the next tile's conversion waits neither for the last S nor the next S for it.
//
// Bound: the tensor pipe and shared memory together.  A key tile of 128 costs a pair of row tiles 4 S and 8 PV
// products of 128 x 128 x 64, 3072 cycles of the tensor pipe at its bf16 rate, and about the same of the
// 128 B/clk shared-memory port (operands 256 KB, conversion 96 KB, raw codes 32 KB); the exponentials are 2048.  A tile
// takes about 6000: the products of a group, its softmax and the next products follow one another, and two groups fill
// half of the gaps.  Sixteen softmax warps instead of eight (two a row quarter) ran 5% slower, and so did loads of the next
// scores ahead of the exponentials.
//
// Measured (H 32 over 8 KV heads): 64 nodes, 32 requests of 1K - 8K tokens 250 us with the combination, 0.59 PFLOP/s of
// 4 D flop a score (0.89 with the second product of the weights); 65 nodes, one request of 4096 tokens 31 us, 21 of them here.
//
// Split: as in kv8_attention_rows.cu, in key tiles of 128: equal ranges of all units' tiles laid end to end, or at most
// one piece a CTA when there are few units.  Pieces leave (m, l, O) and kv8_combine_kernel adds them in order, spread
// over the GPU (one CTA reading all pieces of 256 rows would take longer than the attention at batch 1).
//
// Every mbarrier wait is bounded; a CTA whose wait gave up records status 1, stops and releases its TMEM.
#include "kv8_attention.cuh"
#include "tcgen05.cuh"

namespace mfd {
namespace kv8 {

namespace {

__device__ int gave_up;  // sticky, of all calls on the device

constexpr int kTcThreads = 512;
constexpr int kConv = 6;                 // converter warps
constexpr int kSoftmaxRegs = 152, kOtherRegs = 104;
constexpr int kKt = 128;                 // keys per tile
constexpr int kTileBytes = kKt * kD * 2;  // 32 KB: a bf16 tile, [2 d-halves][128 rows][128 B]
constexpr int kRawBytes = 2 * kKt * kD;   // 32 KB: the codes of K and V
constexpr uint32_t kTries = 1u << 20;
// How far (log2) a score may pass its row's reference within a tile, and the unit of l, 2^u.  1 / sv goes up to 2^100 (a page
// of zeros): the 128 weights of a tile sum to at most 2^(7 + 30 + 100 - 12), those of 2^30 keys in all, within 2^8 of their
// references, to 2^(30 + 8 + 100 - 12), and a key of the largest bf16 values still counts with 16 bits.
constexpr float kFar = 30.f;
constexpr float kUnit = 0.000244140625f, kUnitLog2 = 12.f;  // 2^-u and u
// Tiles of a unit as the cut counts them.  Many units share CTAs, and there a unit counts kUnitTiles more than it has, for
// its queries and its epilogue: otherwise the CTAs that get several short requests end last (32 trees of 65 nodes over 1K
// - 8K tokens 273 us, this way 237).
constexpr int kUnitTiles = 3;
__device__ __forceinline__ int counted_tiles(const AttnParams& p, int len, int units, int ctas) {
    return max(1, (len + kKt - 1) / kKt + (p.nn + kKt - 1) / kKt) + (units > ctas / 2 ? kUnitTiles : 0);
}

// What the producer says of a tile beside its page constants.
struct TileConst {
    float factor[8];  // score factors of its 8 groups, where not all are positive (their constants say 1 then)
    int turned;       // whether that is so
    int pad[3];
};

template <bool PAIR>
struct Layout {
    static constexpr int kRowTiles = PAIR ? 2 : 1;
    static constexpr int kStages = PAIR ? 1 : 2;  // of raw codes; K's and V's halves are filled and freed on their own
    static constexpr int kRing = 8;  // tiles of page constants kept (the producer is at most kStages + 3 ahead of a softmax warp)
    static constexpr int kOffQ = 0;
    static constexpr int kOffK = kOffQ + kRowTiles * kTileBytes;
    static constexpr int kOffV = kOffK + 2 * kTileBytes;
    static constexpr int kOffRaw = kOffV + 2 * kTileBytes;
    static constexpr int kOffConst = kOffRaw + kStages * kRawBytes;  // [kRing][8 groups][4] floats: c, d, 2^-u / sv
    static constexpr int kOffTile = kOffConst + kRing * 8 * 4 * 4;  // [kRing] TileConst
    static constexpr int kOffBar = kOffTile + kRing * (int)sizeof(TileConst);
    static constexpr int kUsed = kOffBar + 512;
    static constexpr int kBytes = kUsed + 1024;  // the base is aligned to 1024 by hand
    static_assert(kBytes <= 227 * 1024, "shared memory");
    // barriers; two of each kind that follows the K and V halves of a stage or two buffers
    static constexpr int kQFull = 0;
    static constexpr int kRawFull = 1;  // + 2 stage + (0: K, 1: V)
    static constexpr int kRawEmpty = kRawFull + 2 * kStages;
    static constexpr int kKFull = kRawEmpty + 2 * kStages;
    static constexpr int kKEmpty = kKFull + 2;
    static constexpr int kVFull = kKEmpty + 2;
    static constexpr int kVEmpty = kVFull + 2;
    static constexpr int kSFull = kVEmpty + 2;
    static constexpr int kPFull = kSFull + 2;
    static constexpr int kPV = kPFull + 2;
    static constexpr int kBars = kPV + 2;
    static_assert(8 * kBars + 32 <= 512, "barriers");
};

constexpr int kSlotRows(bool pair) { return pair ? 256 : 128; }
// floats of a partial: m, l per row, then O as float4 chunks, chunk-major (a warp stores 512 contiguous bytes)
constexpr int64_t kSlotFloats(bool pair) { return (int64_t)kSlotRows(pair) * (2 + kD); }

// One lane of the warp (elected), and the tensor-core instructions issued by it alone while the warp stays together.
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r;
}
__device__ __forceinline__ void umma_if(uint32_t leader, uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, l;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 l, %5, 0;\n\t"
        "@l tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(leader));
}
__device__ __forceinline__ void umma_ts_if(uint32_t leader, uint32_t d_tmem, uint32_t a_tmem, uint64_t b, uint32_t idesc,
                                           uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, l;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 l, %5, 0;\n\t"
        "@l tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b), "r"(idesc), "r"(acc), "r"(leader));
}
__device__ __forceinline__ void commit_if(uint32_t leader, uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred l;\n\tsetp.ne.b32 l, %1, 0;\n\t"
        "@l tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_addr(bar)),
        "r"(leader)
        : "memory");
}

// A TMEM store is asynchronous: whoever reads what it wrote (a later load of the same warp too) waits for it first.
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// What a piece's tiles are (of 128 keys: cached tokens first, then the nodes' own).
struct Tiles {
    int hk, rb;       // KV head, block of rows
    int tp, t1;       // tiles of cached tokens of the request; end of the piece's
    int ntiles;       // the piece's
    int row_base, ntl;  // first row, row tiles in use
    bool alternate;   // key tiles alternate between the groups, which share the rows
    int nsteps;
    uint32_t n_piece, n_tile, n_s0, n_s1;  // pieces, tiles and the groups' steps before
};

template <bool FP8, bool PAIR>
__global__ void __launch_bounds__(kTcThreads, 1)
    kv8_tc_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv, const AttnParams p) {
    using L = Layout<PAIR>;
    constexpr int kStages = L::kStages;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    const uint32_t pad = (1024u - (smem_addr(smem_raw) & 1023u)) & 1023u;
    unsigned char* smem = smem_raw + pad;
    const uint32_t sbase = smem_addr(smem);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kOffBar);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kOffBar + 8 * L::kBars);
    volatile int* s_failed = reinterpret_cast<volatile int*>(smem + L::kOffBar + 8 * L::kBars + 4);
    volatile int* s_odd = s_failed + 1;  // a non-finite own value was met in this piece
    float4* consts = reinterpret_cast<float4*>(smem + L::kOffConst);
    TileConst* tile_consts = reinterpret_cast<TileConst*>(smem + L::kOffTile);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        mbar_init(&bars[L::kQFull], 8);
        for (int i = 0; i < 2 * kStages; ++i) {
            mbar_init(&bars[L::kRawFull + i], 32);
            mbar_init(&bars[L::kRawEmpty + i], kConv);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars[L::kKFull + i], kConv);
            mbar_init(&bars[L::kKEmpty + i], 1);
            mbar_init(&bars[L::kVFull + i], kConv);
            mbar_init(&bars[L::kVEmpty + i], 1);
            mbar_init(&bars[L::kSFull + i], 1);
            mbar_init(&bars[L::kPFull + i], 4);
            mbar_init(&bars[L::kPV + i], 1);
        }
        *s_failed = 0;
        *s_odd = 0;
        mbar_fence_init();
    }
    if (warp == 15) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the combination may be set up (it waits for this grid's end)
    // TMEM columns: O of group t at 128 t, S of group t at 256 + 128 t
    const int RB = (p.rows - p.row0 + 128 * L::kRowTiles - 1) / (128 * L::kRowTiles);
    auto tiles_of = [&](int len) { return counted_tiles(p, len, p.bs * p.c.Hkv * RB, gridDim.x); };
    const Lengths lens(p.c, p.bs);
    const Cut cut = make_cut(lens, tiles_of, p.c.Hkv * RB, gridDim.x);
    int pos, end;
    cut_range(cut, blockIdx.x, pos, end);

    // Every role walks the CTA's pieces in its own loop (below), all meeting at the end of each.
    bool ok = true;
    uint32_t issued = 0;  // producer: raw stages filled
    auto pieces = [&](auto body) {
        uint32_t n_piece = 0, n_tile = 0, n_s[2] = {0u, 0u};  // running counts: the barriers' phases
        Piece pc;
        while (next_piece(lens, tiles_of, cut, blockIdx.x, pos, end, pc)) {
            Tiles x;
            x.hk = pc.u / RB, x.rb = pc.u % RB;
            x.tp = (pc.len + kKt - 1) / kKt;
            x.t1 = min(pc.g1, x.tp + (p.nn + kKt - 1) / kKt);  // (counted tiles that there are not are empty)
            x.ntiles = max(0, x.t1 - pc.g0);
            x.row_base = p.row0 + x.rb * 128 * L::kRowTiles;
            x.ntl = PAIR ? (p.rows - x.row_base > 128 ? 2 : 1) : 1;
            x.alternate = !PAIR || x.ntl == 1;
            x.nsteps = x.alternate ? x.ntiles : 2 * x.ntiles;
            x.n_piece = n_piece, x.n_tile = n_tile, x.n_s0 = n_s[0], x.n_s1 = n_s[1];
            body(pc, x);
            __syncwarp();
            if (!ok) *s_failed = 1;
            tc_fence_before();
            bar_sync<kTcThreads>(0);  // the piece is over for every role
            tc_fence_after();
            if (*s_failed) break;
            n_piece += 1, n_tile += x.ntiles;
            n_s[0] += (x.nsteps + 1) >> 1, n_s[1] += x.nsteps >> 1;
            if (tid == 0) *s_odd = 0;
            bar_sync<kTcThreads>(0);
        }
    };

    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        pieces([&](const Piece& pc, const Tiles& x) {
            // ------------------------------------------------------------ queries into their operand layout
            // (asynchronous copies, all in flight together; a rolled loop, since the code is cold)
#pragma unroll 1
            for (int r = tid >> 4; r < 128 * x.ntl; r += 16) {
                const int row = x.row_base + r, c = tid & 15;
                unsigned char* dst = smem + L::kOffQ + (r >> 7) * kTileBytes + sw128_offset(r & 127, c * 8, 128);
                if (row < p.rows) {
                    const int node = quotient(row, p.G);
                    copy16(dst, p.q + (int64_t)pc.b * p.sq_b + (int64_t)node * p.sq_n +
                                    (int64_t)(x.hk * p.G + row - node * p.G) * p.sq_h + c * 8);
                } else {
                    *reinterpret_cast<uint4*>(dst) = make_uint4(0u, 0u, 0u, 0u);
                }
            }
            copies_commit();
            copies_wait<0>();
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars[L::kQFull]);

            // ------------------------------------------------------------ softmax
            const int grp = warp >> 2, quarter = warp & 3;
            const int rt = quarter * 32 + lane;
            const int row = x.row_base + (x.alternate ? 0 : 128 * grp) + rt;
            const bool live = row < p.rows;
            const bool quarter_live = row - lane < p.rows;
            const int node = live ? row / p.G : 0;
            const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
            const uint32_t s_tm = tmem + lane_off + 256 + 128 * grp, o_tm = tmem + lane_off + 128 * grp;
            // O and l are relative to 2^m; m_next is what m should be (the tiles' maxima).  A tile's weights are formed
            // in one pass against the m of the tiles before it, which bf16's range allows: m only follows when the
            // maximum has passed it by 2^8, before the next tile, and at once where a chunk passes it by 2^kFar.
            float m = -INFINITY, m_next = -INFINITY, l = 0.f;
            int done = 0;  // steps of this group
            auto rescale_o = [&](float alpha) {  // (S of this step is there, so the group's last product is complete)
#pragma unroll 1
                for (int oc = 0; oc < kD; oc += 32) {
                    float o[32];
                    tmem_ld32(o_tm + oc, o);
#pragma unroll
                    for (int j = 0; j < 32; ++j) o[j] *= alpha;
                    tmem_st32(o_tm + oc, o);
                }
                tmem_st_wait();  // (a second rescaling in the step reads O again)
            };
            for (int s = grp; s < x.nsteps; s += 2, ++done) {
                const int tile = pc.g0 + (x.alternate ? s : s >> 1);
                ok = __all_sync(MFD_FULL_MASK, ok & mbar_wait(&bars[L::kSFull + grp], ((grp ? x.n_s1 : x.n_s0) + done) & 1, kTries));
                tc_fence_after();
                if (quarter_live && ok) {
                    const float4* cst = consts + (size_t)((x.n_tile + tile - pc.g0) % L::kRing) * 8;
                    const TileConst& tc = tile_consts[(x.n_tile + tile - pc.g0) % L::kRing];
                    if (tc.turned) {
                        // rare: a factor that is not positive (a K scale of 0, a softmax scale of 0 or below) goes in before the
                        // maximum, which it would turn over, and before the mask, which it would turn into NaN (-inf * 0)
#pragma unroll 1
                        for (int c = 0; c < 4; ++c) {
                            float v[32];
                            tmem_ld32(s_tm + 32 * c, v);
#pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] *= tc.factor[2 * c + (j >> 4)];
                            tmem_st32(s_tm + 32 * c, v);
                        }
                        tmem_st_wait();
                    }
                    // visibility of the tile's keys, 32 a word
                    const int valid = pc.len - tile * kKt;
                    const bool masked = tile >= x.tp || valid < kKt;
                    auto visible = [&](int c) -> uint32_t {
                        if (tile < x.tp)
                            return valid >= 32 * c + 32 ? ~0u : (valid <= 32 * c ? 0u : (1u << (valid - 32 * c)) - 1u);
                        const uint64_t v = live ? visible_word(p, pc.b, node, 2 * (tile - x.tp) + (c >> 1)) : 0ull;
                        return (uint32_t)(v >> (32 * (c & 1)));
                    };
                    const bool behind = m_next > m + 8.f;
                    if (__any_sync(MFD_FULL_MASK, behind)) {
                        const float alpha = behind ? fast_exp2(m - m_next) : 1.f;  // (m is finite: see below)
                        if (behind) m = m_next;
                        l *= alpha;
                        rescale_o(alpha);
                    }
                    uint64_t acc[2] = {0ull, 0ull};
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {  // (rolled: an unrolled step misses the instruction cache)
                        uint32_t u[1][32];
                        tmem_ld32_issue(s_tm + 32 * c, u[0]);
                        tmem_ld_wait(u);
                        if (masked) {
                            const uint32_t vis = visible(c);
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (!((vis >> j) & 1u)) u[0][j] = 0xff800000u;
                        }
                        const float4 k0 = cst[2 * c], k1 = cst[2 * c + 1];  // of 16 keys: one page
                        float top[2];
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            float a[6];
#pragma unroll
                            for (int j = 0; j < 5; ++j)
                                a[j] = fmax3(__uint_as_float(u[0][16 * q + 3 * j]), __uint_as_float(u[0][16 * q + 3 * j + 1]),
                                             __uint_as_float(u[0][16 * q + 3 * j + 2]));
                            a[5] = __uint_as_float(u[0][16 * q + 15]);
                            top[q] = fmaxf(fmax3(a[0], a[1], a[2]), fmax3(a[3], a[4], a[5]));
                        }
                        const float mx = fmaxf(top[0] == -INFINITY ? top[0] : fmaf(top[0], k0.x, k0.y),
                                               top[1] == -INFINITY ? top[1] : fmaf(top[1], k1.x, k1.y));
                        m_next = fmaxf(m_next, mx);
                        const bool far = mx > m + kFar;
                        if (__any_sync(MFD_FULL_MASK, far)) {
                            // a row's first keys, or scores that leap: the reference moves now, by a power of two, so that the
                            // weights already written scale exactly
                            const float up = far ? (m == -INFINITY ? mx : m + ceilf(mx - m)) : m;
                            const float alpha = up == m ? 1.f : fast_exp2(m - up);
                            m = up;
                            l *= alpha;
                            acc[0] = mul2(acc[0], dup2(alpha)), acc[1] = mul2(acc[1], dup2(alpha));
                            if (done >= 1) rescale_o(alpha);
                            const __nv_bfloat162 a2 = __float2bfloat162_rn(alpha);
                            tmem_st_wait();  // the weights of the chunks before are read again
#pragma unroll 1
                            for (int d = 0; d < c; ++d) {
                                uint32_t w[1][32];
                                tmem_ld32_issue(s_tm + 32 * d, w[0]);
                                tmem_ld_wait(w);
#pragma unroll
                                for (int j = 0; j < 32; ++j) {
                                    const __nv_bfloat162 v = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&w[0][j]), a2);
                                    w[0][j] = *reinterpret_cast<const uint32_t*>(&v);
                                }
                                tmem_st32u(s_tm + 32 * d, w[0]);
                            }
                        }
                        const float mr = m == -INFINITY ? 0.f : m;
                        uint32_t hl[32];  // hi pairs, then lo pairs
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            const float4 k = q ? k1 : k0;
                            const uint64_t kc = dup2(k.x), kd = dup2(k.y - mr), ki = dup2(k.z);
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                const int e = 16 * q + 2 * j;
                                float x0, x1;
                                upk2(fma2(pk2(__uint_as_float(u[0][e]), __uint_as_float(u[0][e + 1])), kc, kd), x0, x1);
                                const uint64_t w = pk2(fast_exp2(x0), fast_exp2(x1));
                                acc[j & 1] = fma2(w, ki, acc[j & 1]);
                                split_bf16(w, hl[8 * q + j], hl[16 + 8 * q + j]);
                            }
                        }
                        tmem_st32u(s_tm + 32 * c, hl);  // over the 32 scores they come from
                    }
                    float a0, a1;
                    upk2(add2(acc[0], acc[1]), a0, a1);
                    l += a0 + a1;
                    tmem_st_wait();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars[L::kPFull + grp]);
                if (!ok) break;
            }
            // ------------------------------------------------------------ epilogue
            if (done > 0 && ok) {
                ok = __all_sync(MFD_FULL_MASK, mbar_wait(&bars[L::kPV + grp], ((grp ? x.n_s1 : x.n_s0) + done - 1) & 1, kTries));
                tc_fence_after();
            }
            // x.alternate: the two groups' (m, l) of a row meet in the raw ring (every code is converted by now), and each
            // group finishes 64 columns
            // (l and O come down to the tiles' maximum first: m may be 2^kFar below it)
            const float f_late = m_next > m && m != -INFINITY ? fast_exp2(m - m_next) : 1.f;
            if (m != -INFINITY) m = fmaxf(m, m_next);
            l *= f_late;
            float m_fin = m, l_fin = l, f_own = 1.f, f_oth = 0.f, f_oth_late = 1.f;
            if (x.alternate) {
                float* xch = reinterpret_cast<float*>(smem + L::kOffRaw);
                bar_sync<256>(1);  // (a group without a step has waited for nothing: the other's last product has)
                xch[grp * 128 + rt] = m;
                xch[256 + grp * 128 + rt] = l;
                xch[512 + grp * 128 + rt] = f_late;
                tc_fence_before();
                bar_sync<256>(1);  // (both groups' products are complete: each waited for its own)
                tc_fence_after();
                const float mo = xch[(1 - grp) * 128 + rt], lo = xch[256 + (1 - grp) * 128 + rt];
                f_oth_late = xch[512 + (1 - grp) * 128 + rt];
                m_fin = fmaxf(m, mo);
                f_own = m == -INFINITY ? 0.f : fast_exp2(m - m_fin);
                f_oth = mo == -INFINITY ? 0.f : fast_exp2(mo - m_fin);
                l_fin = l * f_own + lo * f_oth;
                fence_proxy_async_smem();  // (the next piece's copies land here)
            }
            const bool own_used = done > 0, oth_used = x.alternate && (grp == 0 ? x.nsteps > 1 : x.nsteps > 0);
            const bool odd = *s_odd != 0;
            const int own0 = max(pc.g0 - x.tp, 0) * kKt, own1 = min(p.nn, (x.t1 - x.tp) * kKt);  // own keys of this piece
            if (quarter_live && ok) {
                const float inv = l_fin > 0.f ? kUnit / l_fin : (l_fin == 0.f ? 0.f : l_fin);
                const int c_lo = x.alternate ? 64 * grp : 0, c_hi = x.alternate ? c_lo + 64 : kD;
                float* slot = p.part + (int64_t)pc.slot * kSlotFloats(PAIR);
                const int srow = (x.alternate ? 0 : 128 * grp) + rt;
                if (c_lo == 0) {
                    if (pc.pieces > 1) {
                        slot[srow] = m_fin;
                        slot[kSlotRows(PAIR) + srow] = l_fin;
                    } else if (live && p.lse) {
                        p.lse[((int64_t)pc.b * p.n + node) * p.H + x.hk * p.G + row % p.G] =
                            l_fin == 0.f ? -INFINITY : 0.6931471805599453f * (m_fin + (kUnitLog2 + log2f(l_fin)));
                    }
                }
#pragma unroll 1
                for (int oc = c_lo; oc < c_hi; oc += 32) {
                    float o[32];
#pragma unroll
                    for (int j = 0; j < 32; ++j) o[j] = 0.f;
                    if (own_used) {
                        tmem_ld32(o_tm + oc, o);
#pragma unroll
                        for (int j = 0; j < 32; ++j) o[j] = o[j] * f_late * f_own;
                    }
                    if (oth_used) {
                        float o2[32];
                        tmem_ld32(tmem + lane_off + 128 * (1 - grp) + oc, o2);
#pragma unroll
                        for (int j = 0; j < 32; ++j) o[j] = fmaf(o2[j] * f_oth_late, f_oth, o[j]);
                    }
                    if (odd && live) {  // rare: infinities and NaNs of the own values the row sees
                        for (int key = own0; key < own1; ++key) {
                            if (!((visible_word(p, pc.b, node, key >> 6) >> (key & 63)) & 1ull)) continue;
                            const __nv_bfloat16* vr = p.vn + (int64_t)pc.b * p.sn_b + (int64_t)key * p.sn_n +
                                                      (int64_t)x.hk * p.sn_h + oc;
#pragma unroll
                            for (int j = 0; j < 32; ++j) {
                                const float y = __bfloat162float(vr[j]);
                                if (!(fabsf(y) < INFINITY)) o[j] += y;
                            }
                        }
                    }
                    if (pc.pieces > 1) {
                        float4* dst = reinterpret_cast<float4*>(slot + 2 * kSlotRows(PAIR));
#pragma unroll
                        for (int j = 0; j < 32; j += 4)
                            dst[((oc + j) >> 2) * kSlotRows(PAIR) + srow] = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
                    } else if (live) {
                        uint4* dst = reinterpret_cast<uint4*>(p.out + (int64_t)pc.b * p.so_b + (int64_t)node * p.so_n +
                                                              (int64_t)(x.hk * p.G + row % p.G) * p.so_h + oc);
#pragma unroll
                        for (int j = 0; j < 32; j += 8)
                            dst[j >> 3] = make_uint4(pack_bf16(o[j] * inv, o[j + 1] * inv), pack_bf16(o[j + 2] * inv, o[j + 3] * inv),
                                                     pack_bf16(o[j + 4] * inv, o[j + 5] * inv),
                                                     pack_bf16(o[j + 6] * inv, o[j + 7] * inv));
                    }
                }
            }
            tc_fence_before();
        });
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp < 8 + kConv) {
            pieces([&](const Piece& pc, const Tiles& x) {
            // ------------------------------------------------------------ converters
            const int cw = warp - 8;
            for (int i = 0; i < x.ntiles && ok; ++i) {
                const int tile = pc.g0 + i;
                const uint32_t nr = x.n_tile + i, st = nr % kStages;
#pragma unroll 1
                for (int which = 0; which < 2 && ok; ++which) {  // K, then V
                    ok &= mbar_wait(&bars[L::kRawFull + 2 * st + which], (nr / kStages) & 1, kTries);
                    const int buf = which * 2 + (int)(nr & 1);
                    if (nr >= 2) ok &= mbar_wait(&bars[(which ? L::kVEmpty : L::kKEmpty) + (nr & 1)], ((nr >> 1) - 1) & 1, kTries);
                    unsigned char* dst = smem + L::kOffK + buf * kTileBytes;
                    ok = __all_sync(MFD_FULL_MASK, ok);
                    if (!ok) break;
                    if (tile < x.tp) {
                        const int valid = min(kKt, pc.len - tile * kKt);
                        const unsigned char* src = smem + L::kOffRaw + st * kRawBytes + which * (kRawBytes / 2);
                        const int c = lane & 7, h = c >> 2, q = 2 * (c & 3);
                        constexpr int kMine = (32 + kConv - 1) / kConv;  // groups of 4 rows (8 16-byte chunks each) a warp
                        uint4 raw[kMine];                                // all loads first: one latency, not six
#pragma unroll
                        for (int i = 0; i < kMine; ++i) {
                            const int r = (cw + kConv * i) * 4 + (lane >> 3);
                            raw[i] = make_uint4(0u, 0u, 0u, 0u);
                            if (r < valid) raw[i] = *reinterpret_cast<const uint4*>(src + r * kD + c * 16);
                        }
#pragma unroll
                        for (int i = 0; i < kMine; ++i) {
                            const int r = (cw + kConv * i) * 4 + (lane >> 3);
                            if (r >= kKt) break;  // (uniform: whole groups)
                            uint4 y0, y1;
                            bfloats<FP8>(raw[i].x, y0.x, y0.y);
                            bfloats<FP8>(raw[i].y, y0.z, y0.w);
                            bfloats<FP8>(raw[i].z, y1.x, y1.y);
                            bfloats<FP8>(raw[i].w, y1.z, y1.w);
                            unsigned char* base = dst + h * (kTileBytes / 2) + r * 128;
                            // chunks q and q + 1; the upper half's lanes store them in the other order, so the eight
                            // lanes of a row hit eight different bank groups
                            const int first = h ? q + 1 : q, second = h ? q : q + 1;
                            *reinterpret_cast<uint4*>(base + ((first ^ (r & 7)) << 4)) = h ? y1 : y0;
                            *reinterpret_cast<uint4*>(base + ((second ^ (r & 7)) << 4)) = h ? y0 : y1;
                        }
                    } else {  // the nodes' own rows; a non-finite value leaves the product (0 times it is not 0)
                        const __nv_bfloat16* src = (which ? p.vn : p.kn) + (int64_t)pc.b * p.sn_b + (int64_t)x.hk * p.sn_h;
                        const int key0 = (tile - x.tp) * kKt;
                        bool odd = false;
#pragma unroll 4
                        for (int j = cw; j < 64; j += kConv) {
                            const int r = 2 * j + (lane >> 4), c = lane & 15;
                            uint4 cw4 = make_uint4(0u, 0u, 0u, 0u);
                            if (key0 + r < p.nn)
                                cw4 = __ldg(reinterpret_cast<const uint4*>(src + (int64_t)(key0 + r) * p.sn_n + c * 8));
                            if (which) {
                                uint32_t v[4] = {cw4.x, cw4.y, cw4.z, cw4.w};
#pragma unroll
                                for (int u = 0; u < 4; ++u) {
                                    if ((v[u] & 0x7f80u) == 0x7f80u) v[u] &= 0xffff0000u, odd = true;
                                    if ((v[u] & 0x7f800000u) == 0x7f800000u) v[u] &= 0xffffu, odd = true;
                                }
                                cw4 = make_uint4(v[0], v[1], v[2], v[3]);
                            }
                            *reinterpret_cast<uint4*>(dst + sw128_offset(r, c * 8, 128)) = cw4;
                        }
                        if (odd) *s_odd = 1;
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(&bars[(which ? L::kVFull : L::kKFull) + (nr & 1)]);
                        mbar_arrive(&bars[L::kRawEmpty + 2 * st + which]);
                    }
                }
            }
            });
        } else if (warp == 14) {
            pieces([&](const Piece& pc, const Tiles& x) {
            // ------------------------------------------------------------ producer
            const int ppt = kKt >> p.c.page_shift;  // pages per tile; lane j < ppt takes page j
            const int gpp = p.c.page >> 4;
            auto id_of = [&](int tile) {
                const int pg = tile * ppt + lane;
                return (lane < ppt && tile < x.tp && (pg << p.c.page_shift) < pc.len) ? page_id(p.c, pc.b, pg) : -1;
            };
            int id = id_of(pc.g0);
            for (int i = 0; i < x.ntiles && ok; ++i) {
                const int tile = pc.g0 + i;
                const uint32_t nr = x.n_tile + i, st = nr % kStages;
                const int id_next = i + 1 < x.ntiles ? id_of(tile + 1) : -1;
                float4* cst = consts + (size_t)(nr % L::kRing) * 8;
#pragma unroll 1
                for (int which = 0; which < 2; ++which) {
                    uint64_t* bar = &bars[L::kRawFull + 2 * st + which];
                    if (nr >= (uint32_t)kStages)
                        ok = __all_sync(MFD_FULL_MASK, ok & mbar_wait(&bars[L::kRawEmpty + 2 * st + which], (nr / kStages - 1) & 1, kTries));
                    if (!ok) break;
                    if (id >= 0) {
                        const uint32_t bytes = (uint32_t)(p.c.page * kD);
                        mbar_expect_tx(bar, bytes);
                        tma_page(sbase + L::kOffRaw + st * kRawBytes + which * (kRawBytes / 2) + lane * bytes, which ? &tmv : &tmk,
                                 bar, x.hk, id);
                    }
                    if (which == 0) {
                        float4 k = make_float4(p.scale_log2, 0.f, kUnit, 0.f);  // own keys, or behind the request's end
                        if (id >= 0) {
                            const float sk = __ldg(p.c.k_scale + (int64_t)id * p.c.Hkv + x.hk);
                            const float sv = fmaxf(__ldg(p.c.v_scale + (int64_t)id * p.c.Hkv + x.hk), kScaleFloor);
                            k = make_float4(sk * p.scale_log2, __log2f(sv), __frcp_rn(sv) * kUnit, 0.f);
                        }
                        TileConst& tc = tile_consts[nr % L::kRing];
                        const bool turned = __any_sync(MFD_FULL_MASK, !(k.x > 0.f));
                        const float factor = k.x;
                        if (turned) k.x = 1.f;
                        if (lane < ppt)
                            for (int g = 0; g < gpp; ++g) {
                                cst[lane * gpp + g] = k;
                                if (turned) tc.factor[lane * gpp + g] = factor;
                            }
                        if (lane == 0) tc.turned = turned;
                    }
                    // the lanes without a page arrive last (lanes 8 .. 31 never have one), after every constant is stored
                    __syncwarp();
                    if (id < 0) mbar_arrive(bar);
                }
                if (!ok) break;
                id = id_next;
                issued = nr + 1;
            }
            });
            if (*s_failed)  // copies in flight end before the CTA does (bounded)
                for (uint32_t f = issued > kStages ? issued - kStages : 0u; f < issued; ++f)
                    for (int which = 0; which < 2; ++which)
                        mbar_wait(&bars[L::kRawFull + 2 * (f % kStages) + which], (f / kStages) & 1, 1u << 14);
        } else {
            // The whole warp walks the steps and one elected lane issues, by predicate: control flow and descriptors stay
            // uniform, so the operands of an instruction are immediates and uniform registers (a single lane in a branch of
            // its own spent three times the products' duration on moving them there).
            constexpr uint32_t kIdescS = idesc_bf16(128, kKt, 0);
            constexpr uint32_t kIdescO = idesc_bf16(128, kD, 1);
            const uint32_t leader = elect_one();
            const uint64_t qd = sdesc(sbase + L::kOffQ, 16, 1024), kd = sdesc(sbase + L::kOffK, 16, 1024);
            const uint64_t vd = sdesc(sbase + L::kOffV, kTileBytes / 2, 1024);
            pieces([&](const Piece&, const Tiles& x) {
                auto wait = [&](int bar, uint32_t parity) {
                    ok = __all_sync(MFD_FULL_MASK, ok & mbar_wait(&bars[bar], parity, kTries));
                    tc_fence_after();
                };
                auto scores = [&](int s) {
                    const int i = x.alternate ? s : s >> 1, grp = s & 1;
                    const uint32_t nk = x.n_tile + i;
                    if (x.alternate || grp == 0) wait(L::kKFull + (nk & 1), (nk >> 1) & 1);
                    if (!ok) return;
                    const uint64_t k = kd + (uint64_t)((nk & 1) * (kTileBytes >> 4));
                    const uint64_t q = qd + (uint64_t)(x.alternate || grp == 0 ? 0 : kTileBytes >> 4);
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks) {
                        const uint64_t off = (uint64_t)(((ks >> 2) * (kTileBytes / 2) + (ks & 3) * 32) >> 4);
                        umma_if(leader, tmem + 256 + 128 * grp, q + off, k + off, kIdescS, ks > 0);
                    }
                    commit_if(leader, &bars[L::kSFull + grp]);
                    if (x.alternate || grp == 1) commit_if(leader, &bars[L::kKEmpty + (nk & 1)]);
                };
                if (x.nsteps > 0) wait(L::kQFull, x.n_piece & 1);
                if (x.nsteps > 0 && ok) scores(0);
                if (x.nsteps > 1 && ok) scores(1);
#pragma unroll 1
                for (int s = 0; s < x.nsteps && ok; ++s) {
                    const int i = x.alternate ? s : s >> 1, grp = s & 1;
                    const uint32_t nv = x.n_tile + i;
                    if (x.alternate || grp == 0) wait(L::kVFull + (nv & 1), (nv >> 1) & 1);
                    wait(L::kPFull + grp, ((grp ? x.n_s1 : x.n_s0) + (s >> 1)) & 1);
                    if (!ok) break;
                    const uint64_t v = vd + (uint64_t)((nv & 1) * (kTileBytes >> 4));
                    const uint32_t pt = tmem + 256 + 128 * grp;
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks) {  // 16 keys: hi, then lo
                        const uint32_t pa = pt + 32 * (ks >> 1) + 8 * (ks & 1);
                        umma_ts_if(leader, tmem + 128 * grp, pa, v + (uint64_t)(ks * 128), kIdescO, ks > 0 ? 1u : (uint32_t)(s >= 2));
                        umma_ts_if(leader, tmem + 128 * grp, pa + 16, v + (uint64_t)(ks * 128), kIdescO, 1u);
                    }
                    commit_if(leader, &bars[L::kPV + grp]);
                    if (x.alternate || grp == 1) commit_if(leader, &bars[L::kVEmpty + (nv & 1)]);
                    if (s + 2 < x.nsteps) scores(s + 2);
                }
            });
        }
    }
    if (*s_failed && tid == 0) atomicExch(p.status, 1), atomicExch(&gave_up, 1);
    tc_fence_before();
    __syncthreads();
    if (warp == 15) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// Adds up the pieces of every unit that was cut, in their order.  Block x is the CTA boundary (range cut: the first one
// inside its unit; split: the unit's first piece) that answers for a unit, block y 32 of its rows; a warp takes 16
// columns of them, lane = row, so every load of a piece is 512 contiguous bytes.  It is launched while the attention runs and
// waits for its end after finding its unit (2 us of a call less).
template <bool PAIR>
__global__ void __launch_bounds__(256) kv8_combine_kernel(const AttnParams p, int ctas) {
    constexpr int kRowsU = kSlotRows(PAIR);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cta = blockIdx.x;
    const int RB = (p.rows - p.row0 + kRowsU - 1) / kRowsU;
    auto tiles_of = [&](int len) { return counted_tiles(p, len, p.bs * p.c.Hkv * RB, ctas); };
    const Lengths lens(p.c, p.bs);
    const Cut cut = make_cut(lens, tiles_of, p.c.Hkv * RB, ctas);
    int pos, end;
    cut_range(cut, cta, pos, end);
    Piece pc;
    const bool any = next_piece(lens, tiles_of, cut, cta, pos, end, pc);
    // The pieces are complete and visible from here.  (Every CTA waits, so that this grid never ends before the attention's:
    // the next launch waits for this one.)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (!any) return;
    if (cut.split ? (pc.first != cta || pc.pieces == 1) : (pc.g0 == 0 || pc.first != cta - 1)) return;
    const int hk = pc.u / RB, rb = pc.u % RB;
    const int r = blockIdx.y * 32 + lane, row = p.row0 + rb * kRowsU + r;
    if (row - lane >= p.rows) return;
    float mm = -INFINITY;
#pragma unroll 8
    for (int i = 0; i < pc.pieces; ++i) mm = fmaxf(mm, __ldcg(p.part + (int64_t)slot_of(pc, i) * kSlotFloats(PAIR) + r));
    float ll = 0.f;
    float4 v[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) v[c] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = 0; i < pc.pieces; ++i) {
        const float* s = p.part + (int64_t)slot_of(pc, i) * kSlotFloats(PAIR);
        const float mi = __ldcg(s + r), li = __ldcg(s + kRowsU + r);
        const float a = mi == -INFINITY ? 0.f : fast_exp2(mi - mm);
        ll = fmaf(a, li, ll);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const float4 o = __ldcg(reinterpret_cast<const float4*>(s + 2 * kRowsU) + (int64_t)(4 * warp + c) * kRowsU + r);
            v[c].x = fmaf(a, o.x, v[c].x), v[c].y = fmaf(a, o.y, v[c].y);
            v[c].z = fmaf(a, o.z, v[c].z), v[c].w = fmaf(a, o.w, v[c].w);
        }
    }
    if (row >= p.rows) return;
    const float inv = ll > 0.f ? kUnit / ll : (ll == 0.f ? 0.f : ll);
    const int node = row / p.G, head = hk * p.G + row % p.G;
    uint4* dst = reinterpret_cast<uint4*>(p.out + (int64_t)pc.b * p.so_b + (int64_t)node * p.so_n + (int64_t)head * p.so_h +
                                          16 * warp);
#pragma unroll
    for (int c = 0; c < 2; ++c)
        dst[c] = make_uint4(pack_bf16(v[2 * c].x * inv, v[2 * c].y * inv), pack_bf16(v[2 * c].z * inv, v[2 * c].w * inv),
                            pack_bf16(v[2 * c + 1].x * inv, v[2 * c + 1].y * inv),
                            pack_bf16(v[2 * c + 1].z * inv, v[2 * c + 1].w * inv));
    if (p.lse && warp == 0)
        p.lse[((int64_t)pc.b * p.n + node) * p.H + head] = ll == 0.f ? -INFINITY : 0.6931471805599453f * (mm + (kUnitLog2 + log2f(ll)));
}

template <bool FP8, bool PAIR>
int launch_tc_one(const AttnParams& p, int sms, cudaStream_t stream) {
    CUtensorMap tk, tv;
    if (!make_page_map(&tk, p.c.k, p.c) || !make_page_map(&tv, p.c.v, p.c)) {
        set_error("mfd_kv8_attention: could not encode the TMA tensor maps");
        return MFD_ERR_CUDA;
    }
    static bool opted[64];
    cudaError_t e = opt_in_smem((const void*)kv8_tc_kernel<FP8, PAIR>, Layout<PAIR>::kBytes, opted);
    if (e != cudaSuccess) {
        set_error("mfd_kv8_attention: %s", cudaGetErrorString(e));
        return MFD_ERR_CUDA;
    }
    kv8_tc_kernel<FP8, PAIR><<<sms, kTcThreads, Layout<PAIR>::kBytes, stream>>>(tk, tv, p);
    MFD_CHECK_LAUNCH("mfd_kv8_attention");
    const int rows = p.rows - p.row0 < kSlotRows(PAIR) ? p.rows - p.row0 : kSlotRows(PAIR);
    // the combination's launch overlaps the attention (programmatic dependent launch)
    cudaLaunchAttribute overlap;
    overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    overlap.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)sms, (unsigned)((rows + 31) / 32));
    cfg.blockDim = dim3(256);
    cfg.stream = stream;
    cfg.attrs = &overlap, cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kv8_combine_kernel<PAIR>, p, sms);
    if (e != cudaSuccess) {
        set_error("mfd_kv8_attention: %s", cudaGetErrorString(e));
        return MFD_ERR_CUDA;
    }
    MFD_CHECK_LAUNCH("mfd_kv8_attention (combination)");
    return MFD_OK;
}

}  // namespace

size_t tc_workspace(int sms) { return (size_t)sms * 2 * kSlotFloats(true) * sizeof(float); }

int launch_tc(const AttnParams& p, bool pair, int sms, cudaStream_t stream) {
    if (p.fp8) return pair ? launch_tc_one<true, true>(p, sms, stream) : launch_tc_one<true, false>(p, sms, stream);
    return pair ? launch_tc_one<false, true>(p, sms, stream) : launch_tc_one<false, false>(p, sms, stream);
}

}  // namespace kv8
}  // namespace mfd

extern "C" int mfd_kv8_attention_status(int* status, void* stream) {
    cudaError_t e = status ? cudaSuccess : cudaErrorInvalidValue;
    if (e == cudaSuccess)
        e = cudaMemcpyFromSymbolAsync(status, mfd::kv8::gave_up, sizeof(int), 0, cudaMemcpyDeviceToHost, (cudaStream_t)stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize((cudaStream_t)stream);
    if (e != cudaSuccess) {
        mfd::set_error("mfd_kv8_attention_status: %s", cudaGetErrorString(e));
        return MFD_ERR_CUDA;
    }
    return MFD_OK;
}
