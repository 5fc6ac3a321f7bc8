// kv8.cuh -- what the kernels of the 8-bit paged K/V cache share: code conversions, page addressing, the tensor
// instruction of the register kernels, and the limits of the accepted-path lists.
//
// A cached value is code * scale with one float32 scale per (page, KV head, tensor).  Both code types are exact in
// float16 and in bf16 (int8: |c| <= 128; e4m3: 3 fraction bits, 2^-9 .. 448), so products of 16-bit operands lose
// nothing and the page's scale multiplies a finished dot product (K) or is folded into the softmax weight (V).
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <type_traits>

#include "common.cuh"

namespace mfd {
namespace kv8 {

constexpr int kD = 128;                           // head dim: codes per row
constexpr float kScaleFloor = 7.888609052210118e-31f;  // 2^-100, the least scale of a page

// One cache tensor pair of a layer; strides in bytes (= codes).
struct Cache {
    const uint8_t* k;
    const uint8_t* v;
    int64_t sc_p, sc_h, sc_t;
    const float* k_scale;  // [num_pages, Hkv]
    const float* v_scale;
    int64_t num_pages;
    int page, page_shift;  // tokens per page (a power of two) and its log2
    const int32_t* table;
    int64_t table_stride;
    int max_pages;
    const int32_t* lens;
    int Hkv;
};

__device__ __forceinline__ int seq_len(const Cache& c, int b) {
    const int cap = c.max_pages << c.page_shift;
    return min(max(__ldg(c.lens + b), 0), cap);
}
// a page id as read from the table, clamped to the pool
__device__ __forceinline__ int page_id(const Cache& c, int b, int p) {
    return min(max(__ldg(c.table + (int64_t)b * c.table_stride + p), 0), (int)c.num_pages - 1);
}

// four codes of a word as two float16 pairs: (bytes 0, 1) and (bytes 2, 3)
template <bool FP8>
__device__ __forceinline__ void halves(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if (FP8) {
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
            : "=r"(lo), "=r"(hi)
            : "r"(w));
    } else {
        // c + 128 as the low byte of the float16 1024 (bits 0x6400, spacing 1), less 1152: exact
        w ^= 0x80808080u;
        const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
        uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
        const __half2 x = __hsub2(*reinterpret_cast<__half2*>(&a), off);
        const __half2 y = __hsub2(*reinterpret_cast<__half2*>(&b), off);
        lo = *reinterpret_cast<const uint32_t*>(&x);
        hi = *reinterpret_cast<const uint32_t*>(&y);
    }
}

// the same as two bf16 pairs
template <bool FP8>
__device__ __forceinline__ void bfloats(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if (FP8) {  // through float16 (a NaN code stays NaN)
        uint32_t a, b;
        halves<true>(w, a, b);
        const float2 x = __half22float2(*reinterpret_cast<__half2*>(&a)), y = __half22float2(*reinterpret_cast<__half2*>(&b));
        const __nv_bfloat162 u = __floats2bfloat162_rn(x.x, x.y), v = __floats2bfloat162_rn(y.x, y.y);
        lo = *reinterpret_cast<const uint32_t*>(&u);
        hi = *reinterpret_cast<const uint32_t*>(&v);
    } else {
        // the low seven bits on the bf16 128 (bits 0x4300, spacing 1), less 128 or, with the sign bit, 256: exact
        const uint32_t x = __byte_perm(w, 0x43434343u, 0x4140), y = __byte_perm(w, 0x43434343u, 0x4342);
        uint32_t xa = x & 0xff7fff7fu, xb = x & 0xff80ff80u, ya = y & 0xff7fff7fu, yb = y & 0xff80ff80u;
        const __nv_bfloat162 u = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&xa), *reinterpret_cast<__nv_bfloat162*>(&xb));
        const __nv_bfloat162 v = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&ya), *reinterpret_cast<__nv_bfloat162*>(&yb));
        lo = *reinterpret_cast<const uint32_t*>(&u);
        hi = *reinterpret_cast<const uint32_t*>(&v);
    }
}

// A pair of weights as bf16 hi + lo, both cut off instead of rounded (byte moves and one packed subtraction; the rounding
// conversions run at half rate): hi keeps the top 8 bits, lo the next 8, so a weight loses at most 2^-15 of itself.
__device__ __forceinline__ void split_bf16(uint64_t w, uint32_t& hi, uint32_t& lo) {
    const uint64_t top = w & 0xffff0000ffff0000ull;
    const uint64_t left = sub2(w, top);
    hi = __byte_perm((uint32_t)w, (uint32_t)(w >> 32), 0x7632);
    lo = __byte_perm((uint32_t)left, (uint32_t)(left >> 32), 0x7632);
}

// The same as float16 hi + lo, rounded: 22 bits of each down to 2^-24 (the caller lifts the weights well above it).
__device__ __forceinline__ void split_half(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const __half2 r = __floats2half2_rn(a - f.x, b - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&r);
}

// the 8 x 8 transpose of 16-bit values held two a lane (row lane / 4, columns 2 (lane % 4) and the next)
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// bf16 pair -> the two floats
__device__ __forceinline__ float2 bf2(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// the power of two 2^-e that brings a row of largest magnitude mx into (-2, 2), and 2^e.  Both are exact, so a bf16
// query row becomes float16 without loss down to 2^-17 of its largest element (8 bits, the last of them 2^-24, where
// float16 ends); smaller ones lose up to 2^-25 of it, which vanishes against the row's own rounding.  (A zero or non-finite
// row is left as it is.)
__device__ __forceinline__ void row_power(float mx, float& down, float& up) {
    int e = (int)((__float_as_uint(mx) >> 23) & 0xffu) - 127;
    if (mx == 0.f || e == 128) e = 0;
    e = max(e, -126);
    down = e == 127 ? 5.877471754111438e-39f : __uint_as_float((uint32_t)(127 - e) << 23);  // (2^-127 is subnormal)
    up = __uint_as_float((uint32_t)(max(e + 127, 1)) << 23);
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// One asynchronous 16-byte copy into shared memory, and the groups they are waited for in.
__device__ __forceinline__ void copy16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {  // all but the last N groups have landed
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// Where a warp keeps rows of 128 codes in shared memory: 16-byte chunk c of row r.  The eight lanes of a 16-byte access
// that read chunks 2 t (+ 1) of two neighbouring rows, or one chunk of every other row, hit eight different bank groups.
__device__ __forceinline__ int chunk_at(int r, int c) { return r * kD + ((c ^ (r & 7)) << 4); }

// Rows a request lists: counts[b] (or `rows`), cut at the first path entry outside [0, n).  Called by whole warps.
__device__ __forceinline__ int listed_rows(const int64_t* path, int64_t path_stride, int rows, const int32_t* counts,
                                           int n, int b) {
    int c = counts ? min(max(__ldg(counts + b), 0), rows) : rows;
    if (!path) return min(c, n);
    const int lane = threadIdx.x & 31;
    for (int i = 0; i < c; i += 32) {
        int64_t e = 0;
        if (i + lane < c) e = __ldg((const long long*)path + (int64_t)b * path_stride + i + lane);
        const uint32_t bad = __ballot_sync(MFD_FULL_MASK, e < 0 || e >= n);
        if (bad) {
            c = i + __ffs(bad) - 1;
            break;
        }
    }
    return c;
}

// a / b for a >= 0, b > 0.  Small ones (all but extreme cases) by a reciprocal estimate, within one of the quotient, and
// its correction: every CTA starts with a few of these, one after another.
__device__ __forceinline__ int quotient(int a, int b) {
    if (((uint32_t)(a | b) >> 22) != 0) return (int)((uint32_t)a / (uint32_t)b);
    int q = __float2int_rz(__fdividef((float)a, (float)b));
    const int r = a - q * b;
    q += r >= b ? 1 : (r < 0 ? -1 : 0);
    return q;
}

// Work laid end to end over the requests, f(length) * mul (or f(length, request) * mul) of it for each (below 2^31 in all:
// the entry points check); every warp finds its place by itself.  The lengths of the first 32 requests stay in the lanes' registers.
struct Lengths {
    const Cache& c;
    int bs, mine;
    __device__ __forceinline__ Lengths(const Cache& cache, int requests) : c(cache), bs(requests) {
        const int lane = threadIdx.x & 31;
        mine = lane < bs ? seq_len(c, lane) : 0;
    }
    template <class F>
    __device__ __forceinline__ int part(int b0, F f, int& len) const {
        const int b = b0 + (threadIdx.x & 31);
        len = b0 == 0 ? mine : (b < bs ? seq_len(c, b) : 0);
        if (b >= bs) return 0;
        if constexpr (std::is_invocable_v<F, int, int>) return f(len, b);
        else return f(len);
    }
    // the sum over all requests
    template <class F>
    __device__ __forceinline__ int sum(F f) const {
        int total = 0;
        for (int b0 = 0; b0 < bs; b0 += 32) {
            int len;
            total += __reduce_add_sync(MFD_FULL_MASK, part(b0, f, len));
        }
        return total;
    }
    // the request whose range [before, before + f * mul) contains x, its length and before; -1 behind the last
    template <class F>
    __device__ __forceinline__ int find(int x, int mul, F f, int& before, int& len) const {
        const int lane = threadIdx.x & 31;
        int base = 0;
        for (int b0 = 0; b0 < bs; b0 += 32) {
            const int v = part(b0, f, len);
            int inc = v;
            if (bs > 1) {
#pragma unroll 1
                for (int d = 1; d < 32; d <<= 1) {
                    const int o = __shfl_up_sync(MFD_FULL_MASK, inc, d);
                    if (lane >= d) inc += o;
                }
            }
            const uint32_t hit = __ballot_sync(MFD_FULL_MASK, (base + inc) * mul > x);
            if (hit) {
                const int l = __ffs(hit) - 1;
                before = (base + __shfl_sync(MFD_FULL_MASK, inc - v, l)) * mul;
                len = __shfl_sync(MFD_FULL_MASK, len, l);
                return b0 + l;
            }
            base += __shfl_sync(MFD_FULL_MASK, inc, 31);
        }
        return -1;
    }
};

// How the units' work is cut over `ctas` CTAs: few units (split) into pieces of `per`, at most one piece a CTA;
// otherwise equal ranges of `per` end to end, which may begin and end inside a unit.
struct Cut {
    int total, per;
    int per_req;  // units per request
    bool split;
};
template <class F>
__device__ __forceinline__ Cut make_cut(const Lengths& lens, F f, int per_req, int ctas) {
    Cut w;
    w.per_req = per_req;
    w.total = lens.sum(f) * per_req;
    w.split = lens.bs * per_req <= ctas / 2;
    w.per = max(1, quotient(w.total + ctas - 1, ctas));
    if (w.split) {
        // the smallest piece (nearly: 1/16 steps) of which there are at most ctas
        const int step = max(1, w.per >> 4);
        while (lens.sum([&](int len) { return quotient(f(len) + w.per - 1, w.per); }) * per_req > ctas) w.per += step;
    }
    return w;
}
// [begin, end) of CTA `cta`: a range of the work, or (split) a piece's number
__device__ __forceinline__ void cut_range(const Cut& w, int cta, int& begin, int& end) {
    begin = w.split ? cta : (int)min((int64_t)cta * w.per, (int64_t)w.total);
    end = w.split ? begin + 1 : (int)min((int64_t)w.total, (int64_t)begin + w.per);
}

struct Piece {
    int b, len;      // request and its length
    int u;           // unit of the request
    int g0, g1, of;  // the piece's part [g0, g1) of the unit's `of`
    int first;       // the CTA of the unit's first piece
    int pieces;
    int slot;        // this piece's partial record (two a CTA: a range can end one unit and begin another)
    bool second;     // the unit's first piece is its CTA's second record
};
// the next piece of CTA `cta` at `pos` (moved on); false at the end
template <class F>
__device__ __forceinline__ bool next_piece(const Lengths& lens, F f, const Cut& w, int cta, int& pos, int end, Piece& pc) {
    if (pos >= end) return false;
    int before;
    if (w.split) {
        auto pieces_of = [&](int len) { return quotient(f(len) + w.per - 1, w.per); };
        pc.b = lens.find(pos, w.per_req, pieces_of, before, pc.len);
        if (pc.b < 0) return false;
        pc.of = f(pc.len);
        pc.pieces = pieces_of(pc.len);
        const int off = pos - before;
        pc.u = quotient(off, pc.pieces);
        const int i = off - pc.u * pc.pieces;
        pc.g0 = i * w.per;
        pc.g1 = min(pc.of, pc.g0 + w.per);
        pc.first = pos - i;
        pc.slot = 2 * cta;
        pc.second = false;
        pos = end;
    } else {
        pc.b = lens.find(pos, w.per_req, f, before, pc.len);
        if (pc.b < 0) return false;
        pc.of = f(pc.len);
        const int off = pos - before;
        pc.u = quotient(off, pc.of);
        pc.g0 = off - pc.u * pc.of;
        pc.g1 = min(pc.of, pc.g0 + (end - pos));
        const int lo = pos - pc.g0;  // where the unit begins
        pc.first = quotient(lo, w.per);
        pc.pieces = quotient(lo + pc.of - 1, w.per) - pc.first + 1;
        pc.second = pc.first * w.per < lo;
        pc.slot = 2 * cta + (pos == cta * w.per ? 0 : 1);
        pos += pc.g1 - pc.g0;
    }
    return true;
}
// the partial record of piece i of a unit
__device__ __forceinline__ int slot_of(const Piece& pc, int i) {
    return 2 * (pc.first + i) + (pc.second && i == 0 ? 1 : 0);
}
// whether all requests at their capacity are less than 2^31 pieces of work of `tokens` each, and a few a unit (host)
inline bool work_fits(int64_t bs, int64_t per_req, int64_t max_pages, int64_t page, int64_t tokens) {
    const double all = (double)bs * (double)per_req * ((double)max_pages * (double)page / (double)tokens + 16.0);
    return all < 2147483648.0;
}

// over the lanes with the same lane % 4
__device__ __forceinline__ float column_max(float v) {
    v = fmaxf(v, __shfl_xor_sync(MFD_FULL_MASK, v, 4));
    v = fmaxf(v, __shfl_xor_sync(MFD_FULL_MASK, v, 8));
    return fmaxf(v, __shfl_xor_sync(MFD_FULL_MASK, v, 16));
}
__device__ __forceinline__ float column_sum(float v) {
    v += __shfl_xor_sync(MFD_FULL_MASK, v, 4);
    v += __shfl_xor_sync(MFD_FULL_MASK, v, 8);
    return v + __shfl_xor_sync(MFD_FULL_MASK, v, 16);
}
__device__ __forceinline__ float quad_max(float v) {
    v = fmaxf(v, __shfl_xor_sync(MFD_FULL_MASK, v, 1));
    return fmaxf(v, __shfl_xor_sync(MFD_FULL_MASK, v, 2));
}
// SMs of the current device, and the opt-in to a kernel's dynamic shared memory, asked of the driver once per device
int sm_count();
cudaError_t opt_in_smem(const void* kernel, int bytes, bool (&done)[64]);

// host checks shared by the entry points; false after set_error
bool check_cache(const char* who, const void* k, const void* v, int64_t sc_p, int64_t sc_h, int64_t sc_t,
                 int code_dtype, int64_t num_pages, int64_t page_size, const int32_t* table, int64_t max_pages,
                 const int32_t* lens, int64_t bs, int64_t hkv, int64_t head_dim, int* status);

}  // namespace kv8
}  // namespace mfd
