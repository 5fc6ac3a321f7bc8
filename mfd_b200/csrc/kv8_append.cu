// kv8_append.cu -- quantise new K / V rows into the pages of an 8-bit cache (the commit of an accepted path, or a
// prompt), with one scale per page and KV head.
//
//   s' = max(s_open, amax(finite new values of the page) * (1 / qmax), 2^-100),  code = rne(x / s')
//
// and the rows already in the request's open page are rounded again, rne(code * s_open / s'), when its scale grows.
// A tensor's scale only ever grows while its page fills, so a row is rounded again at most as often as the running
// maximum of a page changes.  Multiplication, division and rounding are IEEE float32: the codes are the same whatever
// the launch.
//
// Bound: bytes (each new row read once in bf16, written once in 8 bits; 12 bytes per 4 values at most).  One CTA of
// 256 threads per (touched page, KV head and tensor, request) keeps the page's values in registers between the
// maximum and the rounding, so the rows are read once.  Threads take 16-byte granules of a row (8 values), 16 lanes a
// row, so loads and the 8-byte code stores are contiguous.
//
// Measured (8 KV heads): the accepted paths of 32 requests (17 nodes each at most, pages of 64) 6.3 us, launch and latency; two
// prompts of 8192 tokens (pages of 128) 24.5 us, 3.7 TB/s: a CTA's rows are 256 bytes apart from one another by all heads'.
#include "kv8.cuh"

namespace mfd {
namespace kv8 {

constexpr int kThreads = 256;
constexpr int kRowLanes = 16;                      // lanes per row: 8 values each
constexpr int kRowsPerPass = kThreads / kRowLanes;  // 16

struct AppendParams {
    uint8_t* cache[2];  // K, V
    float* scale[2];
    const __nv_bfloat16* fresh[2];
    int64_t sc_p, sc_h, sc_t;
    int64_t sn_b, sn_n, sn_h;
    int64_t num_pages;
    int page, page_shift, max_pages;
    const int32_t* table;
    int64_t table_stride;
    const int32_t* lens;
    const int64_t* path;
    int64_t path_stride;
    int rows, n, Hkv;
    const int32_t* counts;
    int32_t* new_lens;
    int* status;
};

template <bool FP8>
__device__ __forceinline__ uint32_t encode2(float a, float b) {  // two values already divided by the scale
    constexpr float qmax = FP8 ? 448.f : 127.f;
    a = a == a ? fminf(fmaxf(a, -qmax), qmax) : 0.f;
    b = b == b ? fminf(fmaxf(b, -qmax), qmax) : 0.f;
    if (FP8) {
        uint16_t r;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
        return r;
    }
    return (uint32_t)(__float2int_rn(a) & 0xff) | ((uint32_t)(__float2int_rn(b) & 0xff) << 8);
}
// The codes of 8 finite bf16 values x / s, given r, the float32 nearest to 1 / s: the product x r and one correction by its
// exact remainder (Markstein's theorem on the correctly rounded quotient), two values an instruction.  The result is the
// IEEE quotient for every bf16 x and every scale whose reciprocal is normal and whose remainders are exact, at a fifth of
// the instructions of a division.  (2^23 significands of the scale times 128 of x: none differs.  Below 2^-90 a remainder may be
// subnormal: 1.9999999 * 2^-100 and x = 2^-109 give another e4m3 code.)  Blocks of other scales divide, unless all their values are zero.
constexpr float kFastScaleLo = 5.421010862427522e-20f, kFastScaleHi = 8.507059173023462e+37f;  // 2^-64 and 2^126
template <bool FP8>
__device__ __forceinline__ uint2 encode8(const uint4& x, float s, float r) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    const uint64_t r2 = dup2(r), s2 = dup2(-s);
    uint32_t c[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 f = bf2(w[j]);
        const uint64_t v = pk2(f.x, f.y);
        uint64_t q = mul2(v, r2);
        q = fma2(fma2(q, s2, v), r2, q);
        if (FP8) {
            float a, b;
            upk2(q, a, b);
            uint16_t e;
            asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(e) : "f"(b), "f"(a));
            c[j] = e;
        } else {
            const uint64_t m = add2(q, dup2(12582912.f));  // 1.5 * 2^23: rounds to an integer, the low byte its code
            c[j] = __byte_perm((uint32_t)m, (uint32_t)(m >> 32), 0x0040) & 0xffffu;
        }
    }
    return make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
}
template <bool FP8>
__device__ __forceinline__ float4 decode4(uint32_t w) {
    uint32_t lo, hi;
    halves<FP8>(w, lo, hi);
    const float2 a = __half22float2(*reinterpret_cast<__half2*>(&lo)), b = __half22float2(*reinterpret_cast<__half2*>(&hi));
    return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a < INFINITY ? a : 0.f;  // (false for NaN too)
}

// CTAs an SM the registers are cut for.  A CTA waits for its rows, then for its maximum, then writes, so the others keep the
// memory busy: two prompts of 8192 tokens in pages of 128 take 27 us with 4 (what 64 registers allow), 24.4 with 5 and
// 29 with 8 (rows in local memory); in pages of 64 24.7 with 5, 23.9 with 6 and 22.7 with 8.  Pages of 16 take 32 registers,
// which is 8, uncut (30.9 either way); pages of 32 take 40 uncut (26.7, and 24.7 with 8).  Paths of 17 rows: no difference.
constexpr int ctas_per_sm(int page) { return page == 128 ? 5 : (page == 64 ? 8 : 1); }

// PAGE: tokens per page, kItems rows of 16 lanes a thread
template <bool FP8, int PAGE>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(PAGE)) kv8_append_kernel(const AppendParams p) {
    constexpr int kItems = PAGE / kRowsPerPass;
    constexpr float qmax = FP8 ? 448.f : 127.f;  // (1 / qmax below is the float32 nearest to it)
    __shared__ float warp_max[kThreads / 32];
    const int b = blockIdx.z, which = blockIdx.y & 1, hk = blockIdx.y >> 1;
    const int cap = p.max_pages << p.page_shift;
    const int len = min(max(__ldg(p.lens + b), 0), cap);
    int count = listed_rows(p.path, p.path_stride, p.rows, p.counts, p.n, b);
    const bool over = count > cap - len;
    if (over) count = cap - len;
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) {
        p.new_lens[b] = len + count;
        if (over && p.status) atomicExch(p.status, MFD_ERR_CAPACITY);
    }
    const int first = len >> p.page_shift;
    const int pg = first + (int)blockIdx.x;
    const int lo = max(len - pg * PAGE, 0);                    // slots [lo, hi) of the page are new,
    const int hi = min(len + count - pg * PAGE, PAGE);         // slots [0, lo) hold earlier tokens
    if (hi <= lo) return;
    const int id = __ldg(p.table + (int64_t)b * p.table_stride + pg);
    const int r0 = threadIdx.x / kRowLanes, c = threadIdx.x % kRowLanes;
    const __nv_bfloat16* src = p.fresh[which] + (int64_t)b * p.sn_b + (int64_t)hk * p.sn_h + c * 8;
    uint4 x[kItems];  // 8 bf16 values of slots r0 + 16 i (on their way before the page id is)
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        const int slot = r0 + kRowsPerPass * i;
        x[i] = make_uint4(0u, 0u, 0u, 0u);
        if (slot >= lo && slot < hi) {
            const int row = pg * PAGE + slot - len;
            const int64_t node = p.path ? __ldg((const long long*)p.path + (int64_t)b * p.path_stride + row) : row;
            x[i] = ldg_stream_u4(src + node * p.sn_n);
        }
    }
    if (id < 0 || (int64_t)id >= p.num_pages) {
        if (threadIdx.x == 0 && p.status) atomicExch(p.status, MFD_ERR_CAPACITY);
        return;
    }
    uint8_t* page = p.cache[which] + (int64_t)id * p.sc_p + (int64_t)hk * p.sc_h + c * 8;
    float* scale = p.scale[which] + (int64_t)id * p.Hkv + hk;
    const float open = lo > 0 ? *scale : 0.f;
    // the largest magnitude, two bf16 at a time; a NaN stays one, so that a block with anything non-finite is known
    __nv_bfloat162 top = __float2bfloat162_rn(0.f);
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t a = w[j] & 0x7fff7fffu;
            top = __hmax2_nan(top, *reinterpret_cast<const __nv_bfloat162*>(&a));
        }
    }
    const float2 tops = __bfloat1622float2(top);
    float mx = fmaxf(tops.x, tops.y);
    if (tops.x != tops.x || tops.y != tops.y) mx = INFINITY;
    mx = warp_max_f32(mx);
    if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = mx;
    __syncthreads();  // (also: every thread has read the open page's scale)
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) mx = fmaxf(mx, warp_max[w]);
    const bool finite = mx < INFINITY;  // (of the whole block)
    if (!finite) {
        mx = 0.f;
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
            const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = bf2(w[j]);
                mx = fmaxf(mx, fmaxf(finite_abs(f.x), finite_abs(f.y)));
            }
        }
        mx = warp_max_f32(mx);
        __syncthreads();
        if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = mx;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) mx = fmaxf(mx, warp_max[w]);
    }
    const float s = fmaxf(fmaxf(__fmul_rn(mx, 1.f / qmax), open), kScaleFloor), r = __frcp_rn(s);
    const bool fast = finite && s <= kFastScaleHi && (s >= kFastScaleLo || mx == 0.f);  // (zeros are 0 in any scale)
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        const int slot = r0 + kRowsPerPass * i;
        uint2* dst = reinterpret_cast<uint2*>(page + (int64_t)slot * p.sc_t);
        if (slot >= lo && slot < hi && fast) {
            *dst = encode8<FP8>(x[i], s, r);
        } else if (slot < hi && (slot >= lo || s != open)) {  // rare: rows already there whose scale grows, non-finite blocks, extreme scales
            float f[8];
            if (slot >= lo) {
                const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 g = bf2(w[j]);
                    f[2 * j] = g.x;
                    f[2 * j + 1] = g.y;
                }
            } else {
                const uint2 old = *dst;
                const float4 a = decode4<FP8>(old.x), d = decode4<FP8>(old.y);
                f[0] = __fmul_rn(a.x, open), f[1] = __fmul_rn(a.y, open), f[2] = __fmul_rn(a.z, open);
                f[3] = __fmul_rn(a.w, open), f[4] = __fmul_rn(d.x, open), f[5] = __fmul_rn(d.y, open);
                f[6] = __fmul_rn(d.z, open), f[7] = __fmul_rn(d.w, open);
            }
            uint32_t e[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) e[j] = encode2<FP8>(__fdiv_rn(f[2 * j], s), __fdiv_rn(f[2 * j + 1], s));
            *dst = make_uint2(e[0] | (e[1] << 16), e[2] | (e[3] << 16));
        }
    }
    if (threadIdx.x == 0) *scale = s;
}

int sm_count() {
    static int known[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return current_sm_count();
    if (!known[dev]) known[dev] = current_sm_count();  // (threads that race here store the same number)
    return known[dev];
}

cudaError_t opt_in_smem(const void* kernel, int bytes, bool (&done)[64]) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || (dev < 64 && done[dev])) return e;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && dev < 64) done[dev] = true;
    return e;
}

bool check_cache(const char* who, const void* k, const void* v, int64_t sc_p, int64_t sc_h, int64_t sc_t,
                 int code_dtype, int64_t num_pages, int64_t page_size, const int32_t* table, int64_t max_pages,
                 const int32_t* lens, int64_t bs, int64_t hkv, int64_t head_dim, int* status) {
    *status = MFD_ERR_INVALID;
    if (!k || !v || (bs > 0 && (!table || !lens))) {  // (the tensors of an empty batch have no memory)
        set_error("%s: null pointer", who);
        return false;
    }
    if (code_dtype != MFD_I8 && code_dtype != MFD_E4M3) {
        set_error("%s: codes must be int8 or e4m3", who);
        return false;
    }
    if (bs < 0 || hkv <= 0 || num_pages <= 0 || max_pages <= 0) {
        set_error("%s: invalid sizes (bs %lld, KV heads %lld, pages %lld, table width %lld)", who, (long long)bs,
                  (long long)hkv, (long long)num_pages, (long long)max_pages);
        return false;
    }
    if (sc_p % 16 || sc_h % 16 || sc_t % 16 || (uintptr_t)k % 16 || (uintptr_t)v % 16 || sc_t < kD) {
        set_error("%s: cache rows must be 128 contiguous codes with strides and bases that are multiples of 16", who);
        return false;
    }
    *status = MFD_ERR_UNSUPPORTED;
    if (head_dim != kD) {
        set_error("%s: head dim %lld is not 128", who, (long long)head_dim);
        return false;
    }
    if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128) {
        set_error("%s: page size %lld is not 16, 32, 64 or 128", who, (long long)page_size);
        return false;
    }
    if (max_pages > (int64_t)0x3fffffff / page_size || num_pages > 0x7fffffff || bs > 65535 || hkv > 16384) {
        set_error("%s: sizes beyond this build's limits (2^30 tokens a request, 65535 requests)", who);
        return false;
    }
    *status = MFD_OK;
    return true;
}

template <bool FP8>
static void launch_append(const AppendParams& p, dim3 grid, cudaStream_t st) {
    switch (p.page) {
        case 16: kv8_append_kernel<FP8, 16><<<grid, kThreads, 0, st>>>(p); break;
        case 32: kv8_append_kernel<FP8, 32><<<grid, kThreads, 0, st>>>(p); break;
        case 64: kv8_append_kernel<FP8, 64><<<grid, kThreads, 0, st>>>(p); break;
        default: kv8_append_kernel<FP8, 128><<<grid, kThreads, 0, st>>>(p); break;
    }
}

}  // namespace kv8
}  // namespace mfd

using namespace mfd;

extern "C" int mfd_kv8_append(void* k_cache, void* v_cache, int64_t sc_p, int64_t sc_h, int64_t sc_t, int code_dtype,
                              float* k_scale, float* v_scale, int64_t num_pages, int64_t page_size,
                              const int32_t* page_table, int64_t table_stride, int64_t max_pages,
                              const int32_t* seq_lens, const void* k_new, const void* v_new, int64_t sn_b,
                              int64_t sn_n, int64_t sn_h, int64_t n, const int64_t* path, int64_t path_stride,
                              int64_t rows, const int32_t* counts, int64_t bs, int64_t num_kv_heads, int64_t head_dim,
                              int32_t* new_lens, int* status, void* stream) {
    const char* who = "mfd_kv8_append";
    int st;
    if (!kv8::check_cache(who, k_cache, v_cache, sc_p, sc_h, sc_t, code_dtype, num_pages, page_size, page_table,
                          max_pages, seq_lens, bs, num_kv_heads, head_dim, &st))
        return st;
    if (!k_scale || !v_scale || (bs > 0 && (!k_new || !v_new || !new_lens || new_lens == seq_lens)) || n <= 0 || rows < 0 ||
        (!path && rows > n)) {
        set_error("%s: null pointer, new_lens over seq_lens, or invalid sizes (n %lld, rows %lld)", who, (long long)n,
                  (long long)rows);
        return MFD_ERR_INVALID;
    }
    if (sn_b % 8 || sn_n % 8 || sn_h % 8 || (uintptr_t)k_new % 16 || (uintptr_t)v_new % 16) {
        set_error("%s: new rows need strides that are multiples of 8 elements and 16-byte aligned bases", who);
        return MFD_ERR_INVALID;
    }
    if ((uintptr_t)status % sizeof(int)) {
        set_error("%s: status is not aligned to an int", who);
        return MFD_ERR_INVALID;
    }
    if (n > 0x3fffffff || rows > 0x3fffffff) {
        set_error("%s: too many rows", who);
        return MFD_ERR_UNSUPPORTED;
    }
    if (bs == 0) return MFD_OK;
    kv8::AppendParams p;
    p.cache[0] = (uint8_t*)k_cache;
    p.cache[1] = (uint8_t*)v_cache;
    p.scale[0] = k_scale;
    p.scale[1] = v_scale;
    p.fresh[0] = (const __nv_bfloat16*)k_new;
    p.fresh[1] = (const __nv_bfloat16*)v_new;
    p.sc_p = sc_p, p.sc_h = sc_h, p.sc_t = sc_t;
    p.sn_b = sn_b, p.sn_n = sn_n, p.sn_h = sn_h;
    p.num_pages = num_pages;
    p.page = (int)page_size;
    p.page_shift = __builtin_ctz((unsigned)page_size);
    p.max_pages = (int)max_pages;
    p.table = page_table;
    p.table_stride = table_stride;
    p.lens = seq_lens;
    p.path = path;
    p.path_stride = path_stride;
    p.rows = (int)rows, p.n = (int)n, p.Hkv = (int)num_kv_heads;
    p.counts = counts;
    p.new_lens = new_lens;
    p.status = status;
    // rows land in at most ceil((rows - 1) / page) + 1 pages whatever the open page's fill
    const int64_t touched = rows > 0 ? (rows - 1 + page_size - 1) / page_size + 1 : 1;
    dim3 grid((unsigned)touched, (unsigned)(2 * num_kv_heads), (unsigned)bs);
    if (code_dtype == MFD_E4M3) kv8::launch_append<true>(p, grid, (cudaStream_t)stream);
    else kv8::launch_append<false>(p, grid, (cudaStream_t)stream);
    MFD_CHECK_LAUNCH(who);
    return MFD_OK;
}
