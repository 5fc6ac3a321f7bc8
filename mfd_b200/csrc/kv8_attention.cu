// kv8_attention.cu -- C entry point of the attention over the 8-bit paged cache: checks, and which kernel takes the
// rows.
#include <cudaTypedefs.h>

#include "kv8_attention.cuh"

namespace mfd {
namespace kv8 {

static PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    if (!fn) {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = (PFN_cuTensorMapEncodeTiled_v12000)ptr;
    }
    return fn;
}

bool make_page_map(CUtensorMap* m, const uint8_t* base, const Cache& c) {
    auto fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[4] = {(cuuint64_t)kD, (cuuint64_t)c.page, (cuuint64_t)c.Hkv, (cuuint64_t)c.num_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)c.sc_t, (cuuint64_t)c.sc_h, (cuuint64_t)c.sc_p};
    const cuuint32_t box[4] = {(cuuint32_t)kD, (cuuint32_t)c.page, 1, 1};
    const cuuint32_t estr[4] = {1, 1, 1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<uint8_t*>(base), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace kv8
}  // namespace mfd

using namespace mfd;

static int kv8_rows_total(int64_t n, int64_t H, int64_t Hkv) { return (int)(n * (H / Hkv)); }

// Rows of a (request, KV head) up to which the register kernel takes them all: its unit.  H 32 over 8 KV heads, register
// against tensor-core kernel: 16 rows, 32 requests of 4096 tokens 95 against 147 us, one request 23 against 27; 32 rows,
// 171 against 147 and 23 against 27, one request of 16384 tokens 37 against 39.  (So one request of 17 to 32 rows would be 2 to
// 4 us faster in the register kernel: the rule looks at the rows alone, not at how many units there are.)
constexpr int kRowsAlone = 16;

static bool kv8_sizes_ok(int64_t bs, int64_t n, int64_t H, int64_t Hkv) {
    return bs >= 0 && n > 0 && n <= 4096 && H > 0 && Hkv > 0 && H % Hkv == 0 && H <= 16384;
}

extern "C" size_t mfd_kv8_attention_workspace(int64_t bs, int64_t n, int64_t num_heads, int64_t num_kv_heads) {
    if (!kv8_sizes_ok(bs, n, num_heads, num_kv_heads)) return 0;
    const size_t rows = kv8::rows_workspace(kv8::sm_count()), tc = kv8::tc_workspace(kv8::sm_count());
    return 512 + (kv8_rows_total(n, num_heads, num_kv_heads) <= kRowsAlone || rows > tc ? rows : tc);
}

extern "C" int64_t mfd_kv8_attention_tickets(int64_t bs, int64_t n, int64_t num_heads, int64_t num_kv_heads) {
    if (!kv8_sizes_ok(bs, n, num_heads, num_kv_heads)) return 0;
    return kv8::rows_tickets(bs, num_kv_heads, kv8_rows_total(n, num_heads, num_kv_heads));
}

extern "C" int mfd_kv8_attention(const void* q, int64_t sq_b, int64_t sq_n, int64_t sq_h, const void* k_cache,
                                 const void* v_cache, int64_t sc_p, int64_t sc_h, int64_t sc_t, int code_dtype,
                                 const float* k_scale, const float* v_scale, int64_t num_pages, int64_t page_size,
                                 const int32_t* page_table, int64_t table_stride, int64_t max_pages,
                                 const int32_t* seq_lens, const void* k_new, const void* v_new, int64_t sn_b,
                                 int64_t sn_n, int64_t sn_h, const uint64_t* anc_bits, int64_t anc_words, int64_t bs,
                                 int64_t n, int64_t num_heads, int64_t num_kv_heads, int64_t head_dim, float scale,
                                 void* out, int64_t so_b, int64_t so_n, int64_t so_h, float* lse, void* workspace,
                                 size_t workspace_bytes, unsigned int* tickets, int64_t tickets_len, void* stream) {
    const char* who = "mfd_kv8_attention";
    int st;
    if (!kv8::check_cache(who, k_cache, v_cache, sc_p, sc_h, sc_t, code_dtype, num_pages, page_size, page_table,
                          max_pages, seq_lens, bs, num_kv_heads, head_dim, &st))
        return st;
    if ((bs > 0 && (!q || !out)) || !k_scale || !v_scale || !workspace || !tickets || (k_new == nullptr) != (v_new == nullptr)) {
        set_error("%s: null pointer", who);
        return MFD_ERR_INVALID;
    }
    if (n <= 0 || num_heads <= 0 || num_heads % num_kv_heads || (anc_bits && anc_words < (n + 63) / 64)) {
        set_error("%s: invalid sizes (n %lld, %lld query heads over %lld KV heads, %lld mask words)", who, (long long)n,
                  (long long)num_heads, (long long)num_kv_heads, (long long)anc_words);
        return MFD_ERR_INVALID;
    }
    if (!kv8_sizes_ok(bs, n, num_heads, num_kv_heads)) {
        set_error("%s: more than 4096 nodes or 16384 heads", who);
        return MFD_ERR_UNSUPPORTED;
    }
    if (sq_b % 8 || sq_n % 8 || sq_h % 8 || so_b % 8 || so_n % 8 || so_h % 8 || (uintptr_t)q % 16 ||
        (uintptr_t)out % 16 || (k_new && (sn_b % 8 || sn_n % 8 || sn_h % 8 || (uintptr_t)k_new % 16 || (uintptr_t)v_new % 16))) {
        set_error("%s: rows need strides that are multiples of 8 elements and 16-byte aligned bases", who);
        return MFD_ERR_INVALID;
    }
    const int64_t base = ((uintptr_t)workspace + 255) / 256 * 256 - (uintptr_t)workspace;
    if (workspace_bytes < mfd_kv8_attention_workspace(bs, n, num_heads, num_kv_heads) ||
        tickets_len < mfd_kv8_attention_tickets(bs, n, num_heads, num_kv_heads)) {
        set_error("%s: workspace or tickets too small", who);
        return MFD_ERR_INVALID;
    }
    if (!kv8::work_fits(bs, num_kv_heads * ((kv8_rows_total(n, num_heads, num_kv_heads) + 15) / 16), max_pages, page_size,
                        128) || bs * num_heads * n > 0x7fffffff) {
        set_error("%s: the requests' capacity is beyond this build's limits", who);
        return MFD_ERR_UNSUPPORTED;
    }
    if (bs == 0) return MFD_OK;
    kv8::AttnParams p;
    p.c.k = (const uint8_t*)k_cache, p.c.v = (const uint8_t*)v_cache;
    p.c.sc_p = sc_p, p.c.sc_h = sc_h, p.c.sc_t = sc_t;
    p.c.k_scale = k_scale, p.c.v_scale = v_scale;
    p.c.num_pages = num_pages;
    p.c.page = (int)page_size, p.c.page_shift = __builtin_ctz((unsigned)page_size);
    p.c.table = page_table, p.c.table_stride = table_stride, p.c.max_pages = (int)max_pages;
    p.c.lens = seq_lens;
    p.c.Hkv = (int)num_kv_heads;
    p.fp8 = code_dtype == MFD_E4M3;
    p.q = (const __nv_bfloat16*)q, p.sq_b = sq_b, p.sq_n = sq_n, p.sq_h = sq_h;
    p.kn = (const __nv_bfloat16*)k_new, p.vn = (const __nv_bfloat16*)v_new;
    p.sn_b = sn_b, p.sn_n = sn_n, p.sn_h = sn_h;
    p.anc = anc_bits, p.words = (int)anc_words;
    p.bs = (int)bs, p.n = (int)n, p.H = (int)num_heads, p.G = (int)(num_heads / num_kv_heads);
    p.nn = k_new ? (int)n : 0;
    p.row0 = 0, p.rows = kv8_rows_total(n, num_heads, num_kv_heads);
    p.scale_log2 = scale * kLog2e;
    p.out = (__nv_bfloat16*)out, p.so_b = so_b, p.so_n = so_n, p.so_h = so_h;
    p.lse = lse;
    char* ws = (char*)workspace + base;
    p.status = (int*)ws;
    p.part = (float*)(ws + 256);
    p.tickets = tickets;
    const int sms = kv8::sm_count(), rows = p.rows;
    cudaStream_t s = (cudaStream_t)stream;
    if (rows <= kRowsAlone) return kv8::launch_rows(p, sms, s);
    // Pairs of 128-row tiles; a remainder of a few rows goes to the register kernel instead of a tile of padding (32
    // requests of 4096 tokens, 65 nodes x 4 heads: 309 against 362 us).
    const int rest = rows % 256;
    const bool tail = rows > 256 && rest > 0 && rest <= kRowsAlone && p.nn <= kv8::kRowsMaxOwn;
    // With few units one row tile a CTA.  In place of a second and a third launch the last tile is mostly empty (65 nodes
    // x 4 heads over 4096 tokens: 32 against 60 us at 1 request of 8 KV heads, 43 against 60 at 2, 77 against 76 at 4); in
    // place of pairs more CTAs share the keys (64 nodes x 4 heads, 1 request: 29 against 36 us over 4096 tokens, 53
    // against 58 over 16384; at 2 requests 39 against 39 and 90 against 77).
    const int64_t pairs = bs * num_kv_heads * ((rows + 255) / 256);
    if (pairs <= sms / (tail ? 4 : 16)) return kv8::launch_tc(p, false, sms, s);
    if (tail) p.rows = rows - rest;
    st = kv8::launch_tc(p, rows > 128, sms, s);
    if (st != MFD_OK || !tail) return st;
    p.row0 = rows - rest, p.rows = rows;
    return kv8::launch_rows(p, sms, s);
}
