// kv8_attention.cuh -- parameters shared by the attention kernels over the 8-bit paged cache and their C entry point.
#pragma once

#include <cuda.h>

#include "kv8.cuh"

namespace mfd {
namespace kv8 {

struct AttnParams {
    Cache c;
    bool fp8;  // e4m3 codes, else int8
    const __nv_bfloat16* q;
    int64_t sq_b, sq_n, sq_h;
    const __nv_bfloat16* kn;  // the nodes' own keys and values, or null
    const __nv_bfloat16* vn;
    int64_t sn_b, sn_n, sn_h;
    const uint64_t* anc;  // [bs, n, words] or null: node i sees j <= i
    int words;
    int bs, n, H, G;   // G query heads per KV head; row r of a (request, KV head): node r / G, head r % G
    int nn;            // own keys per request: n, or 0 without k_new
    int row0, rows;    // the rows [row0, rows) of every (request, KV head) this launch computes
    float scale_log2;  // scale * log2(e)
    __nv_bfloat16* out;
    int64_t so_b, so_n, so_h;
    float* lse;  // [bs, n, H] or null
    float* part;
    unsigned int* tickets;
    int* status;
};

// TMA map of a cache tensor's codes: (128, page, KV heads, pages), one page of one head a box
bool make_page_map(CUtensorMap* m, const uint8_t* base, const Cache& c);
__device__ __forceinline__ void tma_page(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int head, int page) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, "
        "%5}], [%6];" ::"r"(dst),
        "l"(map), "r"(0), "r"(0), "r"(head), "r"(page), "r"(smem_addr(bar))
        : "memory");
}
template <int N>
__device__ __forceinline__ void bar_sync(int id) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(N) : "memory");
}

// Own keys a request the register kernel holds in shared memory (larger trees go to the tensor-core kernel).
constexpr int kRowsMaxOwn = 128;
// rows [p.row0, p.rows) with the register kernel (16 rows a unit)
int launch_rows(const AttnParams& p, int sms, cudaStream_t stream);
int64_t rows_tickets(int64_t bs, int64_t hkv, int64_t rows);
size_t rows_workspace(int sms);

// the same with the tensor-core kernel (tiles of 128 rows; pair: two tiles a CTA), and its combination of pieces
int launch_tc(const AttnParams& p, bool pair, int sms, cudaStream_t stream);
size_t tc_workspace(int sms);

// 64 visibility bits of own keys [64 w, 64 w + 64) for a node
__device__ __forceinline__ uint64_t visible_word(const AttnParams& p, int b, int node, int w) {
    const int left = p.nn - 64 * w;
    if (left <= 0) return 0ull;
    uint64_t v;
    if (p.anc) {
        v = w < p.words ? __ldg(p.anc + ((int64_t)b * p.n + node) * p.words + w) : 0ull;
    } else {
        const int upto = node + 1 - 64 * w;
        v = upto <= 0 ? 0ull : (upto >= 64 ? ~0ull : (1ull << upto) - 1ull);
    }
    return left >= 64 ? v : v & ((1ull << left) - 1ull);
}

}  // namespace kv8
}  // namespace mfd
