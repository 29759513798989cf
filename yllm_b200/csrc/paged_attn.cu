// paged_attn.cu -- host side of the paged attention: argument checks, workspace, choice of kernel.
#include "paged.cuh"

#include <algorithm>

namespace yattn {
namespace {

// Workspace: kPagedCounters counters (zero between calls), then the partial rows' (m, l) and o, two slots per CTA and
// two CTAs per SM.  The tiles kernel's slots are the larger ones.
size_t ml_offset() { return kPagedCounters * sizeof(uint32_t); }
size_t workspace_bytes(uint32_t hd) {
    const size_t ctas = std::min<uint32_t>(static_cast<uint32_t>(dev_num_sms()), kPagedMaxPieces);
    return ml_offset() + ctas * kPagedTileRows * (4 * 2 + 4 * static_cast<size_t>(hd)) * sizeof(float);
}

int attn_paged(void* out, uint32_t out_stride, const void* q, uint32_t q_stride, const void* gate,
               uint32_t gate_stride, int act, const uint16_t* kpool, const uint16_t* vpool, uint32_t n_pages,
               uint32_t page_size, const int32_t* tables, uint32_t max_pages, uint32_t table_stride,
               const int32_t* cu_new, const int32_t* kv_len, uint32_t n_seqs, uint32_t n_tokens, uint32_t max_new,
               uint32_t n_heads, uint32_t n_kv, uint32_t hd, uint32_t kv_dim, void* ws, size_t ws_bytes,
               cudaStream_t st, char* err, size_t errlen) {
    if (n_seqs == 0 || n_tokens == 0 || max_new == 0) return 0;
    if (!out || !q || !kpool || !vpool || !tables || !cu_new || !kv_len) {
        set_err(err, errlen, "attn_paged: null pointer argument");
        return -1;
    }
    if (act != YATTN_ACT_F32 && act != YATTN_ACT_F16 && act != YATTN_ACT_BF16) {
        set_err(err, errlen, "attn_paged: unknown activation type %d", act);
        return -1;
    }
    if (!paged_size_ok(page_size)) {
        set_err(err, errlen, "attn_paged: page_size %u not supported (16/32/64/128/256)", page_size);
        return -1;
    }
    if (hd != 64 && hd != 128 && hd != 256) {
        set_err(err, errlen, "attn_paged: head_dim %u not supported (64/128/256)", hd);
        return -1;
    }
    if (n_heads == 0 || n_kv == 0 || n_heads % n_kv != 0 || n_heads > 1024) {
        set_err(err, errlen, "attn_paged: n_heads %u must be a multiple of n_kv_heads %u (1024 at most)", n_heads, n_kv);
        return -1;
    }
    if (kv_dim < n_kv * hd || (kv_dim % 8) != 0 || kv_dim > (1u << 20)) {
        set_err(err, errlen, "attn_paged: kv_dim %u must be >= n_kv_heads*head_dim and a multiple of 8", kv_dim);
        return -1;
    }
    const uint32_t unit = act == YATTN_ACT_F32 ? 4 : 8, cols = n_heads * hd;
    if (q_stride < cols || out_stride < cols || (gate && gate_stride < cols) ||
        ((q_stride | out_stride | (gate ? gate_stride : 0u)) % unit) != 0) {
        set_err(err, errlen, "attn_paged: token strides must cover the heads and be multiples of 16 bytes");
        return -1;
    }
    if ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(gate) |
         reinterpret_cast<uintptr_t>(kpool) | reinterpret_cast<uintptr_t>(vpool) | reinterpret_cast<uintptr_t>(ws)) & 15u) {
        set_err(err, errlen, "attn_paged: out, q, gate, the pools and the workspace must be 16-byte aligned");
        return -1;
    }
    if ((reinterpret_cast<uintptr_t>(tables) | reinterpret_cast<uintptr_t>(cu_new) | reinterpret_cast<uintptr_t>(kv_len)) & 3u) {
        set_err(err, errlen, "attn_paged: tables, cu_new and kv_len must be 4-byte aligned");
        return -1;
    }
    if (max_pages == 0 || (n_seqs > 1 && table_stride < max_pages) ||
        static_cast<uint64_t>(max_pages) * page_size > 0x7fffffffull) {
        set_err(err, errlen, "attn_paged: bad table shape: max_pages %u, table_stride %u", max_pages, table_stride);
        return -1;
    }
    if (n_pages == 0 || static_cast<uint64_t>(n_pages) * page_size > 0x7fffffffull) {
        set_err(err, errlen, "attn_paged: %u pages of %u tokens: more than 2^31-1 rows", n_pages, page_size);
        return -1;
    }
    if (n_seqs > 65535 || static_cast<uint64_t>(n_tokens) * n_heads > 0x7fffffffull) {
        set_err(err, errlen, "attn_paged: too many requests (%u, at most 65535) or tokens (%u)", n_seqs, n_tokens);
        return -1;
    }
    // the schedule's weights (paged.cuh) are summed in 51 bits
    const double tiles = static_cast<double>(n_tokens) * (n_heads / n_kv) / kPagedTileRows + n_seqs;
    if (tiles * (static_cast<double>(max_pages) * page_size + 1024.0) * n_heads > 1e15) {
        set_err(err, errlen, "attn_paged: %u tokens over tables of %u pages: more work than one call can divide", n_tokens,
                max_pages);
        return -1;
    }
    if (!ws || ws_bytes < workspace_bytes(hd)) {
        set_err(err, errlen, "attn_paged: workspace of %zu bytes, %zu needed", ws ? ws_bytes : static_cast<size_t>(0),
                workspace_bytes(hd));
        return -1;
    }
    DevCtx* ctx = dev_ctx(err, errlen);
    if (!ctx) return -1;
    PagedParams p{};
    p.q = q;
    p.gate = gate;
    p.out = out;
    p.tables = tables;
    p.cu = cu_new;
    p.kv_len = kv_len;
    p.q_stride = q_stride;
    p.gate_stride = gate_stride;
    p.out_stride = out_stride;
    p.table_stride = table_stride;
    p.max_pages = max_pages;
    p.n_pages = n_pages;
    p.page_shift = static_cast<uint32_t>(__builtin_ctz(page_size));
    p.n_tokens = n_tokens;
    p.n_seqs = n_seqs;
    p.max_new = std::min(max_new, n_tokens);
    p.n_heads = n_heads;
    p.group = n_heads / n_kv;
    // x / d = x * ceil(2^(31 + l) / d) >> (31 + l) for x < 2^31, l = ceil(log2 d)
    uint32_t l = 0;
    while ((1u << l) < p.group) ++l;
    p.group_s = 31 + l;
    p.group_m = static_cast<uint32_t>(((1ull << p.group_s) + p.group - 1) / p.group);
    p.act = act;
    p.scale_log2 = 1.4426950408889634f / sqrtf(static_cast<float>(hd));
    p.counters = static_cast<uint32_t*>(ws);
    p.part_ml = reinterpret_cast<float*>(static_cast<char*>(ws) + ml_offset());
    p.part_o = p.part_ml + 2 * static_cast<size_t>(kPagedTileRows) *
                               (4 * std::min<uint32_t>(static_cast<uint32_t>(dev_num_sms()), kPagedMaxPieces));
    p.status = ctx->status;
    const uint64_t n_rows = static_cast<uint64_t>(n_pages) * page_size;
    // up to 8 query rows per kv head the warp-level kernel wastes no tensor work on absent rows; above, 128-row tiles
    p.rows_hi = 0xffffffffu;
    if (static_cast<uint64_t>(p.max_new) * p.group <= kPagedRows)
        return paged_rows(p, kpool, vpool, n_rows, kv_dim, hd, n_kv, st, err, errlen);
    // Many requests, most of them of far fewer tokens than the largest: with fp32 activations, whose tiles take four
    // products, those that fit the warp-level kernel go there in a second launch.  From a request's kv head per SM on;
    // the launch costs 8 to 10 us where it finds less (Llama-3-8B shape: 28 single tokens beside 4 chunks 352 -> 314 us,
    // 63 beside one 186 -> 150, but 14 beside 2 76 -> 85).  With 16-bit activations it mostly loses: bf16 221 -> 238
    const bool split = act == YATTN_ACT_F32 && p.group <= kPagedRows &&
                       static_cast<uint64_t>(n_seqs) * n_kv >= static_cast<uint64_t>(ctx->num_sms) &&
                       static_cast<uint64_t>(n_tokens) * 4 <= static_cast<uint64_t>(n_seqs) * p.max_new;
    if (split) p.rows_lo = kPagedRows + 1;
    const int rc = paged_tiles(p, kpool, vpool, n_rows, kv_dim, hd, n_kv, st, err, errlen);
    if (rc != 0 || !split) return rc;
    p.rows_lo = 0;
    p.rows_hi = kPagedRows;
    return paged_rows(p, kpool, vpool, n_rows, kv_dim, hd, n_kv, st, err, errlen);
}

}  // namespace
}  // namespace yattn

using namespace yattn;

extern "C" size_t yattn_attn_paged_workspace_bytes(uint32_t head_dim) { return workspace_bytes(head_dim); }

extern "C" int yattn_attn_paged(void* out, uint32_t out_stride, const void* q, uint32_t q_stride, const void* gate,
                                uint32_t gate_stride, int act, const uint16_t* kpool, const uint16_t* vpool,
                                uint32_t n_pages, uint32_t page_size, const int32_t* tables, uint32_t max_pages,
                                uint32_t table_stride, const int32_t* cu_new, const int32_t* kv_len, uint32_t n_seqs,
                                uint32_t n_tokens, uint32_t max_new, uint32_t n_heads, uint32_t n_kv_heads,
                                uint32_t head_dim, uint32_t kv_dim, void* workspace, size_t workspace_bytes_given,
                                void* stream, char* err, size_t errlen) {
    return attn_paged(out, out_stride, q, q_stride, gate, gate_stride, act, kpool, vpool, n_pages, page_size, tables,
                      max_pages, table_stride, cu_new, kv_len, n_seqs, n_tokens, max_new, n_heads, n_kv_heads,
                      head_dim, kv_dim, workspace, workspace_bytes_given, static_cast<cudaStream_t>(stream), err,
                      errlen);
}
