// paged.cuh -- what the two kernels of the paged attention share: parameters, the schedule, the merge.
//
// Work.  A unit is one head group x one request x one tile of its query rows; it reads the keys its last
// row sees, in blocks of BN.  Lengths are known on the device only, so every CTA finds its own share:
// with w(unit) = kUnitCost + keys laid end to end (head group, then request, then tile), CTA c of A takes
// [c, c+1) * total / A of that line.  A unit that a border cuts is shared by the CTAs on both sides at a
// key block; each leaves (m, l, o) of its piece in a slot of its own and the last one to finish merges
// the pieces in piece order, so the result does not depend on who was last.  The shares are equal
// whatever the lengths: one long context spreads over every SM, and 64 ragged ones fill them evenly.
//
// The line is never built: w summed over a request's tiles has a closed form, so a CTA needs one pass
// over (cu, kv_len) -- a block-wide sum and scan -- and then walks its units in order.
#pragma once

#include "common.cuh"

#include <cuda_bf16.h>

namespace yattn {

struct PagedParams {
    const void* q;
    const void* gate;                 // NULL: none
    void* out;
    const int32_t* tables;
    const int32_t* cu;                // [n_seqs + 1] first token of each request
    const int32_t* kv_len;            // [n_seqs] keys of each request, its new tokens included
    uint64_t q_stride, gate_stride, out_stride;   // elements between tokens
    uint32_t table_stride, max_pages, n_pages, page_shift;
    uint32_t n_tokens, n_seqs, max_new;
    uint32_t n_heads, group;          // query heads, query heads per kv head
    uint32_t hc, n_groups;            // kv heads per unit, units' head groups (n_kv / hc)
    int act;                          // YATTN_ACT_*
    float scale_log2;                 // log2(e) / sqrt(head_dim)
    uint32_t* counters;               // [gridDim.x]: pieces of a cut unit that are done, by its first CTA
    float* part_ml;                   // [2 * gridDim.x][rows][2]
    float* part_o;                    // [2 * gridDim.x][rows][HD]
    int* status;
};

constexpr uint32_t kPagedCounters = 1024;        // most CTAs of a launch
constexpr int kPagedMaxPieces = 5 * 32;          // a cut unit has at most one piece per CTA

// Activations of the call's type, as fp32.
__device__ __forceinline__ float2 ld_act2(const void* p, size_t i, int act) {
    if (act == YATTN_ACT_F32) return *reinterpret_cast<const float2*>(static_cast<const float*>(p) + i);
    const uint32_t w = *reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(p) + i);
    if (act == YATTN_ACT_F16) return h2f2(w);
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float ld_act(const void* p, size_t i, int act) {
    if (act == YATTN_ACT_F32) return static_cast<const float*>(p)[i];
    const uint16_t w = static_cast<const uint16_t*>(p)[i];
    return act == YATTN_ACT_F16 ? h2f(w) : __uint_as_float(static_cast<uint32_t>(w) << 16);
}
__device__ __forceinline__ void st_act(void* p, size_t i, int act, float x) {
    if (act == YATTN_ACT_F32) static_cast<float*>(p)[i] = x;
    else if (act == YATTN_ACT_F16) static_cast<__half*>(p)[i] = __float2half_rn(x);
    else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
}
__device__ __forceinline__ float sigmoid_of(float x) { return 1.0f / (1.0f + __expf(-x)); }

// 2^-e and 2^e with 2^e <= |mx| < 2^(e+1): a q row times 2^-e has its values in (-2, 2), where fp16 hi + lo
// keep about 22 bits of the largest, whatever the row's magnitude.  Zero, infinite and NaN rows: 1.
__device__ __forceinline__ void row_scale(float mx, float& down, float& up) {
    const uint32_t ex = min(max((__float_as_uint(mx) >> 23) & 255u, 1u), 255u);
    if (mx == 0.f || ex == 255u) {
        down = up = 1.f;
        return;
    }
    const uint32_t e = min(ex, 253u);
    down = __uint_as_float((254u - e) << 23);
    up = __uint_as_float(e << 23);
}

// ------------------------------------------------------------------ requests

struct PagedReq {
    int32_t tok0, n, len;   // first token, tokens, keys; n = 0: nothing to do
};
__device__ __forceinline__ PagedReq paged_req(const PagedParams& p, uint32_t r) {
    PagedReq q;
    q.tok0 = p.cu[r];
    const int32_t end = p.cu[r + 1];
    q.len = p.kv_len[r];
    q.n = end - q.tok0;
    if (q.tok0 < 0 || end < q.tok0 || static_cast<uint32_t>(end) > p.n_tokens || q.len < 0 ||
        static_cast<uint32_t>(q.n) > p.max_new ||
        static_cast<uint64_t>(q.len) > (static_cast<uint64_t>(p.max_pages) << p.page_shift)) {
        atomicCAS(p.status, 0, ST_PAGED_BAD_REQUEST);
        q.tok0 = q.n = q.len = 0;
    }
    return q;
}

// A block table entry as the first row of its page, or a row past the pool (tensor copies read zeros there).
__device__ __forceinline__ int32_t paged_row(const PagedParams& p, uint32_t r, uint32_t page_index) {
    const int32_t page = __ldg(p.tables + static_cast<size_t>(r) * p.table_stride + page_index);
    if (static_cast<uint32_t>(page) < p.n_pages) return page << p.page_shift;
    atomicCAS(p.status, 0, ST_PAGED_BAD_PAGE);
    return static_cast<int32_t>(p.n_pages << p.page_shift);
}

// ------------------------------------------------------------------ schedule

struct PagedUnit {
    uint32_t g, r, j;           // head group, request, query tile
    int32_t tok0, n, len;       // the request
    uint32_t kb0, kb1;          // key blocks of this piece
    uint32_t n_pieces;          // 1: the unit is whole
    uint32_t c_first;           // CTA of the unit's first piece
    uint32_t slot;              // this piece's partial slot
    uint32_t done;              // 1: no unit, the list has ended
};

// ROWS: query rows per tile (a row is one token x one head of the group); 0: a request's rows are one tile.
template <int BN, int ROWS> struct PagedSched {
    // keys charged for a unit besides its own, shortest share, and least blocks at a cut
    static constexpr long long kUnitCost = ROWS ? 384 : 192;
    static constexpr long long kMinShare = ROWS ? 512 : 256;
    static constexpr uint32_t kSnap = 1;
    // a share inside a unit holds a block: a unit charges at most BN + 128 keys per block once it has two
    static_assert(kMinShare >= BN + 128 && kUnitCost / kMinShare < 8, "pieces are contiguous and found in one probe");

    const PagedParams& p;
    int lane;
    long long W, total, x0, x1;   // weight of a head group and in all; this CTA's share
    long long base;               // weight of the group's requests before r
    uint32_t n_active, cta, g, r, j;

    __device__ __forceinline__ explicit PagedSched(const PagedParams& pp) : p(pp) {}

    static __device__ __forceinline__ uint32_t tiles(const PagedParams& p, const PagedReq& q) {
        if (!ROWS) return q.n > 0 ? 1u : 0u;
        return (static_cast<uint32_t>(q.n) * p.group + ROWS - 1) / (ROWS ? ROWS : 1);
    }
    // weight of the request's tiles before tile t
    static __device__ __forceinline__ long long before(const PagedParams& p, const PagedReq& q, uint32_t t) {
        if (!ROWS) return t ? kUnitCost + q.len : 0;
        const long long T = t;
        return T * (kUnitCost + max(q.len - q.n, 0)) + T * (T + 1) * (ROWS / 2) / p.group;
    }
    static __device__ __forceinline__ long long weight(const PagedParams& p, const PagedReq& q) {
        return before(p, q, tiles(p, q));
    }
    // key blocks of tile t: up to the last position its rows see
    static __device__ __forceinline__ uint32_t blocks(const PagedParams& p, const PagedReq& q, uint32_t t) {
        return static_cast<uint32_t>(keys(p, q, t) + BN - 1) / BN;
    }
    static __device__ __forceinline__ int32_t keys(const PagedParams& p, const PagedReq& q, uint32_t t) {
        if (!ROWS) return q.len;
        const uint32_t rows = static_cast<uint32_t>(q.n) * p.group;
        const uint32_t last = (min(rows, (t + 1) * ROWS) - 1) / p.group;
        return max(q.len - q.n + static_cast<int32_t>(last) + 1, 0);
    }
    __device__ __forceinline__ long long border(uint32_t c) const {
        return total * static_cast<long long>(c) / static_cast<long long>(n_active);
    }
    // The key block at which a border at x cuts a unit at [us, us + w) of nb blocks.
    static __device__ __forceinline__ uint32_t cut(long long x, long long us, long long w, uint32_t nb) {
        if (x >= us + w) return nb;
        const long long y = x - us - kUnitCost;
        if (y <= 0) return 0;
        const uint32_t t = static_cast<uint32_t>(y * nb / (w - kUnitCost));
        return t < kSnap ? 0u : nb - t < kSnap ? nb : t;
    }

    // Every thread of the block: this CTA's share and the request it starts in.  scratch: 40 long longs of
    // shared memory.  Ends with a block barrier; false: no share.
    __device__ bool locate(long long* scratch) {
        const uint32_t tid = threadIdx.x, nt = blockDim.x, nw = nt / 32, warp = tid / 32;
        lane = static_cast<int>(tid & 31);
        cta = blockIdx.x;
        long long first = 0, sum = 0;   // weight of request tid, and of all of this thread's
        for (uint32_t i = tid; i < p.n_seqs; i += nt) {
            const long long w = weight(p, paged_req(p, i));
            if (i == tid) first = w;
            sum += w;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) scratch[warp] = sum;
        __syncthreads();
        W = 0;
        for (uint32_t w = 0; w < nw; ++w) W += scratch[w];
        total = W * p.n_groups;
        n_active = static_cast<uint32_t>(min(static_cast<long long>(gridDim.x), max(total / kMinShare, 1ll)));
        if (W == 0 || cta >= n_active) return false;   // the whole block
        x0 = border(cta);
        x1 = border(cta + 1);
        g = static_cast<uint32_t>(x0 / W);
        const long long y = x0 - g * W;
        // the request whose weights hold y
        long long carry = 0;
        for (uint32_t chunk = 0; chunk < p.n_seqs; chunk += nt) {
            const uint32_t i = chunk + tid;
            const long long w = chunk == 0 ? first : i < p.n_seqs ? weight(p, paged_req(p, i)) : 0;
            long long s = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long u = __shfl_up_sync(0xffffffffu, s, o);
                if (lane >= o) s += u;
            }
            __syncthreads();                           // the last round's sums have been read
            if (lane == 31) scratch[warp] = s;
            __syncthreads();
            long long at = carry, all = carry;
            for (uint32_t k = 0; k < nw; ++k) {
                if (k < warp) at += scratch[k];
                all += scratch[k];
            }
            if (at + s - w <= y && y < at + s) {
                scratch[32] = i;
                scratch[33] = at + s - w;
            }
            carry = all;
            if (y < carry) break;                      // uniform: found in this chunk
        }
        __syncthreads();
        r = static_cast<uint32_t>(scratch[32]);
        base = scratch[33];
        // the tile of r that holds y: before() grows with t
        const PagedReq q = paged_req(p, r);
        uint32_t lo = 0, hi = tiles(p, q);
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if (base + before(p, q, mid) <= y) lo = mid; else hi = mid;
        }
        j = lo;
        return true;
    }

    // One warp, all lanes: the next unit of the share into u; false when the share has ended.
    __device__ bool next(PagedUnit& u) {
        for (;;) {
            if (g >= p.n_groups) return false;
            const PagedReq q = paged_req(p, r);
            const uint32_t nt = tiles(p, q);
            if (j >= nt) {                             // on to the next request that has work
                base += weight(p, q);
                ++r;
                j = 0;
                for (;;) {
                    if (r >= p.n_seqs) {
                        ++g;
                        if (g >= p.n_groups) return false;
                        r = 0;
                        base = 0;
                    }
                    const uint32_t i = r + lane;
                    const uint32_t m = __ballot_sync(0xffffffffu, i < p.n_seqs && paged_req(p, i).n > 0);
                    if (m) {
                        r += __ffs(m) - 1;
                        break;
                    }
                    r += 32;
                }
                continue;
            }
            const long long us = g * W + base + before(p, q, j);
            const long long w = base + before(p, q, j + 1) + g * W - us;
            if (us >= x1) return false;
            const uint32_t nb = blocks(p, q, j);
            u.g = g;
            u.r = r;
            u.j = j++;
            u.tok0 = q.tok0;
            u.n = q.n;
            u.len = q.len;
            u.kb0 = cut(x0, us, w, nb);
            u.kb1 = cut(x1, us, w, nb);
            u.n_pieces = 1;
            u.c_first = 0;
            u.slot = 0;
            u.done = 0;
            if (nb == 0) {                             // no key to see: whoever holds its start writes zeros
                if (us < x0) continue;
                return true;
            }
            if (u.kb0 >= u.kb1) continue;
            if (u.kb0 > 0 || u.kb1 < nb) {
                // The first piece is the first CTA whose end border cuts past block 0, the last one the first
                // whose end border cuts at nb; between them every CTA has a piece (kMinShare).
                const uint32_t ca = static_cast<uint32_t>(max(us * n_active / total - 2, 0ll)) + lane;
                const bool past = ca < n_active && cut(border(ca + 1), us, w, nb) > 0;
                const long long tail = max(us + w - (BN + 128) * static_cast<long long>(kSnap), 0ll);
                const uint32_t cb = static_cast<uint32_t>(max(tail * n_active / total - 3, 0ll)) + lane;
                const bool whole = cb < n_active && cut(border(cb + 1), us, w, nb) == nb;
                const uint32_t ma = __ballot_sync(0xffffffffu, past), mb = __ballot_sync(0xffffffffu, whole);
                u.c_first = __shfl_sync(0xffffffffu, ca, __ffs(ma) - 1);
                u.n_pieces = __shfl_sync(0xffffffffu, cb, __ffs(mb) - 1) - u.c_first + 1;
                u.slot = 2 * cta + (u.kb0 > 0 ? 0u : 1u);
            }
            return true;
        }
    }
};

// Partial slot of piece i of a cut unit: a first piece ends its CTA's share, any other one begins its CTA's.
__device__ __forceinline__ uint32_t piece_slot(uint32_t c_first, uint32_t i) {
    return i == 0 ? 2 * c_first + 1 : 2 * (c_first + i);
}

// ---------------------------------------------------------------- host side

int paged_rows(const PagedParams& p, const uint16_t* kpool, const uint16_t* vpool, uint64_t n_rows, uint32_t kv_dim,
               uint32_t hd, uint32_t n_kv, cudaStream_t st, char* err, size_t errlen);
int paged_tiles(const PagedParams& p, const uint16_t* kpool, const uint16_t* vpool, uint64_t n_rows, uint32_t kv_dim,
                uint32_t hd, uint32_t n_kv, cudaStream_t st, char* err, size_t errlen);

constexpr uint32_t kPagedRows = 8;      // query rows per kv head the rows kernel takes (an MMA's columns)
constexpr uint32_t kPagedTileRows = 128;

}  // namespace yattn
