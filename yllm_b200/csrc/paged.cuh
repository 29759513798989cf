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
// The line is never built: w summed over a request's tiles has a closed form, so one warp of the CTA needs
// one pass over (cu, kv_len) -- a sum and a scan -- and then walks its units in order.
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
    uint32_t rows_lo, rows_hi;        // requests of rows_lo to rows_hi query rows per kv head are this launch's
    uint32_t group_m, group_s;        // x / group = x * group_m >> group_s for x < 2^31
    uint32_t hc, n_groups;            // kv heads per unit, units' head groups (n_kv / hc)
    int act;                          // YATTN_ACT_*
    float scale_log2;                 // log2(e) / sqrt(head_dim)
    uint32_t* counters;               // [gridDim.x]: pieces of a cut unit that are done, by its first CTA
    float* part_ml;                   // [2 * gridDim.x][rows][2]
    float* part_o;                    // [2 * gridDim.x][rows][HD]: two partials a CTA (tiles: or a folded sum in the second)
    int* status;
};

constexpr uint32_t kPagedCounters = 1024;        // most CTAs of a launch
constexpr int kPagedMaxPieces = 5 * 32;          // decode form: most CTAs, each of which holds a piece of a unit at most
                                                 // (the tiles' merge has no such bound; they run up to two CTAs per SM)

// Activations of the call's type, as fp32.
__device__ __forceinline__ float2 ld_act2(const void* p, size_t i, int act) {
    if (act == YATTN_ACT_F32) return *reinterpret_cast<const float2*>(static_cast<const float*>(p) + i);
    const uint32_t w = *reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(p) + i);
    if (act == YATTN_ACT_F16) return h2f2(w);
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
// N = 2, 4 or 8 consecutive values (N * size aligned): activations out, fp32 in shared or global memory.
template <int N> __device__ __forceinline__ void st_act_vec(void* p, size_t i, int act, const float (&x)[N]) {
    if (act == YATTN_ACT_F32) {
        float* d = static_cast<float*>(p) + i;
        if constexpr (N == 2) *reinterpret_cast<float2*>(d) = make_float2(x[0], x[1]);
        else
#pragma unroll
            for (int k = 0; k < N; k += 4) *reinterpret_cast<float4*>(d + k) = make_float4(x[k], x[k + 1], x[k + 2], x[k + 3]);
        return;
    }
    uint32_t w[N / 2];
#pragma unroll
    for (int k = 0; k < N / 2; ++k) {
        if (act == YATTN_ACT_F16) {
            const __half2 h = __floats2half2_rn(x[2 * k], x[2 * k + 1]);
            w[k] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
            const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * k], x[2 * k + 1]);
            w[k] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
    uint16_t* d = static_cast<uint16_t*>(p) + i;
    if constexpr (N == 2) *reinterpret_cast<uint32_t*>(d) = w[0];
    else if constexpr (N == 4) *reinterpret_cast<uint2*>(d) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint4*>(d) = make_uint4(w[0], w[1], w[2], w[3]);
}
template <int N> __device__ __forceinline__ void ld_vec(const float* p, float (&x)[N]) {
    if constexpr (N == 2) {
        const float2 v = *reinterpret_cast<const float2*>(p);
        x[0] = v.x;
        x[1] = v.y;
    } else {
#pragma unroll
        for (int k = 0; k < N; k += 4) {
            const float4 v = *reinterpret_cast<const float4*>(p + k);
            x[k] = v.x;
            x[k + 1] = v.y;
            x[k + 2] = v.z;
            x[k + 3] = v.w;
        }
    }
}
template <int N> __device__ __forceinline__ void ldcg_vec_n(const float* p, float (&x)[N]) {
    if constexpr (N == 2) {
        const float2 v = __ldcg(reinterpret_cast<const float2*>(p));
        x[0] = v.x;
        x[1] = v.y;
    } else {
#pragma unroll
        for (int k = 0; k < N; k += 4) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(p + k));
            x[k] = v.x;
            x[k + 1] = v.y;
            x[k + 2] = v.z;
            x[k + 3] = v.w;
        }
    }
}
template <int N> __device__ __forceinline__ void st_vec(float* p, const float (&x)[N]) {
    if constexpr (N == 2) *reinterpret_cast<float2*>(p) = make_float2(x[0], x[1]);
    else
#pragma unroll
        for (int k = 0; k < N; k += 4) *reinterpret_cast<float4*>(p + k) = make_float4(x[k], x[k + 1], x[k + 2], x[k + 3]);
}
// (the approximate reciprocal is 1 ulp off; the exact division took a gated unit's 128 per thread 3 us)
__device__ __forceinline__ float sigmoid_of(float x) { return __fdividef(1.0f, 1.0f + __expf(-x)); }

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

__device__ __forceinline__ uint32_t div_group(const PagedParams& p, uint32_t x) {
    return static_cast<uint32_t>(static_cast<uint64_t>(x) * p.group_m >> p.group_s);
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
    const uint32_t rows = static_cast<uint32_t>(q.n) * p.group;
    if (rows < p.rows_lo || rows > p.rows_hi) q.n = 0;
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
    int32_t keys;               // keys that the tile's last row sees
    uint32_t done;              // 1: no unit, the list has ended
};

// a / b; the usual operands fit 32 bits, where the division is several times shorter.
__device__ __forceinline__ long long div_pos(long long a, long long b) {
    if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
    return a / b;
}

// ROWS: query rows per tile (a row is one token x one head of the group); 0: a request's rows are one tile.
// One warp runs it, all lanes.  Weights are in units of 1 / group key where ROWS, so that no sum needs a division.
// PAIR: two CTAs share an SM and hide part of each other's fixed steps.  GATE_KEYS: charged for a unit whose output is
// gated.
template <int BN, int ROWS, bool PAIR = false, int GATE_KEYS = 0> struct PagedSched {
    // Keys charged for a unit besides its own, the least keys of a share where units are cut, the least blocks of a
    // cut unit's first and last piece.  A cut costs a partial's round trip through memory.  Decode form: about
    // 2.5 us, and a block 0.9 us when nothing else runs: shares of 128 beat 512 from 512 keys on (one Llama-3-8B
    // sequence, 1024 keys: 12.0 us against 17.6), and cutting a unit less than about fourfold loses (256 keys:
    // 12.0 us cut, 11.1 whole).
    static constexpr long long kUnitCost = ROWS ? (PAIR ? 384 : 512) : 192;
    static constexpr long long kMinShare = ROWS ? 512 : 128;
    static constexpr uint32_t kSnap = ROWS ? (PAIR ? 128 : 256) / BN : 1;
    static constexpr long long kCutFrom = ROWS ? 2 : 4;   // cut where a unit would get that many shares on average
    static_assert(kUnitCost >= BN && kMinShare >= BN, "a share inside a unit holds a block, so a cut unit's pieces are contiguous CTAs");

    const PagedParams& p;
    int lane;
    long long W, total, x0, x1;   // weight of a head group and in all; this CTA's share
    long long per, rem;           // total = per * n_active + rem: the first rem shares are one longer
    long long base;               // weight of the group's requests before r
    uint32_t n_active, cta, g, r, j;

    __device__ __forceinline__ explicit PagedSched(const PagedParams& pp) : p(pp) {}

    static __device__ __forceinline__ long long unit_keys(const PagedParams& p) {
        return kUnitCost + (GATE_KEYS && p.gate ? GATE_KEYS : 0);
    }
    static __device__ __forceinline__ long long unit_cost(const PagedParams& p) {
        return ROWS ? unit_keys(p) * p.group : kUnitCost;
    }
    static __device__ __forceinline__ long long block_cost(const PagedParams& p) { return ROWS ? BN * static_cast<long long>(p.group) : BN; }
    static __device__ __forceinline__ uint32_t tiles(const PagedParams& p, const PagedReq& q) {
        if (!ROWS) return q.n > 0 ? 1u : 0u;
        return (static_cast<uint32_t>(q.n) * p.group + ROWS - 1) / (ROWS ? ROWS : 1);
    }
    // weight of the request's tiles before tile t: kUnitCost and about the keys its last row sees, each
    static __device__ __forceinline__ long long before(const PagedParams& p, const PagedReq& q, uint32_t t) {
        if (!ROWS) return t ? kUnitCost + q.len : 0;
        const long long T = t;
        return T * ((unit_keys(p) + max(q.len - q.n, 0)) * p.group) + T * (T + 1) * (ROWS / 2);
    }
    static __device__ __forceinline__ long long weight(const PagedParams& p, const PagedReq& q) {
        return before(p, q, tiles(p, q));
    }
    // keys that tile t's rows see: up to its last row's position
    static __device__ __forceinline__ int32_t keys(const PagedParams& p, const PagedReq& q, uint32_t t) {
        if (!ROWS) return q.len;
        const uint32_t rows = static_cast<uint32_t>(q.n) * p.group;
        const uint32_t last = div_group(p, min(rows, (t + 1) * ROWS) - 1);
        return max(q.len - q.n + static_cast<int32_t>(last) + 1, 0);
    }
    __device__ __forceinline__ long long border(uint32_t c) const { return per * c + min(static_cast<long long>(c), rem); }
    // The key block at which a border at x cuts a unit at [us, us + w) of nb blocks.
    __device__ __forceinline__ uint32_t cut(long long x, long long us, long long w, uint32_t nb) const {
        const long long y = x - us - unit_cost(p);
        if (x >= us + w || y >= static_cast<long long>(nb) * block_cost(p)) return nb;
        if (y <= 0) return 0;
        const long long b = y / BN;                      // (BN is a power of two)
        const uint32_t t = !ROWS ? static_cast<uint32_t>(b)
                           : (b >> 31) == 0 ? div_group(p, static_cast<uint32_t>(b)) : static_cast<uint32_t>(b / p.group);
        return t < kSnap ? 0u : nb - t < kSnap ? nb : t;
    }
    // The first CTA whose share ends at x or behind it (0 < x <= total).
    __device__ __forceinline__ uint32_t ends_at(long long x) const {
        const long long head = (per + 1) * rem;       // where the longer shares end
        const long long c = x <= head ? div_pos(x + per, per + 1) : rem + div_pos(x - head + per - 1, per);
        return static_cast<uint32_t>(c) - 1;
    }
    // A sum over the warp of values below 2^51 (the call checks that), in two parts, one reduction instruction each.
    static __device__ __forceinline__ long long warp_sum(long long x) {
        const uint32_t lo = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(x) & 0xffffffu);
        const uint32_t hi = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(x >> 24));
        return (static_cast<long long>(hi) << 24) + lo;
    }

    // This CTA's share and the unit it starts in; false: no share.
    __device__ bool begin() {
        lane = static_cast<int>(threadIdx.x & 31);
        cta = blockIdx.x;
        long long first = 0, sum = 0;                  // weight of request lane, and of all of this lane's
        uint32_t units = 0;                            // tiles of a head group
#pragma unroll 4
        for (uint32_t i = lane; i < p.n_seqs; i += 32) {
            const PagedReq q = paged_req(p, i);
            const long long w = weight(p, q);
            if (i == static_cast<uint32_t>(lane)) first = w;
            sum += w;
            units += tiles(p, q);
        }
        sum = warp_sum(sum);
        units = __reduce_add_sync(0xffffffffu, units);
        W = sum;
        if (W == 0) return false;
        total = W * p.n_groups;
        // as many shares as hold kMinShare keys, or a share per unit where that would cut units into fewer than kCutFrom
        const long long all = static_cast<long long>(units) * p.n_groups, fine = ROWS ? div_pos(total, kMinShare * p.group) : total / kMinShare;
        n_active = static_cast<uint32_t>(min(static_cast<long long>(gridDim.x), fine < kCutFrom * all ? all : fine));
        if (cta >= n_active) return false;
        per = div_pos(total, n_active);
        rem = total - per * n_active;
        x0 = border(cta);
        x1 = border(cta + 1);
        g = static_cast<uint32_t>(div_pos(x0, W));
        const long long y = x0 - g * W;
        // the request whose weights hold y
        long long carry = 0;
        bool found = false;
        auto look = [&](uint32_t chunk, long long w) {
            long long s = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long u = __shfl_up_sync(0xffffffffu, s, o);
                if (lane >= o) s += u;
            }
            const uint32_t m = __ballot_sync(0xffffffffu, carry + s > y);
            if (m) {
                const int k = __ffs(m) - 1;
                r = chunk + k;
                base = carry + __shfl_sync(0xffffffffu, s - w, k);
                found = true;
            } else {
                carry += __shfl_sync(0xffffffffu, s, 31);
            }
        };
#pragma unroll 1
        for (uint32_t chunk = 0; !found && chunk < p.n_seqs; chunk += 32)
            look(chunk, chunk == 0 ? first : chunk + lane < p.n_seqs ? weight(p, paged_req(p, chunk + lane)) : 0);
        // the tile of r that holds y: before() is quadratic in t, so its root (rounded) and a step or two
        j = 0;
        if (ROWS) {
            const PagedReq q = paged_req(p, r);
            const uint32_t nt = tiles(p, q);
            if (nt > 1) {
                const long long in = y - base;
                const float a = static_cast<float>(before(p, q, 1)) * (1.0f / ROWS), c = static_cast<float>(in) * (2.0f / ROWS);
                j = min(nt - 1, static_cast<uint32_t>(c / (a + sqrtf(a * a + c))));
                while (j + 1 < nt && before(p, q, j + 1) <= in) ++j;
                while (before(p, q, j) > in) --j;
            }
        }
        return true;
    }

    // The next unit of the share into u; false when the share has ended.
    __device__ bool next(PagedUnit& u) {
        for (;;) {
            if (g >= p.n_groups) return false;
            const PagedReq q = paged_req(p, r);
            const uint32_t nt = tiles(p, q);
            if (j >= nt) {                             // on to the next request that has work
                base += before(p, q, nt);
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
            const long long at = before(p, q, j), us = g * W + base + at, w = before(p, q, j + 1) - at;
            if (us >= x1) return false;
            u.keys = keys(p, q, j);
            const uint32_t nb = (static_cast<uint32_t>(u.keys) + BN - 1) / BN;
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
                u.kb0 = u.kb1 = 0;
                return true;
            }
            if (u.kb0 >= u.kb1) continue;
            if (u.kb0 > 0 || u.kb1 < nb) {
                // the first piece ends where the unit is first cut behind block 0, the last one where nothing is left
                const long long uc = unit_cost(p), bc = block_cost(p);
                u.c_first = ends_at(us + min(w, uc + kSnap * bc));
                u.n_pieces = ends_at(us + min(w, uc + max(kSnap, nb - kSnap + 1) * bc)) - u.c_first + 1;
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
