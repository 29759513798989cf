// paged_rows.cu -- paged attention for few query rows: requests whose new tokens x heads per kv head fit
// the 8 columns of a warp-level MMA (a decode step of up to 8 heads per kv head, or a few tokens of it).
//
// Math per kv head: S^T = K Q^T and O^T += V^T P^T with tokens and dims on the MMA's M side and the rows
// on its 8 columns, so no tensor work is spent on absent rows; the online softmax runs in the log2 domain.
// q (scaled by a power of two per row) and p are split into fp16 hi + lo, K and V are the cache's fp16:
// the products carry about 22 bits of fp32's 24 for any activation type.
//
// One persistent CTA per SM walks its equal share of the schedule (paged.cuh).  A producer warp fills a
// ring of stages (K and V of 16 tokens per consumer warp) with tensor copies, one per page and lane: the
// lanes look the pages up in the block table one stage ahead, so the lookup's latency is off the stream.
// A copy brings all the unit's dims of min(page, stage) rows (4-D maps); with a copy per 64 dims, 2 KB
// at 16-row pages, the copies' rate was the bound (64 ragged Llama-3-8B sequences: 232 us against 203).
// Units are published ahead of their data, so the consumers fetch q while the first stage is in flight.  Consumer warps own one kv
// head and 16 tokens of each stage; the warps' (m, l, o) meet in the unit's last stage.
//
// Bound: HBM, K and V once.
#include "mma_sync.cuh"
#include "paged.cuh"
#include "tcgen05.cuh"

#include <algorithm>

namespace yattn {
namespace {

// p is carried as 2^7 p (l and o with it; the factor cancels in o / l): p <= 2^8, as m may be stale by 8 binades,
// and the lo plane of an unscaled p under 2^-3 would fall into fp16's subnormals, 2^-25 off whatever p is, which a
// long context adds up.
constexpr float kPUp = 7.f;

template <int HD> struct RowsCfg {
    static constexpr int NCW = HD >= 256 ? 4 : 8;                // consumer warps
    static constexpr int THREADS = 32 * (NCW + 1);
    static constexpr int STAGE = 2 * 16 * NCW * HD * 2;          // K and V of 16 tokens per consumer warp
    static constexpr int NST = HD <= 64 ? 5 : 3;
    static constexpr int HC_MAX = HD <= 128 ? 2 : 1;             // kv heads per unit
    static constexpr int OFF_ML = NST * STAGE;                   // [NCW][8][2] floats
    static constexpr int NU = 4;                                 // unit descriptors in flight
    static constexpr int OFF_UNIT = OFF_ML + NCW * 8 * 2 * 4;    // [NU] units, 64 B apart
    static constexpr int OFF_BAR = OFF_UNIT + NU * 64;
    static constexpr int SMEM = OFF_BAR + (2 * NST + 2 * NU + 2) * 8 + 1024;   // + flags, + alignment slack
    static_assert(sizeof(PagedUnit) <= 64 && SMEM <= 232448, "shared memory");
    static_assert(NCW * 8 * HD * 4 <= STAGE, "the warps' o fit the unit's last stage");
};

template <int HD, int HC>
__global__ void __launch_bounds__(RowsCfg<HD>::THREADS, 1)
    k_paged_rows(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                 const __grid_constant__ PagedParams p) {
    using C = RowsCfg<HD>;
    constexpr int NCW = C::NCW, NST = C::NST, NU = C::NU;
    constexpr int KS = HD / 16;                    // k-steps (QK) and m-tiles (PV)
    constexpr uint32_t TOK = 16u * NCW / HC;       // tokens per stage = keys per block
    constexpr uint32_t TILEB = TOK * HC * HD * 2;
    constexpr uint32_t NPAN = HC * HD / 64;        // 64-dim panels of a stage's K (and V)
    constexpr uint32_t NSL = NCW / HC;             // slice warps per kv head
    using Sched = PagedSched<static_cast<int>(TOK), 0>;

    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
    uint64_t* empty = full + NST;
    uint64_t* u_full = empty + NST;
    uint64_t* u_empty = u_full + NU;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(u_empty + NU);
    int* last_flag = reinterpret_cast<int*>(u_empty + NU + 1);
    float* mrg_ml = reinterpret_cast<float*>(smem + C::OFF_ML);
    auto unit_at = [&](uint32_t i) { return reinterpret_cast<PagedUnit*>(smem + C::OFF_UNIT + (i % NU) * 64); };

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < NST; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], NCW);
        }
        for (int s = 0; s < NU; ++s) {
            mbar_init(&u_full[s], 1);
            mbar_init(&u_empty[s], NCW);
        }
        *abort_flag = 0;
        fence_mbar_init();
    }
    // (the producer looks for its share meanwhile)
    Sched sched(p);
    const bool share = warp == NCW && sched.begin();
    __syncthreads();

    if (warp == NCW) {
        // ================= producer =================
        if (lane == 0) {
            prefetch_tensormap(&kmap);
            prefetch_tensormap(&vmap);
        }
        const uint32_t page = 1u << p.page_shift;
        const uint32_t box = min(page, TOK);                  // rows of a copy
        const uint32_t per_block = TOK / box;                 // pages of a stage
        // this lane's copy: K (even) or V (odd) of page lane / 2 of the stage (8 pages at most)
        const uint32_t i_pg = lane >> 1, i_v = lane & 1;
        const bool mine = i_pg < per_block;
        uint32_t gi = 0, ui = 0;
        bool ok = true;
        auto publish = [&](const PagedUnit& u) -> bool {
            if (ui >= static_cast<uint32_t>(NU) &&
                !warp_wait_bounded(&u_empty[ui % NU], ((ui / NU) & 1u) ^ 1u, p.status, ST_PAGED_TIMEOUT, abort_flag))
                return false;
            if (lane == 0) {
                *unit_at(ui) = u;
                mbar_arrive(&u_full[ui % NU]);
            }
            ++ui;
            return true;
        };
        PagedUnit u;
        auto claim = [&](uint32_t s) -> bool {
            return gi < static_cast<uint32_t>(NST) ||
                   warp_wait_bounded(&empty[s], ((gi / NST) & 1u) ^ 1u, p.status, ST_PAGED_TIMEOUT, abort_flag);
        };
        while (ok && share && sched.next(u)) {
            ok = publish(u);
            if (!ok) break;
            const uint32_t nt = max(1u, u.kb1 - u.kb0);
            const int32_t pan0 = static_cast<int32_t>(u.g * NPAN);
            // row of this lane's copy in block b, or -1 behind the request's last key
            auto row_of = [&](uint32_t b) -> int32_t {
                const uint32_t key = b * TOK + i_pg * box;
                if (!mine || key >= static_cast<uint32_t>(u.len)) return -1;
                return paged_row(p, u.r, key >> p.page_shift) + static_cast<int32_t>(key & (page - 1));
            };
            int32_t row = u.kb1 > u.kb0 ? row_of(u.kb0) : -1;
            for (uint32_t i = 0; i < nt; ++i, ++gi) {
                const uint32_t s = gi % NST;
                if (!claim(s)) {
                    ok = false;
                    break;
                }
                const uint32_t n_copy = __popc(__ballot_sync(0xffffffffu, row >= 0));
                if (lane == 0) mbar_arrive_expect_tx(&full[s], n_copy * box * (NPAN * 128));
                __syncwarp();
                if (row >= 0)
                    tma_load_4d(smem + s * C::STAGE + i_v * TILEB + i_pg * box * (NPAN * 128), i_v ? &vmap : &kmap, 0,
                                0, pan0, row >> 3, &full[s]);
                row = i + 1 < nt ? row_of(u.kb0 + i + 1) : -1;
            }
        }
        u.done = 1;
        if (ok) publish(u);                                   // the end of the list
        // no copy may still be in flight when the CTA exits (consumers stop early on an abort)
        volatile int dummy = 0;
        for (uint32_t b = gi > static_cast<uint32_t>(NST) ? gi - NST : 0; b < gi; ++b)
            mbar_wait_bounded(&full[b % NST], (b / NST) & 1u, p.status, ST_PAGED_TIMEOUT, &dummy);
        return;
    }

    // ================= consumers =================
    const uint32_t hl = warp % HC, sl = warp / HC;            // kv head of the unit, 16-token slice of a stage
    const int g8 = lane >> 2, t4 = lane & 3;                  // fragment row (token, dim, query row), column pair
    const uint32_t rk = 16 * sl + (lane & 15), rv = 16 * sl + (lane & 7) + ((lane >> 4) & 1) * 8;
    const uint32_t hpan = hl * (HD / 64);
    // a tile is 1024-byte atoms (8 rows of a 64-dim panel, 16-byte chunk c of row r at c ^ (r & 7)), panels then
    // 8-row groups
    auto k_addr = [&](uint32_t kt, int kk) -> uint32_t {      // K fragment, k-step kk
        return kt + ((rk >> 3) * NPAN + hpan + (kk >> 2)) * 1024 + (lane & 7) * 128 +
               ((static_cast<uint32_t>(((kk & 3) << 1) + (lane >> 4)) ^ (lane & 7)) << 4);
    };
    auto v_addr = [&](uint32_t vt, int mt) -> uint32_t {      // V^T fragment, m-tile mt
        return vt + ((rv >> 3) * NPAN + hpan + (mt >> 2)) * 1024 + (lane & 7) * 128 +
               ((static_cast<uint32_t>(((mt & 3) << 1) + ((lane >> 3) & 1)) ^ (lane & 7)) << 4);
    };

    // query rows of a kv head: row f is token f / group, head f % group.  This lane's row of the Q fragment (g8)
    // and of S^T's columns (2 t4, 2 t4 + 1)
    const uint32_t tok_q = g8 / p.group, head_q = g8 % p.group;
    const int32_t tok_a = 2 * t4 / p.group, tok_b = (2 * t4 + 1) / p.group;
    uint32_t tb = 0;   // stages of this CTA's earlier units
    for (uint32_t ui = 0;; ++ui) {
        const bool got = warp_wait_bounded(&u_full[ui % NU], (ui / NU) & 1u, p.status, ST_PAGED_TIMEOUT, abort_flag);
        if (!named_bar_and(1, 32 * NCW, got)) return;
        const PagedUnit u = *unit_at(ui);
        __syncwarp();
        if (lane == 0) mbar_arrive(&u_empty[ui % NU]);
        if (u.done) return;
        const uint32_t nt = max(1u, u.kb1 - u.kb0);
        const uint32_t rows = static_cast<uint32_t>(u.n) * p.group;            // query rows per kv head, <= 8
        const uint32_t head0 = (u.g * HC + hl) * p.group;                      // first query head of this kv head

        // Q^T as the MMA B operand (column g8 = row g8), scaled to (-2, 2)
        uint32_t qhi[KS][2], qlo[KS][2];
        float up;
        {
            const bool hv = static_cast<uint32_t>(g8) < rows;
            const size_t qa = (u.tok0 + static_cast<size_t>(hv ? tok_q : 0)) * p.q_stride +
                              static_cast<size_t>(head0 + (hv ? head_q : 0)) * HD + 2 * t4;
            float2 xa[KS], xb[KS];
            float mx = 0.f;
            auto load = [&](auto pair) {
#pragma unroll
                for (int kk = 0; kk < KS; ++kk) {
                    xa[kk] = hv ? pair(qa + kk * 16) : make_float2(0.f, 0.f);
                    xb[kk] = hv ? pair(qa + kk * 16 + 8) : make_float2(0.f, 0.f);
                }
            };
            if (p.act == YATTN_ACT_F32) load([&](size_t i) { return ld_act2(p.q, i, YATTN_ACT_F32); });
            else if (p.act == YATTN_ACT_F16) load([&](size_t i) { return ld_act2(p.q, i, YATTN_ACT_F16); });
            else load([&](size_t i) { return ld_act2(p.q, i, YATTN_ACT_BF16); });
#pragma unroll
            for (int kk = 0; kk < KS; ++kk)
                mx = fmaxf(mx, fmaxf(fmaxf(fabsf(xa[kk].x), fabsf(xa[kk].y)), fmaxf(fabsf(xb[kk].x), fabsf(xb[kk].y))));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            float down;
            row_scale(mx, down, up);
#pragma unroll
            for (int kk = 0; kk < KS; ++kk) {
                split_h2(xa[kk].x * down, xa[kk].y * down, qhi[kk][0], qlo[kk][0]);
                split_h2(xb[kk].x * down, xb[kk].y * down, qhi[kk][1], qlo[kk][1]);
            }
        }
        // columns of S^T: how many keys each sees
        const float sc_a = p.scale_log2 * __shfl_sync(0xffffffffu, up, 8 * t4);
        const float sc_b = p.scale_log2 * __shfl_sync(0xffffffffu, up, 8 * t4 + 4);
        const int32_t seen0 = u.len - u.n + 1;
        const int32_t see_a = static_cast<uint32_t>(2 * t4) < rows ? seen0 + tok_a : 0;
        const int32_t see_b = static_cast<uint32_t>(2 * t4 + 1) < rows ? seen0 + tok_b : 0;

        float oc[KS][4];
#pragma unroll
        for (int mt = 0; mt < KS; ++mt) oc[mt][0] = oc[mt][1] = oc[mt][2] = oc[mt][3] = 0.f;
        float m_a = -INFINITY, m_b = -INFINITY, l_a = 0.f, l_b = 0.f;

        for (uint32_t i = 0; i < nt; ++i) {
            const uint32_t gi = tb + i, s = gi % NST;
            if (!warp_wait_bounded(&full[s], (gi / NST) & 1u, p.status, ST_PAGED_TIMEOUT, abort_flag)) break;
            const int32_t key0 = static_cast<int32_t>((u.kb0 + i) * TOK + 16 * sl);   // this warp's first key
            const int nvalid = u.kb1 > u.kb0 ? max(0, min(16, u.len - key0)) : 0;
            if (nvalid > 0) {
                const uint32_t kt = smem_u32(smem + s * C::STAGE), vt = kt + TILEB;
                // ---- S^T = K Q^T: four chains (q hi / lo x even / odd k-step) hide the MMA latency ----
                float sc[4] = {}, sc1[4] = {}, sc2[4] = {}, sc3[4] = {};
#pragma unroll
                for (int kk = 0; kk < KS; kk += 2) {
                    uint32_t a[4], b[4];
                    ldsm_x4(k_addr(kt, kk), a);
                    ldsm_x4(k_addr(kt, kk + 1), b);
                    mma16816(sc, a, qhi[kk][0], qhi[kk][1]);
                    mma16816(sc1, b, qhi[kk + 1][0], qhi[kk + 1][1]);
                    mma16816(sc2, a, qlo[kk][0], qlo[kk][1]);
                    mma16816(sc3, b, qlo[kk + 1][0], qlo[kk + 1][1]);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) sc[r] = (sc[r] + sc1[r]) + (sc2[r] + sc3[r]);
                // tokens g8 and g8 + 8, rows a and b; masked by each row's last key (which also drops the
                // stale rows behind the request's last key)
                const int32_t k0 = key0 + g8, k1 = k0 + 8;
                const float s0 = k0 < see_a ? sc[0] * sc_a : -INFINITY, s1 = k0 < see_b ? sc[1] * sc_b : -INFINITY;
                const float s2 = k1 < see_a ? sc[2] * sc_a : -INFINITY, s3 = k1 < see_b ? sc[3] * sc_b : -INFINITY;
                // m moves only where a score passes it by more than 8 binades: rarely, and then with all that hangs on it
                const bool grow = fmaxf(s0, s2) > m_a + 8.f || fmaxf(s1, s3) > m_b + 8.f;
                if (__any_sync(0xffffffffu, grow)) {
                    float mx_a = fmaxf(m_a, fmaxf(s0, s2)), mx_b = fmaxf(m_b, fmaxf(s1, s3));
#pragma unroll
                    for (int o = 4; o <= 16; o <<= 1) {
                        mx_a = fmaxf(mx_a, __shfl_xor_sync(0xffffffffu, mx_a, o));
                        mx_b = fmaxf(mx_b, __shfl_xor_sync(0xffffffffu, mx_b, o));
                    }
                    // (a row that has seen no key yet keeps m = -inf)
                    const float al_a = mx_a == -INFINITY ? 1.f : ex2_approx(m_a - mx_a);
                    const float al_b = mx_b == -INFINITY ? 1.f : ex2_approx(m_b - mx_b);
                    m_a = mx_a;
                    m_b = mx_b;
                    l_a *= al_a;
                    l_b *= al_b;
#pragma unroll
                    for (int mt = 0; mt < KS; ++mt) {
                        oc[mt][0] *= al_a;
                        oc[mt][1] *= al_b;
                        oc[mt][2] *= al_a;
                        oc[mt][3] *= al_b;
                    }
                }
                const float mp_a = (m_a == -INFINITY ? 0.f : m_a) - kPUp, mp_b = (m_b == -INFINITY ? 0.f : m_b) - kPUp;
                const float p0 = ex2_approx(s0 - mp_a), p1 = ex2_approx(s1 - mp_b);
                const float p2 = ex2_approx(s2 - mp_a), p3 = ex2_approx(s3 - mp_b);
                // row sums stay per lane (this lane's tokens); the lanes of a column add up at the unit's end
                l_a += p0 + p2;
                l_b += p1 + p3;
                // P^T as the MMA's B operand, fp16 hi and lo planes: tokens x rows to rows x tokens, 8 x 8 at a time
                uint32_t ph0, ph1, pl0, pl1;
                {
                    uint32_t h01, l01, h23, l23;
                    split_h2(p0, p1, h01, l01);
                    split_h2(p2, p3, h23, l23);
                    ph0 = movmatrix_t(h01);
                    ph1 = movmatrix_t(h23);
                    pl0 = movmatrix_t(l01);
                    pl1 = movmatrix_t(l23);
                }
                // ---- O^T = O^T + V^T P^T.  V rows behind the request's last key hold whatever the page
                // held (or nothing was copied): 0 * NaN would poison the sum, so those lanes are zeroed. ----
                uint32_t vm01 = 0xffffffffu, vm23 = 0xffffffffu;
                if (nvalid < 16) {
                    vm01 = (2 * t4 < nvalid ? 0x0000ffffu : 0u) | (2 * t4 + 1 < nvalid ? 0xffff0000u : 0u);
                    vm23 = (2 * t4 + 8 < nvalid ? 0x0000ffffu : 0u) | (2 * t4 + 9 < nvalid ? 0xffff0000u : 0u);
                }
#pragma unroll
                for (int mt = 0; mt < KS; ++mt) {
                    uint32_t a[4];
                    ldsm_x4_t(v_addr(vt, mt), a);
                    a[0] &= vm01;
                    a[1] &= vm01;
                    a[2] &= vm23;
                    a[3] &= vm23;
                    // a sum of its own, added in fp32: the tensor core truncates where it adds to an accumulator,
                    // and over a long context those half ulps all point towards zero
                    float d[4] = {};
                    mma16816(d, a, pl0, pl1);
                    mma16816(d, a, ph0, ph1);
#pragma unroll
                    for (int r = 0; r < 4; ++r) oc[mt][r] += d[r];
                }
            }
            __syncwarp();
            if (lane == 0 && i + 1 < nt) mbar_arrive(&empty[s]);   // the last stage: after the merge below
        }
#pragma unroll
        for (int o = 4; o <= 16; o <<= 1) {
            l_a += __shfl_xor_sync(0xffffffffu, l_a, o);
            l_b += __shfl_xor_sync(0xffffffffu, l_b, o);
        }

        // ---- the warps' (m, l, o) meet in the unit's last stage; every warp reaches these barriers ----
        const uint32_t s_last = (tb + nt - 1) % NST;
        float* mrg_o = reinterpret_cast<float*>(smem + s_last * C::STAGE);       // [NCW][8][HD]
        named_bar_sync(1, 32 * NCW);
        {
            const int ra = 2 * t4, rb = 2 * t4 + 1;
            if (g8 == 0) {
                *reinterpret_cast<float4*>(&mrg_ml[(warp * 8 + ra) * 2]) = make_float4(m_a, l_a, m_b, l_b);
            }
#pragma unroll
            for (int mt = 0; mt < KS; ++mt) {
                const int d0 = mt * 16 + g8, d1 = d0 + 8;
                mrg_o[(warp * 8 + ra) * HD + d0] = oc[mt][0];
                mrg_o[(warp * 8 + ra) * HD + d1] = oc[mt][2];
                mrg_o[(warp * 8 + rb) * HD + d0] = oc[mt][1];
                mrg_o[(warp * 8 + rb) * HD + d1] = oc[mt][3];
            }
        }
        named_bar_sync(1, 32 * NCW);
        constexpr int DPL = HD / 32;                          // dims [lane * DPL, +DPL) of a row are this lane's
        const bool whole = u.n_pieces == 1;
        // one warp per (kv head, query row)
        auto finish = [&](uint32_t h, uint32_t f, const float (&acc)[DPL], float l) {
            const uint32_t tk = f / p.group;
            const float inv = u.len - u.n + static_cast<int32_t>(tk) < 0 ? 0.f : 1.0f / l;   // no key seen: zeros
            const size_t tok = u.tok0 + static_cast<size_t>(tk);
            const size_t col = static_cast<size_t>((u.g * HC + h) * p.group + f - tk * p.group) * HD + lane * DPL;
            float x[DPL];
#pragma unroll
            for (int i = 0; i < DPL; ++i) x[i] = acc[i] * inv;
            if (p.gate) {
#pragma unroll
                for (int i = 0; i < DPL; i += 2) {
                    const float2 g = ld_act2(p.gate, tok * p.gate_stride + col + i, p.act);
                    x[i] *= sigmoid_of(g.x);
                    x[i + 1] *= sigmoid_of(g.y);
                }
            }
            st_act_vec<DPL>(p.out, tok * p.out_stride + col, p.act, x);
        };
        for (uint32_t row = warp; row < HC * rows; row += NCW) {
            const uint32_t h = row >= rows ? 1 : 0, f = row - h * rows;          // HC <= 2
            float M = -INFINITY, l = 0.f, acc[DPL], mw[NSL], o[DPL];
#pragma unroll
            for (uint32_t j = 0; j < NSL; ++j) {
                mw[j] = mrg_ml[((h + j * HC) * 8 + f) * 2];
                M = fmaxf(M, mw[j]);
            }
#pragma unroll
            for (int i = 0; i < DPL; ++i) acc[i] = 0.f;
#pragma unroll
            for (uint32_t j = 0; j < NSL; ++j) {
                const uint32_t at = (h + j * HC) * 8 + f;
                const float sc = mw[j] == -INFINITY ? 0.f : ex2_approx(mw[j] - M);
                l += sc * mrg_ml[at * 2 + 1];
                ld_vec<DPL>(mrg_o + at * HD + lane * DPL, o);
#pragma unroll
                for (int i = 0; i < DPL; ++i) acc[i] += sc * o[i];
            }
            if (whole) {
                finish(h, f, acc, l);
            } else {
                const size_t at = static_cast<size_t>(u.slot) * (HC * 8) + h * 8 + f;
                st_vec<DPL>(p.part_o + at * HD + lane * DPL, acc);
                if (lane == 0) *reinterpret_cast<float2*>(&p.part_ml[at * 2]) = make_float2(M, l);
            }
        }
        fence_proxy_async_smem();      // the o written here before the tensor copies that reuse the stage
        named_bar_sync(1, 32 * NCW);   // every warp is done with the stage
        if (lane == 0) mbar_arrive(&empty[s_last]);
        tb += nt;
        if (whole) continue;

        // ---- the last piece of the unit to arrive merges them all, in piece order ----
        __threadfence();
        named_bar_sync(1, 32 * NCW);
        if (threadIdx.x == 0) *last_flag = atomicInc(&p.counters[u.c_first], u.n_pieces - 1) == u.n_pieces - 1;
        named_bar_sync(1, 32 * NCW);
        if (!*last_flag) continue;
        __threadfence();
        for (uint32_t row = warp; row < HC * rows; row += NCW) {
            const uint32_t h = row >= rows ? 1 : 0, f = row - h * rows;
            // row (h, f) of piece i: slot 2 c_first + 1, then every second one from 2 (c_first + 1)
            auto at = [&](uint32_t i) { return static_cast<size_t>(piece_slot(u.c_first, i)) * (HC * 8) + h * 8 + f; };
            float2 ml[kPagedMaxPieces / 32];          // lane: pieces lane, lane + 32, ..
            float M = -INFINITY, l = 0.f, acc[DPL], o0[DPL];
            ldcg_vec_n<DPL>(p.part_o + at(0) * HD + lane * DPL, o0);
#pragma unroll
            for (int c = 0; c < kPagedMaxPieces / 32; ++c) {
                const uint32_t i = c * 32 + lane;
                ml[c] = make_float2(-INFINITY, 0.f);
                if (i < u.n_pieces) ml[c] = __ldcg(reinterpret_cast<const float2*>(&p.part_ml[at(i) * 2]));
                M = fmaxf(M, ml[c].x);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
            float w[kPagedMaxPieces / 32];
#pragma unroll
            for (int c = 0; c < kPagedMaxPieces / 32; ++c) {
                w[c] = ml[c].x == -INFINITY ? 0.f : ex2_approx(ml[c].x - M);
                l += w[c] * ml[c].y;
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
            const float w0 = __shfl_sync(0xffffffffu, w[0], 0);
#pragma unroll
            for (int i = 0; i < DPL; ++i) acc[i] = w0 * o0[i];
            constexpr uint32_t FLY = 32 / DPL;         // pieces' loads in flight
            constexpr uint32_t STEP = 2 * HC * 8 * HD; // floats between consecutive pieces
            const float* src = p.part_o + at(1) * HD + lane * DPL;
#pragma unroll
            for (int c = 0; c < kPagedMaxPieces / 32; ++c) {
                for (uint32_t k = c * 32u; k < min(u.n_pieces, c * 32u + 32u); k += FLY) {   // pieces [k, k + FLY)
                    float o[FLY][DPL];
#pragma unroll
                    for (uint32_t y = 0; y < FLY; ++y) {
#pragma unroll
                        for (int i = 0; i < DPL; ++i) o[y][i] = 0.f;
                        if (k + y >= 1 && k + y < u.n_pieces)
                            ldcg_vec_n<DPL>(src + static_cast<size_t>(k) * STEP + static_cast<int>(y - 1) * static_cast<int>(STEP), o[y]);
                    }
#pragma unroll
                    for (uint32_t y = 0; y < FLY; ++y) {
                        const float wy = __shfl_sync(0xffffffffu, w[c], (k + y) & 31);
#pragma unroll
                        for (int i = 0; i < DPL; ++i) acc[i] += wy * o[y][i];
                    }
                }
            }
            finish(h, f, acc, l);
        }
    }
}

template <int HD, int HC>
int launch(const PagedParams& p, const CUtensorMap& mk, const CUtensorMap& mv, uint32_t ctas, cudaStream_t st,
           char* err, size_t errlen) {
    using C = RowsCfg<HD>;
    static bool attr_done[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && !attr_done[dev]) {
        cudaError_t e = cudaFuncSetAttribute(k_paged_rows<HD, HC>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e != cudaSuccess) {
            set_err(err, errlen, "attn_paged: smem attribute (%d bytes): %s", C::SMEM, cudaGetErrorString(e));
            return -1;
        }
        attr_done[dev] = true;
    }
    k_paged_rows<HD, HC><<<ctas, C::THREADS, C::SMEM, st>>>(mk, mv, p);
    YATTN_CHECK_LAUNCH(err, errlen, "attn_paged");
    return 0;
}

}  // namespace

int paged_rows(const PagedParams& pp, const uint16_t* kpool, const uint16_t* vpool, uint64_t n_rows, uint32_t kv_dim,
               uint32_t hd, uint32_t n_kv, cudaStream_t st, char* err, size_t errlen) {
    PagedParams p = pp;
    p.hc = hd <= 128 && n_kv % 2 == 0 ? 2 : 1;
    p.n_groups = n_kv / p.hc;
    const uint32_t ncw = hd >= 256 ? 4 : 8, tok = 16 * ncw / p.hc;
    const uint32_t box = std::min(1u << p.page_shift, tok);
    CUtensorMap mk, mv;
    const uint32_t panels = p.hc * hd / 64;
    if (encode_page_map(&mk, kpool, kv_dim, n_rows, n_kv * hd, box, panels, err, errlen) ||
        encode_page_map(&mv, vpool, kv_dim, n_rows, n_kv * hd, box, panels, err, errlen))
        return -1;
    const uint32_t ctas = std::min<uint32_t>(static_cast<uint32_t>(dev_num_sms()), kPagedMaxPieces);
    switch (hd) {
        case 64: return p.hc == 2 ? launch<64, 2>(p, mk, mv, ctas, st, err, errlen)
                                  : launch<64, 1>(p, mk, mv, ctas, st, err, errlen);
        case 128: return p.hc == 2 ? launch<128, 2>(p, mk, mv, ctas, st, err, errlen)
                                   : launch<128, 1>(p, mk, mv, ctas, st, err, errlen);
        default: return launch<256, 1>(p, mk, mv, ctas, st, err, errlen);
    }
}

}  // namespace yattn
