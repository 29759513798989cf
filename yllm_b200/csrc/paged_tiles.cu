// paged_tiles.cu -- paged attention of token chunks on tcgen05 / TMEM / TMA: 128-row query tiles.
//
// A tile's rows are (token, head of the kv head's group) pairs, token-major, so a kv head's K and V are read
// once for all its query heads, any group size fills the tile, and one ragged batch may mix long chunks
// with single tokens.  Math per key block of BN keys, in the log2 domain with a running maximum m:
//     S = Q K^T,  P = 2^(S c - m),  l = l 2^(m_old - m) + sum P,  O = O 2^(m_old - m) + P V.
// fp32 activations (PREC): q = hi + lo and P = hi + lo in fp16, each q row scaled by a power of two into (-2, 2)
// first (row_scale()), four products for about 22 bits.  16-bit activations: one plane of each, half the
// products.  fp16 q is taken as it is, bf16 q where fp16 holds it to 2^-19 of its neighbours' largest (where it
// is fetched, below), else scaled as fp32 is.  P's half step 2^-11 is far below the output's own rounding at bf16
// and equal to it at fp16, where it adds to it: fp16 outputs are off by 1.15 (20 keys) to 1.45 (30,000 keys) times
// what fp32 arithmetic rounded once is.  P carries a factor 2^7 (it cancels in O / l): kPUp.
// The tensor core truncates where it adds to an accumulator, always towards zero, so PREC issues Q_lo K before
// Q_hi K, sums at most 256 keys of P V in one accumulator and adds those sums in fp32 (the fold below).  Over 8700 keys the result was off
// by 1.1e-5 without that, 2.6e-6 with sums of 1024 keys, 0.9e-6 with 256 (elementary fp32 operations: 1.3e-6),
// for 1 % of the time at head_dim 128 and 15 % at 256, where the fold goes through global memory.  16-bit
// activations sum 8192 keys, through global memory too: the drift stays under 2^-14 of the result, far below its
// rounding.  With one accumulator it was 2.3e-4 over 131,072 keys and 4e-3 over 2^20.
//
// A persistent CTA, or a pair of them, per SM walks its share of the schedule (paged.cuh).  Alone, a CTA's warps:
//   0-7  softmax: row r of the tile (TMEM lane r) belongs to warps r/32 and r/32 + 4, which halve each
//        block's columns.  They fetch Q, turn S into P in place, rescale O when m grows by more than 2^8,
//        and write the unit's rows or partials.  Rows are fetched and written through a warp's 2 KB of
//        shared memory, whole 64-byte runs at a time: with a row per lane every access touched 32 lines,
//        and a gated unit at head_dim 256 spent 12 us on its way out.
//   8, 10  K and V blocks by tensor copies into their rings, one copy per page and lane (4-D maps).
//   9    MMA issue.  S runs up to NSB blocks ahead of the softmax.
//   11   the schedule: units into a ring of four descriptors, so finding the next unit is off the others' path.
// In a pair (16-bit activations, head_dim 64 and 128) a CTA has half of the SM's shared and tensor memory: blocks
// of 64 keys, two S buffers at head_dim 128, four softmax warps with a whole row per thread, K, MMA, V and schedule
// warps 4 to 7.  One CTA's Q, first S and rows out, and its waits for S, fall into the other's products and
// exponentials: 785 cycles of the SM per 64 keys of a tile against 1,000.
// V rows behind the last key the tile sees hold whatever the page held: the PV product stops at the 16-key
// step that holds that key, and the rows after it in that step are zeroed in shared memory first.
#include "paged.cuh"
#include "tcgen05.cuh"

#include <algorithm>
#include <type_traits>

namespace yattn {
namespace {

constexpr int BM = static_cast<int>(kPagedTileRows);
constexpr int NU = 4;                    // unit descriptors in flight
// P's factor: m may be stale by 8 binades, and fp16 ends below 2^16
constexpr float kPUp = 7.f;

// PAIR: two CTAs per SM, 16-bit activations up to head_dim 128
template <int HD, bool PREC, bool PAIR> struct TCfg {
    static_assert(!PAIR || (!PREC && HD <= 128), "two CTAs' tensor and shared memory");
    static constexpr int SPLIT = PAIR ? 1 : 2;              // threads per row
    static constexpr int NSW = 4 * SPLIT, THREADS = 32 * (NSW + 4);
    // registers per thread after the split
    static constexpr int REGS_SOFTMAX = PAIR ? 168 : 200, REGS_REST = PAIR ? 88 : 104;
    static constexpr int BN = HD >= 256 || PAIR ? 64 : 128;
    static constexpr bool LO_SMEM = PREC && HD <= 128;      // Q_lo in shared memory; head_dim 256: in TMEM
    static constexpr int KST = HD >= 256 || (HD == 128 && (PREC || PAIR)) ? 2 : 3;    // K ring depth
    static constexpr int VST = HD >= 128 ? 2 : 3;           // V ring depth: V(j) is needed two blocks after K(j)
    static constexpr int Q_BYTES = BM * HD * 2;
    static constexpr int KV_BYTES = BN * HD * 2;
    static constexpr int OFF_Q = 0;
    static constexpr int OFF_QLO = OFF_Q + Q_BYTES;
    static constexpr int OFF_K = OFF_QLO + (LO_SMEM ? Q_BYTES : 0);
    static constexpr int OFF_V = OFF_K + KST * KV_BYTES;
    static constexpr int OFF_STG = OFF_V + VST * KV_BYTES;  // per softmax warp: 32 rows x 64 B
    static constexpr int OFF_X = OFF_STG + NSW * 2048;        // [2 blocks][2 halves][BM] floats: row maxima / sums
    static constexpr int OFF_UP = OFF_X + (SPLIT - 1) * 2 * 2 * BM * 4;   // [BM] floats: the rows' powers of two
    static constexpr int OFF_U = OFF_UP + BM * 4;           // [NU] units, 64 B apart
    static constexpr int OFF_BAR = OFF_U + NU * 64;
    static constexpr int SMEM = OFF_BAR + 320 + 1024;       // + barriers, + alignment slack
    static constexpr uint32_t TMEM_COLS = PAIR ? 256 : 512;
    static constexpr int NSB = PREC || (PAIR && HD == 128) ? 2 : 3;                // S buffers: b at columns [b*BN, (b+1)*BN)
    static constexpr uint32_t COL_S = 0;
    static constexpr uint32_t COL_QLO = NSB * BN;           // head_dim 256, PREC: HD/2 columns
    static constexpr uint32_t COL_O = PREC ? 256 : NSB * BN;
    // The fp32 sum of the folded O: beside O, or where TMEM is full (16 bits, head_dim 256) in global memory
    static constexpr bool FOLD_TMEM = PREC && HD <= 128;
    static constexpr uint32_t COL_F = COL_O + HD;
    static constexpr uint32_t FOLD = (PREC ? 256 : 8192) / BN;             // blocks per fold
    static_assert(COL_O + HD * (FOLD_TMEM ? 2 : 1) <= TMEM_COLS && NSB * BN <= static_cast<int>(COL_O), "TMEM columns");
    static_assert(!PREC || LO_SMEM || COL_QLO + HD / 2 <= COL_O, "Q_lo columns");
    static_assert(SMEM <= (PAIR ? 115712 : 232448) && sizeof(PagedUnit) <= 64, "shared memory");
};

template <int KST, int VST> struct TBars {
    uint64_t k_full[KST], k_empty[KST], v_full[VST], v_empty[VST];
    uint64_t s_full[3], p_full[3], pv_done[3];   // per S buffer
    uint64_t o_done, q_full, mma_drain;
    uint64_t u_full[NU], u_empty[NU];
    uint32_t tmem_base;
    int abort_flag, last_flag;
};

__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }

// A warp's 32 rows of 64 bytes through 2 KB of shared memory, 16-byte chunk c of row r at c ^ (r / 2 & 3): from
// four lanes a row (lane: rows lane / 4 + 8 i) to a row per lane, and back.
__device__ __forceinline__ void stage_in(uint8_t* stg, int lane, const uint4 (&raw)[4], uint32_t (&w)[16]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int rr = i * 8 + (lane >> 2);
        *reinterpret_cast<uint4*>(stg + rr * 64 + (((lane & 3) ^ ((rr >> 1) & 3)) << 4)) = raw[i];
    }
    __syncwarp();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint4 v = *reinterpret_cast<const uint4*>(stg + lane * 64 + ((k ^ ((lane >> 1) & 3)) << 4));
        w[4 * k] = v.x;
        w[4 * k + 1] = v.y;
        w[4 * k + 2] = v.z;
        w[4 * k + 3] = v.w;
    }
    __syncwarp();
}
__device__ __forceinline__ void stage_out(uint8_t* stg, int lane, const uint32_t (&w)[16], uint4 (&raw)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
        *reinterpret_cast<uint4*>(stg + lane * 64 + ((k ^ ((lane >> 1) & 3)) << 4)) =
            make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int rr = i * 8 + (lane >> 2);
        raw[i] = *reinterpret_cast<const uint4*>(stg + rr * 64 + (((lane & 3) ^ ((rr >> 1) & 3)) << 4));
    }
    __syncwarp();
}

template <int HD, int ACT, bool PAIR>
__global__ void __launch_bounds__(TCfg<HD, ACT == YATTN_ACT_F32, PAIR>::THREADS, PAIR ? 2 : 1)
    k_paged_tiles(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const __grid_constant__ PagedParams p) {
    constexpr bool PREC = ACT == YATTN_ACT_F32;
    using C = TCfg<HD, PREC, PAIR>;
    constexpr int NSW = C::NSW, SPLIT = C::SPLIT, HW = HD / SPLIT;   // softmax warps, threads per row, their columns of O
    constexpr int BN = C::BN, HB = BN / SPLIT, KST = C::KST, VST = C::VST, NPAN = HD / 64;
    constexpr uint32_t NSB = C::NSB, FOLD = C::FOLD;
    // Charging 256 keys for the gate's way in: 8 gated chunks of the qwen3.5 shape 213 -> 200 us, of the Llama-3-8B shape
    // 262 -> 246 (fp32 412 -> 386); at head_dim 64, with half the columns, it loses 3 %
    using Sched = PagedSched<BN, BM, PAIR, HD >= 128 ? 256 : 0>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sQ = smem + C::OFF_Q;
    uint8_t* sK = smem + C::OFF_K;
    uint8_t* sV = smem + C::OFF_V;
    float* xch = reinterpret_cast<float*>(smem + C::OFF_X);
    using Bars = TBars<KST, VST>;
    static_assert(sizeof(Bars) <= 320, "barriers");
    Bars* bars = reinterpret_cast<Bars*>(smem + C::OFF_BAR);
    volatile int* abort_flag = &bars->abort_flag;
    auto unit_at = [&](uint32_t i) { return reinterpret_cast<PagedUnit*>(smem + C::OFF_U + (i % NU) * 64); };
    int* const status = p.status;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < KST; ++s) {
            mbar_init(&bars->k_full[s], 1);
            mbar_init(&bars->k_empty[s], 1);
        }
        for (int s = 0; s < VST; ++s) {
            mbar_init(&bars->v_full[s], 1);
            mbar_init(&bars->v_empty[s], 1);
        }
        for (int s = 0; s < 3; ++s) {
            mbar_init(&bars->s_full[s], 1);
            mbar_init(&bars->p_full[s], NSW);
            mbar_init(&bars->pv_done[s], 1);
        }
        mbar_init(&bars->o_done, 1);
        mbar_init(&bars->q_full, NSW);
        mbar_init(&bars->mma_drain, 1);
        for (int s = 0; s < NU; ++s) {
            mbar_init(&bars->u_full[s], 1);
            mbar_init(&bars->u_empty[s], 3 + NSW);    // K, V, MMA and the softmax warps
        }
        bars->abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 0) tmem_alloc(&bars->tmem_base, C::TMEM_COLS);
    Sched sched(p);                              // (its warp looks for the share meanwhile)
    bool more = warp == NSW + 3 && sched.begin();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = warp_uniform(bars->tmem_base);

    // Unit ui of the list, for one warp: waits for its descriptor.  false: the list has ended (or a wait gave up).
    auto get_unit = [&](uint32_t ui, PagedUnit& u) -> bool {
        if (!warp_wait_bounded(&bars->u_full[ui % NU], (ui / NU) & 1u, status, ST_PAGED_TIMEOUT, abort_flag)) return false;
        u = *unit_at(ui);
        return !u.done;
    };
    auto put_unit = [&](uint32_t ui) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->u_empty[ui % NU]);
    };
    // registers move to the softmax warps (the launcher checks the sum against the launch's)
    if (warp >= NSW) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REGS_REST));
        if (warp == NSW + 3) {
            // ================= schedule =================
            uint32_t ui = 0;
            bool ok = true;
            for (;;) {
                PagedUnit u;
                more = more && sched.next(u);
                if (ui >= NU)
                    ok = warp_wait_bounded(&bars->u_empty[ui % NU], ((ui / NU) & 1u) ^ 1u, status, ST_PAGED_TIMEOUT, abort_flag);
                if (ok && lane == 0) {
                    u.done = more ? 0u : 1u;
                    *unit_at(ui) = u;
                    mbar_arrive(&bars->u_full[ui % NU]);
                }
                if (!ok || !more) break;
                // its rows of q and of the gate on their way to L2, a few units ahead of their use
                const uint32_t row0 = u.j * BM, rows = min(static_cast<uint32_t>(BM), static_cast<uint32_t>(u.n) * p.group - row0);
#pragma unroll 1
                for (uint32_t i = lane; i < rows; i += 32) {
                    const uint32_t tk = div_group(p, row0 + i);
                    const size_t tok = static_cast<size_t>(u.tok0) + tk, col = (u.g * p.group + row0 + i - tk * p.group) * HD;
                    constexpr int ES = PREC ? 4 : 2;
                    const char* q = static_cast<const char*>(p.q) + (tok * p.q_stride + col) * ES;
                    const char* gt = static_cast<const char*>(p.gate) + (tok * p.gate_stride + col) * ES;
#pragma unroll 1
                    for (int c = 0; c < HD * ES; c += 128) {
                        prefetch_l2(q + c);
                        if (p.gate) prefetch_l2(gt + c);
                    }
                }
                ++ui;
            }
        } else if (warp == NSW || warp == NSW + 2) {
            // ================= K / V copies =================
            const bool is_v = warp == NSW + 2;
            const CUtensorMap* map = is_v ? &tmV : &tmK;
            uint8_t* ring = is_v ? sV : sK;
            uint64_t* full = is_v ? bars->v_full : bars->k_full;
            uint64_t* empty = is_v ? bars->v_empty : bars->k_empty;
            const uint32_t depth = is_v ? VST : KST;
            if (lane == 0) prefetch_tensormap(map);
            const uint32_t page = 1u << p.page_shift, box = min(page, static_cast<uint32_t>(BN));
            const uint32_t i_pg = lane;                               // this lane's page of a block (8 at most)
            const bool mine = i_pg < BN / box;
            uint32_t s = 0, ph = 0, issued = 0;                       // ring stage, its pass's parity, blocks in all
            bool ok = true;
            PagedUnit u;
            for (uint32_t ui = 0; ok && get_unit(ui, u); ++ui) {
                const uint32_t kend = static_cast<uint32_t>(u.keys);
                auto row_of = [&](uint32_t b) -> int32_t {
                    const uint32_t key = b * BN + i_pg * box;
                    if (!mine || key >= kend) return -1;
                    return paged_row(p, u.r, key >> p.page_shift) + static_cast<int32_t>(key & (page - 1));
                };
                int32_t row = u.kb1 > u.kb0 ? row_of(u.kb0) : -1;
                for (uint32_t b = u.kb0; b < u.kb1; ++b) {
                    if (issued >= depth &&
                        !warp_wait_bounded(&empty[s], ph ^ 1u, status, ST_PAGED_TIMEOUT, abort_flag)) {
                        ok = false;
                        break;
                    }
                    const uint32_t n_copy = __popc(__ballot_sync(0xffffffffu, row >= 0));
                    if (lane == 0) mbar_arrive_expect_tx(&full[s], n_copy * box * (HD * 2));
                    __syncwarp();
                    if (row >= 0)
                        tma_load_4d(ring + s * C::KV_BYTES + i_pg * box * (HD * 2), map, 0, 0, static_cast<int32_t>(u.g * NPAN),
                                    row >> 3, &full[s]);
                    ++issued;
                    if (++s == depth) {
                        s = 0;
                        ph ^= 1u;
                    }
                    row = b + 1 < u.kb1 ? row_of(b + 1) : -1;
                }
                put_unit(ui);
            }
            // no copy may still be landing when the CTA exits
            volatile int dummy = 0;
            for (uint32_t b = issued > depth ? issued - depth : 0; b < issued; ++b)
                mbar_wait_bounded(&full[b % depth], (b / depth) & 1u, status, ST_PAGED_TIMEOUT, &dummy);
        } else {
            // ================= MMA =================
            constexpr uint32_t IDESC_QK = idesc_f16(BM, BN, 0);
            constexpr uint32_t IDESC_PV = idesc_f16(BM, HD, 1);
            // an operand at base + off has the base's descriptor + off / 16
            const uint64_t dq0 = sdesc_sw128(sQ, 16, 1024);
            // K and V tiles: 1024-byte atoms of 8 rows x 64 dims, panels 1024 B and row groups NPAN * 1024 B apart
            const uint64_t dk0 = sdesc_sw128(sK, 16, NPAN * 1024);
            const uint64_t dv0 = sdesc_sw128(sV, 1024, NPAN * 1024);
            uint32_t ks = 0, kph = 0, vs = 0, vph = 0;      // ring stages and parities
            uint32_t s_sb = 0, pv_sb = 0, pv_ph = 0;        // S buffer of the next S product, of the next PV product
            uint32_t qph = 0;
            bool ok = true;
            PagedUnit u;
            for (uint32_t ui = 0; ok && get_unit(ui, u); ++ui) {
                const uint32_t nb = u.kb1 - u.kb0;
                if (nb == 0) {
                    put_unit(ui);
                    continue;
                }
                const int32_t kend = u.keys;
                ok = warp_wait_bounded(&bars->q_full, qph, status, ST_PAGED_TIMEOUT, abort_flag);
                qph ^= 1u;
                tc_fence_after();
                // S = Q K^T of the next block into the next S buffer; that buffer's last P was consumed by a PV product
                // issued earlier, and the tensor core runs one thread's MMAs in order
                auto do_s = [&]() -> bool {
                    if (!warp_wait_bounded(&bars->k_full[ks], kph, status, ST_PAGED_TIMEOUT, abort_flag)) return false;
                    tc_fence_after();
                    const uint64_t dk = dk0 + warp_uniform((ks * C::KV_BYTES) >> 4);
                    const uint32_t d = tmem + C::COL_S + warp_uniform(s_sb * BN);
                    if (elect_one()) {
                        if constexpr (PREC) {   // Q_lo K^T first: the accumulator's truncations are relative to what it holds
#pragma unroll
                            for (int kk = 0; kk < HD / 16; ++kk) {
                                const uint64_t b = dk + (((kk >> 2) * 1024 + (kk & 3) * 32) >> 4);
                                if constexpr (C::LO_SMEM)
                                    umma_f16(d, dq0 + ((C::OFF_QLO - C::OFF_Q + (kk >> 2) * (BM * 128) + (kk & 3) * 32) >> 4), b,
                                             IDESC_QK, kk > 0 ? 1u : 0u);
                                else
                                    umma_f16_ts(d, tmem + C::COL_QLO + 8 * kk, b, IDESC_QK, kk > 0 ? 1u : 0u);
                            }
                        }
#pragma unroll
                        for (int kk = 0; kk < HD / 16; ++kk) {
                            const uint64_t a = dq0 + (((kk >> 2) * (BM * 128) + (kk & 3) * 32) >> 4);
                            const uint64_t b = dk + (((kk >> 2) * 1024 + (kk & 3) * 32) >> 4);
                            umma_f16(d, a, b, IDESC_QK, PREC || kk > 0 ? 1u : 0u);
                        }
                        umma_commit(&bars->s_full[s_sb]);
                        umma_commit(&bars->k_empty[ks]);
                    }
                    __syncwarp();
                    if (++s_sb == NSB) s_sb = 0;
                    if (++ks == KST) {
                        ks = 0;
                        kph ^= 1u;
                    }
                    return true;
                };
                // O += P V: keys [16 kk, +16) of a plane are the 8 columns at 32 (kk/2) + 16 plane + 8 (kk%2)
                auto do_pv = [&](uint32_t jj) -> bool {
                    if (!warp_wait_bounded(&bars->p_full[pv_sb], pv_ph, status, ST_PAGED_TIMEOUT, abort_flag) ||
                        !warp_wait_bounded(&bars->v_full[vs], vph, status, ST_PAGED_TIMEOUT, abort_flag))
                        return false;
                    tc_fence_after();
                    const int valid = min(BN, kend - static_cast<int32_t>((u.kb0 + jj) * BN));   // >= 1
                    const int steps = (valid + 15) >> 4;
                    if (valid & 15) {   // the rest of the last 16-key step
                        const int zrows = steps * 16 - valid;
                        for (int i = lane; i < zrows * NPAN * 8; i += 32) {
                            const int row = valid + i / (NPAN * 8), c = i % (NPAN * 8);
                            *reinterpret_cast<uint4*>(sV + vs * C::KV_BYTES + ((row >> 3) * NPAN + (c >> 3)) * 1024 + (row & 7) * 128 + (c & 7) * 16) =
                                make_uint4(0u, 0u, 0u, 0u);
                        }
                        fence_proxy_async_smem();
                        __syncwarp();
                    }
                    const uint32_t pcol = tmem + C::COL_S + warp_uniform(pv_sb * BN);
                    const uint64_t dv = dv0 + warp_uniform((vs * C::KV_BYTES) >> 4);
                    if (elect_one()) {
                        const bool fresh = jj % FOLD == 0;                    // the sum so far has been folded
#pragma unroll
                        for (int plane = 0; plane < (PREC ? 2 : 1); ++plane)
#pragma unroll
                            for (int kk = 0; kk < BN / 16; ++kk)
                                if (kk < steps)
                                    umma_f16_ts(tmem + C::COL_O, pcol + 32 * (kk >> 1) + 16 * plane + 8 * (kk & 1),
                                                dv + ((kk * 2 * NPAN * 1024) >> 4), IDESC_PV,
                                                (!fresh || plane > 0 || kk > 0) ? 1u : 0u);
                        umma_commit(&bars->v_empty[vs]);
                        umma_commit(&bars->pv_done[pv_sb]);
                    }
                    __syncwarp();
                    if (++pv_sb == NSB) {
                        pv_sb = 0;
                        pv_ph ^= 1u;
                    }
                    if (++vs == VST) {
                        vs = 0;
                        vph ^= 1u;
                    }
                    return true;
                };
                for (uint32_t jj = 0; ok && jj < nb && jj < NSB; ++jj) ok = do_s();
                for (uint32_t jj = 0; ok && jj < nb; ++jj) {
                    ok = do_pv(jj);
                    if (ok && jj + NSB < nb) ok = do_s();
                }
                if (ok && elect_one()) umma_commit(&bars->o_done);
                put_unit(ui);
            }
            // every MMA issued so far completes before TMEM is freed
            if (elect_one()) {
                umma_commit(&bars->mma_drain);
                volatile int dummy = 0;
                mbar_wait_bounded(&bars->mma_drain, 0, status, ST_PAGED_TIMEOUT, &dummy);
            }
            __syncwarp();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REGS_SOFTMAX));
        // ================= softmax warps =================
        const int qd = warp & 3, h = warp >> 2;          // TMEM lane quadrant, half of each block's columns (SPLIT 1: 0)
        const int r = qd * 32 + lane;                    // row of the tile
        const uint32_t trow = tmem + (static_cast<uint32_t>(qd * 32) << 16);
        uint32_t sb = 0, sph = 0, pb = 0, pph = 0;       // S buffer of this block / of the last one, and parities
        uint32_t oph = 0;
        uint8_t* stg = smem + C::OFF_STG + warp * 2048;
        float* s_up = reinterpret_cast<float*>(smem + C::OFF_UP);
        // Waits' results are ANDed over the warps that meet at the next barrier, so all of them leave together.
        for (uint32_t ui = 0;; ++ui) {
            PagedUnit u;
            const bool got = get_unit(ui, u);
            if (!named_bar_and(5, 32 * NSW, got)) break;      // the end, or a wait that gave up
            const uint32_t nb = u.kb1 - u.kb0;
            const uint32_t row0 = u.j * BM, rows = min(static_cast<uint32_t>(BM), static_cast<uint32_t>(u.n) * p.group - row0);
            const bool work = static_cast<uint32_t>(qd * 32) < rows;      // this warp has a live row
            // this thread's row (padding rows: the last one again) and the column of its head
            const uint32_t f = row0 + min(static_cast<uint32_t>(r), rows - 1);
            const uint32_t tk = div_group(p, f);
            const uint32_t hcol = (u.g * p.group + f - tk * p.group) * HD;
            const int32_t qpos = u.len - u.n + static_cast<int32_t>(tk);   // last key this row sees
            const int32_t qpos_min = u.len - u.n + static_cast<int32_t>(div_group(p, row0));
            // the threads of these rows meet: the warp, or the two that halve the columns
            auto rows_and = [&](bool x) -> bool { return SPLIT == 1 ? x : named_bar_and(1 + qd, 64, x); };
            // Columns [c, c + 32) of this half's rows, a row per lane, gated and rounded, out through the warp's
            // staging; g: their gate values from ld_gate(), in the staging's order.  All lanes.
            constexpr int ES = PREC ? 4 : 2, CW = 64 / ES, SUBS = 32 / CW;   // columns of a 64-byte run, runs
            // lane: 16 bytes of rows lane / 4 + 8 i of the warp
            auto run_at = [&](int c, int i, size_t& token, size_t& col) -> bool {
                const int rr = i * 8 + (lane >> 2);
                token = static_cast<size_t>(u.tok0) + __shfl_sync(0xffffffffu, tk, rr);
                col = __shfl_sync(0xffffffffu, hcol, rr) + static_cast<size_t>(h * HW + c + (lane & 3) * (16 / ES));
                return static_cast<uint32_t>(qd * 32 + rr) < rows;
            };
            auto ld_gate = [&](int c, uint4 (&g)[SUBS * 4]) {
                if (!p.gate) return;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    size_t token, col;
                    const bool in = run_at(c, i, token, col);
#pragma unroll
                    for (int sub = 0; sub < SUBS; ++sub) {
                        g[sub * 4 + i] = make_uint4(0u, 0u, 0u, 0u);
                        if (in)
                            g[sub * 4 + i] = __ldg(reinterpret_cast<const uint4*>(
                                static_cast<const char*>(p.gate) + (token * p.gate_stride + col + sub * CW) * ES));
                    }
                }
            };
            auto write_out = [&](int c, const float (&x)[32], const uint4 (&g)[SUBS * 4]) {
#pragma unroll
                for (int sub = 0; sub < SUBS; ++sub) {
                    float y[CW];
#pragma unroll
                    for (int i = 0; i < CW; ++i) y[i] = x[sub * CW + i];
                    uint32_t w[16];
                    if (p.gate) {
                        const uint4 raw[4] = {g[sub * 4], g[sub * 4 + 1], g[sub * 4 + 2], g[sub * 4 + 3]};
                        stage_in(stg, lane, raw, w);
                        if constexpr (PREC) {
#pragma unroll
                            for (int i = 0; i < CW; ++i) y[i] *= sigmoid_of(__uint_as_float(w[i]));
                        } else {
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const float2 t = ACT == YATTN_ACT_F16
                                                     ? h2f2(w[i])
                                                     : make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
                                y[2 * i] *= sigmoid_of(t.x);
                                y[2 * i + 1] *= sigmoid_of(t.y);
                            }
                        }
                    }
                    if constexpr (PREC) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(y[i]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            if (ACT == YATTN_ACT_F16) {
                                w[i] = h2_bits(__floats2half2_rn(y[2 * i], y[2 * i + 1]));
                            } else {
                                const __nv_bfloat162 b = __floats2bfloat162_rn(y[2 * i], y[2 * i + 1]);
                                w[i] = *reinterpret_cast<const uint32_t*>(&b);
                            }
                        }
                    }
                    uint4 raw[4];
                    stage_out(stg, lane, w, raw);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        size_t token, col;
                        if (run_at(c + sub * CW, i, token, col))
                            *reinterpret_cast<uint4*>(static_cast<char*>(p.out) + (token * p.out_stride + col) * ES) = raw[i];
                    }
                }
            };
            const bool folded = nb > FOLD;
            float m_run = -INFINITY, l_run = 0.f, l_row = 0.f;   // log2 units; l_run: this half's columns
            uint4 g[SUBS * 4];                           // the gate of the next 32 columns, a step ahead
            bool ok = true;
            // ---- O and the folded sum, 32 columns of this half at a time ----
            const uint32_t ocol = trow + C::COL_O + h * HW, fcol = trow + C::COL_F + h * HW;
            const int quad0 = h * (HW / 4);              // this half's first column quad
            auto quads = [&](uint32_t slot) {            // partials by column quads: a warp's accesses are whole lines
                return reinterpret_cast<float4*>(p.part_o) + (static_cast<size_t>(slot) * (HD / 4) + quad0) * BM + r;
            };
            // (the slot of the piece that ends this CTA's share: the last one to be written, from these very sums)
            float4* const fsum = quads(2 * blockIdx.x + 1);
            auto ld_fold = [&](int c, float (&x)[32]) {
                if constexpr (C::FOLD_TMEM) {
                    uint32_t rr[32];
                    tmem_ld32(fcol + c, rr);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; ++i) x[i] = __uint_as_float(rr[i]);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float4 v = fsum[(c / 4 + i) * BM];
                        x[4 * i] = v.x;
                        x[4 * i + 1] = v.y;
                        x[4 * i + 2] = v.z;
                        x[4 * i + 3] = v.w;
                    }
                }
            };
            auto st_fold = [&](int c, const float (&x)[32]) {
                if constexpr (C::FOLD_TMEM) {
                    uint32_t rr[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) rr[i] = __float_as_uint(x[i]);
                    tmem_st32(fcol + c, rr);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        fsum[(c / 4 + i) * BM] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
                }
            };
            auto ld_o = [&](int c, float (&x)[32], bool folded) {           // the whole sum so far
                uint32_t rr[32];
                tmem_ld32(ocol + c, rr);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i) x[i] = __uint_as_float(rr[i]);
                if (folded) {
                    float y[32];
                    ld_fold(c, y);
#pragma unroll
                    for (int i = 0; i < 32; ++i) x[i] += y[i];
                }
            };
            if (nb > 0) {
                float up = 1.f;
                // ---- Q, each row scaled by its power of two: hi to shared memory, lo (PREC) beside it or to TMEM ----
                if constexpr (!PREC || C::LO_SMEM) {
                    // a warp fetches RPW rows, LPR lanes a row, 16 bytes a lane
                    constexpr int ES = PREC ? 4 : 2, EL = 16 / ES, LPR = HD / EL, RPI = 32 / LPR, RPW = BM / NSW, NI = RPW / RPI;
                    uint4 raw[NI];
#pragma unroll
                    for (int i = 0; i < NI; ++i) {
                        const uint32_t row = warp * RPW + i * RPI + lane / LPR;
                        const uint32_t fr = row0 + min(row, rows - 1), tr = div_group(p, fr);
                        const size_t at = (static_cast<size_t>(u.tok0) + tr) * p.q_stride +
                                          (u.g * p.group + fr - tr * p.group) * HD + (lane % LPR) * EL;
                        raw[i] = __ldg(reinterpret_cast<const uint4*>(static_cast<const char*>(p.q) + at * ES));
                    }
                    // fp16 goes as it is; bf16 too where fp16 holds this warp's rows: every 8 neighbours below 2^15 and, unless
                    // all zero, with one of 2^-6 or more, so what falls under fp16's normal range is off by 2^-25, which is
                    // 2^-19 of its row's largest (bf16 itself rounds at 2^-9).  Else scaled as fp32 is
                    bool plain = ACT == YATTN_ACT_F16;
                    if constexpr (ACT == YATTN_ACT_BF16) {
                        bool fits = true;
#pragma unroll
                        for (int i = 0; i < NI; ++i) {
                            uint32_t hi = 0, lo = 0;
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const uint32_t w = k == 0 ? raw[i].x : k == 1 ? raw[i].y : k == 2 ? raw[i].z : raw[i].w;
                                hi = max(hi, w & 0x7fff7fffu);
                                lo = max(lo, w & 0x7fffu);
                            }
                            const uint32_t top = max(hi >> 16, lo);   // the largest of 8 values, as bf16 bits
                            fits = fits && (top == 0 || (top >= 0x3c80u && top < 0x4700u));
                        }
                        plain = __all_sync(0xffffffffu, fits);
                        if (plain) {
#pragma unroll
                            for (int i = 0; i < NI; ++i) {
                                uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
                                for (int k = 0; k < 4; ++k)
                                    w[k] = h2_bits(__floats2half2_rn(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xffff0000u)));
                                raw[i] = make_uint4(w[0], w[1], w[2], w[3]);
                            }
                        }
                    }
                    if (plain) {
#pragma unroll
                        for (int i = 0; i < NI; ++i) {
                            const uint32_t row = warp * RPW + i * RPI + lane / LPR;
                            if (lane % LPR == 0) s_up[row] = 1.f;
                            *reinterpret_cast<uint4*>(sQ + sw128_offset(row, (lane % LPR) * EL, BM)) = raw[i];
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < NI; ++i) {
                            const uint32_t row = warp * RPW + i * RPI + lane / LPR;
                            const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
                            float x[EL], mx = 0.f;
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                if constexpr (PREC) {
                                    x[k] = __uint_as_float(w[k]);
                                } else {
                                    const float2 t = ACT == YATTN_ACT_F16
                                                         ? h2f2(w[k])
                                                         : make_float2(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xffff0000u));
                                    x[2 * k] = t.x;
                                    x[2 * k + 1] = t.y;
                                }
                            }
#pragma unroll
                            for (int k = 0; k < EL; ++k) mx = fmaxf(mx, fabsf(x[k]));
                            if constexpr (LPR == 32) {               // (magnitudes order as their bits)
                                mx = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(mx)));
                            } else {
#pragma unroll
                                for (int o = LPR / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                            }
                            float down, rup;
                            row_scale(mx, down, rup);
                            if (lane % LPR == 0) s_up[row] = rup;
                            uint32_t hi[EL / 2], lo[EL / 2];
#pragma unroll
                            for (int k = 0; k < EL / 2; ++k) {
                                const float a = x[2 * k] * down, b = x[2 * k + 1] * down;
                                const __half2 hv = __floats2half2_rn(a, b);
                                hi[k] = h2_bits(hv);
                                const float2 fv = __half22float2(hv);
                                lo[k] = h2_bits(__floats2half2_rn(a - fv.x, b - fv.y));
                            }
                            uint8_t* dst = sQ + sw128_offset(row, (lane % LPR) * EL, BM);
                            if constexpr (PREC) {
                                *reinterpret_cast<uint2*>(dst) = make_uint2(hi[0], hi[1]);
                                *reinterpret_cast<uint2*>(dst + (C::OFF_QLO - C::OFF_Q)) = make_uint2(lo[0], lo[1]);
                            } else {
                                *reinterpret_cast<uint4*>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                            }
                        }
                    }
                    fence_proxy_async_smem();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bars->q_full);
                    named_bar_sync(5, 32 * NSW);                                   // s_up of every row
                    up = s_up[r];
                } else {
                    // head_dim 256, fp32: a row's half per lane, in two passes (its largest value, then the planes)
                    constexpr int CH = 64;                                    // columns in registers at a time
                    float x[CH];
                    const size_t qi = (static_cast<size_t>(u.tok0) + tk) * p.q_stride + hcol + h * (HD / 2);
                    auto load = [&](int c) {
                        const float4* src = reinterpret_cast<const float4*>(static_cast<const float*>(p.q) + qi + c);
#pragma unroll
                        for (int i = 0; i < CH / 4; ++i) {
                            const float4 v = __ldg(src + i);
                            x[4 * i] = v.x;
                            x[4 * i + 1] = v.y;
                            x[4 * i + 2] = v.z;
                            x[4 * i + 3] = v.w;
                        }
                    };
                    float mx = 0.f;
#pragma unroll 1
                    for (int c = HD / 2 - CH; c >= 0; c -= CH) {              // ends with columns [0, CH) in x
                        load(c);
#pragma unroll
                        for (int i = 0; i < CH; ++i) mx = fmaxf(mx, fabsf(x[i]));
                    }
                    xch[h * BM + r] = mx;
                    named_bar_sync(1 + qd, 64);                               // the row's two halves
                    mx = fmaxf(xch[r], xch[BM + r]);
                    named_bar_sync(1 + qd, 64);                               // read before the first block's maxima
                    float down;
                    row_scale(mx, down, up);
#pragma unroll 1
                    for (int c = 0; c < HD / 2; c += CH) {
                        if (c > 0) load(c);
                        const int d0 = h * (HD / 2) + c;
#pragma unroll
                        for (int i = 0; i < CH; i += 32) {
                            uint32_t hi[16], lo[16];
#pragma unroll
                            for (int k = 0; k < 16; ++k) {
                                const float a = x[i + 2 * k] * down, b = x[i + 2 * k + 1] * down;
                                const __half2 hv = __floats2half2_rn(a, b);
                                hi[k] = h2_bits(hv);
                                const float2 fv = __half22float2(hv);
                                lo[k] = h2_bits(__floats2half2_rn(a - fv.x, b - fv.y));
                            }
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                *reinterpret_cast<uint4*>(sQ + sw128_offset(r, d0 + i + 8 * k, BM)) =
                                    make_uint4(hi[4 * k], hi[4 * k + 1], hi[4 * k + 2], hi[4 * k + 3]);
                            tmem_st16(trow + C::COL_QLO + (d0 + i) / 2, lo);
                        }
                    }
                    tmem_wait_st();
                    fence_proxy_async_smem();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bars->q_full);
                }
                const float sl2 = p.scale_log2 * up;
                for (uint32_t j = 0; j < nb; ++j) {
                    const bool have = warp_wait_bounded(&bars->s_full[sb], sph, status, ST_PAGED_TIMEOUT, abort_flag);
                    if (!work) {                             // no live row: P's lanes stay as they are, nothing reads them
                        if (!rows_and(have)) {
                            ok = false;
                            break;
                        }
                    } else {
                        const uint32_t scol = trow + C::COL_S + sb * BN + h * HB;
                        float sv[HB];
                        if (have) {
                            tc_fence_after();
#pragma unroll
                            for (int c = 0; c < HB / 32; ++c) {
                                uint32_t rr[32];
                                tmem_ld32(scol + c * 32, rr);
#pragma unroll
                                for (int i = 0; i < 32; ++i) sv[c * 32 + i] = __uint_as_float(rr[i]);
                            }
                            tmem_wait_ld();
                        } else {
#pragma unroll
                            for (int c = 0; c < HB; ++c) sv[c] = -INFINITY;
                        }
                        // causal mask; also drops the stale rows behind the last key (their S may be NaN)
                        const int32_t kbase = static_cast<int32_t>((u.kb0 + j) * BN) + h * HB;
                        if (static_cast<int32_t>((u.kb0 + j + 1) * BN) - 1 > qpos_min) {
#pragma unroll
                            for (int c = 0; c < HB; ++c)
                                if (kbase + c > qpos) sv[c] = -INFINITY;
                        }
                        float mx4[4] = {sv[0], sv[1], sv[2], sv[3]};
#pragma unroll
                        for (int c = 4; c < HB; c += 4) {
                            mx4[0] = fmaxf(mx4[0], sv[c]);
                            mx4[1] = fmaxf(mx4[1], sv[c + 1]);
                            mx4[2] = fmaxf(mx4[2], sv[c + 2]);
                            mx4[3] = fmaxf(mx4[3], sv[c + 3]);
                        }
                        float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
                        float* xb = xch + (j & 1) * (2 * BM);
                        if constexpr (SPLIT == 2) xb[h * BM + r] = mx;
                        if (!rows_and(have)) {
                            ok = false;
                            break;
                        }
                        if constexpr (SPLIT == 2) mx = fmaxf(xb[r], xb[BM + r]);
                        mx *= sl2;
                        const float m_new = fmaxf(m_run, mx);
                        const bool grow = m_new > m_run + 8.0f;          // a stale m costs nothing up to 2^8
                        const float m_use = grow ? m_new : m_run;
                        const float alpha = grow ? ex2_approx(m_run - m_use) : 1.0f;
                        const float m_sub = (m_use == -INFINITY ? 0.f : m_use) - kPUp;   // no key yet: p = 0
                        const float2 sl2x2 = make_float2(sl2, sl2), negm = make_float2(-m_sub, -m_sub);
                        const float2 neg1 = make_float2(-1.f, -1.f);
                        float2 rs2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                        for (int c = 0; c < HB / 32; ++c) {   // 32 keys: 16 columns of P hi, then 16 of P lo
                            uint32_t hi[16], lo[16];
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const float2 x = __ffma2_rn(make_float2(sv[c * 32 + 2 * i], sv[c * 32 + 2 * i + 1]), sl2x2, negm);
                                const float2 pp = make_float2(ex2_approx(x.x), ex2_approx(x.y));
                                rs2[i & 1] = __fadd2_rn(rs2[i & 1], pp);
                                const __half2 hv = __floats2half2_rn(pp.x, pp.y);
                                hi[i] = h2_bits(hv);
                                if constexpr (PREC) {
                                    const float2 d = __ffma2_rn(__half22float2(hv), neg1, pp);
                                    lo[i] = h2_bits(__floats2half2_rn(d.x, d.y));
                                }
                            }
                            tmem_st16(scol + c * 32, hi);
                            if constexpr (PREC) tmem_st16(scol + c * 32 + 16, lo);
                        }
                        l_run = l_run * alpha + ((rs2[0].x + rs2[0].y) + (rs2[1].x + rs2[1].y));
                        m_run = m_use;
                        // ---- O rescale (rare) or fold, this half's columns: the last block's PV must have
                        // finished.  Both halves of the rows see the same `grow`. ----
                        const bool fold = j >= 1 && j % FOLD == 0;
                        if (j >= 1 && (fold || __any_sync(0xffffffffu, grow))) {
                            const bool done = warp_wait_bounded(&bars->pv_done[pb], pph, status, ST_PAGED_TIMEOUT, abort_flag);
                            if (!rows_and(done)) {
                                ok = false;
                                break;
                            }
                            tc_fence_after();
                            const bool folded = j > FOLD;
#pragma unroll 1
                            for (int c = 0; c < HW; c += 32) {
                                float x[32];
                                ld_o(c, x, fold && folded);
#pragma unroll
                                for (int i = 0; i < 32; ++i) x[i] *= alpha;
                                if (fold) {
                                    st_fold(c, x);
                                    continue;
                                }
                                uint32_t rr[32];
#pragma unroll
                                for (int i = 0; i < 32; ++i) rr[i] = __float_as_uint(x[i]);
                                tmem_st32(ocol + c, rr);
                                if (folded) {
                                    ld_fold(c, x);
#pragma unroll
                                    for (int i = 0; i < 32; ++i) x[i] *= alpha;
                                    st_fold(c, x);
                                }
                            }
                        }
                        tmem_wait_st();
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bars->p_full[sb]);
                    pb = sb;
                    pph = sph;
                    if (++sb == NSB) {
                        sb = 0;
                        sph ^= 1u;
                    }
                }
                if (work) ld_gate(0, g);
                // ---- the unit's rows: the slot that block nb-1 did not use is free (both halves have read it) ----
                ok = ok && warp_wait_bounded(&bars->o_done, oph, status, ST_PAGED_TIMEOUT, abort_flag);
                oph ^= 1u;
                float* xl = xch + (nb & 1) * (2 * BM);
                if constexpr (SPLIT == 2) xl[h * BM + r] = l_run;
                if (!named_bar_and(5, 32 * NSW, ok)) break;       // every softmax warp
                tc_fence_after();
                l_row = l_run;
                if constexpr (SPLIT == 2) {
                    l_row = xl[r] + xl[BM + r];
                    named_bar_sync(1 + qd, 64);              // read before the next unit's Q maxima
                }
            } else if (work) {                           // no key to see: zeros
                ld_gate(0, g);
            }
            // ---- the unit's rows, or a piece's (m, l, o) and, of the last piece to arrive, the merged rows ----
            bool write = work;
            float M = -INFINITY;
            // a row that sees no key is zeros; one whose keys all score -inf has l = 0 and comes out as 0 / 0
            float inv = qpos < 0 ? 0.f : 1.0f / l_row;
            auto ml_of = [&](uint32_t i) {
                return __ldcg(reinterpret_cast<const float2*>(
                    &p.part_ml[(static_cast<size_t>(piece_slot(u.c_first, i)) * BM + r) * 2]));
            };
            if (u.n_pieces > 1) {
                if (h == 0)
                    *reinterpret_cast<float2*>(&p.part_ml[(static_cast<size_t>(u.slot) * BM + r) * 2]) = make_float2(m_run, l_row);
                if (work) {
                    float4* po = quads(u.slot);
#pragma unroll 1
                    for (int c = 0; c < HW; c += 32) {
                        float x[32];
                        ld_o(c, x, folded);
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            po[(c / 4 + i) * BM] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
                    }
                }
                __threadfence();
                named_bar_sync(5, 32 * NSW);
                if (threadIdx.x == 0)
                    bars->last_flag = atomicInc(&p.counters[u.c_first], u.n_pieces - 1) == u.n_pieces - 1;
                named_bar_sync(5, 32 * NSW);
                write = bars->last_flag && work;
                if (write) {
                    __threadfence();
                    float l = 0.f;
#pragma unroll 4
                    for (uint32_t i = 0; i < u.n_pieces; ++i) M = fmaxf(M, ml_of(i).x);
#pragma unroll 4
                    for (uint32_t i = 0; i < u.n_pieces; ++i) {
                        const float2 ml = ml_of(i);
                        l += (ml.x == -INFINITY ? 0.f : ex2_approx(ml.x - M)) * ml.y;
                    }
                    inv = qpos < 0 ? 0.f : 1.0f / l;
                }
            }
            if (write) {
#pragma unroll 1
                for (int c = 0; c < HW; c += 32) {
                    uint4 g_next[SUBS * 4];
                    if (c + 32 < HW) ld_gate(c + 32, g_next);
                    float x[32];
                    if (u.n_pieces > 1) {                // in piece order
#pragma unroll
                        for (int i = 0; i < 32; ++i) x[i] = 0.f;
#pragma unroll 1
                        for (uint32_t i = 0; i < u.n_pieces; i += 2) {      // two pieces' loads in flight
                            const uint32_t i1 = min(i + 1, u.n_pieces - 1);
                            const float4* s0 = quads(piece_slot(u.c_first, i)) + (c / 4) * BM;
                            const float4* s1 = quads(piece_slot(u.c_first, i1)) + (c / 4) * BM;
                            const float m0 = ml_of(i).x, m1 = ml_of(i1).x;
                            float4 o0[8], o1[8];
#pragma unroll
                            for (int k = 0; k < 8; ++k) {
                                o0[k] = __ldcg(s0 + k * BM);
                                o1[k] = __ldcg(s1 + k * BM);
                            }
                            const float w0 = (m0 == -INFINITY ? 0.f : ex2_approx(m0 - M)) * inv;
                            const float w1 = i1 == i ? 0.f : (m1 == -INFINITY ? 0.f : ex2_approx(m1 - M)) * inv;
#pragma unroll
                            for (int k = 0; k < 8; ++k) {
                                x[4 * k] += w0 * o0[k].x + w1 * o1[k].x;
                                x[4 * k + 1] += w0 * o0[k].y + w1 * o1[k].y;
                                x[4 * k + 2] += w0 * o0[k].z + w1 * o1[k].z;
                                x[4 * k + 3] += w0 * o0[k].w + w1 * o1[k].w;
                            }
                        }
                    } else if (nb > 0) {
                        ld_o(c, x, folded);
#pragma unroll
                        for (int i = 0; i < 32; ++i) x[i] *= inv;
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) x[i] = 0.f;
                    }
                    write_out(c, x, g);
#pragma unroll
                    for (int i = 0; i < SUBS * 4; ++i) g[i] = g_next[i];
                }
            }
            tc_fence_before();
            put_unit(ui);
        }
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    if (warp == 0) tmem_dealloc(tmem, C::TMEM_COLS);
}

template <int HD, int ACT, bool PAIR>
int launch(const PagedParams& p, const CUtensorMap& mk, const CUtensorMap& mv, uint32_t ctas, cudaStream_t st,
           char* err, size_t errlen) {
    using C = TCfg<HD, ACT == YATTN_ACT_F32, PAIR>;
    static bool attr_done[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && !attr_done[dev]) {
        cudaError_t e = cudaFuncSetAttribute(k_paged_tiles<HD, ACT, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e != cudaSuccess) {
            set_err(err, errlen, "attn_paged: smem attribute (%d bytes): %s", C::SMEM, cudaGetErrorString(e));
            return -1;
        }
        // an increase past what the block was launched with would wait for ever
        cudaFuncAttributes at{};
        e = cudaFuncGetAttributes(&at, k_paged_tiles<HD, ACT, PAIR>);
        if (e != cudaSuccess || at.numRegs * C::THREADS < 32 * C::NSW * C::REGS_SOFTMAX + 128 * C::REGS_REST) {
            set_err(err, errlen, "attn_paged: built with %d registers a thread, too few for the register split", at.numRegs);
            return -1;
        }
        attr_done[dev] = true;
    }
    k_paged_tiles<HD, ACT, PAIR><<<ctas * (PAIR ? 2 : 1), C::THREADS, C::SMEM, st>>>(mk, mv, p);
    YATTN_CHECK_LAUNCH(err, errlen, "attn_paged");
    return 0;
}

}  // namespace

int paged_tiles(const PagedParams& pp, const uint16_t* kpool, const uint16_t* vpool, uint64_t n_rows, uint32_t kv_dim,
                uint32_t hd, uint32_t n_kv, cudaStream_t st, char* err, size_t errlen) {
    PagedParams p = pp;
    p.hc = 1;
    p.n_groups = n_kv;
    const uint32_t sms = static_cast<uint32_t>(dev_num_sms());
    // Two CTAs per SM from a tile per SM on: below that most SMs would hold one of them, slower than a CTA that has
    // the SM to itself (bf16, Llama-3-8B: 4096-token prompt 177 us against 197, 300 tokens behind 700: 31 against 27)
    const bool pair = hd <= 128 && p.act != YATTN_ACT_F32 &&
                      static_cast<uint64_t>(p.n_tokens) * p.n_heads >= static_cast<uint64_t>(sms) * kPagedTileRows;
    const uint32_t bn = hd >= 256 || pair ? 64 : 128, box = std::min(1u << p.page_shift, bn);
    CUtensorMap mk, mv;
    if (encode_page_map(&mk, kpool, kv_dim, n_rows, n_kv * hd, box, hd / 64, err, errlen) ||
        encode_page_map(&mv, vpool, kv_dim, n_rows, n_kv * hd, box, hd / 64, err, errlen))
        return -1;
    const uint32_t ctas = std::min<uint32_t>(sms, kPagedMaxPieces);
    auto run = [&](auto tag) -> int {
        constexpr int HD = decltype(tag)::value;
        if constexpr (HD <= 128) {
            if (pair)
                return p.act == YATTN_ACT_F16 ? launch<HD, YATTN_ACT_F16, true>(p, mk, mv, ctas, st, err, errlen)
                                              : launch<HD, YATTN_ACT_BF16, true>(p, mk, mv, ctas, st, err, errlen);
        }
        switch (p.act) {
            case YATTN_ACT_F32: return launch<HD, YATTN_ACT_F32, false>(p, mk, mv, ctas, st, err, errlen);
            case YATTN_ACT_F16: return launch<HD, YATTN_ACT_F16, false>(p, mk, mv, ctas, st, err, errlen);
            default: return launch<HD, YATTN_ACT_BF16, false>(p, mk, mv, ctas, st, err, errlen);
        }
    };
    switch (hd) {
        case 64: return run(std::integral_constant<int, 64>{});
        case 128: return run(std::integral_constant<int, 128>{});
        default: return run(std::integral_constant<int, 256>{});
    }
}

}  // namespace yattn
