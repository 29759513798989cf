// page_step.cu -- block tables, slot maps and the page queue of one serving step, from request lengths.
//
// Request r holds kv_len[r] cached tokens in ceil(kv_len / page) pages and gets new_len[r] more (or, at
// -1, has ended).  With the exclusive prefix sums over the requests
//     cu[r]   of max(new_len, 0),
//     take[r] of ceil((kv_len + new) / page) - ceil(kv_len / page),
//     back[r] of the ended requests' page counts,
// token t = cu[r] + i sits at position kv_len[r] + i, the k-th page handed out (request order, then page
// order) is ring[(head + k) mod n_pages], and the ended requests' pages go behind the queue's tail in the
// same order.  Nothing depends on another block's output: a token in a page handed out by this very call
// takes that page from the queue, not from the table.  So one launch of many blocks needs no grid barrier;
// each block repeats the prefix sums (n_seqs values, three sums in one pass over shared memory) and takes
// a grid-strided share of the tokens, of the new table entries and of the returned pages.
//
// The inputs (lengths, queue state) are not written, so a repeated call gives the same answer, and the
// queue's written entries [head + count, ..) and read entries [head, ..) never overlap.
//
// Page numbers are checked where they are used (602), not before the verdict: that takes every block another dependent
// load before it can decide (1 request 3.5 to 3.9 us, 512 with chunks 5.6 to 6.6, and 16 with the returned ones).
//
// Bound: latency.  The bytes are 16 per request, 8 per token and 4 per page touched (under 1 MB at 512
// requests); a call is the launch, two dependent loads, the sums and one search.
#include "common.cuh"

#include <algorithm>
#include <atomic>

namespace yattn {
namespace {

constexpr int kThreads = 512;
constexpr uint32_t kMaxSeqs = 16384;   // three prefix arrays in shared memory: 192 KB

struct StepParams {
    int32_t* kv_len_out;
    int32_t* cu_new;
    int32_t* slots;
    int32_t* positions;
    int32_t* state_out;
    int32_t* tables;
    int32_t* ring;
    const int32_t* state;
    const int32_t* kv_len;
    const int32_t* new_len;
    uint32_t max_tokens, max_pages, table_stride, n_pages, n_seqs, page_shift;
    int* status;
};

// Last index r of pre[0..n] (non-decreasing) with pre[r] <= x; x < pre[n].
__device__ __forceinline__ uint32_t owner(const int32_t* pre, uint32_t n, int32_t x) {
    uint32_t lo = 0, hi = n;   // pre[lo] <= x < pre[hi]
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (pre[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(kThreads) k_page_step(const StepParams p) {
    extern __shared__ int32_t sm[];
    int32_t* cu = sm;                        // [n + 1] each
    int32_t* take = cu + p.n_seqs + 1;
    int32_t* back = take + p.n_seqs + 1;
    __shared__ long long w_new[kThreads / 32];
    __shared__ int32_t w_take[kThreads / 32], w_back[kThreads / 32];
    const uint32_t n = p.n_seqs, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int32_t pm = (1 << p.page_shift) - 1;
    const int32_t head = p.state[0], count = p.state[1];

    long long c_new = 0;                     // sums of the requests before this chunk of kThreads
    int32_t c_take = 0, c_back = 0;
    bool over = false, bad = false;
    for (uint32_t base = 0; base < n; base += kThreads) {
        const uint32_t r = base + tid;
        long long a = 0;
        int32_t b = 0, c = 0;
        if (r < n) {
            const int32_t len = p.kv_len[r], add = p.new_len[r];
            const uint32_t held = (static_cast<uint32_t>(len) + pm) >> p.page_shift;
            if (len < 0 || add < -1 || held > p.max_pages) {
                bad = true;
            } else if (add < 0) {
                c = static_cast<int32_t>(held);
            } else {
                const unsigned long long to = (static_cast<unsigned long long>(len) + add + pm) >> p.page_shift;
                if (to > p.max_pages) {
                    over = true;
                } else {
                    a = add;
                    b = static_cast<int32_t>(to - held);
                }
            }
        }
        const long long a0 = a;
        const int32_t b0 = b, c0 = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long ua = __shfl_up_sync(0xffffffffu, a, o);
            const int32_t ub = __shfl_up_sync(0xffffffffu, b, o), uc = __shfl_up_sync(0xffffffffu, c, o);
            if (lane >= static_cast<uint32_t>(o)) {
                a += ua;
                b += ub;
                c += uc;
            }
        }
        if (lane == 31) {
            w_new[warp] = a;
            w_take[warp] = b;
            w_back[warp] = c;
        }
        __syncthreads();
        for (uint32_t w = 0; w < kThreads / 32; ++w) {
            if (w == warp && r < n) {   // exclusive sums; a total past 32 bits is refused below
                cu[r] = static_cast<int32_t>(c_new + a - a0);
                take[r] = c_take + b - b0;
                back[r] = c_back + c - c0;
            }
            c_new += w_new[w];
            c_take += w_take[w];
            c_back += w_back[w];
        }
        __syncthreads();                     // the warps' sums are read before the next chunk's replace them
    }
    bad = bad || head < 0 || count < 0 || static_cast<uint32_t>(head) >= p.n_pages ||
          static_cast<uint32_t>(count) > p.n_pages;
    const int any_bad = __syncthreads_or(bad), any_over = __syncthreads_or(over);
    // every block reaches the same verdict
    int32_t verdict = 0;
    if (any_bad || static_cast<long long>(count) + c_back > static_cast<long long>(p.n_pages)) verdict = -3;
    else if (any_over) verdict = -2;
    else if (c_new > static_cast<long long>(p.max_tokens)) verdict = -1;
    else if (c_take > count) verdict = c_take - count;
    const bool go = verdict == 0;
    const int32_t total = go ? static_cast<int32_t>(c_new) : 0;
    if (tid == 0) {
        cu[n] = total;
        take[n] = c_take;
        back[n] = c_back;
    }
    __syncthreads();

    const uint32_t first = blockIdx.x * kThreads + tid, stride = gridDim.x * kThreads;
    auto queued = [&](int32_t k) -> int32_t {   // the k-th queue entry from the head, k < n_pages
        const uint32_t at = static_cast<uint32_t>(head) + static_cast<uint32_t>(k);
        return p.ring[at >= p.n_pages ? at - p.n_pages : at];
    };
    for (uint32_t t = first; t < p.max_tokens; t += stride) {
        int32_t slot = -1, pos = 0;
        if (t < static_cast<uint32_t>(total)) {
            const uint32_t r = owner(cu, n, static_cast<int32_t>(t));
            const int32_t len = p.kv_len[r];
            pos = len + static_cast<int32_t>(t) - cu[r];
            const int32_t pg = pos >> p.page_shift, held = (len + pm) >> p.page_shift;
            const int32_t page = pg < held ? p.tables[static_cast<size_t>(r) * p.table_stride + pg]
                                           : queued(take[r] + pg - held);
            if (page >= 0 && static_cast<uint32_t>(page) < p.n_pages)
                slot = (page << p.page_shift) + (pos & pm);
            else
                atomicCAS(p.status, 0, ST_PAGED_BAD_PAGE);
        }
        p.slots[t] = slot;
        p.positions[t] = pos;
    }
    for (uint32_t r = first; r <= n; r += stride) {
        p.cu_new[r] = go ? cu[r] : 0;
        if (r < n) {
            const int32_t len = p.kv_len[r], add = p.new_len[r];
            p.kv_len_out[r] = !go ? len : add < 0 ? 0 : len + add;
        }
    }
    if (first == 0) {
        int32_t h = head + c_take;
        if (go && static_cast<uint32_t>(h) >= p.n_pages) h -= static_cast<int32_t>(p.n_pages);
        *reinterpret_cast<int4*>(p.state_out) =
            go ? make_int4(h, count - c_take + c_back, 0, total) : make_int4(head, count, verdict, 0);
    }
    if (!go) return;
    for (uint32_t k = first; k < static_cast<uint32_t>(c_take); k += stride) {
        const uint32_t r = owner(take, n, static_cast<int32_t>(k));
        const int32_t held = (p.kv_len[r] + pm) >> p.page_shift;
        p.tables[static_cast<size_t>(r) * p.table_stride + held + (k - take[r])] = queued(static_cast<int32_t>(k));
    }
    for (uint32_t k = first; k < static_cast<uint32_t>(c_back); k += stride) {
        const uint32_t r = owner(back, n, static_cast<int32_t>(k));
        const int32_t page = p.tables[static_cast<size_t>(r) * p.table_stride + (k - back[r])];
        if (page < 0 || static_cast<uint32_t>(page) >= p.n_pages) atomicCAS(p.status, 0, ST_PAGED_BAD_PAGE);
        uint32_t at = static_cast<uint32_t>(head) + static_cast<uint32_t>(count);   // < 2 * n_pages
        if (at >= p.n_pages) at -= p.n_pages;
        at += k;
        p.ring[at >= p.n_pages ? at - p.n_pages : at] = page;
    }
}

bool overlap(const void* a, size_t an, const void* b, size_t bn) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + bn && y < x + an;
}

}  // namespace
}  // namespace yattn

using namespace yattn;

extern "C" int yattn_page_step(int32_t* kv_len_out, int32_t* cu_new, int32_t* slots, int32_t* positions,
                               uint32_t max_tokens, int32_t* state_out, int32_t* tables, uint32_t max_pages,
                               uint32_t table_stride, int32_t* ring, uint32_t n_pages, const int32_t* state,
                               const int32_t* kv_len, const int32_t* new_len, uint32_t n_seqs, uint32_t page_size,
                               void* stream, char* err, size_t errlen) {
    if (!kv_len_out || !cu_new || !state_out || !tables || !ring || !state || !kv_len || !new_len ||
        (max_tokens && (!slots || !positions))) {
        set_err(err, errlen, "page_step: null pointer argument");
        return -1;
    }
    if (!paged_size_ok(page_size)) {
        set_err(err, errlen, "page_step: page_size %u not supported (16/32/64/128/256)", page_size);
        return -1;
    }
    if (n_seqs == 0 || n_seqs > kMaxSeqs) {
        set_err(err, errlen, "page_step: %u requests (1 to %u)", n_seqs, kMaxSeqs);
        return -1;
    }
    if (max_pages == 0 || table_stride < max_pages ||
        static_cast<uint64_t>(max_pages) * page_size > 0x7fffffffull ||
        static_cast<uint64_t>(max_pages) * n_seqs > 0x7fffffffull) {
        set_err(err, errlen, "page_step: bad table shape: max_pages %u, table_stride %u, %u requests", max_pages,
                table_stride, n_seqs);
        return -1;
    }
    if (n_pages == 0 || static_cast<uint64_t>(n_pages) * page_size > 0x7fffffffull || max_tokens > 0x7fffffffu) {
        set_err(err, errlen, "page_step: %u pages of %u tokens, %u token slots: more than 2^31-1 rows", n_pages,
                page_size, max_tokens);
        return -1;
    }
    const uintptr_t all = reinterpret_cast<uintptr_t>(kv_len_out) | reinterpret_cast<uintptr_t>(cu_new) |
                          reinterpret_cast<uintptr_t>(slots) | reinterpret_cast<uintptr_t>(positions) |
                          reinterpret_cast<uintptr_t>(tables) | reinterpret_cast<uintptr_t>(ring) |
                          reinterpret_cast<uintptr_t>(state) | reinterpret_cast<uintptr_t>(kv_len) |
                          reinterpret_cast<uintptr_t>(new_len);
    if ((all & 3u) || (reinterpret_cast<uintptr_t>(state_out) & 15u)) {
        set_err(err, errlen, "page_step: arrays must be 4-byte aligned, state_out 16-byte aligned");
        return -1;
    }
    // blocks run in any order: an output over an input would be read back by a later block
    const size_t nb = static_cast<size_t>(n_seqs) * 4;
    const void* ins[3] = {kv_len, new_len, state};
    const size_t in_n[3] = {nb, nb, 8};
    const void* outs[5] = {kv_len_out, cu_new, slots, positions, state_out};
    const size_t out_n[5] = {nb, nb + 4, static_cast<size_t>(max_tokens) * 4, static_cast<size_t>(max_tokens) * 4, 16};
    for (int i = 0; i < 5; ++i)
        for (int j = 0; j < 3; ++j)
            if (outs[i] && overlap(outs[i], out_n[i], ins[j], in_n[j])) {
                set_err(err, errlen, "page_step: an output overlaps kv_len, new_len or state: use separate buffers");
                return -1;
            }
    DevCtx* ctx = dev_ctx(err, errlen);
    if (!ctx) return -1;
    StepParams p{};
    p.kv_len_out = kv_len_out;
    p.cu_new = cu_new;
    p.slots = slots;
    p.positions = positions;
    p.state_out = state_out;
    p.tables = tables;
    p.ring = ring;
    p.state = state;
    p.kv_len = kv_len;
    p.new_len = new_len;
    p.max_tokens = max_tokens;
    p.max_pages = max_pages;
    p.table_stride = table_stride;
    p.n_pages = n_pages;
    p.n_seqs = n_seqs;
    p.page_shift = static_cast<uint32_t>(__builtin_ctz(page_size));
    p.status = ctx->status;
    const size_t smem = 3 * (static_cast<size_t>(n_seqs) + 1) * 4;
    // the limit is the kernel's, not the call's: raised once to what the largest call needs, so that no other thread's
    // call finds it lower than its own size
    static std::atomic<bool> attr_done[64];
    if (!attr_done[ctx->device].load(std::memory_order_acquire)) {
        constexpr int kMaxSmem = 3 * (static_cast<int>(kMaxSeqs) + 1) * 4;
        cudaError_t e = cudaFuncSetAttribute(k_page_step, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
        if (e != cudaSuccess) {
            set_err(err, errlen, "page_step: smem attribute (%d bytes): %s", kMaxSmem, cudaGetErrorString(e));
            return -1;
        }
        attr_done[ctx->device].store(true, std::memory_order_release);
    }
    // a token a thread up to one block per SM; the prefix sums are repeated in every block
    const uint32_t work = std::max(max_tokens, n_seqs + 1);
    const uint32_t blocks = std::min<uint32_t>((work + kThreads - 1) / kThreads, static_cast<uint32_t>(ctx->num_sms));
    k_page_step<<<blocks, kThreads, smem, static_cast<cudaStream_t>(stream)>>>(p);
    YATTN_CHECK_LAUNCH(err, errlen, "page_step");
    return 0;
}
