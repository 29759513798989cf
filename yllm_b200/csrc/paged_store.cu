// paged_store.cu -- QK-norm, RoPE and the K/V store of ragged tokens into a paged cache.
//
// Per token t (position pos, cache row slot):
//     x' = x * w / sqrt(mean(x^2) + eps)          per q and k head, if norm weights are given
//     (a, b) -> (a c - b s, a s + b c)            pair j of a q or k head, angle = pos * theta^(-2j/n)
//     q_out[t] = q', kpool[slot] = fp16(k'), vpool[slot] = fp16(v)
// The pairs are those of the contiguous store (rope.cu).  The angle differs on purpose: there it is one
// fp32 multiply, as in the reference's engine, which at position 100,000 is off by up to 2^-8 rad (half
// an ulp of the angle); here it is a product in 64 bits, reduced to a half turn before it is rounded, so
// sine and cosine are off by 2^-22 or less, absolute, however far the position: 2^-24 or so for the angle's
// rounding and 2 ulp for sincospif, which is 2^-22 of the pair's norm.
//
// A thread holds two VEC-element chunks of one head, VEC * size = 16 bytes, placed so that both elements
// of each of its pairs are its own (half-split pairs: chunk c and chunk c + n/2; neighbour pairs and
// unrotated dims: two chunks in a row).  So a head is hd / (2 VEC) consecutive lanes (4 to 32), its sum of
// squares is a shuffle reduction among them, and every global access is a 16-byte vector (8 for the fp16
// rows of fp32 activations).
//
// A CTA covers a token's heads (or a slice of them, where they pass 512 threads) and walks over tokens
// with the next token's loads in flight, so the chain of one token -- load, norm, rotate, store -- hides
// behind the others.  Sines and cosines, shared by a token's heads, go through shared memory, two buffers
// in turn and four tokens at a time: with one barrier per token the barrier was the kernel's largest stall
// (the fp64 angle and sincospif of one warp behind it; 16384 tokens of the qwen3.5 shape took 161 us).
// The norm weights are read from global memory once per CTA.
//
// Bound: HBM.  q, k and v are read once, q_out and the cache rows written once.
#include "common.cuh"

#include <cuda_bf16.h>

#include <algorithm>
#include <cmath>

namespace yattn {
namespace {

constexpr int kMaxPairs = 128;   // head_dim <= 256

struct StoreParams {
    void* q_out;
    const void* q;
    const void* k;
    const void* v;
    uint16_t* kpool;
    uint16_t* vpool;
    const int32_t* slots;
    const int32_t* positions;
    const void* q_w;                 // QK-norm weights [hd]; NULL: no norm
    const void* k_w;
    uint32_t norm_f16;
    float eps;
    uint64_t q_stride, k_stride, v_stride, qo_stride;   // elements between tokens
    uint64_t n_rows;                 // rows of each pool
    uint32_t n_tokens, n_heads, n_kv, kv_dim;
    uint32_t group;                  // tokens per barrier, 1 to kGroup
    uint32_t neighbour;              // pairs (2j, 2j+1); else (j, j + n_dims/2)
    uint32_t n_dims;
    int* status;
    double half_turns[kMaxPairs];    // theta^(-2j/n_dims) / pi: half turns per position
};

// 16 bytes of activations as fp32, and back (rounded to nearest).
__device__ __forceinline__ void widen(const uint4& v, const float*, float (&x)[4]) {
    x[0] = __uint_as_float(v.x);
    x[1] = __uint_as_float(v.y);
    x[2] = __uint_as_float(v.z);
    x[3] = __uint_as_float(v.w);
}
__device__ __forceinline__ void widen(const uint4& v, const __half*, float (&x)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = h2f2(w[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void widen(const uint4& v, const __nv_bfloat16*, float (&x)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void store_vec(float* p, const float (&x)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ void store_vec(__half* p, const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void store_vec(__nv_bfloat16* p, const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
// Cache rows: the engine's rounding, as every other store into the cache.  From 2^-14 up it adds half a
// step to the magnitude and truncates, which leaves an fp16 value; smaller ones and NaN take the long form.
__device__ __forceinline__ uint32_t cache_bits(float x) {
    const uint32_t b = __float_as_uint(x);
    if ((b & 0x7fffffffu) - 0x38800000u <= 0x7f800000u - 0x38800000u)
        return __half_as_ushort(__float2half_rn(__uint_as_float((b + 0x1000u) & 0xffffe000u)));
    return engine_f32_to_f16(x);
}
template <int VEC> __device__ __forceinline__ void store_cache(uint16_t* p, const float (&x)[VEC]) {
    uint32_t w[VEC / 2];
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) w[i] = cache_bits(x[2 * i]) | cache_bits(x[2 * i + 1]) << 16;
    if constexpr (VEC == 4)
        *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// N floats from 16-byte aligned shared memory.
template <int N> __device__ __forceinline__ void lds(const float* p, float (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        const float4 v = *reinterpret_cast<const float4*>(p + i);
        x[i] = v.x;
        x[i + 1] = v.y;
        x[i + 2] = v.z;
        x[i + 3] = v.w;
    }
}

constexpr uint32_t kGroup = 4;   // most tokens per barrier

template <typename T, int HD>
__global__ void __launch_bounds__(512, sizeof(T) == 4 ? 3 : 2) k_paged_store(const __grid_constant__ StoreParams p) {
    constexpr int VEC = 16 / sizeof(T);
    constexpr uint32_t LPH = HD / (2 * VEC);          // lanes per head
    static_assert(LPH <= 32 && (LPH & (LPH - 1)) == 0, "a head lies in one warp");
    __shared__ __align__(16) float s_cos[2][kGroup][kMaxPairs], s_sin[2][kGroup][kMaxPairs];
    __shared__ __align__(16) float s_w[2][HD];        // QK-norm weights of q and k heads
    const uint32_t half = p.n_dims / 2;
    // this thread's item: two chunks of a q, k or v head, the same for every token
    const uint32_t item = blockIdx.y * blockDim.x + threadIdx.x;
    const uint32_t head = item / LPH, u = item % LPH;
    const bool live = head < p.n_heads + 2 * p.n_kv;
    const bool is_q = head < p.n_heads, is_v = head >= p.n_heads + p.n_kv;
    const uint32_t h = is_q ? head : is_v ? head - p.n_heads - p.n_kv : head - p.n_heads;
    const bool split = !p.neighbour && !is_v && u * VEC < half;
    const uint32_t ea = split ? u * VEC : u * 2 * VEC;
    const uint32_t eb = split ? ea + half : ea + VEC;
    const T* src = static_cast<const T*>(is_q ? p.q : is_v ? p.v : p.k) + h * HD;
    const uint64_t src_stride = is_q ? p.q_stride : is_v ? p.v_stride : p.k_stride;
    uint16_t* pool = (is_v ? p.vpool : p.kpool) + h * HD;
    auto fetch = [&](size_t t, uint4& ra, uint4& rb) {
        if (live) {
            const T* row = src + t * src_stride;
            ra = __ldcs(reinterpret_cast<const uint4*>(row + ea));
            rb = __ldcs(reinterpret_cast<const uint4*>(row + eb));
        }
    };

    auto process = [&](size_t t, int32_t slot, const uint4& ra, const uint4& rb, const float* cs, const float* sn) {
        float a[VEC], b[VEC];
        widen(ra, static_cast<const T*>(nullptr), a);
        widen(rb, static_cast<const T*>(nullptr), b);
        if (p.q_w) {                                  // every lane of the warp takes part
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < VEC; ++i) ss += a[i] * a[i] + b[i] * b[i];
#pragma unroll
            for (uint32_t o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (!is_v) {
                const float m = ss * (1.0f / HD) + p.eps;
                float inv = rsqrtf(m);
                // one Newton step: rsqrt.approx is 2 ulp off.  Where the squares passed fp32, 1 / sqrt(m) = 0 stays, and
                // x goes times it before w: x w may pass fp32 as well
                inv = m < INFINITY ? inv * (1.5f - 0.5f * m * inv * inv) : inv;
                float wa[VEC], wb[VEC];
                lds(s_w[is_q ? 0 : 1] + ea, wa);
                lds(s_w[is_q ? 0 : 1] + eb, wb);
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    a[i] = a[i] * inv * wa[i];
                    b[i] = b[i] * inv * wb[i];
                }
            }
        }
        if (split) {
            float c[VEC], s[VEC];
            lds(cs + ea, c);
            lds(sn + ea, s);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float x = a[i], y = b[i];
                a[i] = x * c[i] - y * s[i];
                b[i] = x * s[i] + y * c[i];
            }
        } else if (p.neighbour && !is_v) {            // pairs ea/2 .. ea/2 + VEC - 1: chunk a's, then chunk b's
            float c[VEC], s[VEC];
            lds(cs + ea / 2, c);
            lds(sn + ea / 2, s);
#pragma unroll
            for (int i = 0; i < VEC / 2; ++i) {
                const float xa = a[2 * i], ya = a[2 * i + 1], xb = b[2 * i], yb = b[2 * i + 1];
                a[2 * i] = xa * c[i] - ya * s[i];
                a[2 * i + 1] = xa * s[i] + ya * c[i];
                b[2 * i] = xb * c[VEC / 2 + i] - yb * s[VEC / 2 + i];
                b[2 * i + 1] = xb * s[VEC / 2 + i] + yb * c[VEC / 2 + i];
            }
        }
        if (!live) {
        } else if (is_q) {
            T* dst = static_cast<T*>(p.q_out) + t * p.qo_stride + h * HD;
            store_vec(dst + ea, a);
            store_vec(dst + eb, b);
        } else if (static_cast<uint64_t>(slot) < p.n_rows) {
            uint16_t* dst = pool + static_cast<size_t>(slot) * p.kv_dim;
            store_cache<VEC>(dst + ea, a);
            store_cache<VEC>(dst + eb, b);
        } else if (u == 0) {
            atomicCAS(p.status, 0, ST_PAGED_BAD_PAGE);
        }
    };

    const size_t n = p.n_tokens, group = p.group;
    size_t t = blockIdx.x * group;                    // < n_tokens
    uint4 ra = {}, rb = {};
    fetch(t, ra, rb);
    int32_t slot = p.slots[t];
    if (p.q_w) {                                      // published by the first group's barrier
        for (uint32_t i = threadIdx.x; i < 2 * HD; i += blockDim.x) {
            const void* w = i < HD ? p.q_w : p.k_w;
            const uint32_t e = i % HD;
            s_w[i / HD][e] = p.norm_f16 ? h2f(static_cast<const uint16_t*>(w)[e]) : static_cast<const float*>(w)[e];
        }
    }
    // this thread's first pair of a group, whose position is loaded a group ahead
    const uint32_t j0 = threadIdx.x % half, k0 = threadIdx.x / half;
    const double f0 = p.half_turns[j0];
    int32_t pos0 = k0 < group && t + k0 < n ? p.positions[t + k0] : 0;
    for (uint32_t buf = 0; t < n; buf ^= 1) {
        const size_t t_next = t + gridDim.x * group;  // the next group
        for (uint32_t i = threadIdx.x; i < group * half; i += blockDim.x) {
            const bool first = i == threadIdx.x;
            const uint32_t k = first ? k0 : i / half, j = first ? j0 : i % half;
            if (t + k >= n) break;
            double ht = first ? pos0 * f0 : p.positions[t + k] * p.half_turns[j];
            ht -= 2.0 * rint(0.5 * ht);               // [-1, 1] half turns
            sincospif(static_cast<float>(ht), &s_sin[buf][k][j], &s_cos[buf][k][j]);
        }
        pos0 = k0 < group && t_next + k0 < n ? p.positions[t_next + k0] : 0;
        __syncthreads();
        for (uint32_t k = 0; k < group && t < n; ++k) {
            const size_t tn = k + 1 < group && t + 1 < n ? t + 1 : t_next;
            uint4 na = {}, nb = {};
            int32_t nslot = -1;
            if (tn < n) {
                fetch(tn, na, nb);
                nslot = p.slots[tn];
            }
            if (slot >= 0) process(t, slot, ra, rb, s_cos[buf][k], s_sin[buf][k]);   // else a padded token
            const bool last = tn == t_next;
            t = tn;
            ra = na;
            rb = nb;
            slot = nslot;
            if (last) break;
        }
    }
}

template <typename T, int HD>
int launch_store(const StoreParams& p, uint32_t sms, cudaStream_t st, char* err, size_t errlen) {
    constexpr uint32_t LPH = HD / (2 * (16 / sizeof(T)));
    const uint32_t items = (p.n_heads + 2 * p.n_kv) * LPH;
    const uint32_t slices = (items + 511) / 512;
    const uint32_t threads = ((items + slices - 1) / slices + 31) / 32 * 32;
    // as many CTAs as the SMs hold, at 42 registers a thread for fp32 and 64 for 16-bit activations (twice the
    // values a thread, which 42 would spill): 8192 Llama-3-8B tokens in fp32 take 62 us against 74 at 64. Each CTA
    // walks over every gridDim.x-th group of tokens
    const uint32_t resident = std::max(1u, std::min(16u, (sizeof(T) == 4 ? 1536u : 1024u) / threads));
    const uint32_t most = std::max(1u, sms * resident / slices);
    StoreParams q = p;
    // tokens per barrier: 4 once a CTA has more than 8 of them, as long as few, 1 or 2, which spreads them more evenly
    // (fp16 qwen3-0.6b shape with norms: 700 tokens 6.1 us against 8.9 with 4, 2048 11.0 against 12.4, 2600 13.9
    // against 16.4; from 8 on 4 is as fast or faster)
    q.group = p.n_tokens <= 4 * most ? 1 : p.n_tokens <= 8 * most ? 2 : kGroup;
    const uint32_t ctas = std::min((p.n_tokens + q.group - 1) / q.group, most);
    k_paged_store<T, HD><<<dim3(ctas, slices), threads, 0, st>>>(q);
    YATTN_CHECK_LAUNCH(err, errlen, "rope_store_kv_paged");
    return 0;
}

template <typename T>
int dispatch_store(const StoreParams& p, uint32_t hd, uint32_t sms, cudaStream_t st, char* err, size_t errlen) {
    switch (hd) {
        case 64: return launch_store<T, 64>(p, sms, st, err, errlen);
        case 128: return launch_store<T, 128>(p, sms, st, err, errlen);
        default: return launch_store<T, 256>(p, sms, st, err, errlen);
    }
}

}  // namespace
}  // namespace yattn

using namespace yattn;

extern "C" int yattn_rope_store_kv_paged(void* q_out, uint32_t q_out_stride, const void* q, uint32_t q_stride,
                                         const void* k, uint32_t k_stride, const void* v, uint32_t v_stride, int act,
                                         uint16_t* kpool, uint16_t* vpool, uint64_t n_rows, const int32_t* slots,
                                         const int32_t* positions, uint32_t n_tokens, uint32_t n_heads,
                                         uint32_t n_kv_heads, uint32_t head_dim, uint32_t kv_dim, int rope_kind,
                                         uint32_t n_rope_dims, float theta, const YattnQkNorm* qk_norm, void* stream,
                                         char* err, size_t errlen) {
    if (n_tokens == 0) return 0;
    if (!q_out || !q || !k || !v || !kpool || !vpool || !slots || !positions) {
        set_err(err, errlen, "rope_store_kv_paged: null pointer argument");
        return -1;
    }
    if (act != YATTN_ACT_F32 && act != YATTN_ACT_F16 && act != YATTN_ACT_BF16) {
        set_err(err, errlen, "rope_store_kv_paged: unknown activation type %d", act);
        return -1;
    }
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) {
        set_err(err, errlen, "rope_store_kv_paged: head_dim %u not supported (64/128/256)", head_dim);
        return -1;
    }
    if (n_heads == 0 || n_kv_heads == 0 || n_kv_heads > n_heads || n_heads > 1024 ||
        kv_dim < n_kv_heads * head_dim || (kv_dim % 8) != 0) {
        set_err(err, errlen, "rope_store_kv_paged: bad geometry n_heads=%u n_kv_heads=%u head_dim=%u kv_dim=%u",
                n_heads, n_kv_heads, head_dim, kv_dim);
        return -1;
    }
    if (rope_kind < 0 || rope_kind > 2) {
        set_err(err, errlen, "rope_store_kv_paged: rope_kind %d (0 llama, 1 qwen, 2 mrope)", rope_kind);
        return -1;
    }
    const uint32_t n_dims = rope_kind == 2 ? n_rope_dims : head_dim;
    if (n_dims == 0 || (n_dims % 16) != 0 || n_dims > head_dim) {
        set_err(err, errlen, "rope_store_kv_paged: %u rotated dims for head_dim %u (a multiple of 16)", n_dims,
                head_dim);
        return -1;
    }
    if (!(theta > 0.f) || !std::isfinite(theta)) {
        set_err(err, errlen, "rope_store_kv_paged: theta must be positive and finite");
        return -1;
    }
    const uint32_t size = act == YATTN_ACT_F32 ? 4 : 2, unit = 16 / size;
    if (q_stride < n_heads * head_dim || q_out_stride < n_heads * head_dim || k_stride < n_kv_heads * head_dim ||
        v_stride < n_kv_heads * head_dim || ((q_stride | q_out_stride | k_stride | v_stride) % unit) != 0) {
        set_err(err, errlen, "rope_store_kv_paged: token strides must cover the heads and be multiples of 16 bytes");
        return -1;
    }
    if ((reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) |
         reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(kpool) | reinterpret_cast<uintptr_t>(vpool)) & 15u) {
        set_err(err, errlen, "rope_store_kv_paged: q_out, q, k, v and the pools must be 16-byte aligned");
        return -1;
    }
    if ((reinterpret_cast<uintptr_t>(slots) | reinterpret_cast<uintptr_t>(positions)) & 3u) {
        set_err(err, errlen, "rope_store_kv_paged: slots and positions must be 4-byte aligned");
        return -1;
    }
    if (n_rows == 0 || n_rows > 0x7fffffffull || n_tokens > 0x7fffffffu) {
        set_err(err, errlen, "rope_store_kv_paged: %llu pool rows, %u tokens", static_cast<unsigned long long>(n_rows),
                n_tokens);
        return -1;
    }
    StoreParams p{};
    if (qk_norm) {
        if (!qk_norm->q_w || !qk_norm->k_w) {
            set_err(err, errlen, "rope_store_kv_paged: QK-norm needs both the q and the k weights");
            return -1;
        }
        if ((reinterpret_cast<uintptr_t>(qk_norm->q_w) | reinterpret_cast<uintptr_t>(qk_norm->k_w)) &
            (qk_norm->w_f16 ? 1u : 3u)) {
            set_err(err, errlen, "rope_store_kv_paged: QK-norm weights must be aligned to their element size");
            return -1;
        }
        p.q_w = qk_norm->q_w;
        p.k_w = qk_norm->k_w;
        p.norm_f16 = qk_norm->w_f16 ? 1u : 0u;
        p.eps = qk_norm->eps;
    }
    DevCtx* ctx = dev_ctx(err, errlen);
    if (!ctx) return -1;
    p.q_out = q_out;
    p.q = q;
    p.k = k;
    p.v = v;
    p.kpool = kpool;
    p.vpool = vpool;
    p.slots = slots;
    p.positions = positions;
    p.q_stride = q_stride;
    p.k_stride = k_stride;
    p.v_stride = v_stride;
    p.qo_stride = q_out_stride;
    p.n_rows = n_rows;
    p.n_tokens = n_tokens;
    p.n_heads = n_heads;
    p.n_kv = n_kv_heads;
    p.kv_dim = kv_dim;
    p.neighbour = rope_kind == 0;
    p.n_dims = n_dims;
    p.status = ctx->status;
    // the frequencies of the last (theta, n_dims) of this host thread: 128 powers cost more than the launch
    static thread_local struct {
        float theta;
        uint32_t n_dims;
        double f[kMaxPairs];
    } freq = {0.f, 0, {}};
    if (freq.theta != theta || freq.n_dims != n_dims) {
        for (uint32_t j = 0; j < n_dims / 2; ++j)
            freq.f[j] = std::pow(static_cast<double>(theta), -2.0 * j / n_dims) / 3.14159265358979323846;
        freq.theta = theta;
        freq.n_dims = n_dims;
    }
    std::copy(freq.f, freq.f + n_dims / 2, p.half_turns);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (act) {
        case YATTN_ACT_F32: return dispatch_store<float>(p, head_dim, static_cast<uint32_t>(ctx->num_sms), st, err, errlen);
        case YATTN_ACT_F16: return dispatch_store<__half>(p, head_dim, static_cast<uint32_t>(ctx->num_sms), st, err, errlen);
        default: return dispatch_store<__nv_bfloat16>(p, head_dim, static_cast<uint32_t>(ctx->num_sms), st, err, errlen);
    }
}
