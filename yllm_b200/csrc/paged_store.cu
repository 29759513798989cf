// paged_store.cu -- QK-norm, RoPE and the K/V store of ragged tokens into a paged cache.
//
// Per token t (position pos, cache row slot):
//     x' = x * w / sqrt(mean(x^2) + eps)          per q and k head, if norm weights are given
//     (a, b) -> (a c - b s, a s + b c)            pair j of a q or k head, angle = pos * theta^(-2j/n)
//     q_out[t] = q', kpool[slot] = fp16(k'), vpool[slot] = fp16(v)
// The pairs are those of the contiguous store (rope.cu).  The angle differs on purpose: there it is one
// fp32 multiply, as in the reference's engine, which at position 100,000 is off by up to 2^-8 rad (half
// an ulp of the angle); here it is a product in 64 bits, reduced to a half turn before it is rounded, so
// every angle is good to 1 ulp of its sine and cosine however far the position.
//
// One CTA per token.  A thread holds two VEC-element chunks of one head, VEC * size = 16 bytes, placed so
// that both elements of each of its pairs are its own (half-split pairs: chunk c and chunk c + n/2;
// neighbour pairs and unrotated dims: two chunks in a row).  So a head is hd / (2 VEC) consecutive lanes
// (4 to 32), its sum of squares is a shuffle reduction among them, and every global access is a 16-byte
// vector (8 for the fp16 rows of fp32 activations).  The token's sines and cosines, n/2 pairs shared by
// all its heads, are computed once by the first threads while the row's loads are in flight.
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
    uint32_t n_heads, n_kv, kv_dim;
    uint32_t neighbour;              // pairs (2j, 2j+1); else (j, j + n_dims/2)
    uint32_t n_dims;
    int* status;
    double half_turns[kMaxPairs];    // theta^(-2j/n_dims) / pi: half turns per position
};

// VEC consecutive activations as fp32 (16 bytes read), and back (rounded to nearest).
__device__ __forceinline__ void load_vec(const float* p, float (&x)[4]) {
    const float4 v = __ldcs(reinterpret_cast<const float4*>(p));
    x[0] = v.x;
    x[1] = v.y;
    x[2] = v.z;
    x[3] = v.w;
}
__device__ __forceinline__ void load_vec(const __half* p, float (&x)[8]) {
    const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = h2f2(w[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void load_vec(const __nv_bfloat16* p, float (&x)[8]) {
    const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p));
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
// Cache rows: the engine's rounding, as every other store into the cache.
template <int VEC> __device__ __forceinline__ void store_cache(uint16_t* p, const float (&x)[VEC]) {
    uint32_t w[VEC / 2];
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i)
        w[i] = engine_f32_to_f16(x[2 * i]) | static_cast<uint32_t>(engine_f32_to_f16(x[2 * i + 1])) << 16;
    if constexpr (VEC == 4)
        *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ float norm_w(const StoreParams& p, const void* w, uint32_t e) {
    return p.norm_f16 ? h2f(static_cast<const uint16_t*>(w)[e]) : static_cast<const float*>(w)[e];
}

template <typename T, int HD>
__global__ void __launch_bounds__(512) k_paged_store(const __grid_constant__ StoreParams p) {
    constexpr int VEC = 16 / sizeof(T);
    constexpr uint32_t LPH = HD / (2 * VEC);          // lanes per head
    static_assert(LPH <= 32 && (LPH & (LPH - 1)) == 0, "a head lies in one warp");
    __shared__ float2 s_cs[kMaxPairs];
    const size_t t = blockIdx.x;
    const int32_t slot = p.slots[t];
    if (slot < 0) return;                             // a padded token: nothing is read or written
    const uint32_t half = p.n_dims / 2;
    const uint32_t n_items = (p.n_heads + 2 * p.n_kv) * LPH;
    bool ready = false;
    for (uint32_t base = 0; base < n_items; base += blockDim.x) {
        const uint32_t item = base + threadIdx.x;
        const uint32_t head = item / LPH, u = item % LPH;   // q heads, k heads, v heads
        const bool live = item < n_items;
        const bool is_q = head < p.n_heads, is_v = head >= p.n_heads + p.n_kv;
        const uint32_t h = is_q ? head : is_v ? head - p.n_heads - p.n_kv : head - p.n_heads;
        // this thread's two chunks of the head
        uint32_t ea = u * 2 * VEC, eb = ea + VEC;
        const bool split = !p.neighbour && !is_v && u * VEC < half;
        if (split) {
            ea = u * VEC;
            eb = ea + half;
        }
        float a[VEC], b[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) a[i] = b[i] = 0.f;
        if (live) {
            const T* src = is_q ? static_cast<const T*>(p.q) + t * p.q_stride
                                : is_v ? static_cast<const T*>(p.v) + t * p.v_stride
                                       : static_cast<const T*>(p.k) + t * p.k_stride;
            load_vec(src + h * HD + ea, a);
            load_vec(src + h * HD + eb, b);
        }
        if (!ready) {                                 // while those loads are in flight
            const double pos = static_cast<double>(p.positions[t]);
            for (uint32_t j = threadIdx.x; j < half; j += blockDim.x) {
                double ht = pos * p.half_turns[j];
                ht -= 2.0 * rint(0.5 * ht);           // [-1, 1] half turns
                float s, c;
                sincospif(static_cast<float>(ht), &s, &c);
                s_cs[j] = make_float2(c, s);
            }
            __syncthreads();
            ready = true;
        }
        if (p.q_w) {                                  // every lane of the warp takes part
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < VEC; ++i) ss += a[i] * a[i] + b[i] * b[i];
#pragma unroll
            for (uint32_t o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (live && !is_v) {
                const float inv = 1.0f / sqrtf(ss * (1.0f / HD) + p.eps);
                const void* w = is_q ? p.q_w : p.k_w;
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    a[i] = a[i] * norm_w(p, w, ea + i) * inv;
                    b[i] = b[i] * norm_w(p, w, eb + i) * inv;
                }
            }
        }
        if (!live) continue;
        if (!is_v) {
            if (split) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float2 cs = s_cs[ea + i];
                    const float x = a[i], y = b[i];
                    a[i] = x * cs.x - y * cs.y;
                    b[i] = x * cs.y + y * cs.x;
                }
            } else if (p.neighbour) {
#pragma unroll
                for (int i = 0; i < VEC; i += 2) {
                    const float2 ca = s_cs[(ea + i) / 2], cb = s_cs[(eb + i) / 2];
                    const float xa = a[i], ya = a[i + 1], xb = b[i], yb = b[i + 1];
                    a[i] = xa * ca.x - ya * ca.y;
                    a[i + 1] = xa * ca.y + ya * ca.x;
                    b[i] = xb * cb.x - yb * cb.y;
                    b[i + 1] = xb * cb.y + yb * cb.x;
                }
            }
        }
        if (is_q) {
            T* dst = static_cast<T*>(p.q_out) + t * p.qo_stride + h * HD;
            store_vec(dst + ea, a);
            store_vec(dst + eb, b);
        } else if (static_cast<uint64_t>(slot) < p.n_rows) {
            uint16_t* dst = (is_v ? p.vpool : p.kpool) + static_cast<size_t>(slot) * p.kv_dim + h * HD;
            store_cache<VEC>(dst + ea, a);
            store_cache<VEC>(dst + eb, b);
        } else if (u == 0) {
            atomicCAS(p.status, 0, ST_PAGED_BAD_PAGE);
        }
    }
}

template <typename T, int HD>
int launch_store(const StoreParams& p, uint32_t n_tokens, cudaStream_t st, char* err, size_t errlen) {
    constexpr uint32_t LPH = HD / (2 * (16 / sizeof(T)));
    const uint32_t items = (p.n_heads + 2 * p.n_kv) * LPH;
    // one pass over the token's items where they fit a block of 512, else equal passes
    const uint32_t passes = (items + 511) / 512;
    const uint32_t threads = ((items + passes - 1) / passes + 31) / 32 * 32;
    k_paged_store<T, HD><<<n_tokens, threads, 0, st>>>(p);
    YATTN_CHECK_LAUNCH(err, errlen, "rope_store_kv_paged");
    return 0;
}

template <typename T>
int dispatch_store(const StoreParams& p, uint32_t hd, uint32_t n_tokens, cudaStream_t st, char* err, size_t errlen) {
    switch (hd) {
        case 64: return launch_store<T, 64>(p, n_tokens, st, err, errlen);
        case 128: return launch_store<T, 128>(p, n_tokens, st, err, errlen);
        default: return launch_store<T, 256>(p, n_tokens, st, err, errlen);
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
        case YATTN_ACT_F32: return dispatch_store<float>(p, head_dim, n_tokens, st, err, errlen);
        case YATTN_ACT_F16: return dispatch_store<__half>(p, head_dim, n_tokens, st, err, errlen);
        default: return dispatch_store<__nv_bfloat16>(p, head_dim, n_tokens, st, err, errlen);
    }
}
