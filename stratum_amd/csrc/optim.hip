// What a training step does to its gradients and parameters (gfx950): the norm
// of all gradients, and one AdamW step over all tensors, each in few launches.
//
//   norm      out[0] = |g| / c, out[1] = min(1, max_norm / (out[0] + 1e-6)) / c, c the loss scale;
//             out[1] = NaN where the norm is not finite
//   AdamW     g' = scale g;  m = b1 m + (1 - b1) g';  v = b2 v + (1 - b2) g' g'
//             p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//             and nothing at all where scale is not finite
//
// Both are bound by HBM: the norm reads every gradient once; a step reads p, g, m
// and v and writes p, m and v. All arithmetic is fp32 in the order above, one rounding
// each (no contraction), so that a plain evaluation gives the same states bit for bit.
//
// Tensors travel as kernel arguments (pointers and sizes, one launch for up to
// kAdamTensors / kNormTensors of them); a work-group finds its tensor by a ballot over
// the prefix sums of work-groups.
//
// States in 8 bits. Blocks of 256 elements of a tensor share an fp32 scale, their
// largest magnitude. A code holds a magnitude q of K + 1 bits (K = 6 below a sign bit
// for m, K = 7 for v, which has no sign): q = 0 is zero, otherwise with k = floor(log2 q)
//     level(q) = (7 q + 7 - 6 * 2^k) * 2^(2 k - 3 - 3 K),
// i.e. linear segments between powers of 8 of which the one from 1/8 to 1 holds 2^K
// levels and every lower one half as many as the next. The segments' ends, 1 among
// them, are levels, so the largest element of a block is kept exactly. A magnitude
// takes the nearest level of its segment (ties to the even step from the lower end);
// below the lowest level, 8^-K, the nearer of it and zero. A second moment that is
// not zero never becomes zero (it takes the lowest level): with a first moment left,
// a zero would divide by eps alone in a later step. Levels are dyadic, so the code is
// arithmetic both ways: no table, no LDS.
#include "nf4_common.h"

namespace stm {
namespace {

constexpr int kBlock8 = 256;      // elements per scale of an 8-bit state
constexpr int kAdamTensors = 56;  // tensors per launch (below 4 KB of kernel arguments)
constexpr int kNormTensors = 160;
constexpr int kTile = 2048;       // elements per work-group: 256 threads of 8
constexpr int kNormTile = 16384;  // elements per work-group of the norm

struct AdamArgs {
    stm_adamw_tensor t[kAdamTensors];
    int first[kAdamTensors];  // first work-group of tensor i
    int count;
    float beta1, beta2, rest1, rest2;  // rest = 1 - beta
    float decay, step_size, inv_root2, eps;
    const float* scale;
};
static_assert(sizeof(AdamArgs) <= 4096, "kernel arguments");

struct NormArgs {
    const void* g[kNormTensors];
    int64_t n[kNormTensors];
    int first[kNormTensors];
    int count;
};
static_assert(sizeof(NormArgs) <= 4096, "kernel arguments");

// The tensor that work-group b belongs to: the last one whose first work-group is at
// or before b. Every lane of the wave takes part.
template <int CAP>
__device__ __forceinline__ int tensor_of(const int* first, int count, int b, int lane) {
    int below = 0;
#pragma unroll
    for (int i0 = 0; i0 < CAP; i0 += 64) {
        const int i = i0 + lane;
        below += __popcll(__ballot(i < count && first[i < count ? i : 0] <= b));
    }
    return __builtin_amdgcn_readfirstlane(below - 1);
}

// ------------------------------------------------------------ element access
struct F32 {
    static constexpr int tag = STM_F32;
};

template <typename T>
__device__ __forceinline__ void load8(const void* base, int64_t i, int64_t n, bool vec, float (&f)[8]) {
    if constexpr (T::tag == STM_F32) {
        const float* p = reinterpret_cast<const float*>(base) + i;
        if (vec && i + 8 <= n) {
            const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
            f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = i + e < n ? p[e] : 0.0f;
        }
    } else {
        const uint16_t* p = reinterpret_cast<const uint16_t*>(base) + i;
        if (vec && i + 8 <= n) {
            const uint4 v = *reinterpret_cast<const uint4*>(p);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                f[2 * e] = T::to_f32((uint16_t)(w[e] & 0xFFFFu));
                f[2 * e + 1] = T::to_f32((uint16_t)(w[e] >> 16));
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = i + e < n ? T::to_f32(p[e]) : 0.0f;
        }
    }
}

template <typename T>
__device__ __forceinline__ void store8(void* base, int64_t i, int64_t n, bool vec, const float (&f)[8]) {
    if constexpr (T::tag == STM_F32) {
        float* p = reinterpret_cast<float*>(base) + i;
        if (vec && i + 8 <= n) {
            reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
            reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (i + e < n) p[e] = f[e];
        }
    } else {
        uint16_t* p = reinterpret_cast<uint16_t*>(base) + i;
        if (vec && i + 8 <= n) {
            *reinterpret_cast<uint4*>(p) = make_uint4(T::pack2(f[0], f[1]), T::pack2(f[2], f[3]), T::pack2(f[4], f[5]),
                                                      T::pack2(f[6], f[7]));
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (i + e < n) p[e] = T::from_f32(f[e]);
        }
    }
}

__device__ __forceinline__ void load_codes(const uint8_t* base, int64_t i, int64_t n, bool vec, uint32_t (&c)[8]) {
    const uint8_t* p = base + i;
    if (vec && i + 8 <= n) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
#pragma unroll
        for (int e = 0; e < 4; ++e) c[e] = (v.x >> (8 * e)) & 255u, c[4 + e] = (v.y >> (8 * e)) & 255u;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) c[e] = i + e < n ? p[e] : 0u;
    }
}

__device__ __forceinline__ void store_codes(uint8_t* base, int64_t i, int64_t n, bool vec, const uint32_t (&c)[8]) {
    uint8_t* p = base + i;
    if (vec && i + 8 <= n) {
        uint2 v;
        v.x = c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
        v.y = c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24;
        *reinterpret_cast<uint2*>(p) = v;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (i + e < n) p[e] = (uint8_t)c[e];
    }
}

// ------------------------------------------------------------ the 8-bit code
// level(q) for q in 0..2^(K+1) - 1
template <int K>
__device__ __forceinline__ float level8(uint32_t q) {
    const int k = 31 - __builtin_clz(q | 1u);
    const float a = (float)(int)(7u * q + 7u - (6u << k));
    const float l = a * __uint_as_float((uint32_t)(127 + 2 * k - 3 - 3 * K) << 23);
    return q ? l : 0.0f;
}

template <bool SIGNED>
__device__ __forceinline__ float decode8(uint32_t code, float scale) {
    if constexpr (SIGNED) {
        const float v = level8<6>(code & 127u);
        return (code & 128u ? -v : v) * scale;
    } else {
        return level8<7>(code) * scale;
    }
}

// 1 / scale, or 0 for a block whose scale has no finite reciprocal that is normal
// (zero, subnormal, infinite, NaN): its codes are zero (v: the lowest level).
__device__ __forceinline__ float inverse_scale(float top) { return top >= 0x1p-126f ? 1.0f / top : 0.0f; }

template <bool SIGNED>
__device__ __forceinline__ uint32_t encode8(float x, float inv) {
    constexpr int K = SIGNED ? 6 : 7;
    const float s = fminf(fabsf(x) * inv, 1.0f);  // 1 also for an infinite x (inv is 0)
    // segment z: 8^-(z+1) <= s < 8^-z (z = K: everything below), from the exponent
    const int e = 126 - (int)(__float_as_uint(s) >> 23);
    int z = e <= 0 ? 0 : (e * 43) >> 7;  // e / 3 for e <= 127
    z = z < K ? z : K;
    const float y = s * __uint_as_float((uint32_t)(127 + 3 * z) << 23);
    // steps from the segment's lower end, 2^(K - z) of them between 1/8 and 1
    const float per = __uint_as_float(__float_as_uint(8.0f / 7.0f) + ((uint32_t)(K - z) << 23));
    const float j = z == K ? y : (y - 0.125f) * per;
    const int q = (1 << (K - z)) - 1 + (int)rintf(j);
    if constexpr (SIGNED) return (uint32_t)q | (x < 0.0f ? 128u : 0u);
    return (uint32_t)(q == 0 && x > 0.0f ? 1 : q);
}

// The largest magnitude of the 32 lanes that share a block (8 elements each). Compared
// as integers: the order of non-negative floats, with NaN above everything.
__device__ __forceinline__ float block_top(const float (&f)[8]) {
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t b = __float_as_uint(f[e]) & 0x7FFFFFFFu;
        top = top > b ? top : b;
    }
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t o = (uint32_t)__shfl_xor((int)top, d);
        top = top > o ? top : o;
    }
    return __uint_as_float(top);
}

// ------------------------------------------------------------ AdamW
template <typename P, typename G, int BITS>
__global__ __launch_bounds__(256) void k_adamw(AdamArgs a) {
    float scale = 1.0f;
    if (a.scale) {
        scale = *a.scale;
        if (!(fabsf(scale) < INFINITY)) return;  // the whole launch alike
    }
    const int lane = threadIdx.x & 63;
    const int ti = tensor_of<kAdamTensors>(a.first, a.count, (int)blockIdx.x, lane);
    const stm_adamw_tensor t = a.t[ti];
    const int64_t n = t.n, i = ((int64_t)blockIdx.x - a.first[ti]) * kTile + threadIdx.x * 8;
    auto al = [](const void* p, uintptr_t b) { return ((uintptr_t)p & (b - 1)) == 0; };
    const bool vp = al(t.param, 16), vg = al(t.grad, 16);
    const bool vs = al(t.exp_avg, BITS == 8 ? 8 : 16) && al(t.exp_avg_sq, BITS == 8 ? 8 : 16);

    float p[8], g[8], m[8], v[8];
    load8<G>(t.grad, i, n, vg, g);
    if (t.master)
        load8<F32>(t.master, i, n, al(t.master, 16), p);
    else
        load8<P>(t.param, i, n, vp, p);
    if constexpr (BITS == 32) {
        load8<F32>(t.exp_avg, i, n, vs, m);
        load8<F32>(t.exp_avg_sq, i, n, vs, v);
    } else {
        uint32_t cm[8], cv[8];
        load_codes((const uint8_t*)t.exp_avg, i, n, vs, cm);
        load_codes((const uint8_t*)t.exp_avg_sq, i, n, vs, cv);
        const int64_t b = i / kBlock8;
        const float sm = i < n ? t.exp_avg_scale[b] : 0.0f, sv = i < n ? t.exp_avg_sq_scale[b] : 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) m[e] = decode8<true>(cm[e], sm), v[e] = decode8<false>(cv[e], sv);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float ge = g[e] * scale;
        m[e] = m[e] * a.beta1 + ge * a.rest1;
        v[e] = v[e] * a.beta2 + ge * a.rest2 * ge;
        const float d = sqrtf(v[e]) * a.inv_root2 + a.eps;
        p[e] = p[e] * a.decay - a.step_size * m[e] / d;
    }
    if (t.master) store8<F32>(t.master, i, n, al(t.master, 16), p);
    store8<P>(t.param, i, n, vp, p);
    if constexpr (BITS == 32) {
        store8<F32>(t.exp_avg, i, n, vs, m);
        store8<F32>(t.exp_avg_sq, i, n, vs, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (i + e >= n) m[e] = v[e] = 0.0f;  // past the tensor: no part in the block's scale
        const float tm = block_top(m), tv = block_top(v);
        const float im = inverse_scale(tm), iv = inverse_scale(tv);
        uint32_t cm[8], cv[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) cm[e] = encode8<true>(m[e], im), cv[e] = encode8<false>(v[e], iv);
        store_codes((uint8_t*)t.exp_avg, i, n, vs, cm);
        store_codes((uint8_t*)t.exp_avg_sq, i, n, vs, cv);
        if ((lane & 31) == 0 && i < n) {
            t.exp_avg_scale[i / kBlock8] = tm;
            t.exp_avg_sq_scale[i / kBlock8] = tv;
        }
    }
}

template <typename P, typename G>
void launch_adamw(const AdamArgs& a, int bits, unsigned grid, hipStream_t st) {
    if (bits == 8)
        hipLaunchKernelGGL((k_adamw<P, G, 8>), dim3(grid), dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((k_adamw<P, G, 32>), dim3(grid), dim3(256), 0, st, a);
}

template <typename P>
void launch_adamw(const AdamArgs& a, int grad_dtype, int bits, unsigned grid, hipStream_t st) {
    if (grad_dtype == STM_F32)
        launch_adamw<P, F32>(a, bits, grid, st);
    else if (grad_dtype == STM_BF16)
        launch_adamw<P, BF16>(a, bits, grid, st);
    else
        launch_adamw<P, F16>(a, bits, grid, st);
}

// ------------------------------------------------------------ 8-bit states as values
template <bool SIGNED>
__global__ __launch_bounds__(256) void k_state_values(const uint8_t* __restrict__ codes,
                                                      const float* __restrict__ scales, int64_t n,
                                                      float* __restrict__ out, int vec) {
    for (int64_t i = (blockIdx.x * (int64_t)256 + threadIdx.x) * 8; i < n; i += (int64_t)gridDim.x * kTile) {
        uint32_t c[8];
        float f[8];
        load_codes(codes, i, n, vec, c);
        const float s = scales[i / kBlock8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = decode8<SIGNED>(c[e], s);
        store8<F32>(out, i, n, vec, f);
    }
}

template <bool SIGNED>
__global__ __launch_bounds__(256) void k_state_codes(const float* __restrict__ x, int64_t n,
                                                     uint8_t* __restrict__ codes, float* __restrict__ scales,
                                                     int vec) {
    // whole waves stay in the loop together: a block's 32 lanes meet in the reduction
    for (int64_t base = blockIdx.x * (int64_t)kTile; base < n; base += (int64_t)gridDim.x * kTile) {
        const int64_t i = base + threadIdx.x * 8;
        float f[8];
        load8<F32>(x, i, n, vec, f);
        const float top = block_top(f), inv = inverse_scale(top);
        uint32_t c[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) c[e] = encode8<SIGNED>(f[e], inv);
        store_codes(codes, i, n, vec, c);
        if ((threadIdx.x & 31) == 0 && i < n) scales[i / kBlock8] = top;
    }
}

// ------------------------------------------------------------ gradient norm
// Sum of v over the work-group's 256 threads, in a fixed order; valid in thread 0.
__device__ __forceinline__ double group_sum(double v, double* lds) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    return lds[0] + lds[1] + lds[2] + lds[3];
}

// Squares are summed in fp64: exact products of the 16-bit types, no overflow for any
// fp32 gradient, and an order of its own would not show in the fp32 result.
template <typename G>
__global__ __launch_bounds__(256) void k_norm_partial(NormArgs a, double* __restrict__ partial) {
    __shared__ double lds[4];
    const int ti = tensor_of<kNormTensors>(a.first, a.count, (int)blockIdx.x, threadIdx.x & 63);
    const void* g = a.g[ti];
    const int64_t n = a.n[ti], base = ((int64_t)blockIdx.x - a.first[ti]) * kNormTile;
    const bool vec = ((uintptr_t)g & 15) == 0;
    double sum = 0.0;
#pragma unroll 4
    for (int k = 0; k < kNormTile / kTile; ++k) {
        float f[8];
        load8<G>(g, base + k * kTile + threadIdx.x * 8, n, vec, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fma((double)f[e], (double)f[e], sum);
    }
    sum = group_sum(sum, lds);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

__global__ __launch_bounds__(256) void k_norm_final(const double* __restrict__ partial, int64_t count, double max_norm,
                                                    double loss_scale, float* __restrict__ out) {
    __shared__ double lds[4];
    double sum = 0.0;
    for (int64_t i = threadIdx.x; i < count; i += 256) sum += partial[i];
    sum = group_sum(sum, lds);
    if (threadIdx.x == 0) {
        const double norm = sqrt(sum) / loss_scale;
        const double factor = max_norm / (norm + 1e-6);
        out[0] = (float)norm;
        out[1] = norm < (double)INFINITY ? (float)((factor < 1.0 ? factor : 1.0) / loss_scale) : NAN;
    }
}

int64_t norm_groups(int64_t n) { return (n + kNormTile - 1) / kNormTile; }

bool valid_dtype(int dt) { return dt == STM_F16 || dt == STM_BF16 || dt == STM_F32; }

}  // namespace
}  // namespace stm

using namespace stm;

extern "C" int stm_adamw_step(int count, const stm_adamw_tensor* tensors, int param_dtype, int grad_dtype,
                              int state_bits, double lr, double beta1, double beta2, double eps, double weight_decay,
                              int64_t step, const float* grad_scale, void* stream) {
    if (count < 0 || (count && !tensors)) return set_error(STM_ERR_INVALID, "adamw_step: bad tensor list");
    if (!valid_dtype(param_dtype) || !valid_dtype(grad_dtype))
        return set_error(STM_ERR_INVALID, "adamw_step: unknown dtype");
    if (state_bits != 8 && state_bits != 32)
        return set_error(STM_ERR_INVALID, "adamw_step: states have 8 or 32 bits, got %d", state_bits);
    if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0))
        return set_error(STM_ERR_INVALID, "adamw_step: betas must lie in [0, 1)");
    if (step < 1) return set_error(STM_ERR_INVALID, "adamw_step: the first step is step 1");
    for (int i = 0; i < count; ++i) {
        const stm_adamw_tensor& t = tensors[i];
        if (t.n < 0) return set_error(STM_ERR_INVALID, "adamw_step: tensor %d has a negative size", i);
        if (t.n == 0) continue;
        if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq ||
            (state_bits == 8 && (!t.exp_avg_scale || !t.exp_avg_sq_scale)))
            return set_error(STM_ERR_INVALID, "adamw_step: tensor %d has a null pointer", i);
        const uintptr_t pa = param_dtype == STM_F32 ? 4 : 2, ga = grad_dtype == STM_F32 ? 4 : 2;
        const uintptr_t sa = state_bits == 32 ? 4 : 1;
        if (!aligned(t.param, pa) || !aligned(t.grad, ga) || !aligned(t.master, 4) || !aligned(t.exp_avg, sa) ||
            !aligned(t.exp_avg_sq, sa) || !aligned(t.exp_avg_scale, 4) || !aligned(t.exp_avg_sq_scale, 4))
            return set_error(STM_ERR_INVALID, "adamw_step: tensor %d is not aligned to its elements", i);
        if ((t.n + kTile - 1) / kTile > 0x3FFFFFFF)
            return set_error(STM_ERR_UNSUPPORTED, "adamw_step: tensor %d is too large", i);
    }
    AdamArgs a;
    a.beta1 = (float)beta1;
    a.beta2 = (float)beta2;
    a.rest1 = (float)(1.0 - beta1);
    a.rest2 = (float)(1.0 - beta2);
    a.decay = (float)(1.0 - lr * weight_decay);
    a.step_size = (float)(lr / (1.0 - pow(beta1, (double)step)));
    a.inv_root2 = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)step)));
    a.eps = (float)eps;
    a.scale = grad_scale;
    for (int i = 0; i < count;) {
        a.count = 0;
        int64_t groups = 0;
        while (i < count && a.count < kAdamTensors) {
            const int64_t g = (tensors[i].n + kTile - 1) / kTile;
            if (groups + g > 0x3FFFFFFF) break;
            if (g) {
                a.t[a.count] = tensors[i];
                a.first[a.count++] = (int)groups;
                groups += g;
            }
            ++i;
        }
        if (!groups) continue;
        if (param_dtype == STM_F32)
            launch_adamw<F32>(a, grad_dtype, state_bits, (unsigned)groups, (hipStream_t)stream);
        else if (param_dtype == STM_BF16)
            launch_adamw<BF16>(a, grad_dtype, state_bits, (unsigned)groups, (hipStream_t)stream);
        else
            launch_adamw<F16>(a, grad_dtype, state_bits, (unsigned)groups, (hipStream_t)stream);
        const int rc = check_launch("adamw_step");
        if (rc) return rc;
    }
    return STM_OK;
}

extern "C" int stm_state8_values(const uint8_t* codes, const float* scales, int64_t n, int is_signed, float* out,
                                 void* stream) {
    if (n < 0) return set_error(STM_ERR_INVALID, "state8_values: negative size");
    if (n == 0) return STM_OK;
    if (!codes || !scales || !out) return set_error(STM_ERR_INVALID, "state8_values: null pointer");
    if (!aligned(scales, 4) || !aligned(out, 4)) return set_error(STM_ERR_INVALID, "state8_values: unaligned fp32");
    const int vec = aligned(codes, 8) && aligned(out, 16);
    const int64_t tiles = (n + kTile - 1) / kTile;
    const dim3 grid((unsigned)(tiles < 65536 ? tiles : 65536));
    if (is_signed)
        hipLaunchKernelGGL(k_state_values<true>, grid, dim3(256), 0, (hipStream_t)stream, codes, scales, n, out, vec);
    else
        hipLaunchKernelGGL(k_state_values<false>, grid, dim3(256), 0, (hipStream_t)stream, codes, scales, n, out, vec);
    return check_launch("state8_values");
}

extern "C" int stm_state8_codes(const float* x, int64_t n, int is_signed, uint8_t* codes, float* scales,
                                void* stream) {
    if (n < 0) return set_error(STM_ERR_INVALID, "state8_codes: negative size");
    if (n == 0) return STM_OK;
    if (!codes || !scales || !x) return set_error(STM_ERR_INVALID, "state8_codes: null pointer");
    if (!aligned(scales, 4) || !aligned(x, 4)) return set_error(STM_ERR_INVALID, "state8_codes: unaligned fp32");
    const int vec = aligned(codes, 8) && aligned(x, 16);
    const int64_t tiles = (n + kTile - 1) / kTile;
    const dim3 grid((unsigned)(tiles < 65536 ? tiles : 65536));
    if (is_signed)
        hipLaunchKernelGGL(k_state_codes<true>, grid, dim3(256), 0, (hipStream_t)stream, x, n, codes, scales, vec);
    else
        hipLaunchKernelGGL(k_state_codes<false>, grid, dim3(256), 0, (hipStream_t)stream, x, n, codes, scales, vec);
    return check_launch("state8_codes");
}

extern "C" int64_t stm_grad_norm_workspace_bytes(int count, const int64_t* n) {
    if (count < 0 || (count && !n)) return set_error(STM_ERR_INVALID, "grad_norm: bad tensor list");
    int64_t groups = 0;
    for (int i = 0; i < count; ++i) {
        if (n[i] < 0) return set_error(STM_ERR_INVALID, "grad_norm: tensor %d has a negative size", i);
        groups += norm_groups(n[i]);
    }
    return groups * 8;
}

extern "C" int stm_grad_norm(int count, const void* const* grads, const int64_t* n, int dtype, double max_norm,
                             double loss_scale, float* out, void* workspace, int64_t workspace_bytes, void* stream) {
    const int64_t need = stm_grad_norm_workspace_bytes(count, n);
    if (need < 0) return (int)need;
    if (count && !grads) return set_error(STM_ERR_INVALID, "grad_norm: bad tensor list");
    if (!valid_dtype(dtype)) return set_error(STM_ERR_INVALID, "grad_norm: unknown dtype");
    if (!out || !aligned(out, 4)) return set_error(STM_ERR_INVALID, "grad_norm: out must be two floats");
    if (!(max_norm >= 0.0) || !(loss_scale > 0.0 && loss_scale < (double)INFINITY))
        return set_error(STM_ERR_INVALID, "grad_norm: max_norm must not be negative, loss_scale positive and finite");
    if (need && (!workspace || !aligned(workspace, 8) || workspace_bytes < need))
        return set_error(STM_ERR_INVALID, "grad_norm: the workspace needs %lld bytes", (long long)need);
    for (int i = 0; i < count; ++i) {
        if (n[i] == 0) continue;
        if (!grads[i] || !aligned(grads[i], dtype == STM_F32 ? 4 : 2))
            return set_error(STM_ERR_INVALID, "grad_norm: tensor %d is null or not aligned to its elements", i);
        if (norm_groups(n[i]) > 0x3FFFFFFF) return set_error(STM_ERR_UNSUPPORTED, "grad_norm: tensor %d is too large", i);
    }
    double* partial = (double*)workspace;
    NormArgs a;
    for (int i = 0; i < count;) {
        a.count = 0;
        int64_t groups = 0;
        while (i < count && a.count < kNormTensors) {
            const int64_t g = norm_groups(n[i]);
            if (groups + g > 0x3FFFFFFF) break;
            if (g) {
                a.g[a.count] = grads[i];
                a.n[a.count] = n[i];
                a.first[a.count++] = (int)groups;
                groups += g;
            }
            ++i;
        }
        if (!groups) continue;
        const dim3 grid((unsigned)groups), block(256);
        if (dtype == STM_F32)
            hipLaunchKernelGGL(k_norm_partial<F32>, grid, block, 0, (hipStream_t)stream, a, partial);
        else if (dtype == STM_BF16)
            hipLaunchKernelGGL(k_norm_partial<BF16>, grid, block, 0, (hipStream_t)stream, a, partial);
        else
            hipLaunchKernelGGL(k_norm_partial<F16>, grid, block, 0, (hipStream_t)stream, a, partial);
        const int rc = check_launch("grad_norm");
        if (rc) return rc;
        partial += groups;
    }
    hipLaunchKernelGGL(k_norm_final, dim3(1), dim3(256), 0, (hipStream_t)stream, (const double*)workspace, need / 8,
                       max_norm, loss_scale, out);
    return check_launch("grad_norm");
}
