// What a training step does to its gradients and parameters (gfx950): the norm
// of all gradients, and one AdamW step over all tensors, each in few launches.
//
//   norm      out[0] = |g| / c, out[1] = min(1, max_norm / (out[0] + 1e-6)) / c, c the loss scale;
//             out[1] = NaN where out[0] is not finite
//   AdamW     g' = scale g;  m = b1 m + (1 - b1) g';  v = b2 v + (1 - b2) g' g'
//             p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//             and nothing at all where scale is not finite
//
// Both are bound by HBM: the norm reads every gradient once; a step reads p, g, m
// and v and writes p, m and v (with 8-bit states some 90 vector instructions an element are as
// much: 176 M bf16 elements 377 us, their 1.77 GB 328). All arithmetic is fp32 in the order above, one rounding
// each (no contraction), so that a plain evaluation gives the same states bit for bit.
//
// Tensors travel as kernel arguments (pointers and sizes, one launch for up to
// kAdamTensors / kNormTensors of them), those of a long AdamW list in a table in device
// memory; a work-group finds its tensor by a search in the prefix sums of work-groups.
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
#include <type_traits>

#include "nf4_common.h"

namespace stm {
namespace {

constexpr int kBlock8 = 256;      // elements per scale of an 8-bit state
constexpr int kAdamTensors = 56;  // tensors per launch (below 4 KB of kernel arguments)
constexpr int kNormTensors = 254;
// Rows of 256 elements per wave: with one, a 32-bit step of 42 M elements takes 219 us, with two
// 227, with four 240 (four accesses of a lane stand between a row's loads and its stores); an
// 8-bit step of 176 M 394, 377 and 388 (two rows share a division).
constexpr int rows_of(int bits) { return bits == 8 ? 2 : 1; }
constexpr int tile_of(int bits) { return 4 * rows_of(bits) * kBlock8; }  // elements per work-group
constexpr int kRows = rows_of(8), kTile = tile_of(8);                    // of the conversions
constexpr int kNormThreads = 512, kNormTile = 16384;  // elements per work-group of the norm

struct AdamNumbers {
    float beta1, beta2, rest1, rest2;  // rest = 1 - beta
    float decay, step_size, inv_root2, eps;
    const float* scale;
};

// Up to kAdamTensors tensors in the kernel's arguments,
struct AdamArgs {
    stm_adamw_tensor t[kAdamTensors];
    int first[kAdamTensors];  // first work-group of tensor i
    int count;
    AdamNumbers h;
};
static_assert(sizeof(AdamArgs) <= 4096, "kernel arguments");

// or any number in a table in device memory: `count` tensors, then their first work-groups.
struct AdamTable {
    const stm_adamw_tensor* t;
    const int* first;
    int count;
    AdamNumbers h;
};

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct NormArgs {
    const void* g[kNormTensors];
    int first[kNormTensors + 1];  // first work-group of tensor i; of `count`: all of them
    int last[kNormTensors];       // elements of tensor i's last work-group
    int count;
};
static_assert(sizeof(NormArgs) <= 4096, "kernel arguments");

// The tensor that work-group b belongs to: the last one whose first work-group is at or
// before b. Every read is uniform (scalar loads of the kernel arguments).
__device__ __forceinline__ int tensor_of(const int* first, int count, int b) {
    int lo = 0, hi = count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (first[mid] <= b)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

// ------------------------------------------------------------ element access
struct F32 {
    static constexpr int tag = STM_F32;
};

// Four elements at i of a tensor of n; `vec`: the base is aligned for one access.
template <typename T>
__device__ __forceinline__ void load4(const void* base, int64_t i, int64_t n, bool vec, float (&f)[4]) {
    if constexpr (T::tag == STM_F32) {
        const float* p = reinterpret_cast<const float*>(base) + i;
        if (vec && i + 4 <= n) {
            const float4 a = *reinterpret_cast<const float4*>(p);
            f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] = i + e < n ? p[e] : 0.0f;
        }
    } else {
        const uint16_t* p = reinterpret_cast<const uint16_t*>(base) + i;
        if (vec && i + 4 <= n) {
            const uint2 v = *reinterpret_cast<const uint2*>(p);
            f[0] = T::to_f32((uint16_t)(v.x & 0xFFFFu)), f[1] = T::to_f32((uint16_t)(v.x >> 16));
            f[2] = T::to_f32((uint16_t)(v.y & 0xFFFFu)), f[3] = T::to_f32((uint16_t)(v.y >> 16));
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] = i + e < n ? T::to_f32(p[e]) : 0.0f;
        }
    }
}

template <typename T>
__device__ __forceinline__ void store4(void* base, int64_t i, int64_t n, bool vec, const float (&f)[4]) {
    if constexpr (T::tag == STM_F32) {
        float* p = reinterpret_cast<float*>(base) + i;
        if (vec && i + 4 <= n) {
            *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i + e < n) p[e] = f[e];
        }
    } else {
        uint16_t* p = reinterpret_cast<uint16_t*>(base) + i;
        if (vec && i + 4 <= n) {
            *reinterpret_cast<uint2*>(p) = make_uint2(T::pack2(f[0], f[1]), T::pack2(f[2], f[3]));
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i + e < n) p[e] = T::from_f32(f[e]);
        }
    }
}

// x as the type holds it.
template <typename T>
__device__ __forceinline__ float rounded(float x) {
    if constexpr (T::tag == STM_F32)
        return x;
    else
        return T::to_f32(T::from_f32(x));
}

// Four codes in a word, element 0 in the low byte.
__device__ __forceinline__ uint32_t load_codes(const uint8_t* base, int64_t i, int64_t n, bool vec) {
    const uint8_t* p = base + i;
    if (vec && i + 4 <= n) return *reinterpret_cast<const uint32_t*>(p);
    uint32_t c = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) c |= i + e < n ? (uint32_t)p[e] << (8 * e) : 0u;
    return c;
}

__device__ __forceinline__ void store_codes(uint8_t* base, int64_t i, int64_t n, bool vec, uint32_t c) {
    uint8_t* p = base + i;
    if (vec && i + 4 <= n) {
        *reinterpret_cast<uint32_t*>(p) = c;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (i + e < n) p[e] = (uint8_t)(c >> (8 * e));
    }
}

// ------------------------------------------------------------ the 8-bit code
// Value of magnitude q, given as a float: exact up to the product with the scale.
template <int K>
__device__ __forceinline__ float level8(float q) {
    const float top = __uint_as_float(__float_as_uint(q) & 0xFF800000u);  // 2^k, 0 for q = 0
    const float a = fmaf(top, -6.0f, fmaf(q, 7.0f, 7.0f));
    return a * top * (top * __uint_as_float((uint32_t)(127 - 3 - 3 * K) << 23));
}

// Values of the four codes of a word.
template <bool SIGNED>
__device__ __forceinline__ void decode4(uint32_t c, float scale, float (&f)[4]) {
    const uint32_t q = SIGNED ? c & 0x7F7F7F7Fu : c;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float v = level8<SIGNED ? 6 : 7>((float)((q >> (8 * e)) & 255u)) * scale;
        f[e] = SIGNED ? __uint_as_float(__float_as_uint(v) ^ ((c << (24 - 8 * e)) & 0x80000000u)) : v;
    }
}

// 1 / scale, or 0 for a block whose scale has no finite reciprocal that is normal
// (zero, subnormal, infinite, NaN): its codes are zero (v: the lowest level).
__device__ __forceinline__ float inverse_scale(float top) { return top >= 0x1p-126f ? 1.0f / top : 0.0f; }

// Code of x in a block with that inverse scale. With s = |x| inv in segment z (8^-(z+1) <= s <
// 8^-z; z = K: everything below), n = 2^(K-z) and c = 8/7 n, the step above the segment's
// lower end is j = rint((8^z s - 1/8) c). The difference is exact in fp32, so one fma of s with
// 8^z c and -c/8 gives the product rounded once, as the formula does; the rounding to a
// whole number is that of adding 1.5 * 2^23. In the last segment j = rint(8^K s).
template <bool SIGNED>
__device__ __forceinline__ uint32_t encode8(float x, float inv) {
    constexpr int K = SIGNED ? 6 : 7;
    constexpr uint32_t kC = 0x3F924925u, kMagic = 0x4B400000u;  // 8/7; 1.5 * 2^23
    const float s = fminf(fabsf(x) * inv, 1.0f);  // 1 also for an infinite x (inv is 0)
    // z from the biased exponent E: floor((126 - E) / 3), in [0, K]
    const int E = (int)(__float_as_uint(s) >> 23);
    int z = (126 * 43 - 43 * E) >> 7;  // exact for 0 <= 126 - E <= 126
    z = z < 0 ? 0 : z;
    const bool last = z >= K;
    z = last ? K : z;
    const float mul = __uint_as_float(last ? (uint32_t)(127 + 3 * K) << 23 : kC + ((uint32_t)(2 * z + K) << 23));
    const float sub = last ? 0.0f : __uint_as_float(kC + ((uint32_t)(K - 3 - z) << 23));
    const uint32_t j = __float_as_uint(fmaf(s, mul, -sub) + 12582912.0f);
    const uint32_t q = j + (((1u << K) >> z) - 1u - kMagic);
    if constexpr (SIGNED) return q | ((__float_as_uint(x) >> 24) & 128u);
    const uint32_t some = __float_as_uint(x) < 1u ? 0u : 1u;
    return q > some ? q : some;
}

// The largest magnitude of a wave's 256 elements, the same in every lane. Compared as
// integers: the order of non-negative floats, with NaN above everything.
__device__ __forceinline__ float block_top(const float (&f)[4]) {
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t b = __float_as_uint(f[e]) & 0x7FFFFFFFu;
        top = top > b ? top : b;
    }
    auto step = [&](auto ctrl) {  // the maximum with another lane's, zero where there is none
        const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, decltype(ctrl)::value, 0xF, 0xF, false);
        top = top > o ? top : o;
    };
    step(std::integral_constant<int, 0x111>());  // row_shr 1, 2, 4, 8: lane 15 of every row of 16 has its row's
    step(std::integral_constant<int, 0x112>());
    step(std::integral_constant<int, 0x114>());
    step(std::integral_constant<int, 0x118>());
    step(std::integral_constant<int, 0x142>());  // row_bcast 15, 31: lane 63 has the wave's
    step(std::integral_constant<int, 0x143>());
    return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)top, 63));
}

template <bool SIGNED>
__device__ __forceinline__ uint32_t encode4(const float (&f)[4], float inv) {
    uint32_t c = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) c |= encode8<SIGNED>(f[e], inv) << (8 * e);
    return c;
}

// ------------------------------------------------------------ AdamW
// A work-group takes kTile consecutive elements of one tensor: wave w, kRows rows of 256
// elements, four a lane, so that every access of a wave is one contiguous piece and a row is a
// block of an 8-bit state. All loads are issued before the first result is needed.
//
// FULL: the tile lies inside its tensor and every base is aligned for whole accesses; then no
// access has a test of its own (8-bit states of 176 M elements: 400 -> 377 us).
//
// FOLLOW: an element of the parameter that is not its master rounded was written by something
// else since the last step, and replaces the master. No other trace of such a write is certain (a
// tensor's version counts no write through .data), so the parameter is read as well: 42 M bf16 elements
// with masters 240 -> 255 us, with 8-bit states 145 -> 162.
template <typename P, typename G, int BITS, bool FOLLOW, bool FULL>
__device__ __forceinline__ void adamw_tile(const AdamNumbers& a, const stm_adamw_tensor& t, int64_t base, int lane,
                                           float scale, bool vp, bool vg, bool vs, bool vm) {
    constexpr int kRows = rows_of(BITS);
    const int64_t n = FULL ? INT64_MAX : t.n;
    float p[kRows][4], g[kRows][4], m[kRows][4], v[kRows][4];
    [[maybe_unused]] float held[kRows][4];  // FOLLOW: the parameter beside its master
    [[maybe_unused]] uint32_t cm[kRows], cv[kRows];
    [[maybe_unused]] float sm[kRows], sv[kRows], tops[2 * kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        const int64_t i = base + r * kBlock8;
        load4<G>(t.grad, i, n, vg, g[r]);
        if (t.master)
            load4<F32>(t.master, i, n, vm, p[r]);
        else
            load4<P>(t.param, i, n, vp, p[r]);
        if constexpr (FOLLOW) load4<P>(t.param, i, n, vp, held[r]);
        if constexpr (BITS == 32) {
            load4<F32>(t.exp_avg, i, n, vs, m[r]);
            load4<F32>(t.exp_avg_sq, i, n, vs, v[r]);
        } else {
            cm[r] = load_codes((const uint8_t*)t.exp_avg, i, n, vs);
            cv[r] = load_codes((const uint8_t*)t.exp_avg_sq, i, n, vs);
            sm[r] = FULL || i < n ? t.exp_avg_scale[i / kBlock8] : 0.0f;
            sv[r] = FULL || i < n ? t.exp_avg_sq_scale[i / kBlock8] : 0.0f;
        }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        const int64_t i = base + r * kBlock8;
        if constexpr (BITS == 8) {
            decode4<true>(cm[r], sm[r], m[r]);
            decode4<false>(cv[r], sv[r], v[r]);
        }
        if constexpr (FOLLOW) {
#pragma unroll
            for (int e = 0; e < 4; ++e) p[r][e] = rounded<P>(p[r][e]) == held[r][e] ? p[r][e] : held[r][e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float ge = g[r][e] * scale;
            m[r][e] = m[r][e] * a.beta1 + ge * a.rest1;
            v[r][e] = v[r][e] * a.beta2 + ge * a.rest2 * ge;
            // the update's root and reciprocal are the instructions' (one ulp each): it is added to p,
            // where its last bits do not count, and neither state depends on it
            const float d = __builtin_amdgcn_sqrtf(v[r][e]) * a.inv_root2 + a.eps;
            p[r][e] = p[r][e] * a.decay - a.step_size * m[r][e] * __builtin_amdgcn_rcpf(d);
        }
        if (t.master) store4<F32>(t.master, i, n, vm, p[r]);
        store4<P>(t.param, i, n, vp, p[r]);
        if constexpr (BITS == 32) {
            store4<F32>(t.exp_avg, i, n, vs, m[r]);
            store4<F32>(t.exp_avg_sq, i, n, vs, v[r]);
        } else {
            if (!FULL && i + 4 > n) {  // past the tensor: no part in the block's scale
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (i + e >= n) m[r][e] = v[r][e] = 0.0f;
            }
            tops[2 * r] = block_top(m[r]);
            tops[2 * r + 1] = block_top(v[r]);
        }
    }
    if constexpr (BITS == 8) {
        // one division for the wave's scales: lane i inverts number i
        float mine = tops[0];
#pragma unroll
        for (int k = 1; k < 2 * kRows; ++k) mine = lane == k ? tops[k] : mine;
        const int inverse = (int)__float_as_uint(inverse_scale(mine));
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const int64_t i = base + r * kBlock8;
            const float im = __uint_as_float((uint32_t)__builtin_amdgcn_readlane(inverse, 2 * r));
            const float iv = __uint_as_float((uint32_t)__builtin_amdgcn_readlane(inverse, 2 * r + 1));
            store_codes((uint8_t*)t.exp_avg, i, n, vs, encode4<true>(m[r], im));
            store_codes((uint8_t*)t.exp_avg_sq, i, n, vs, encode4<false>(v[r], iv));
            if (lane == 0 && (FULL || i < n)) {
                t.exp_avg_scale[i / kBlock8] = tops[2 * r];
                t.exp_avg_sq_scale[i / kBlock8] = tops[2 * r + 1];
            }
        }
    }
}

template <typename P, typename G, int BITS, bool FOLLOW, typename Args>
__global__ __launch_bounds__(256) void k_adamw(Args args) {
    const AdamNumbers& a = args.h;
    float scale = 1.0f;
    if (a.scale) {
        scale = *a.scale;
        if (!(fabsf(scale) < INFINITY)) return;  // the whole launch alike
    }
    const int lane = threadIdx.x & 63;
    const int ti = tensor_of(args.first, args.count, (int)blockIdx.x);
    const stm_adamw_tensor t = args.t[ti];
    const int64_t tile = ((int64_t)blockIdx.x - args.first[ti]) * tile_of(BITS);
    const int64_t base = tile + (threadIdx.x >> 6) * (rows_of(BITS) * kBlock8) + lane * 4;
    auto al = [](const void* p, uintptr_t b) { return ((uintptr_t)p & (b - 1)) == 0; };
    const bool vp = al(t.param, P::tag == STM_F32 ? 16 : 8), vg = al(t.grad, G::tag == STM_F32 ? 16 : 8);
    const bool vs = al(t.exp_avg, BITS == 8 ? 4 : 16) && al(t.exp_avg_sq, BITS == 8 ? 4 : 16), vm = al(t.master, 16);
    if (vp && vg && vs && vm && tile + tile_of(BITS) <= t.n)
        adamw_tile<P, G, BITS, FOLLOW, true>(a, t, base, lane, scale, true, true, true, true);
    else
        adamw_tile<P, G, BITS, FOLLOW, false>(a, t, base, lane, scale, vp, vg, vs, vm);
}

// How a step is asked for: its types, the bits of a state, and whether masters follow their parameters.
struct AdamKind {
    int param_dtype, grad_dtype, bits;
    bool follow;
};

template <typename P, typename G, typename Args>
void launch_adamw(const Args& a, const AdamKind& k, unsigned grid, hipStream_t st) {
    const dim3 block(256);
    if (k.bits == 8 && k.follow)
        hipLaunchKernelGGL((k_adamw<P, G, 8, true, Args>), dim3(grid), block, 0, st, a);
    else if (k.bits == 8)
        hipLaunchKernelGGL((k_adamw<P, G, 8, false, Args>), dim3(grid), block, 0, st, a);
    else if (k.follow)
        hipLaunchKernelGGL((k_adamw<P, G, 32, true, Args>), dim3(grid), block, 0, st, a);
    else
        hipLaunchKernelGGL((k_adamw<P, G, 32, false, Args>), dim3(grid), block, 0, st, a);
}

template <typename P, typename Args>
void launch_adamw(const Args& a, const AdamKind& k, unsigned grid, hipStream_t st) {
    if (k.grad_dtype == STM_F32)
        launch_adamw<P, F32>(a, k, grid, st);
    else if (k.grad_dtype == STM_BF16)
        launch_adamw<P, BF16>(a, k, grid, st);
    else
        launch_adamw<P, F16>(a, k, grid, st);
}

template <typename Args>
int launch_adamw(const Args& a, const AdamKind& k, int64_t grid, hipStream_t st) {
    if (k.param_dtype == STM_F32)
        launch_adamw<F32>(a, k, (unsigned)grid, st);
    else if (k.param_dtype == STM_BF16)
        launch_adamw<BF16>(a, k, (unsigned)grid, st);
    else
        launch_adamw<F16>(a, k, (unsigned)grid, st);
    return check_launch("adamw_step");
}

// ------------------------------------------------------------ 8-bit states as values
template <bool SIGNED>
__global__ __launch_bounds__(256) void k_state_values(const uint8_t* __restrict__ codes,
                                                      const float* __restrict__ scales, int64_t n,
                                                      float* __restrict__ out, int vec) {
    const int lane = threadIdx.x & 63;
    const int64_t base = (int64_t)blockIdx.x * kTile + (threadIdx.x >> 6) * (kRows * kBlock8) + lane * 4;
    uint32_t c[kRows];
    float s[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        const int64_t i = base + r * kBlock8;
        c[r] = load_codes(codes, i, n, vec);
        s[r] = i < n ? scales[i / kBlock8] : 0.0f;
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        float f[4];
        decode4<SIGNED>(c[r], s[r], f);
        store4<F32>(out, base + r * kBlock8, n, vec, f);
    }
}

template <bool SIGNED>
__global__ __launch_bounds__(256) void k_state_codes(const float* __restrict__ x, int64_t n,
                                                     uint8_t* __restrict__ codes, float* __restrict__ scales,
                                                     int vec) {
    const int lane = threadIdx.x & 63;
    const int64_t base = (int64_t)blockIdx.x * kTile + (threadIdx.x >> 6) * (kRows * kBlock8) + lane * 4;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        const int64_t i = base + r * kBlock8;
        float f[4];
        load4<F32>(x, i, n, vec, f);
        const float top = block_top(f);
        store_codes(codes, i, n, vec, encode4<SIGNED>(f, inverse_scale(top)));
        if (lane == 0 && i < n) scales[i / kBlock8] = top;
    }
}

// ------------------------------------------------------------ gradient norm
// Sum of v over the work-group's threads, in a fixed order.
template <int THREADS>
__device__ __forceinline__ double group_sum(double v, double (&lds)[THREADS / 64]) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int i = 1; i < THREADS / 64; ++i) v += lds[i];
    return v;
}

// Squares are summed in fp64: exact products of the 16-bit types, no overflow for any
// fp32 gradient, and an order of its own would not show in the fp32 result.
//
// A whole tile of an aligned tensor is asked for at once, 16 bytes a lane and load; the last
// tile of a tensor, and tensors that start between, four elements at a time with bounds.
// 84 M elements in bf16 (168 MB, 448 tensors): 38.5 us where four elements a load took 52;
// 168 M in fp32 120 us (5.6 TB/s), against 133. (256 threads: the same.)
template <typename G>
__global__ __launch_bounds__(kNormThreads) void k_norm_partial(NormArgs a, double* __restrict__ partial) {
    __shared__ double lds[kNormThreads / 64];
    const int ti = tensor_of(a.first, a.count, (int)blockIdx.x);
    const void* g = a.g[ti];
    const int64_t base = ((int64_t)blockIdx.x - a.first[ti]) * kNormTile;
    const int64_t n = (int64_t)(a.first[ti + 1] - a.first[ti] - 1) * kNormTile + a.last[ti];
    double sum = 0.0;
    auto add = [&](float f) { sum = fma((double)f, (double)f, sum); };
    if (((uintptr_t)g & 15) == 0 && base + kNormTile <= n) {
        constexpr int kBytes = G::tag == STM_F32 ? 4 : 2, kLoads = kNormTile * kBytes / (16 * kNormThreads);
        const u32x4* src = reinterpret_cast<const u32x4*>(reinterpret_cast<const uint8_t*>(g) + base * kBytes);
        u32x4 raw[kLoads];
#pragma unroll
        for (int j = 0; j < kLoads; ++j) raw[j] = src[j * kNormThreads + threadIdx.x];
#pragma unroll
        for (int j = 0; j < kLoads; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t word = raw[j][e];
                if constexpr (G::tag == STM_F32) {
                    add(__uint_as_float(word));
                } else {
                    add(G::to_f32((uint16_t)(word & 0xFFFFu)));
                    add(G::to_f32((uint16_t)(word >> 16)));
                }
            }
    } else {
        const bool vec = ((uintptr_t)g & (G::tag == STM_F32 ? 15 : 7)) == 0;
#pragma unroll 4
        for (int j = 0; j < kNormTile; j += 4 * kNormThreads) {
            float f[4];
            load4<G>(g, base + j + threadIdx.x * 4, n, vec, f);
#pragma unroll
            for (int e = 0; e < 4; ++e) add(f[e]);
        }
    }
    sum = group_sum<kNormThreads>(sum, lds);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// One work-group with eight loads a thread in flight: the 5 120 partial sums of 84 M elements.
constexpr int kFinalThreads = 1024;
__global__ __launch_bounds__(kFinalThreads) void k_norm_final(const double* __restrict__ partial, int64_t count,
                                                              double max_norm, double loss_scale,
                                                              float* __restrict__ out) {
    __shared__ double lds[kFinalThreads / 64];
    double sum = 0.0;
    for (int64_t i = threadIdx.x; i < count; i += 8 * kFinalThreads) {  // eight loads in flight
        double v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = i + j * kFinalThreads < count ? partial[i + j * kFinalThreads] : 0.0;
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += v[j];
    }
    sum = group_sum<kFinalThreads>(sum, lds);
    if (threadIdx.x == 0) {
        const double norm = sqrt(sum) / loss_scale;
        const double factor = max_norm / (norm + 1e-6);
        out[0] = (float)norm;  // as it is returned: infinite also where only fp32 ends
        out[1] = out[0] < INFINITY ? (float)((factor < 1.0 ? factor : 1.0) / loss_scale) : NAN;
    }
}

int64_t norm_groups(int64_t n) { return (n + kNormTile - 1) / kNormTile; }

bool valid_dtype(int dt) { return dt == STM_F16 || dt == STM_BF16 || dt == STM_F32; }

}  // namespace
}  // namespace stm

using namespace stm;

// Work-groups of a launch: HIP takes fewer than 2^32 threads. What needs more goes in several launches.
constexpr int64_t most_groups(int threads) { return ((int64_t)1 << 32) / threads - 1; }
constexpr int64_t kMostGroups = most_groups(256);  // of a step and of the conversions
constexpr int64_t kMostElements = (int64_t)1 << 48;

static int adamw_kind(int param_dtype, int grad_dtype, int state_bits, AdamKind& k) {
    if (!valid_dtype(param_dtype) || !valid_dtype(grad_dtype))
        return set_error(STM_ERR_INVALID, "adamw_step: unknown dtype");
    k = {param_dtype, grad_dtype, state_bits & ~STM_ADAMW_FOLLOW, (state_bits & STM_ADAMW_FOLLOW) != 0};
    if (k.bits != 8 && k.bits != 32)
        return set_error(STM_ERR_INVALID, "adamw_step: states have 8 or 32 bits, got %d", k.bits);
    return STM_OK;
}

static int check_adamw_tensors(int count, const stm_adamw_tensor* tensors, const AdamKind& k) {
    if (count < 0 || (count && !tensors)) return set_error(STM_ERR_INVALID, "adamw_step: bad tensor list");
    for (int i = 0; i < count; ++i) {
        const stm_adamw_tensor& t = tensors[i];
        if (t.n < 0) return set_error(STM_ERR_INVALID, "adamw_step: tensor %d has a negative size", i);
        if (t.n == 0) continue;
        if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq ||
            (k.bits == 8 && (!t.exp_avg_scale || !t.exp_avg_sq_scale)))
            return set_error(STM_ERR_INVALID, "adamw_step: tensor %d has a null pointer", i);
        const uintptr_t pa = k.param_dtype == STM_F32 ? 4 : 2, ga = k.grad_dtype == STM_F32 ? 4 : 2;
        const uintptr_t sa = k.bits == 32 ? 4 : 1;
        if (!aligned(t.param, pa) || !aligned(t.grad, ga) || !aligned(t.master, 4) || !aligned(t.exp_avg, sa) ||
            !aligned(t.exp_avg_sq, sa) || !aligned(t.exp_avg_scale, 4) || !aligned(t.exp_avg_sq_scale, 4))
            return set_error(STM_ERR_INVALID, "adamw_step: tensor %d is not aligned to its elements", i);
        if (t.n > kMostElements)
            return set_error(STM_ERR_UNSUPPORTED, "adamw_step: tensor %d is too large", i);
    }
    return STM_OK;
}

static int adamw_numbers(double lr, double beta1, double beta2, double eps, double weight_decay, int64_t step,
                         const float* grad_scale, AdamNumbers& h) {
    if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0))
        return set_error(STM_ERR_INVALID, "adamw_step: betas must lie in [0, 1)");
    if (step < 1) return set_error(STM_ERR_INVALID, "adamw_step: the first step is step 1");
    h.beta1 = (float)beta1;
    h.beta2 = (float)beta2;
    h.rest1 = (float)(1.0 - beta1);
    h.rest2 = (float)(1.0 - beta2);
    h.decay = (float)(1.0 - lr * weight_decay);
    h.step_size = (float)(lr / (1.0 - pow(beta1, (double)step)));
    h.inv_root2 = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)step)));
    h.eps = (float)eps;
    h.scale = grad_scale;
    return STM_OK;
}

// Elements [start, start + n) of a tensor, start a multiple of a tile's elements.
static stm_adamw_tensor piece_of(const stm_adamw_tensor& t, int64_t start, int64_t n, const AdamKind& k) {
    auto at = [&](const void* p, int bytes) { return (void*)((uintptr_t)p + (uintptr_t)(start * bytes)); };
    auto floats = [&](float* p, int64_t i) { return p ? p + i : nullptr; };
    const int state = k.bits == 32 ? 4 : 1;
    return {at(t.param, k.param_dtype == STM_F32 ? 4 : 2), at(t.grad, k.grad_dtype == STM_F32 ? 4 : 2),
            floats(t.master, start), at(t.exp_avg, state), at(t.exp_avg_sq, state),
            floats(t.exp_avg_scale, start / kBlock8), floats(t.exp_avg_sq_scale, start / kBlock8), n};
}

extern "C" int stm_adamw_step(int count, const stm_adamw_tensor* tensors, int param_dtype, int grad_dtype,
                              int state_bits, double lr, double beta1, double beta2, double eps, double weight_decay,
                              int64_t step, const float* grad_scale, void* stream) {
    AdamArgs a;
    AdamKind k;
    int rc = adamw_kind(param_dtype, grad_dtype, state_bits, k);
    if (rc == STM_OK) rc = adamw_numbers(lr, beta1, beta2, eps, weight_decay, step, grad_scale, a.h);
    if (rc == STM_OK) rc = check_adamw_tensors(count, tensors, k);
    if (rc != STM_OK) return rc;
    const int64_t tile = tile_of(k.bits);
    int64_t done = 0;  // tiles of tensor i that earlier launches hold
    for (int i = 0; i < count;) {
        a.count = 0;
        int64_t groups = 0;
        while (i < count && a.count < kAdamTensors && groups < kMostGroups) {
            const int64_t all = (tensors[i].n + tile - 1) / tile, left = all - done;
            const int64_t g = left < kMostGroups - groups ? left : kMostGroups - groups;
            if (g) {
                const int64_t start = done * tile, rest = tensors[i].n - start;
                a.t[a.count] = piece_of(tensors[i], start, rest < g * tile ? rest : g * tile, k);
                a.first[a.count++] = (int)groups;
                groups += g;
                done += g;
            }
            if (done == all) ++i, done = 0;
        }
        if (!groups) continue;
        rc = launch_adamw(a, k, groups, (hipStream_t)stream);
        if (rc != STM_OK) return rc;
    }
    return STM_OK;
}

extern "C" int64_t stm_adamw_table_bytes(int count) {
    if (count < 0) return set_error(STM_ERR_INVALID, "adamw_table: bad tensor list");
    return (int64_t)count * (int64_t)(sizeof(stm_adamw_tensor) + sizeof(int));
}

extern "C" int stm_adamw_fill_table(int count, const stm_adamw_tensor* tensors, int param_dtype, int grad_dtype,
                                    int state_bits, void* table) {
    AdamKind k;
    int rc = adamw_kind(param_dtype, grad_dtype, state_bits, k);
    if (rc == STM_OK) rc = check_adamw_tensors(count, tensors, k);
    if (rc != STM_OK) return rc;
    if (count && (!table || !aligned(table, 8))) return set_error(STM_ERR_INVALID, "adamw_table: bad table");
    auto* t = static_cast<stm_adamw_tensor*>(table);
    auto* first = reinterpret_cast<int*>(t + count);
    const int64_t tile = tile_of(k.bits);
    int64_t groups = 0;
    for (int i = 0; i < count; ++i) {
        t[i] = tensors[i];
        first[i] = (int)groups;
        groups += (tensors[i].n + tile - 1) / tile;
        if (groups > kMostGroups) return set_error(STM_ERR_UNSUPPORTED, "adamw_table: too many elements");
    }
    return (int)groups;
}

extern "C" int stm_adamw_step_table(int count, const void* table, int groups, int param_dtype, int grad_dtype,
                                    int state_bits, double lr, double beta1, double beta2, double eps,
                                    double weight_decay, int64_t step, const float* grad_scale, void* stream) {
    AdamTable a;
    AdamKind k;
    int rc = adamw_kind(param_dtype, grad_dtype, state_bits, k);
    if (rc == STM_OK) rc = adamw_numbers(lr, beta1, beta2, eps, weight_decay, step, grad_scale, a.h);
    if (rc != STM_OK) return rc;
    if (count < 0 || groups < 0 || groups > kMostGroups || (groups && (!count || !table || !aligned(table, 8))))
        return set_error(STM_ERR_INVALID, "adamw_step_table: bad table");
    if (!groups) return STM_OK;
    a.t = static_cast<const stm_adamw_tensor*>(table);
    a.first = reinterpret_cast<const int*>(a.t + count);
    a.count = count;
    return launch_adamw(a, k, groups, (hipStream_t)stream);
}

extern "C" int stm_state8_values(const uint8_t* codes, const float* scales, int64_t n, int is_signed, float* out,
                                 void* stream) {
    if (n < 0) return set_error(STM_ERR_INVALID, "state8_values: negative size");
    if (n == 0) return STM_OK;
    if (!codes || !scales || !out) return set_error(STM_ERR_INVALID, "state8_values: null pointer");
    if (!aligned(scales, 4) || !aligned(out, 4)) return set_error(STM_ERR_INVALID, "state8_values: unaligned fp32");
    const int vec = aligned(codes, 4) && aligned(out, 16);
    auto* kernel = is_signed ? k_state_values<true> : k_state_values<false>;
    for (int64_t i = 0; i < n; i += kMostGroups * kTile) {
        const int64_t m = n - i < kMostGroups * kTile ? n - i : kMostGroups * kTile;
        hipLaunchKernelGGL(kernel, dim3((unsigned)((m + kTile - 1) / kTile)), dim3(256), 0, (hipStream_t)stream, codes + i,
                           scales + i / kBlock8, m, out + i, vec);
        const int rc = check_launch("state8_values");
        if (rc != STM_OK) return rc;
    }
    return STM_OK;
}

extern "C" int stm_state8_codes(const float* x, int64_t n, int is_signed, uint8_t* codes, float* scales,
                                void* stream) {
    if (n < 0) return set_error(STM_ERR_INVALID, "state8_codes: negative size");
    if (n == 0) return STM_OK;
    if (!codes || !scales || !x) return set_error(STM_ERR_INVALID, "state8_codes: null pointer");
    if (!aligned(scales, 4) || !aligned(x, 4)) return set_error(STM_ERR_INVALID, "state8_codes: unaligned fp32");
    const int vec = aligned(codes, 4) && aligned(x, 16);
    auto* kernel = is_signed ? k_state_codes<true> : k_state_codes<false>;
    for (int64_t i = 0; i < n; i += kMostGroups * kTile) {
        const int64_t m = n - i < kMostGroups * kTile ? n - i : kMostGroups * kTile;
        hipLaunchKernelGGL(kernel, dim3((unsigned)((m + kTile - 1) / kTile)), dim3(256), 0, (hipStream_t)stream, x + i, m,
                           codes + i, scales + i / kBlock8, vec);
        const int rc = check_launch("state8_codes");
        if (rc != STM_OK) return rc;
    }
    return STM_OK;
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
        if (norm_groups(n[i]) > most_groups(kNormThreads)) return set_error(STM_ERR_UNSUPPORTED, "grad_norm: tensor %d is too large", i);
    }
    double* partial = (double*)workspace;
    NormArgs a;
    for (int i = 0; i < count;) {
        a.count = 0;
        int64_t groups = 0;
        while (i < count && a.count < kNormTensors) {
            const int64_t g = norm_groups(n[i]);
            if (groups + g > most_groups(kNormThreads)) break;
            if (g) {
                a.g[a.count] = grads[i];
                a.last[a.count] = (int)(n[i] - (g - 1) * kNormTile);
                a.first[a.count++] = (int)groups;
                groups += g;
            }
            ++i;
        }
        if (!groups) continue;
        a.first[a.count] = (int)groups;
        const dim3 grid((unsigned)groups), block(kNormThreads);
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
    hipLaunchKernelGGL(k_norm_final, dim3(1), dim3(kFinalThreads), 0, (hipStream_t)stream, (const double*)workspace, need / 8,
                       max_norm, loss_scale, out);
    return check_launch("grad_norm");
}
