// Rows of 16- or 32-bit elements, 8 at a time, and reductions over the lanes of a wave (gfx950).
#pragma once

#include "nf4_common.h"

namespace stm {

struct F32 {
    static constexpr int tag = STM_F32;
    __device__ static inline float to_f32(float v) { return v; }
    __device__ static inline float from_f32(float v) { return v; }
};

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// 16 bytes at an element's alignment (the typedef's alignment does not pass through a template's argument).
#define STM_LOOSE(NAME, A)                                                                        \
    struct NAME {                                                                                 \
        typedef u32x4_t __attribute__((aligned(A))) type;                                         \
        template <bool STREAM>                                                                    \
        static __device__ __forceinline__ u32x4_t load(const void* p) {                           \
            if constexpr (STREAM) return __builtin_nontemporal_load(static_cast<const type*>(p)); \
            return *static_cast<const type*>(p);                                                  \
        }                                                                                         \
        template <bool STREAM>                                                                    \
        static __device__ __forceinline__ void store(u32x4_t v, void* p) {                        \
            if constexpr (STREAM)                                                                 \
                __builtin_nontemporal_store(v, static_cast<type*>(p));                            \
            else                                                                                  \
                *static_cast<type*>(p) = v;                                                       \
        }                                                                                         \
    }
STM_LOOSE(Loose2, 2);
STM_LOOSE(Loose4, 4);
#undef STM_LOOSE

// 8 consecutive elements of a row as they lie in memory. STREAM: what is read or written will not be met again soon, so the
// caches need not keep it. A row starts wherever its width puts it, so the 16-byte accesses are declared with the
// alignment of one element: the hardware takes them at any address.
template <typename Tr>
struct Eight {
    typedef uint16_t elem;
    u32x4_t v;

    // the first n elements at p (n < 8 at a row's end; n <= 0: none), zeros behind them
    template <bool STREAM = false>
    __device__ __forceinline__ void load(const void* base, int64_t at, int n) {
        const elem* p = static_cast<const elem*>(base) + at;
        if (n >= 8) {
            v = Loose2::load<STREAM>(p);
            return;
        }
        v = u32x4_t{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) v[i / 2] |= (uint32_t)p[i] << (16 * (i % 2));
    }
    template <bool STREAM = false>
    __device__ __forceinline__ void store(void* base, int64_t at, int n) const {
        elem* p = static_cast<elem*>(base) + at;
        if (n >= 8) {
            Loose2::store<STREAM>(v, p);
            return;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = (uint16_t)(v[i / 2] >> (16 * (i % 2)));
    }
    __device__ __forceinline__ float get(int i) const {
        return Tr::to_f32((uint16_t)(v[i / 2] >> (16 * (i % 2))));
    }
    __device__ __forceinline__ void set(const float (&f)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = Tr::pack2(f[2 * i], f[2 * i + 1]);
    }
    __device__ __forceinline__ void clear() { v = u32x4_t{0, 0, 0, 0}; }
};

template <>
struct Eight<F32> {
    typedef float elem;
    u32x4_t v[2];

    template <bool STREAM = false>
    __device__ __forceinline__ void load(const void* base, int64_t at, int n) {
        const elem* p = static_cast<const elem*>(base) + at;
        if (n >= 8) {
            v[0] = Loose4::load<STREAM>(p);
            v[1] = Loose4::load<STREAM>(p + 4);
            return;
        }
        clear();
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) v[i / 4][i % 4] = __float_as_uint(p[i]);
    }
    template <bool STREAM = false>
    __device__ __forceinline__ void store(void* base, int64_t at, int n) const {
        elem* p = static_cast<elem*>(base) + at;
        if (n >= 8) {
            Loose4::store<STREAM>(v[0], p);
            Loose4::store<STREAM>(v[1], p + 4);
            return;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = __uint_as_float(v[i / 4][i % 4]);
    }
    __device__ __forceinline__ float get(int i) const { return __uint_as_float(v[i / 4][i % 4]); }
    __device__ __forceinline__ void set(const float (&f)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i / 4][i % 4] = __float_as_uint(f[i]);
    }
    __device__ __forceinline__ void clear() { v[0] = v[1] = u32x4_t{0, 0, 0, 0}; }
};

// ------------------------------------------------------------ lanes
// op(v, the other lane's v), the other one 1, 2, 4, 8, 16 or 32 away, where all lanes of each smaller group hold one value
// already: within 16 lanes a DPP move (swap neighbours, swap pairs, mirror 8, mirror 16), across them the two row swaps,
// which give every lane both values. op commutes.
template <int STEP, typename Op>
__device__ __forceinline__ uint32_t with_other(uint32_t v, Op op) {
    if constexpr (STEP <= 8) {
        constexpr int ctrl = STEP == 1 ? 0xB1 : STEP == 2 ? 0x4E : STEP == 4 ? 0x141 : 0x140;
        return op(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, 0xF, 0xF, true));
    } else if constexpr (STEP == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return op(r[0], r[1]);
    } else {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return op(r[0], r[1]);
    }
}

// The other lane's value itself.
template <int STEP>
__device__ __forceinline__ uint32_t across(uint32_t v) {
    if constexpr (STEP <= 8) {
        return with_other<STEP>(v, [](uint32_t, uint32_t o) { return o; });
    } else if constexpr (STEP == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return (threadIdx.x & 16) ? r[0] : r[1];
    } else {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return (threadIdx.x & 32) ? r[0] : r[1];
    }
}

// Combine over groups of LANES lanes; every lane of a group gets the same value (op commutes).
template <int LANES, int STEP = 1, typename Op>
__device__ __forceinline__ uint32_t over_lanes(uint32_t v, Op op) {
    if constexpr (STEP < LANES) {
        return over_lanes<LANES, STEP * 2>(with_other<STEP>(v, op), op);
    } else {
        return v;
    }
}

template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
    return __uint_as_float(over_lanes<LANES>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }));
}

template <int LANES>
__device__ __forceinline__ float lanes_max(float v) {
    return __uint_as_float(over_lanes<LANES>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }));
}

template <int LANES>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
    return over_lanes<LANES>(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}

template <int LANES>
__device__ __forceinline__ uint32_t lanes_min(uint32_t v) {
    return over_lanes<LANES>(v, [](uint32_t a, uint32_t b) { return a < b ? a : b; });
}

// 64-bit keys: the largest upper half, then the largest lower half among its holders.
template <int LANES>
__device__ __forceinline__ uint64_t lanes_max(uint64_t v) {
    const uint32_t hi = lanes_max<LANES>((uint32_t)(v >> 32));
    const uint32_t lo = lanes_max<LANES>((uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
    return (uint64_t)hi << 32 | lo;
}

template <int LANES, int STEP = 1>
__device__ __forceinline__ double lanes_sum(double v) {
    if constexpr (STEP < LANES) {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const uint64_t o = (uint64_t)across<STEP>((uint32_t)(u >> 32)) << 32 | across<STEP>((uint32_t)u);
        return lanes_sum<LANES, STEP * 2>(v + __builtin_bit_cast(double, o));
    } else {
        return v;
    }
}

}  // namespace stm
