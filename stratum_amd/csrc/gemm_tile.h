// Device code that the tile kernels share: matrix instructions, the LDS swizzle, the
// global -> LDS copies, the tile order over the XCDs, and the gated epilogue.
#pragma once

#include "nf4_kernels.h"

#ifndef STM_GROUP_M
#define STM_GROUP_M 4
#endif

namespace stm {
namespace {

template <typename Tr>
__device__ __forceinline__ f32x16_t mfma(const uint4& a, const uint4& b, const f32x16_t& c) {
    if constexpr (Tr::tag == STM_BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b),
                                                       c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c,
                                                      0, 0, 0);
}

template <typename Tr>
__device__ __forceinline__ f32x4_t mfma16(const uint4& a, const uint4& b, const f32x4_t& c) {
    if constexpr (Tr::tag == STM_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b),
                                                       c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c,
                                                      0, 0, 0);
}

#ifndef STM_SWZ
#define STM_SWZ 1
#endif
__device__ __forceinline__ int swz_key(int row) { return STM_SWZ ? ((row >> 1) & 7) : (row & 7); }
__device__ __forceinline__ int swz(int row, int chunk) { return row * 8 + (chunk ^ swz_key(row)); }

typedef __attribute__((address_space(3))) uint4 lds_uint4;
typedef int v2i32_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint32_t lds_offset(const uint4* p) {
    return (uint32_t)(size_t)((const lds_uint4*)(p));
}

// 16 bytes global -> LDS for every lane of the wave; the LDS destination is
// lds_base + 16 * lane (lds_base wave-uniform, in M0). Issued as inline asm so
// the compiler does not treat every later LDS read as dependent on it (it
// cannot tell the two LDS buffers apart and would wait for the copy before the
// MFMA operand reads of the other buffer); completion is awaited explicitly
// with wait_vmem() before the barrier that publishes the buffer.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma16(const void* src, uint32_t lds_base) {
    __asm__ volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds_base), "v"(src)
                     : "memory", "m0");
}
// 4 bytes global -> LDS for every lane; destination lds_base + 4 * lane.
__device__ __forceinline__ void dma4(const void* src, uint32_t lds_base) {
    __asm__ volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dword %1, off" ::"s"(lds_base), "v"(src)
                     : "memory", "m0");
}
// The same copy from a wave-uniform 64-bit base plus a 32-bit per-lane byte offset
// (global_load_lds with an SGPR base: no 64-bit address arithmetic per copy).
__device__ __forceinline__ void dma16_s(const void* base, uint32_t voff, uint32_t lds_base) {
    const uint64_t b = (uint64_t)(size_t)base;
    const uint64_t sb = ((uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(b >> 32)) << 32) |
                        (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)b);
    const void* sbase = (const void*)(size_t)sb;
    __asm__ volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds_base), "v"(voff), "s"(sbase)
                     : "memory", "m0");
}
#pragma clang diagnostic pop

// s_waitcnt vmcnt(0) (expcnt, lgkmcnt left at their maxima). Emitted through the
// builtin so the compiler's own wait-count bookkeeping sees it and inserts no
// further waits for the weight registers loaded before it.
__device__ __forceinline__ void wait_vmem() { __builtin_amdgcn_s_waitcnt(0x0F70); }

// Tile order: work-groups are dispatched round-robin over the 8 XCDs, so ids
// i, i + 8, i + 16, ... share an L2. Give each XCD a contiguous run of tiles and
// walk them GROUP_M activation tiles at a time so concurrently running tiles on
// one XCD reuse the same activation rows and weight rows. With 32 CUs per XCD,
// GROUP_M = 4 runs 4 activation x 8 weight tiles together; measured at
// M = 8192 on W [14336, 4096] it fetches 735 MB per forward from beyond L2
// (GROUP_M = 8: 1072 MB, 2: 820 MB) and is 1-4 % faster.
__device__ __forceinline__ void tile_coords(int64_t pid, int64_t ntm, int64_t ntn, int64_t& tm, int64_t& tn,
                                            bool xcd_runs = true) {
    const int64_t T = ntm * ntn;
    const int64_t T8 = (T / 8) * 8;
    if (xcd_runs && pid < T8) pid = (pid % 8) * (T / 8) + pid / 8;
    const int64_t per_group = (int64_t)STM_GROUP_M * ntn;
    const int64_t grp = pid / per_group;
    const int64_t first = grp * STM_GROUP_M;
    const int64_t gsize = (ntm - first) < STM_GROUP_M ? (ntm - first) : STM_GROUP_M;
    const int64_t in = pid % per_group;
    tm = first + in % gsize;
    tn = in / gsize;
}

template <int FA, int FB>
__device__ __forceinline__ void zero_acc(f32x16_t (&acc)[FA][FB]) {
#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
        for (int j = 0; j < FB; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.0f;
}

// An opaque copy of the lane index. Values computed from it stay after the point
// where it is taken: per-work-item lane offsets are recomputed per item, and
// epilogue addresses after the main loop, instead of being computed once up
// front and held (spilled) across the main loop.
__device__ __forceinline__ int opaque_lane(int lane) {
    __asm__ volatile("" : "+v"(lane));
    return lane;
}

// ActStage with a wave-uniform base and 32-bit byte offsets (the tile's rows
// must lie within 4 GiB of the base).
template <int BM, int NW>
struct ActStageS {
    static constexpr int XI = BM / (8 * NW);
    const uint16_t* base;
    uint32_t off[XI];
    uint32_t lds[2][XI];

    __device__ __forceinline__ void init(const uint16_t* b, int64_t ld, int64_t m0, int64_t rows, const uint4* buf0,
                                         const uint4* buf1, int wave, int lane) {
        base = b;
#pragma unroll
        for (int i = 0; i < XI; ++i) {
            const int r0 = (wave * XI + i) * 8;
            const int r = r0 + (lane >> 3);
            const int c = (lane & 7) ^ swz_key(r);
            int64_t row = m0 + r;
            row = row < rows ? row : rows - 1;
            off[i] = (uint32_t)((row * ld + c * 8) * 2);
            lds[0][i] = __builtin_amdgcn_readfirstlane(lds_offset(buf0 + r0 * 8));
            lds[1][i] = __builtin_amdgcn_readfirstlane(lds_offset(buf1 + r0 * 8));
        }
    }
    __device__ __forceinline__ void issue(int64_t k0, int buf) const {
#pragma unroll
        for (int i = 0; i < XI; ++i) dma16_s(base + k0, off[i], lds[buf][i]);
    }
};

// ------------------------------------------------------------ gated forward
// h = silu(x Wg^T) * (x Wu^T) for the stacked weight W = [Wg; Wu] of N = 2 I rows, and its
// backward dgu = [dh u silu'(g) | dh silu(g)] with g and u computed again: the
// kernels of the plain forward over W's rows in another order, in which a gate row and
// the up row of the same output column reach the same lane, and an epilogue on the fp32
// sums (one rounding where the product and the SwiGLU pass as two kernels make two, and
// no [M, 2 I] tensor written and read between them).

// Physical row of output column c of part 0 (gate) or 1 (up); columns past I only feed
// outputs that are never stored.
__device__ __forceinline__ int64_t gated_row(int64_t c, int part, int64_t I) {
    return part * I + (c < I ? c : I - 1);
}

__device__ __forceinline__ float gate_sigmoid(float g) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * g));
}
__device__ __forceinline__ float gate_fwd(float g, float u) { return g * gate_sigmoid(g) * u; }
__device__ __forceinline__ void gate_bwd(float g, float u, float dh, float& dg, float& du) {
    const float s = gate_sigmoid(g), gs = g * s;
    du = dh * gs;
    dg = dh * u * (s + gs * (1.0f - s));
}

// Epilogue of a wave that holds gate columns [c0, c0 + 32) in acc[0] and up columns in
// acc[1] over 32 FB rows: MODE 1 stores h [rows, I], MODE 2 reads dh [rows, I] and
// stores dgu [rows, 2 I], MODE 3 stores h and the sums (g.sums [rows, 2 I], fp32). Through LDS as store_tile_lds (rows of four 16-byte chunks
// per output, chunk slot c ^ (row % 4)), half of the fragments (an odd number: one) at a time. I % 8 == 0.
//
// dgu is rounded to 16 bits because the input gradient's matrix instructions take no more; dx then has the error
// of that rounding beside its own: against 64 bits 2.34e-3 in bf16 and 2.94e-4 in fp16 (relative
// norms), where a product of fp32 values, rounded once, has 1.66e-3 and 2.08e-4. dgu held as two 16-bit
// parts would take that away at twice the product's time.
template <typename Tr, int FB, int MODE>
__device__ __forceinline__ void store_gated(const f32x16_t (&acc)[2][FB], const GemmArgs& g, int c0, int orow_base,
                                            int orows, int lane, uint4* stage) {
    constexpr int NP = FB % 2 ? FB : 2, FP = FB / NP, RP = 32 * FP;
    constexpr int PARTS = MODE == 2 ? 2 : 1;
    const int I = (int)(g.N / 2), ld = PARTS * I, hi = lane >> 5;
    uint8_t* st = reinterpret_cast<uint8_t*>(stage);
    uint16_t* out = reinterpret_cast<uint16_t*>(g.out);
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        if (orow_base + p * RP >= orows) break;  // no valid row left (uniform)
#pragma unroll
        for (int jj = 0; jj < FP; ++jj) {
            const int rr = 32 * jj + (lane & 31);
            uint2 dh[4];
            if constexpr (MODE == 2) {
                const int row = orow_base + p * RP + rr;
                const uint16_t* src = reinterpret_cast<const uint16_t*>(g.dh) + (int64_t)(row < orows ? row : orows - 1) * I;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int col = c0 + 8 * q + 4 * hi;
                    dh[q] = *reinterpret_cast<const uint2*>(src + (col < I ? col : 0));
                }
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                // four columns at a time out of the accumulators
                f32x4_t a, b;
#pragma unroll
                for (int e = 0; e < 4; ++e) a[e] = acc[0][p * FP + jj][4 * q + e], b[e] = acc[1][p * FP + jj][4 * q + e];
                __asm__ volatile("" : "+v"(a), "+v"(b));
                float v[4], w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if constexpr (MODE != 2) {
                        v[e] = gate_fwd(a[e], b[e]);
                    } else {
                        const uint32_t d = e < 2 ? dh[q].x : dh[q].y;
                        gate_bwd(a[e], b[e], Tr::to_f32((uint16_t)(e & 1 ? d >> 16 : d & 0xFFFFu)), v[e], w[e]);
                    }
                }
                if constexpr (MODE == 3) {
                    const int row = orow_base + p * RP + rr, col = c0 + 8 * q + 4 * hi;
                    float* dst = g.sums + ((int64_t)row * 2 * I + col);
                    if (row < orows && col < I) *reinterpret_cast<f32x4_t*>(dst) = a, *reinterpret_cast<f32x4_t*>(dst + I) = b;
                }
                const int slot = q ^ (rr & 3);
                uint2 pk;
                pk.x = Tr::pack2(v[0], v[1]);
                pk.y = Tr::pack2(v[2], v[3]);
                *reinterpret_cast<uint2*>(st + rr * 64 + slot * 16 + 8 * hi) = pk;
                if constexpr (MODE == 2) {
                    pk.x = Tr::pack2(w[0], w[1]);
                    pk.y = Tr::pack2(w[2], w[3]);
                    *reinterpret_cast<uint2*>(st + RP * 64 + rr * 64 + slot * 16 + 8 * hi) = pk;
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
#pragma unroll
        for (int part = 0; part < PARTS; ++part)
#pragma unroll
            for (int it = 0; it < RP / 16; ++it) {
                const int rr = 16 * it + lane / 4, c = lane % 4;
                const uint4 v = stage[part * RP * 4 + rr * 4 + (c ^ (rr & 3))];
                const int orow = orow_base + p * RP + rr, col = c0 + 8 * c;
                if (orow < orows && col < I)
                    *reinterpret_cast<uint4*>(out + ((int64_t)orow * ld + part * I + col)) = v;
            }
    }
}

}  // namespace
}  // namespace stm
