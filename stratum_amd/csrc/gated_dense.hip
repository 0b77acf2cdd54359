// The gated block with many rows (gfx950): h = silu(x Wg^T) * (x Wu^T) and its backward
// dgu = [dh u silu'(g) | dh silu(g)] on a weight that was dequantized once, into the
// tiles of k_dequantize_tiles.
//
// Bound by the matrix pipes at the clock that this load leaves. Work-group tile 256 rows
// x 128 output columns, i.e. 256 rows of the weight (a gate and an up row per column);
// eight waves in two groups of four. Wave (wm, wn) owns rows [128 wm, + 128) and columns
// [32 wn, + 32): fragment 0 the gate rows, fragment 1 the up rows of the same columns, so
// the epilogue has both sums of a column in one lane (store_gated). 2 x 4 tiles of
// v_mfma_f32_32x32x16, 128 accumulators.
//
// The reduction goes in steps of 32. The two groups alternate: while one issues a step's
// 16 matrix instructions, the other reads its operands of the step from LDS (12 reads of
// 16 bytes a lane) and issues copies, so that the matrix pipe of every SIMD, which holds
// one wave of each group, always has work queued. A barrier ends each such phase; group 1
// runs one phase behind group 0: step h is read in phases 2 h and 2 h + 1. The tiles of a
// step (16 KB of x, 16 KB of the weight) lie in a ring of four buffers; step h + 3 is copied
// global -> LDS while step h is read, into the buffer that group 1 left a phase ago, and has
// six phases to land. A copy counts in vmcnt; four of them per step and wave, waited for
// two steps behind.
//
// Measured on 8192 rows, W [2 x 14336, 4096] (the library's plain product of these
// sizes: 1215 us), us: steps of 64 in two buffers, copies at the start of the phase
// 1622; copies behind the operand reads 1474; weight in tiles 1452; steps of 32 in four
// buffers 1420 (five: 1429). Without copies 1240, without the epilogue as well 1210: what
// is left is the copies' share of LDS and L1, of which x, read in rows with a stride of
// 2 K bytes, has 60 us (tiles as the weight's: 1354, but with the kernel that makes them the
// call went from 1502 to 1485, and on [2 x 5632, 2048] from 313 to 317). Copies issued
// between the matrix instructions: 1543-1576. The weight straight into registers: 1628.
#include "gemm_tile.h"

namespace stm {
namespace {

struct DenseArgs {
    GemmArgs g;         // a = x, out, dh, M, N = 2 I, K
    const uint16_t* w;  // tiles of the dequantized weight
};

constexpr int kRing = 4;

__device__ __forceinline__ void phase_barrier() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
}
__device__ __forceinline__ void wait_lds() { __builtin_amdgcn_s_waitcnt(0xC07F); }
// at most N memory operations of the wave in flight
template <int N>
__device__ __forceinline__ void wait_vmem_but() {
    __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | ((N >> 4) << 14));
}

// A tile's row is four 16-byte chunks: chunk c sits in slot c ^ (row / 4) % 4, so that the 16
// rows of one LDS pass hit 16 different 16-byte bank groups.
__device__ __forceinline__ int slot32(int row, int chunk) { return row * 4 + (chunk ^ ((row >> 2) & 3)); }

template <typename Tr, int MODE>
__global__ __launch_bounds__(512) void k_gated_dense(DenseArgs d) {
    constexpr int BM = 256, BN = 256, BK = 32;
    const GemmArgs& g = d.g;
    const int tid = threadIdx.x, lane0 = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 2, wn = wave & 3;
    __shared__ uint4 sx[kRing][BM * 4], sw[kRing][BN * 4];

    const int64_t K = g.K, N = g.N;
    const int H = (int)(K / BK);  // even, at least 2
    const int64_t ntm = (g.M + BM - 1) / BM, ntn = (N + BN - 1) / BN, tiles = ntm * ntn;
    for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        int64_t tm, tn;
        tile_coords(t, ntm, ntn, tm, tn);
        const int64_t m0 = tm * BM, c0 = tn * (BN / 2);
        const int lane = opaque_lane(lane0);

        // copies: wave w takes rows [32 w, + 32) of both tiles, 16 rows (1 KB) an instruction;
        // rows past M repeat the last one and are never stored
        const uint16_t* x = reinterpret_cast<const uint16_t*>(g.a);
        uint32_t xoff[2], woff[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = wave * 32 + 16 * i + (lane >> 2), c = (lane & 3) ^ ((r >> 2) & 3);
            const int64_t row = m0 + r < g.M ? m0 + r : g.M - 1;
            xoff[i] = (uint32_t)((row * K + c * 8) * 2);
            woff[i] = (uint32_t)(wave * 2048 + i * 1024 + lane * 16);
        }
        auto copy = [&](int h, int b) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                dma16_s(d.w + (tn * H + h) * (BN * BK), woff[i], lds_offset(&sw[b][(wave * 32 + 16 * i) * 4]));
                dma16_s(x + (int64_t)h * BK, xoff[i], lds_offset(&sx[b][(wave * 32 + 16 * i) * 4]));
            }
        };

        f32x16_t acc[2][4];
        zero_acc(acc);
#pragma unroll
        for (int h = 0; h < kRing - 1; ++h)
            if (h < H) copy(h, h);
        wait_vmem();
        phase_barrier();
        if (wm) phase_barrier();
        int b = 0, fill = kRing - 1;  // step h is in buffer b, step h + 3 goes into `fill`
        for (int h = 0; h < H; ++h) {
            uint4 a[2][4], w[2][2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int ch = 2 * j + (lane >> 5);
#pragma unroll
                for (int i = 0; i < 2; ++i) w[j][i] = sw[b][slot32(64 * wn + 32 * i + (lane & 31), ch)];
#pragma unroll
                for (int f = 0; f < 4; ++f) a[j][f] = sx[b][slot32(128 * wm + 32 * f + (lane & 31), ch)];
            }
            __builtin_amdgcn_sched_barrier(0);
            if (h + kRing - 1 < H) copy(h + kRing - 1, fill);
            __builtin_amdgcn_sched_barrier(0);
            wait_lds();
            // step h + 1 has landed before the barrier that lets group 0 read it: this wave's
            // copies of steps h + 2 and h + 3 may be in flight
            if (wm) {
                if (h + kRing <= H)
                    wait_vmem_but<8>();
                else
                    wait_vmem();
            }
            phase_barrier();
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int f = 0; f < 4; ++f) acc[i][f] = mfma<Tr>(w[j][i], a[j][f], acc[i][f]);
            __builtin_amdgcn_s_setprio(0);
            __builtin_amdgcn_sched_barrier(0);
            if (!wm) {
                if (h + kRing <= H)
                    wait_vmem_but<8>();
                else
                    wait_vmem();
            }
            phase_barrier();
            fill = b;
            b = b + 1 == kRing ? 0 : b + 1;
        }
        if (!wm) phase_barrier();  // group 1's last phase
        // every wave is done with the ring: 8 KB of it each for the epilogue
        const int lane_e = opaque_lane(lane);
        store_gated<Tr, 4, MODE>(acc, g, (int)(c0 + 32 * wn), (int)(m0 + 128 * wm), (int)g.M, lane_e,
                                 &sx[0][0] + wave * 512);
        __syncthreads();
    }
}

}  // namespace

int launch_gated_dense(const GemmArgs& g, const void* w, int mode, int dtype, unsigned grid, hipStream_t stream) {
    DenseArgs d;
    d.g = g;
    d.w = (const uint16_t*)w;
#define STM_GD_LAUNCH(TR, MODE) hipLaunchKernelGGL((k_gated_dense<TR, MODE>), dim3(grid), dim3(512), 0, stream, d)
    if (dtype == STM_BF16 && mode == 1)
        STM_GD_LAUNCH(BF16, 1);
    else if (dtype == STM_BF16)
        STM_GD_LAUNCH(BF16, 2);
    else if (mode == 1)
        STM_GD_LAUNCH(F16, 1);
    else
        STM_GD_LAUNCH(F16, 2);
#undef STM_GD_LAUNCH
    return check_launch("gated (dense)");
}

}  // namespace stm
