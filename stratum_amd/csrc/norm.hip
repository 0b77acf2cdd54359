// Root-mean-square norm over rows, with the residual's addition before it (gfx950).
//
//   s = x (+ residual),  r = 1 / sqrt(mean(s^2) + eps),  y = s r w,  h = s rounded to the residual's type
//
// backward, with n = s r and t = w dy:
//
//   ds = r (t - n mean(t n)) (+ dh),  dw = sum over rows of dy n
//
// ds is the gradient of x and of the residual. Everything between a load and a store is fp32; y comes from the sum
// before its rounding to h, so each output is rounded once. The backward's s is h where h is exact (x without a residual,
// an fp32 stream) and x + residual again where h has 16 bits: with h as it was rounded a weight's gradient is 2.4e-3 off
// (bf16, 763 rows of 5058) and not the 1.8e-3 of its own rounding, and ds differs by 2.1e-4 ([8192, 4096] bf16) from
// the plain form's.
//
// Bound by bytes. One pass: a row stays in registers between its sum and its result, 8 elements of a thread in one access.
// A row belongs to 8 to 64 lanes of a wave (no barrier), or to 128 to 1024 threads.
#include <type_traits>

#include "nf4_kernels.h"
#include "rows.h"

namespace stm {
namespace {

// 8 elements of a row whose type is known at run time only (the residual's, the weight's): f32 is uniform.
template <typename Tr>
__device__ __forceinline__ void load_as(const void* p, bool f32, int64_t at, int n, float (&f)[8]) {
    if (f32) {
        Eight<F32> e;
        e.load(p, at, n);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = e.get(i);
    } else {
        Eight<Tr> e;
        e.load(p, at, n);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = e.get(i);
    }
}

template <typename Tr>
__device__ __forceinline__ void store_as(void* p, bool f32, int64_t at, int n, const float (&f)[8]) {
    if (f32) {
        Eight<F32> e;
        e.set(f);
        e.store(p, at, n);
    } else {
        Eight<Tr> e;
        e.set(f);
        e.store(p, at, n);
    }
}

// 8 elements of such a row before their conversion, so that a load can be under way while an earlier row is worked on.
template <typename Tr>
struct Loaded {
    u32x4_t v[2];

    __device__ __forceinline__ void load(const void* p, bool f32, int64_t at, int n) {
        if (f32) {
            Eight<F32> e;
            e.load(p, at, n);
            v[0] = e.v[0], v[1] = e.v[1];
        } else {
            Eight<Tr> e;
            e.load(p, at, n);
            if constexpr (sizeof(e) == 32)
                v[0] = e.v[0], v[1] = e.v[1];
            else
                v[0] = __builtin_bit_cast(u32x4_t, e);
        }
    }
    __device__ __forceinline__ void get(bool f32, float (&f)[8]) const {
        if (f32 || sizeof(Eight<Tr>) == 32) {
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(v[i / 4][i % 4]);
        } else if constexpr (sizeof(Eight<Tr>) == 16) {
            const Eight<Tr> e = __builtin_bit_cast(Eight<Tr>, v[0]);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = e.get(i);
        }
    }
};

// A work-group holds one row of T threads, or 256 / T of them.
template <int T>
constexpr int kBlock = T <= 256 ? 256 : T;

// Sum over the T threads of a row; every one of them gets it. Above a wave through LDS, `turn` alternating between two
// buffers so that one barrier a sum is enough.
template <int T>
__device__ __forceinline__ float row_sum(float v, int turn) {
    if constexpr (T <= 64) {
        return lanes_sum<T>(v);
    } else {
        __shared__ float part[2][kBlock<T> / 64];
        v = lanes_sum<64>(v);
        float* p = part[turn & 1];
        if ((threadIdx.x & 63) == 0) p[threadIdx.x / 64] = v;
        __syncthreads();
        p += threadIdx.x / T * (T / 64);
        float s = p[0];
#pragma unroll
        for (int i = 1; i < T / 64; ++i) s += p[i];
        return s;
    }
}

struct NormFwd {
    const void *x, *res, *w;
    void *y, *h;
    float* rstd;
    int64_t rows;
    int cols;
    float eps;
    bool res32, w32;
};

// T threads a row, NV vectors of 8 a thread: cols <= 8 T NV.
template <typename Tr, int T, int NV>
__global__ __launch_bounds__(kBlock<T>) void k_rms_fwd(NormFwd a) {
    constexpr int SLOTS = kBlock<T> / T;
    const int t = threadIdx.x % T;
    int turn = 0;
    for (int64_t first = (int64_t)blockIdx.x * SLOTS; first < a.rows; first += (int64_t)gridDim.x * SLOTS, ++turn) {
        const int64_t row = first + threadIdx.x / T;
        const bool on = row < a.rows;
        const int64_t at = row * a.cols;
        float s[NV][8];
        float q = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = 8 * (t + T * v), n = on ? a.cols - c : 0;
            load_as<Tr>(a.x, false, at + c, n, s[v]);
            if (a.res) {
                float r[8];
                load_as<Tr>(a.res, a.res32, at + c, n, r);
#pragma unroll
                for (int i = 0; i < 8; ++i) s[v][i] += r[i];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) q = __builtin_fmaf(s[v][i], s[v][i], q);
        }
        q = row_sum<T>(q, turn);
        const float r = 1.0f / sqrtf(q / (float)a.cols + a.eps);
        if (on && t == 0 && a.rstd) a.rstd[row] = r;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = 8 * (t + T * v), n = on ? a.cols - c : 0;
            float w[8], y[8];
            load_as<Tr>(a.w, a.w32, c, n, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = s[v][i] * r * w[i];
            store_as<Tr>(a.y, false, at + c, n, y);
            if (a.h) store_as<Tr>(a.h, a.res32, at + c, n, s[v]);
        }
    }
}

// Rows too long for registers: two passes over them, 1024 threads a row.
template <typename Tr>
__global__ __launch_bounds__(1024) void k_rms_fwd_long(NormFwd a) {
    int turn = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, ++turn) {
        const int64_t at = row * a.cols;
        float q = 0.0f;
        for (int c = 8 * threadIdx.x; c < a.cols; c += 8 * 1024) {
            float s[8], r[8];
            load_as<Tr>(a.x, false, at + c, a.cols - c, s);
            if (a.res) {
                load_as<Tr>(a.res, a.res32, at + c, a.cols - c, r);
#pragma unroll
                for (int i = 0; i < 8; ++i) s[i] += r[i];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) q = __builtin_fmaf(s[i], s[i], q);
        }
        q = row_sum<1024>(q, turn);
        const float rstd = 1.0f / sqrtf(q / (float)a.cols + a.eps);
        if (threadIdx.x == 0 && a.rstd) a.rstd[row] = rstd;
        for (int c = 8 * threadIdx.x; c < a.cols; c += 8 * 1024) {
            float s[8], r[8], w[8], y[8];
            load_as<Tr>(a.x, false, at + c, a.cols - c, s);
            if (a.res) {
                load_as<Tr>(a.res, a.res32, at + c, a.cols - c, r);
#pragma unroll
                for (int i = 0; i < 8; ++i) s[i] += r[i];
            }
            load_as<Tr>(a.w, a.w32, c, a.cols - c, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = s[i] * rstd * w[i];
            store_as<Tr>(a.y, false, at + c, a.cols - c, y);
            if (a.h) store_as<Tr>(a.h, a.res32, at + c, a.cols - c, s);
        }
    }
}

struct NormBwd {
    const void *dy, *dh, *h, *w;
    const void* res;  // in h's 16-bit type: h is x, and this its residual (null: h is the sum)
    const float* rstd;
    void *dx, *dres;
    float* dw_part;  // [groups of the grid, cols], or null
    int64_t rows;
    int cols;
    bool h32, w32;
};

// T threads a row, 8 columns each: cols <= 8 T. DW: a thread's columns are the same in every row of its work-group, so the
// weight's gradient gathers in registers over the rows that the group takes (gridDim rows apart), then over the group's
// row slots in LDS, and leaves as one row of partial sums; k_rms_dw adds those rows up in a fixed order. The next row is
// then asked for before this one's sum: few groups, so that there are few partial sums, would leave the memory idle in
// between. bf16 with a residual's gradient, us in a graph with the sum of the parts, look-ahead / none (x and residual read
// again): [8192, 5120] 66 / 74 (80 / 85), [4096, 8192] 54 / 56 (66 / 67), [8192, 4096] 55 / 54 (70 / 67), [131072, 128]
// 32 / 32 (39 / 38); the prologue costs a short launch 1 ([1021, 2050] 14.4 / 13.2). Without the weight's gradient
// [8192, 4096] takes 52 (62).
template <typename Tr, int T, bool DW>
__global__ __launch_bounds__(kBlock<T>) void k_rms_bwd(NormBwd a) {
    constexpr int SLOTS = kBlock<T> / T;
    const int t = threadIdx.x % T, slot = threadIdx.x / T, c = 8 * t;
    const int64_t stride = (int64_t)gridDim.x * SLOTS;
    float dw[8] = {};
    Loaded<Tr> dy, h, res, dh, weight;
    float rstd = 0.0f;
    auto ask = [&](int64_t row) {
        const bool on = row < a.rows;
        const int n = on ? a.cols - c : 0;
        rstd = on ? a.rstd[row] : 0.0f;
        dy.load(a.dy, false, row * a.cols + c, n);
        h.load(a.h, a.h32, row * a.cols + c, n);
        if (a.res) res.load(a.res, false, row * a.cols + c, n);
        if (a.dh) dh.load(a.dh, a.h32, row * a.cols + c, n);
    };
    int turn = 0;
    int64_t first = (int64_t)blockIdx.x * SLOTS;
    if (DW) ask(first + slot);
    weight.load(a.w, a.w32, c, a.cols - c);
    for (; first < a.rows; first += stride, ++turn) {
        const int64_t row = first + slot;
        if (!DW) ask(row);
        const float r = rstd;
        float g[8], n_[8], e[8], w[8];  // t = w dy, n = h r
        float dot = 0.0f;
        dy.get(false, g);
        h.get(a.h32, n_);
        if (a.res) {
            float s[8];
            res.get(false, s);
#pragma unroll
            for (int i = 0; i < 8; ++i) n_[i] += s[i];
        }
        if (a.dh) dh.get(a.h32, e);
        weight.get(a.w32, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            n_[i] *= r;
            if (DW) dw[i] = __builtin_fmaf(g[i], n_[i], dw[i]);
            g[i] *= w[i];
            dot = __builtin_fmaf(g[i], n_[i], dot);
        }
        if (DW) ask(row + stride);
        const float mean = row_sum<T>(dot, turn) / (float)a.cols;
        const int n = row < a.rows ? a.cols - c : 0;
        float d[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            d[i] = r * (g[i] - n_[i] * mean);
            if (a.dh) d[i] += e[i];
        }
        if (a.dx) store_as<Tr>(a.dx, false, row * a.cols + c, n, d);
        if (a.dres) store_as<Tr>(a.dres, a.h32, row * a.cols + c, n, d);
    }
    if (!DW) return;
    float* out = a.dw_part + (int64_t)blockIdx.x * a.cols;
    if constexpr (SLOTS > 1) {
        // slot by slot into one row of LDS, each column by the thread that owns it
        __shared__ float sum[8 * T];
        for (int k = 0; k < SLOTS; ++k) {
            if (slot == k) {
#pragma unroll
                for (int i = 0; i < 8; ++i) sum[c + i] = k ? sum[c + i] + dw[i] : dw[i];
            }
            __syncthreads();
        }
        for (int i = threadIdx.x; i < a.cols; i += kBlock<T>) out[i] = sum[i];
    } else {
        store_as<F32>(out, true, c, a.cols - c, dw);
    }
}

// Rows too long for that (with a second vector a thread the registers do not do): two passes, 1024 threads a row.
template <typename Tr>
__device__ __forceinline__ void load_sum(const NormBwd& a, int64_t at, int n, float (&h)[8]) {
    load_as<Tr>(a.h, a.h32, at, n, h);
    if (a.res) {
        float r[8];
        load_as<Tr>(a.res, false, at, n, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] += r[i];
    }
}

template <typename Tr>
__global__ __launch_bounds__(1024) void k_rms_bwd_long(NormBwd a) {
    int turn = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, ++turn) {
        const int64_t at = row * a.cols;
        const float r = a.rstd[row];
        float dot = 0.0f;
        for (int c = 8 * threadIdx.x; c < a.cols; c += 8 * 1024) {
            float g[8], h[8], w[8];
            load_as<Tr>(a.dy, false, at + c, a.cols - c, g);
            load_sum<Tr>(a, at + c, a.cols - c, h);
            load_as<Tr>(a.w, a.w32, c, a.cols - c, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) dot = __builtin_fmaf(g[i] * w[i], h[i] * r, dot);
        }
        const float mean = row_sum<1024>(dot, turn) / (float)a.cols;
        for (int c = 8 * threadIdx.x; c < a.cols; c += 8 * 1024) {
            float g[8], h[8], w[8];
            load_as<Tr>(a.dy, false, at + c, a.cols - c, g);
            load_sum<Tr>(a, at + c, a.cols - c, h);
            load_as<Tr>(a.w, a.w32, c, a.cols - c, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) g[i] = r * (g[i] * w[i] - h[i] * r * mean);
            if (a.dh) {
                load_as<Tr>(a.dh, a.h32, at + c, a.cols - c, h);
#pragma unroll
                for (int i = 0; i < 8; ++i) g[i] += h[i];
            }
            if (a.dx) store_as<Tr>(a.dx, false, at + c, a.cols - c, g);
            if (a.dres) store_as<Tr>(a.dres, a.h32, at + c, a.cols - c, g);
        }
    }
}

// The weight's gradient of rows too long for registers: a thread's 8 columns, rows blockIdx.y, + gridDim.y, ...
template <typename Tr>
__global__ __launch_bounds__(256) void k_rms_dw_long(NormBwd a) {
    const int64_t c = 8 * ((int64_t)blockIdx.x * 256 + threadIdx.x);
    const int n = (int)min((int64_t)8, a.cols - c);
    if (n <= 0) return;
    float dw[8] = {};
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        float g[8], h[8];
        const float r = a.rstd[row];
        load_as<Tr>(a.dy, false, row * a.cols + c, n, g);
        load_sum<Tr>(a, row * a.cols + c, n, h);
#pragma unroll
        for (int i = 0; i < 8; ++i) dw[i] = __builtin_fmaf(g[i], h[i] * r, dw[i]);
    }
    store_as<F32>(a.dw_part + (int64_t)blockIdx.y * a.cols, true, c, n, dw);
}

// Sum of `parts` rows of partial sums: 32 columns a work-group, its 32 row slots added up in LDS. A slot's rows are
// asked for eight at a time.
template <typename Tr>
__global__ __launch_bounds__(1024) void k_rms_dw(const float* __restrict__ part, int parts, int cols, void* dw,
                                                 bool w32) {
    __shared__ float sum[32][33];
    const int slot = threadIdx.x / 32;
    for (int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x % 32; c - threadIdx.x % 32 < cols; c += (int64_t)gridDim.x * 32) {
        float s = 0.0f;
        if (c < cols)
            for (int p0 = slot; p0 < parts; p0 += 32 * 8) {
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = p0 + 32 * i < parts ? part[(int64_t)(p0 + 32 * i) * cols + c] : 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) s += v[i];
            }
        sum[slot][threadIdx.x % 32] = s;
        __syncthreads();
        if (slot == 0 && c < cols) {
            for (int k = 1; k < 32; ++k) s += sum[k][threadIdx.x];
            if (w32)
                static_cast<float*>(dw)[c] = s;
            else
                static_cast<typename Eight<Tr>::elem*>(dw)[c] = Tr::from_f32(s);
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------ which form
constexpr int64_t kMostGroups = 1 << 21;  // of 1024 threads; the kernels loop over what is left

unsigned row_groups(int64_t rows, int per) {
    const int64_t groups = (rows + per - 1) / per;
    return (unsigned)(groups < kMostGroups ? groups : kMostGroups);
}

constexpr int64_t kForwardCols = 1024 * 4 * 8, kBackwardCols = 1024 * 8;  // what registers hold of a row

// Threads of a row: one vector each, up to 8192 columns; whole pairs of waves where that is more than a wave of them
// ([8192, 5120] backward: 640 threads 67, 1024 80). More vectors a thread are slower, whether a wave then needs no
// barrier or not ([8192, 4096] bf16 with a residual, us forward / backward of h alone: 64 threads of 8 vectors 55 / 115, 128
// of 4 55 / 61, 256 of 2 51 / 52, 512 of 1 49 / 48; [4096, 8192]: 256 57 / 59, 512 53 / 55, 1024 51 / 50).
int row_threads(int64_t cols) {
    const int64_t vecs = (cols + 7) / 8;
    if (vecs > 256) return vecs < 1024 ? (int)(vecs + 127) / 128 * 128 : 1024;
    int t = 8;
    while (t < vecs) t *= 2;
    return t;
}

// Groups of the backward's grid that write partial sums: as many as give each of the 256 compute units up to 1024 threads
// and the same work; half or twice as many are within a tenth of them or slower (bf16 with a residual's gradient, us in a
// graph: [8192, 4096], 512 threads, 256 groups 51, 384 57, 512 55, 768 59, 1024 58; [40000, 2048], 256 threads, 256 159, 512
// 115, 1024 127; [131072, 128], 256 threads, 512 31, 1024 32, 2048 36; [8192, 5120], 640 threads, 256 66, 384 78, 512 70;
// [1021, 2050], 384 threads, 256 16, 512 14, 1021 21).
int dw_groups(int64_t rows, int64_t cols) {
    if (cols > kBackwardCols) return (int)(rows < 256 ? rows : 256);
    const int t = row_threads(cols), slots = t <= 256 ? 256 / t : 1, threads = t <= 256 ? 256 : t;
    const int64_t groups = (rows + slots - 1) / slots, most = 256 * (1024 / threads);
    return (int)(groups < most ? groups : most);
}

template <typename F>
int each_form(int t, int nv, F f) {
#define STM_FORM(T, NV) \
    if (t == T && nv <= NV) return f(std::integral_constant<int, T>{}, std::integral_constant<int, NV>{})
    STM_FORM(8, 1);
    STM_FORM(16, 1);
    STM_FORM(32, 1);
    STM_FORM(64, 1);
    STM_FORM(128, 1);
    STM_FORM(256, 1);
    STM_FORM(384, 1);
    STM_FORM(512, 1);
    STM_FORM(640, 1);
    STM_FORM(768, 1);
    STM_FORM(896, 1);
    STM_FORM(1024, 1);
    STM_FORM(1024, 2);
    STM_FORM(1024, 4);
#undef STM_FORM
    return set_error(STM_ERR_UNSUPPORTED, "rms_norm: no form of %d threads and %d vectors", t, nv);
}

template <typename Tr>
int fwd(const NormFwd& a, hipStream_t st) {
    if (a.cols > kForwardCols) {
        hipLaunchKernelGGL(k_rms_fwd_long<Tr>, dim3(row_groups(a.rows, 1)), dim3(1024), 0, st, a);
        return check_launch("rms_norm_fwd");
    }
    const int t = row_threads(a.cols), nv = (a.cols + 8 * t - 1) / (8 * t);
    return each_form(t, nv, [&](auto T, auto NV) {
        constexpr int per = kBlock<T.value> / T.value;
        hipLaunchKernelGGL((k_rms_fwd<Tr, T.value, NV.value>), dim3(row_groups(a.rows, per)),
                           dim3(kBlock<T.value>), 0, st, a);
        return check_launch("rms_norm_fwd");
    });
}

template <typename Tr>
int bwd(const NormBwd& a, void* dweight, hipStream_t st) {
    const int parts = a.dw_part ? dw_groups(a.rows, a.cols) : 0;
    if (a.rows == 0) {  // no row: the weight's gradient is zero
    } else if (a.cols > kBackwardCols) {
        if (a.dx || a.dres) hipLaunchKernelGGL(k_rms_bwd_long<Tr>, dim3(row_groups(a.rows, 1)), dim3(1024), 0, st, a);
        if (a.dw_part)
            hipLaunchKernelGGL(k_rms_dw_long<Tr>, dim3((unsigned)((a.cols + 2047) / 2048), (unsigned)parts), dim3(256), 0,
                               st, a);
    } else {
        const int rc = each_form(row_threads(a.cols), 1, [&](auto T, auto) {
            constexpr int per = kBlock<T.value> / T.value;
            if (a.dw_part)
                hipLaunchKernelGGL((k_rms_bwd<Tr, T.value, true>), dim3((unsigned)parts), dim3(kBlock<T.value>), 0, st, a);
            else
                hipLaunchKernelGGL((k_rms_bwd<Tr, T.value, false>), dim3(row_groups(a.rows, per)), dim3(kBlock<T.value>), 0, st,
                                   a);
            return STM_OK;
        });
        if (rc) return rc;
    }
    if (dweight)
        hipLaunchKernelGGL(k_rms_dw<Tr>, dim3(row_groups(a.cols, 32)), dim3(1024), 0, st, a.dw_part, parts, a.cols, dweight, a.w32);
    return check_launch("rms_norm_bwd");
}

// Sizes and types that every call shares.
int check_rows(const char* what, int64_t rows, int64_t cols, int dtype, int w_dtype) {
    if (rows < 0 || cols < 0) return set_error(STM_ERR_INVALID, "%s: negative size", what);
    if (dtype < 0 || dtype > STM_F32) return set_error(STM_ERR_INVALID, "%s: dtype must be fp16, bf16 or fp32", what);
    if (w_dtype != dtype && w_dtype != STM_F32)
        return set_error(STM_ERR_INVALID, "%s: the weight must be of the rows' type or fp32", what);
    if (rows >= (1ll << 31) || cols >= (1ll << 30) || (rows && cols > (1ll << 60) / rows))
        return set_error(STM_ERR_UNSUPPORTED, "%s: [%lld, %lld] is too large", what, (long long)rows, (long long)cols);
    return STM_OK;
}

// Elements lie on multiples of their size.
bool lies(const void* p, int dtype) { return aligned(p, dtype == STM_F32 ? 4 : 2); }

}  // namespace
}  // namespace stm

using namespace stm;

extern "C" int stm_rms_norm_fwd(const void* x, const void* residual, int residual_dtype, const void* weight,
                                int weight_dtype, void* y, void* h, float* rstd, int64_t rows, int64_t cols, double eps,
                                int dtype, void* stream) {
    const char* what = "rms_norm_fwd";
    int rc = check_rows(what, rows, cols, dtype, weight_dtype);
    if (rc) return rc;
    if (residual && residual_dtype != dtype && residual_dtype != STM_F32)
        return set_error(STM_ERR_INVALID, "%s: the residual must be of x's type or fp32", what);
    if (!(eps >= 0.0)) return set_error(STM_ERR_INVALID, "%s: eps must not be negative", what);
    if (rows == 0 || cols == 0) return STM_OK;
    if (!x || !weight || !y) return set_error(STM_ERR_INVALID, "%s: null pointer", what);
    if (!residual != !h) return set_error(STM_ERR_INVALID, "%s: a residual and its sum come together", what);
    if (!lies(x, dtype) || !lies(y, dtype) || !lies(residual, residual_dtype) || !lies(h, residual_dtype) ||
        !lies(weight, weight_dtype) || !lies(rstd, STM_F32))
        return set_error(STM_ERR_INVALID, "%s: pointers must be aligned to their elements", what);
    const NormFwd a{x,    residual, weight, y, h, rstd, rows, (int)cols, (float)eps, residual && residual_dtype == STM_F32,
                    weight_dtype == STM_F32};
    hipStream_t st = (hipStream_t)stream;
    return dtype == STM_BF16 ? fwd<BF16>(a, st) : dtype == STM_F16 ? fwd<F16>(a, st) : fwd<F32>(a, st);
}

extern "C" int64_t stm_rms_norm_workspace_bytes(int64_t rows, int64_t cols) {
    const int rc = check_rows("rms_norm_workspace_bytes", rows, cols, STM_F32, STM_F32);
    if (rc) return rc;
    return rows && cols ? (int64_t)dw_groups(rows, cols) * cols * 4 : 0;
}

extern "C" int stm_rms_norm_bwd(const void* dy, const void* dh, const void* h, const void* residual, int h_dtype,
                                const float* rstd, const void* weight, int weight_dtype, void* dx, void* dresidual, void* dweight, int64_t rows,
                                int64_t cols, int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* what = "rms_norm_bwd";
    int rc = check_rows(what, rows, cols, dtype, weight_dtype);
    if (rc) return rc;
    if (h_dtype != dtype && h_dtype != STM_F32) return set_error(STM_ERR_INVALID, "%s: h must be of dy's type or fp32", what);
    if (residual && h_dtype == STM_F32)
        return set_error(STM_ERR_INVALID, "%s: a residual apart from its sum is taken in 16 bits", what);
    if (cols == 0) return STM_OK;
    if (rows && (!dy || !h || !rstd || !weight)) return set_error(STM_ERR_INVALID, "%s: null pointer", what);
    if (!lies(dy, dtype) || !lies(dx, dtype) || !lies(dh, h_dtype) || !lies(h, h_dtype) || !lies(residual, h_dtype) ||
        !lies(dresidual, h_dtype) ||
        !lies(weight, weight_dtype) || !lies(dweight, weight_dtype) || !lies(rstd, STM_F32) || !lies(workspace, STM_F32))
        return set_error(STM_ERR_INVALID, "%s: pointers must be aligned to their elements", what);
    if (dweight && rows) {
        const int64_t need = stm_rms_norm_workspace_bytes(rows, cols);
        if (!workspace || workspace_bytes < need)
            return set_error(STM_ERR_INVALID, "%s: the weight's gradient needs a workspace of %lld bytes, got %lld", what,
                             (long long)need, (long long)(workspace ? workspace_bytes : 0));
    }
    if (rows == 0 && !dweight) return STM_OK;
    if (!dx && !dresidual && !dweight) return STM_OK;
    const NormBwd a{dy, dh, h, weight, residual, rstd, dx, dresidual,
                    dweight && rows ? static_cast<float*>(workspace) : nullptr, rows, (int)cols, h_dtype == STM_F32,
                    weight_dtype == STM_F32};
    hipStream_t st = (hipStream_t)stream;
    return dtype == STM_BF16 ? bwd<BF16>(a, dweight, st) : dtype == STM_F16 ? bwd<F16>(a, dweight, st) : bwd<F32>(a, dweight, st);
}
