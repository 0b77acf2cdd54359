// The operators around the experts' products of a sparse layer (gfx950):
//
//   route     the experts of every token and their weights, from the router's logits, and its gradient
//   sort      the slots (token, j) in the order of their experts: where each expert's rows begin, and both directions
//   gather    the tokens' rows in that order
//   combine   the experts' rows back to their tokens, weighted, and its gradients (without weights: gather's gradient)
//
// n = tokens * top_k slots; slot t * top_k + j. offsets[e] .. offsets[e + 1] are expert e's rows; slots[p] is the slot of
// row p, positions[slot] its row (-1 for a slot without an expert). Whatever these hold, no access leaves the tensors.
#include <type_traits>

#include "nf4_kernels.h"
#include "rows.h"

namespace stm {
namespace {

constexpr unsigned kMostGroups = 1u << 23;  // of 256 threads; the kernels loop over what is left

unsigned groups_for(int64_t items, int per) {
    const int64_t g = (items + per - 1) / per;
    return (unsigned)(g < (int64_t)kMostGroups ? (g > 0 ? g : 1) : kMostGroups);
}

// ------------------------------------------------------------ route
// A token belongs to LANES lanes, lane l holds experts l * VPL .. l * VPL + VPL - 1, so that among equal keys the lowest
// lane, and in it the first of its values, is the lowest expert.
//
// Keys are unsigned integers in the order of the values they stand for, 0 for an expert that cannot be chosen (-inf), NaN
// above all. Without a bias and without sums over groups the scores are in the order of the logits, which are compared as
// they are (32 bits, exact). Otherwise score + bias is computed in 64 bits: two experts whose keys differ by less than an
// fp32 rounding are still told apart, and the same ones are found as by any other program that computes them so.
//
// One key is taken per round: the maximum over a lane's values, over the lanes (DPP), the first lane that holds it.
struct Route {
    const void* logits;
    const float* bias;
    const uint8_t* mask;
    float* weights;
    int32_t* experts;
    int64_t tokens;
    int E, top_k, groups, top_groups;
    bool sigmoid, sums, renorm;
    float scale;
};

__device__ __forceinline__ uint32_t key_of(float f) {
    if (f != f) return 0xFFFFFFFFu;
    if (f == -INFINITY) return 0u;
    const uint32_t u = __float_as_uint(f + 0.0f);  // -0 and +0 are equal
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ uint64_t key_of(double f) {
    if (f != f) return ~0ull;
    if (f == -INFINITY) return 0ull;
    const uint64_t u = __builtin_bit_cast(uint64_t, f + 0.0);
    return u >> 63 ? ~u : u | 1ull << 63;
}

__device__ __forceinline__ double value_of(uint64_t k) {
    if (k == ~0ull) return __builtin_nan("");
    return __builtin_bit_cast(double, k >> 63 ? k & ~(1ull << 63) : ~k);
}

__device__ __forceinline__ float sigmoid_of(float x) {  // accurate on both sides
    const float e = expf(-fabsf(x));
    return (x < 0.0f ? e : 1.0f) / (1.0f + e);
}

// The logit of one expert.
template <typename Tr>
__device__ __forceinline__ float logit(const void* logits, int64_t at) {
    return Tr::to_f32(static_cast<const typename Eight<Tr>::elem*>(logits)[at]);
}

// Best of LANES lanes: its key to all of them, and which lane of the token holds it first.
template <int LANES, typename Key>
__device__ __forceinline__ Key take(Key best, int* lane) {
    const Key top = lanes_max<LANES>(best);
    const uint64_t holders = __ballot(best == top);
    const int first = threadIdx.x & 63 & ~(LANES - 1);
    *lane = __ffsll((unsigned long long)(LANES == 64 ? holders : holders >> first & ((1ull << (LANES % 64)) - 1))) - 1;
    return top;
}

template <int LANES>
__device__ __forceinline__ int from_lane(int v, int lane) {
    if constexpr (LANES == 64) return __builtin_amdgcn_readlane(v, __builtin_amdgcn_readfirstlane(lane));
    return __shfl(v, lane, LANES);
}

template <typename Tr, int LANES, int VPL, typename Key>
__global__ __launch_bounds__(256) void k_route(Route a) {
    constexpr int TOKENS = 256 / LANES;
    __shared__ Key grouped[256 * VPL];
    const int l = threadIdx.x % LANES;
    for (int64_t first = (int64_t)blockIdx.x * TOKENS; first < a.tokens; first += (int64_t)gridDim.x * TOKENS) {
        const int64_t token = first + threadIdx.x / LANES;
        const bool on = token < a.tokens && !(a.mask && !a.mask[token]);
        const int64_t row = token * a.E;
        float x[VPL];
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const int e = l * VPL + i;
            x[i] = on && e < a.E ? logit<Tr>(a.logits, row + e) : -INFINITY;
            top = fmaxf(top, x[i]);
        }
        top = lanes_max<LANES>(top);
        Key key[VPL];
        bool spoiled = false;  // no score of the token is a number
        if constexpr (sizeof(Key) == 4) {
#pragma unroll
            for (int i = 0; i < VPL; ++i) key[i] = key_of(x[i]);
        } else {
            double s[VPL], total = 0.0;
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                s[i] = a.sigmoid ? 1.0 / (1.0 + exp(-(double)x[i])) : exp((double)x[i] - (double)top);
                total += x[i] == -INFINITY ? 0.0 : s[i];
            }
            if (!a.sigmoid) {
                total = lanes_sum<LANES>(total);
                spoiled = total != total;
#pragma unroll
                for (int i = 0; i < VPL; ++i) s[i] /= total;
            }
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                const int e = l * VPL + i;
                if (a.bias && e < a.E) s[i] += (double)a.bias[e];
                key[i] = x[i] == -INFINITY ? 0 : key_of(s[i]);
            }
        }
        if (a.groups > 1) {
            // lane g reads its group's keys back from LDS (groups <= LANES)
            Key* mine = grouped + (threadIdx.x / LANES) * LANES * VPL;
#pragma unroll
            for (int i = 0; i < VPL; ++i) mine[l * VPL + i] = key[i];
            __syncthreads();
            const int size = a.E / a.groups;
            Key best = 0, second = 0;
            if (l < a.groups)
                for (int i = 0; i < size; ++i) {
                    const Key k = mine[l * size + i];
                    second = k > best ? best : k > second ? k : second;
                    best = k > best ? k : best;
                }
            if constexpr (sizeof(Key) == 8)
                if (a.sums && best && second) best = key_of(value_of(best) + value_of(second));
            uint64_t kept = 0;
            for (int j = 0; j < a.top_groups; ++j) {
                int g;
                if (take<LANES>(best, &g)) kept |= 1ull << g;
                if (l == g) best = 0;
            }
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                const int e = l * VPL + i;
                if (e < a.E && !(kept >> (e / size) & 1)) key[i] = 0;
            }
            __syncthreads();
        }
        int chosen = -1;  // lane j: the token's j-th expert
        for (int j = 0; j < a.top_k; ++j) {
            Key best = key[0];
            int at = 0;
#pragma unroll
            for (int i = 1; i < VPL; ++i)
                if (key[i] > best) best = key[i], at = i;
            int holder;
            const Key most = take<LANES>(best, &holder);
            const int e = from_lane<LANES>(l * VPL + at, holder);
            if (l == j && most) chosen = e;
            if (l == holder) {
#pragma unroll
                for (int i = 0; i < VPL; ++i)
                    if (i == at) key[i] = 0;
            }
        }
        // the weights, each lane one
        const float c = chosen >= 0 ? logit<Tr>(a.logits, row + chosen) : -INFINITY;
        float p = 0.0f, total = 1.0f;
        if (!a.sigmoid) {
            // renormalised, the scores' common factor drops out: the largest chosen logit takes its place
            const float m = a.renorm ? lanes_max<LANES>(c) : top;
            p = chosen >= 0 ? expf(c - m) : 0.0f;
            if (a.renorm) {
                total = lanes_sum<LANES>(p);
            } else {
                total = 0.0f;
#pragma unroll
                for (int i = 0; i < VPL; ++i) total += x[i] == -INFINITY ? 0.0f : expf(x[i] - top);
                total = lanes_sum<LANES>(total);
            }
        } else if (a.renorm) {
            // sigmoid(c) = exp(min(c, 0)) / (1 + exp(-|c|)); a common factor keeps the largest of them near one
            const float low = fminf(c, 0.0f), m = lanes_max<LANES>(low);
            p = chosen >= 0 ? (c != c ? c : expf(low - m) / (1.0f + expf(-fabsf(c)))) : 0.0f;
            total = lanes_sum<LANES>(p);
        } else {
            p = chosen >= 0 ? sigmoid_of(c) : 0.0f;
        }
        if (token < a.tokens && l < a.top_k) {
            a.weights[token * a.top_k + l] = chosen < 0 ? 0.0f : spoiled ? __builtin_nanf("") : a.scale * (p / total);
            a.experts[token * a.top_k + l] = chosen;
        }
    }
}

// p_j = the weight before its scale, s_j the score, d_j = scale dw_j.
//   renormalised: softmax  dl_j = p_j (d_j - sum d p), other experts none;   sigmoid  the same times (1 - s_j)
//   else:         softmax  dl_e = s_e (d_e - sum d s), d_e = 0 where not chosen;   sigmoid  dl_j = d_j s_j (1 - s_j)
struct RouteBwd {
    const float* dweights;
    const void* logits;
    const int32_t* experts;
    void* dlogits;
    int64_t tokens;
    int E, top_k;
    bool sigmoid, renorm;
    float scale;
};

template <typename Tr, int LANES, int VPL>
__global__ __launch_bounds__(256) void k_route_bwd(RouteBwd a) {
    constexpr int TOKENS = 256 / LANES;
    __shared__ float scattered[256 * VPL];
    const int l = threadIdx.x % LANES;
    float* mine = scattered + (threadIdx.x / LANES) * LANES * VPL;
    for (int64_t first = (int64_t)blockIdx.x * TOKENS; first < a.tokens; first += (int64_t)gridDim.x * TOKENS) {
        const int64_t token = first + threadIdx.x / LANES;
        const bool on = token < a.tokens;
        const int64_t row = token * a.E;
        int chosen = on && l < a.top_k ? a.experts[token * a.top_k + l] : -1;
        if (chosen >= a.E) chosen = -1;
        const float d = chosen >= 0 ? a.scale * a.dweights[token * a.top_k + l] : 0.0f;
        const float c = chosen >= 0 ? logit<Tr>(a.logits, row + chosen) : -INFINITY;
        const bool any = lanes_max<LANES>((uint32_t)(chosen >= 0));
        const bool whole = !a.sigmoid && !a.renorm;  // every expert has a gradient
        float s[VPL], g, dot = 0.0f;
        if (whole) {
            float top = -INFINITY, total = 0.0f;
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                const int e = l * VPL + i;
                s[i] = any && e < a.E ? logit<Tr>(a.logits, row + e) : -INFINITY;
                top = fmaxf(top, s[i]);
            }
            top = lanes_max<LANES>(top);
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                s[i] = s[i] == -INFINITY ? 0.0f : expf(s[i] - top);
                total += s[i];
            }
            total = lanes_sum<LANES>(total);
#pragma unroll
            for (int i = 0; i < VPL; ++i) s[i] = any ? s[i] / total : 0.0f;
            dot = lanes_sum<LANES>(chosen >= 0 ? d * (expf(c - top) / total) : 0.0f);
            g = d;
        } else if (a.renorm) {
            const float low = a.sigmoid ? fminf(c, 0.0f) : c, m = lanes_max<LANES>(low);
            float p = chosen >= 0 ? (c != c ? c : expf(low - m)) : 0.0f;
            if (a.sigmoid && chosen >= 0) p /= 1.0f + expf(-fabsf(c));
            p /= lanes_sum<LANES>(p);
            dot = lanes_sum<LANES>(chosen >= 0 ? d * p : 0.0f);
            g = p * (d - dot) * (a.sigmoid ? sigmoid_of(-c) : 1.0f);
        } else {
            g = d * sigmoid_of(c) * sigmoid_of(-c);
        }
#pragma unroll
        for (int i = 0; i < VPL; ++i) mine[l * VPL + i] = 0.0f;
        __syncthreads();
        if (chosen >= 0) mine[chosen] = g;
        __syncthreads();
        typename Eight<Tr>::elem* out = static_cast<typename Eight<Tr>::elem*>(a.dlogits);
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const int e = l * VPL + i;
            float v = mine[e];
            if (whole) v = s[i] * (v - dot);
            if (on && e < a.E) out[row + e] = Tr::from_f32(v);
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------ sort
// A counting sort by expert that keeps the slots' order (so equal inputs give equal outputs): a work-group takes a
// stretch of slots, each of its 8 waves an eighth of it in order, 64 slots at a time. Counts first; where there is more
// than one work-group they go to memory, and a second launch sums those of the work-groups before its own.
constexpr int kSortWaves = 8, kSortThreads = 64 * kSortWaves, kSortExperts = 1024, kSortGroups = 64;

struct Sort {
    const int32_t* experts;
    int64_t n, stretch;  // slots, and those of a work-group (a multiple of 64 * kSortWaves)
    int E, groups;
    int32_t *offsets, *slots, *positions;
    int32_t* counts;  // [groups, E]
};

// The wave's slots of a stretch.
__device__ __forceinline__ void wave_part(const Sort& a, int64_t* begin, int64_t* end) {
    const int64_t part = a.stretch / kSortWaves;
    *begin = blockIdx.x * a.stretch + (threadIdx.x / 64) * part;
    *end = *begin + part < a.n ? *begin + part : a.n;
}

__device__ __forceinline__ void count_slots(const Sort& a, int (*cnt)[kSortExperts]) {
    for (int i = threadIdx.x; i < kSortWaves * a.E; i += kSortThreads) cnt[i / a.E][i % a.E] = 0;
    __syncthreads();
    int64_t begin, end;
    wave_part(a, &begin, &end);
    for (int64_t i = begin + (threadIdx.x & 63); i < end; i += 64) {
        const int e = a.experts[i];
        if ((unsigned)e < (unsigned)a.E) atomicAdd(&cnt[threadIdx.x / 64][e], 1);
    }
    __syncthreads();
}

__global__ __launch_bounds__(kSortThreads) void k_sort_count(Sort a) {
    __shared__ int cnt[kSortWaves][kSortExperts];
    count_slots(a, cnt);
    for (int e = threadIdx.x; e < a.E; e += kSortThreads) {
        int s = 0;
        for (int w = 0; w < kSortWaves; ++w) s += cnt[w][e];
        a.counts[(int64_t)blockIdx.x * a.E + e] = s;
    }
}

__global__ __launch_bounds__(kSortThreads) void k_sort(Sort a) {
    __shared__ int cnt[kSortWaves][kSortExperts];
    __shared__ int total[kSortExperts + 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    count_slots(a, cnt);
    // per expert: all rows, and those before this work-group's
    for (int e = threadIdx.x; e < a.E; e += kSortThreads) {
        int before = 0, all = 0;
        if (a.groups == 1) {
            for (int w = 0; w < kSortWaves; ++w) all += cnt[w][e];
        } else {
            for (int g = 0; g < a.groups; ++g) {
                const int c = a.counts[(int64_t)g * a.E + e];
                before += g < (int)blockIdx.x ? c : 0;
                all += c;
            }
        }
        total[e] = all;
        for (int w = 0; w < kSortWaves; ++w) {
            const int c = cnt[w][e];
            cnt[w][e] = before;
            before += c;
        }
    }
    __syncthreads();
    if (wave == 0) {  // exclusive sums over the experts, a run of them a lane
        const int run = (a.E + 63) / 64;
        int s = 0;
        for (int e = lane * run; e < min((lane + 1) * run, a.E); ++e) s += total[e];
        int upto = s;
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(upto, d);
            upto += lane >= d ? o : 0;
        }
        int at = upto - s;
        for (int e = lane * run; e < min((lane + 1) * run, a.E); ++e) {
            const int c = total[e];
            total[e] = at;
            at += c;
        }
        if (lane == 63) total[a.E] = upto;
    }
    __syncthreads();
    if (blockIdx.x == 0)
        for (int e = threadIdx.x; e <= a.E; e += kSortThreads) a.offsets[e] = total[e];
    int64_t begin, end;
    wave_part(a, &begin, &end);
    const int live = total[a.E];
    volatile int* next = cnt[wave];
    for (int64_t i0 = begin; i0 < end; i0 += 64) {
        const int64_t i = i0 + lane;
        int e = i < end ? a.experts[i] : -1;
        const bool has = (unsigned)e < (unsigned)a.E;
        if (!has) e = 0;
        // the lanes of this expert
        uint64_t same = __ballot(has);
        for (int b = 1; b < a.E; b <<= 1) {
            const uint64_t ones = __ballot(e & b);
            same &= e & b ? ones : ~ones;
        }
        const int rank = __popcll(same & ((1ull << lane) - 1));
        const int at = has ? next[e] : 0;
        __builtin_amdgcn_wave_barrier();
        if (has && rank == 0) next[e] = at + __popcll(same);
        __builtin_amdgcn_wave_barrier();
        if (i < end) {
            const int p = has ? total[e] + at + rank : -1;
            a.positions[i] = p;
            if (has) a.slots[p] = (int32_t)i;
        }
    }
    // the slots without an expert leave as many rows over
    for (int64_t i = blockIdx.x * a.stretch + threadIdx.x; i < min((int64_t)(blockIdx.x + 1) * a.stretch, a.n);
         i += kSortThreads)
        if (i >= live) a.slots[i] = -1;
}

int sort_groups(int64_t n, int64_t* stretch) {
    constexpr int64_t unit = kSortThreads;
    int64_t s = 1024;
    if ((n + s - 1) / s > kSortGroups) s = (n + kSortGroups - 1) / kSortGroups;
    s = (s + unit - 1) / unit * unit;
    if (n <= 2048) s = 2048;  // one launch
    *stretch = s;
    return (int)((n + s - 1) / s);
}

// ------------------------------------------------------------ rows by expert, and back
// A wave takes 512 columns of a token, 8 a lane; the token's positions are uniform.
struct Rows {
    const void *in, *other;    // gather: x; combine: y and the residual; its gradients: dout and y
    const float* weights;      // null: ones
    const int32_t *positions, *offsets;
    void* out;
    float* dweights;
    int64_t tokens, hidden, rows;  // rows: of the experts' side
    int top_k, E;
    bool wide;  // the tokens' side (residual and out, dout) is fp32 whatever y is
};

// 8 elements of a row of the tokens' side.
template <typename Tr>
__device__ __forceinline__ void load_stream(const void* p, bool wide, int64_t at, int n, float (&f)[8]) {
    if (wide) {
        Eight<F32> e;
        e.load(p, at, n);
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = e.get(k);
    } else {
        Eight<Tr> e;
        e.load(p, at, n);
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = e.get(k);
    }
}

// Rows from offsets[E] on belong to no slot: zeros. Called by all waves, `wave` of `waves`.
template <typename Tr>
__device__ __forceinline__ void clear_tail(const Rows& a, void* out, int64_t wave, int64_t waves) {
    int64_t live = a.offsets[a.E];
    if (live < 0) live = 0;
    if (live >= a.rows) return;
    const int64_t chunks = (a.hidden + 511) / 512;
    Eight<Tr> zero;
    zero.clear();
    for (int64_t i = live * chunks + wave; i < a.rows * chunks; i += waves) {
        const int64_t row = i / chunks, c = (i - row * chunks) * 512 + 8 * (threadIdx.x & 63);
        const int64_t n = a.hidden - c;
        zero.store(out, row * a.hidden + c, n < 8 ? (int)n : 8);
    }
}

template <typename Tr>
__global__ __launch_bounds__(256) void k_gather(Rows a) {
    const int64_t chunks = (a.hidden + 511) / 512, waves = (int64_t)gridDim.x * 4;
    const int64_t wave = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int64_t i = wave; i < a.tokens * chunks; i += waves) {
        const int64_t token = i / chunks, c = (i - token * chunks) * 512 + 8 * (threadIdx.x & 63);
        const int64_t left = a.hidden - c;
        const int n = left < 8 ? (int)left : 8;
        Eight<Tr> v;
        v.load(a.in, token * a.hidden + c, n);
        for (int j = 0; j < a.top_k; ++j) {
            const int64_t p = a.positions[token * a.top_k + j];
            if (p >= 0 && p < a.rows) v.store(a.out, p * a.hidden + c, n);
        }
    }
    clear_tail<Tr>(a, a.out, wave, waves);
}

template <typename Tr>
__global__ __launch_bounds__(256) void k_combine(Rows a) {
    const int64_t chunks = (a.hidden + 511) / 512, waves = (int64_t)gridDim.x * 4;
    const int64_t wave = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int64_t i = wave; i < a.tokens * chunks; i += waves) {
        const int64_t token = i / chunks, c = (i - token * chunks) * 512 + 8 * (threadIdx.x & 63);
        const int64_t left = a.hidden - c;
        const int n = left < 8 ? (int)left : 8;
        float s[8] = {};
        if (a.other) load_stream<Tr>(a.other, a.wide, token * a.hidden + c, n, s);
        for (int j = 0; j < a.top_k; ++j) {
            const int64_t slot = token * a.top_k + j, p = a.positions[slot];
            if (p < 0 || p >= a.rows) continue;
            const float w = a.weights ? a.weights[slot] : 1.0f;
            Eight<Tr> y;
            y.load(a.in, p * a.hidden + c, n);
#pragma unroll
            for (int k = 0; k < 8; ++k) s[k] = __builtin_fmaf(w, y.get(k), s[k]);
        }
        if (a.wide) {
            Eight<F32> o;
            o.set(s);
            o.store(a.out, token * a.hidden + c, n);
        } else {
            Eight<Tr> o;
            o.set(s);
            o.store(a.out, token * a.hidden + c, n);
        }
    }
}

// A work-group takes a token: its waves walk the columns, and their sums meet in LDS. J slots at a time.
template <typename Tr, int J>
__global__ __launch_bounds__(256) void k_combine_bwd(Rows a) {
    __shared__ float part[4][J];
    const int lane = threadIdx.x & 63, w4 = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int64_t token = blockIdx.x; token < a.tokens; token += gridDim.x) {
        for (int j0 = 0; j0 < a.top_k; j0 += J) {
            float dot[J] = {};
            for (int64_t c = 8 * threadIdx.x; c < a.hidden; c += 2048) {
                const int64_t left = a.hidden - c;
                const int n = left < 8 ? (int)left : 8;
                float d[8];
                load_stream<Tr>(a.in, a.wide, token * a.hidden + c, n, d);
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    if (j0 + j >= a.top_k) continue;
                    const int64_t slot = token * a.top_k + j0 + j, p = a.positions[slot];
                    if (p < 0 || p >= a.rows) continue;
                    if (a.dweights) {
                        Eight<Tr> y;
                        y.load(a.other, p * a.hidden + c, n);
#pragma unroll
                        for (int k = 0; k < 8; ++k) dot[j] = __builtin_fmaf(d[k], y.get(k), dot[j]);
                    }
                    if (a.out) {
                        const float w = a.weights[slot];
                        float g[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) g[k] = w * d[k];
                        Eight<Tr> o;
                        o.set(g);
                        o.store(a.out, p * a.hidden + c, n);
                    }
                }
            }
            if (!a.dweights) continue;
#pragma unroll
            for (int j = 0; j < J; ++j) {
                dot[j] = lanes_sum<64>(dot[j]);
                if (lane == 0) part[w4][j] = dot[j];
            }
            __syncthreads();
            if (threadIdx.x < J && j0 + (int)threadIdx.x < a.top_k)
                a.dweights[token * a.top_k + j0 + threadIdx.x] =
                    part[0][threadIdx.x] + part[1][threadIdx.x] + part[2][threadIdx.x] + part[3][threadIdx.x];
            __syncthreads();
        }
    }
    if (a.out) clear_tail<Tr>(a, a.out, (int64_t)blockIdx.x * 4 + w4, (int64_t)gridDim.x * 4);
}

bool known(int dtype) { return dtype == STM_F16 || dtype == STM_BF16 || dtype == STM_F32; }
bool lies(const void* p, int dtype) { return aligned(p, dtype == STM_F32 ? 4 : 2); }

// f(type, lanes, values a lane) of the form that holds a token's experts.
template <typename Tr, typename F>
int each_width(int E, F f) {
    using std::integral_constant;
    if (E <= 8) return f(Tr{}, integral_constant<int, 8>{}, integral_constant<int, 1>{});
    if (E <= 16) return f(Tr{}, integral_constant<int, 16>{}, integral_constant<int, 1>{});
    if (E <= 32) return f(Tr{}, integral_constant<int, 32>{}, integral_constant<int, 1>{});
    if (E <= 64) return f(Tr{}, integral_constant<int, 64>{}, integral_constant<int, 1>{});
    if (E <= 128) return f(Tr{}, integral_constant<int, 64>{}, integral_constant<int, 2>{});
    if (E <= 256) return f(Tr{}, integral_constant<int, 64>{}, integral_constant<int, 4>{});
    if (E <= 512) return f(Tr{}, integral_constant<int, 64>{}, integral_constant<int, 8>{});
    return f(Tr{}, integral_constant<int, 64>{}, integral_constant<int, 16>{});
}

template <typename F>
int each_route(int dtype, int E, F f) {
    if (dtype == STM_BF16) return each_width<BF16>(E, f);
    if (dtype == STM_F16) return each_width<F16>(E, f);
    return each_width<F32>(E, f);
}

int check_route(const char* what, int64_t tokens, int E, int top_k, int score, int dtype) {
    if (tokens < 0) return set_error(STM_ERR_INVALID, "%s: negative size", what);
    if (!known(dtype)) return set_error(STM_ERR_INVALID, "%s: dtype must be fp16, bf16 or fp32", what);
    if (E < 1 || E > kSortExperts)
        return set_error(STM_ERR_UNSUPPORTED, "%s: 1 to %d experts, got %d", what, kSortExperts, E);
    if (top_k < 1 || top_k > E || top_k > 64)
        return set_error(STM_ERR_INVALID, "%s: top_k must be from 1 to min(experts, 64), got %d", what, top_k);
    if (score != STM_MOE_SOFTMAX && score != STM_MOE_SIGMOID)
        return set_error(STM_ERR_INVALID, "%s: unknown score %d", what, score);
    if (tokens >= (1ll << 31) / top_k) return set_error(STM_ERR_UNSUPPORTED, "%s: 2^31 slots or more", what);
    return STM_OK;
}

int check_rows(const char* what, int64_t tokens, int top_k, int64_t hidden, int dtype) {
    if (tokens < 0 || hidden < 0 || top_k < 0) return set_error(STM_ERR_INVALID, "%s: negative size", what);
    if (!known(dtype)) return set_error(STM_ERR_INVALID, "%s: dtype must be fp16, bf16 or fp32", what);
    if (top_k && tokens >= (1ll << 31) / top_k) return set_error(STM_ERR_UNSUPPORTED, "%s: 2^31 slots or more", what);
    if (tokens >= (1ll << 31) || hidden >= (1ll << 28))
        return set_error(STM_ERR_UNSUPPORTED, "%s: %lld tokens of %lld columns are too many", what, (long long)tokens,
                         (long long)hidden);
    return STM_OK;
}

template <typename F>
int each_type(int dtype, F f) {
    return dtype == STM_BF16 ? f(BF16{}) : dtype == STM_F16 ? f(F16{}) : f(F32{});
}

}  // namespace
}  // namespace stm

using namespace stm;

extern "C" int stm_moe_route(const void* logits, const float* bias, const uint8_t* mask, float* weights, int32_t* experts,
                             int64_t tokens, int num_experts, int top_k, int score, int groups, int top_groups,
                             int group_sums, int renormalize, double scale, int dtype, void* stream) {
    const char* what = "moe_route";
    const int rc = check_route(what, tokens, num_experts, top_k, score, dtype);
    if (rc) return rc;
    if (groups < 1 || groups > 64 || num_experts % groups)
        return set_error(STM_ERR_INVALID, "%s: %d experts do not make %d groups (1 to 64)", what, num_experts, groups);
    if (top_groups < 1 || top_groups > groups)
        return set_error(STM_ERR_INVALID, "%s: %d of %d groups", what, top_groups, groups);
    if (top_k > num_experts / groups * top_groups)
        return set_error(STM_ERR_INVALID, "%s: %d groups hold fewer than %d experts", what, top_groups, top_k);
    if (tokens == 0) return STM_OK;
    if (!logits || !weights || !experts) return set_error(STM_ERR_INVALID, "%s: null pointer", what);
    if (!lies(logits, dtype) || !aligned(bias, 4) || !aligned(weights, 4) || !aligned(experts, 4))
        return set_error(STM_ERR_INVALID, "%s: pointers must be aligned to their elements", what);
    const bool sums = group_sums && groups > 1;
    const Route a{logits, bias, mask, weights, experts, tokens, num_experts, top_k, groups, top_groups,
                  score == STM_MOE_SIGMOID, sums, renormalize != 0, (float)scale};
    return each_route(dtype, num_experts, [&](auto tr, auto lanes, auto vpl) {
        const dim3 grid(groups_for(tokens, 256 / lanes.value)), block(256);
        if (bias || sums)
            hipLaunchKernelGGL((k_route<decltype(tr), lanes.value, vpl.value, uint64_t>), grid, block, 0,
                               (hipStream_t)stream, a);
        else
            hipLaunchKernelGGL((k_route<decltype(tr), lanes.value, vpl.value, uint32_t>), grid, block, 0,
                               (hipStream_t)stream, a);
        return check_launch(what);
    });
}

extern "C" int stm_moe_route_bwd(const float* dweights, const void* logits, const int32_t* experts, void* dlogits,
                                 int64_t tokens, int num_experts, int top_k, int score, int renormalize, double scale,
                                 int dtype, void* stream) {
    const char* what = "moe_route_bwd";
    const int rc = check_route(what, tokens, num_experts, top_k, score, dtype);
    if (rc) return rc;
    if (tokens == 0) return STM_OK;
    if (!dweights || !logits || !experts || !dlogits) return set_error(STM_ERR_INVALID, "%s: null pointer", what);
    if (!lies(logits, dtype) || !lies(dlogits, dtype) || !aligned(dweights, 4) || !aligned(experts, 4))
        return set_error(STM_ERR_INVALID, "%s: pointers must be aligned to their elements", what);
    const RouteBwd a{dweights, logits, experts, dlogits, tokens, num_experts, top_k, score == STM_MOE_SIGMOID,
                     renormalize != 0, (float)scale};
    return each_route(dtype, num_experts, [&](auto tr, auto lanes, auto vpl) {
        hipLaunchKernelGGL((k_route_bwd<decltype(tr), lanes.value, vpl.value>), dim3(groups_for(tokens, 256 / lanes.value)),
                           dim3(256), 0, (hipStream_t)stream, a);
        return check_launch(what);
    });
}

static int check_sort(const char* what, int64_t n, int num_experts) {
    if (n < 0 || n >= (1ll << 31)) return set_error(STM_ERR_INVALID, "%s: 0 to 2^31 - 1 slots", what);
    if (num_experts < 1 || num_experts > kSortExperts)
        return set_error(STM_ERR_UNSUPPORTED, "%s: 1 to %d experts, got %d", what, kSortExperts, num_experts);
    return STM_OK;
}

extern "C" int64_t stm_moe_sort_workspace_bytes(int64_t slots, int num_experts) {
    const int rc = check_sort("moe_sort_workspace_bytes", slots, num_experts);
    if (rc) return rc;
    int64_t stretch;
    const int groups = sort_groups(slots, &stretch);
    return groups > 1 ? (int64_t)groups * num_experts * 4 : 0;
}

extern "C" int stm_moe_sort(const int32_t* experts, int64_t n, int num_experts, int32_t* offsets, int32_t* slots,
                            int32_t* positions, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* what = "moe_sort";
    const int rc = check_sort(what, n, num_experts);
    if (rc) return rc;
    if (!offsets || (n && (!experts || !slots || !positions))) return set_error(STM_ERR_INVALID, "%s: null pointer", what);
    if (!aligned(offsets, 4) || !aligned(experts, 4) || !aligned(slots, 4) || !aligned(positions, 4) || !aligned(workspace, 4))
        return set_error(STM_ERR_INVALID, "%s: pointers must be aligned to their elements", what);
    Sort a{experts, n, 0, num_experts, 0, offsets, slots, positions, static_cast<int32_t*>(workspace)};
    a.groups = sort_groups(n, &a.stretch);
    if (a.groups < 1) a.groups = 1;
    if (a.groups > 1) {
        const int64_t need = (int64_t)a.groups * num_experts * 4;
        if (!workspace || workspace_bytes < need)
            return set_error(STM_ERR_INVALID, "%s: needs a workspace of %lld bytes, got %lld", what, (long long)need,
                             (long long)(workspace ? workspace_bytes : 0));
        hipLaunchKernelGGL(k_sort_count, dim3(a.groups), dim3(kSortThreads), 0, (hipStream_t)stream, a);
    }
    hipLaunchKernelGGL(k_sort, dim3(a.groups), dim3(kSortThreads), 0, (hipStream_t)stream, a);
    return check_launch(what);
}

extern "C" int stm_moe_gather(const void* x, const int32_t* positions, const int32_t* offsets, int num_experts, void* out,
                              int64_t tokens, int top_k, int64_t hidden, int dtype, void* stream) {
    const char* what = "moe_gather";
    const int rc = check_rows(what, tokens, top_k, hidden, dtype);
    if (rc) return rc;
    if (num_experts < 1) return set_error(STM_ERR_INVALID, "%s: no experts", what);
    if (tokens == 0 || hidden == 0 || top_k == 0) return STM_OK;
    if (!x || !positions || !offsets || !out) return set_error(STM_ERR_INVALID, "%s: null pointer", what);
    if (!lies(x, dtype) || !lies(out, dtype) || !aligned(positions, 4) || !aligned(offsets, 4))
        return set_error(STM_ERR_INVALID, "%s: pointers must be aligned to their elements", what);
    const Rows a{x, nullptr, nullptr, positions, offsets, out, nullptr, tokens, hidden, tokens * top_k, top_k, num_experts, false};
    return each_type(dtype, [&](auto tr) {
        hipLaunchKernelGGL(k_gather<decltype(tr)>, dim3(groups_for(tokens * ((hidden + 511) / 512), 4)), dim3(256), 0,
                           (hipStream_t)stream, a);
        return check_launch(what);
    });
}

extern "C" int stm_moe_combine(const void* y, int64_t y_rows, const float* weights, const int32_t* positions,
                               const void* residual, void* out, int out_dtype, int64_t tokens, int top_k, int64_t hidden,
                               int dtype, void* stream) {
    const char* what = "moe_combine";
    const int rc = check_rows(what, tokens, top_k, hidden, dtype);
    if (rc) return rc;
    if (out_dtype != dtype && out_dtype != STM_F32)
        return set_error(STM_ERR_INVALID, "%s: the output must be of y's type or fp32", what);
    if (y_rows < 0 || y_rows > tokens * top_k)
        return set_error(STM_ERR_INVALID, "%s: %lld rows for %lld slots", what, (long long)y_rows,
                         (long long)(tokens * top_k));
    if (tokens == 0 || hidden == 0) return STM_OK;
    if ((y_rows && !y) || (top_k && !positions) || !out) return set_error(STM_ERR_INVALID, "%s: null pointer", what);
    if (!lies(y, dtype) || !lies(out, out_dtype) || !lies(residual, out_dtype) || !aligned(positions, 4) || !aligned(weights, 4))
        return set_error(STM_ERR_INVALID, "%s: pointers must be aligned to their elements", what);
    const Rows a{y, residual, weights, positions, nullptr, out, nullptr, tokens, hidden, y_rows, top_k, 0, out_dtype == STM_F32};
    return each_type(dtype, [&](auto tr) {
        hipLaunchKernelGGL(k_combine<decltype(tr)>, dim3(groups_for(tokens * ((hidden + 511) / 512), 4)), dim3(256), 0,
                           (hipStream_t)stream, a);
        return check_launch(what);
    });
}

extern "C" int stm_moe_combine_bwd(const void* dout, int dout_dtype, const void* y, int64_t y_rows, const float* weights,
                                   const int32_t* positions, const int32_t* offsets, int num_experts, void* dy,
                                   float* dweights, int64_t tokens, int top_k, int64_t hidden, int dtype, void* stream) {
    const char* what = "moe_combine_bwd";
    const int rc = check_rows(what, tokens, top_k, hidden, dtype);
    if (rc) return rc;
    if (num_experts < 1) return set_error(STM_ERR_INVALID, "%s: no experts", what);
    if (dout_dtype != dtype && dout_dtype != STM_F32)
        return set_error(STM_ERR_INVALID, "%s: dout must be of y's type or fp32", what);
    if (y_rows < 0 || y_rows > tokens * top_k)
        return set_error(STM_ERR_INVALID, "%s: %lld rows for %lld slots", what, (long long)y_rows,
                         (long long)(tokens * top_k));
    if (tokens == 0 || top_k == 0 || (!dy && !dweights)) return STM_OK;
    if (!positions || (hidden && (!dout || (y_rows && ((dweights && !y) || (dy && (!weights || !offsets)))))))
        return set_error(STM_ERR_INVALID, "%s: null pointer", what);
    if (!lies(dout, dout_dtype) || !lies(y, dtype) || !lies(dy, dtype) || !aligned(positions, 4) || !aligned(weights, 4) ||
        !aligned(offsets, 4) || !aligned(dweights, 4))
        return set_error(STM_ERR_INVALID, "%s: pointers must be aligned to their elements", what);
    const Rows a{dout, y, weights, positions, offsets, y_rows ? dy : nullptr, dweights, tokens, hidden, y_rows, top_k, num_experts,
                 dout_dtype == STM_F32};
    return each_type(dtype, [&](auto tr) {
        const dim3 grid((unsigned)(tokens < (1 << 22) ? tokens : 1 << 22)), block(256);
        hipStream_t st = (hipStream_t)stream;
        if (top_k <= 1)
            hipLaunchKernelGGL((k_combine_bwd<decltype(tr), 1>), grid, block, 0, st, a);
        else if (top_k <= 2)
            hipLaunchKernelGGL((k_combine_bwd<decltype(tr), 2>), grid, block, 0, st, a);
        else if (top_k <= 4)
            hipLaunchKernelGGL((k_combine_bwd<decltype(tr), 4>), grid, block, 0, st, a);
        else
            hipLaunchKernelGGL((k_combine_bwd<decltype(tr), 8>), grid, block, 0, st, a);
        return check_launch(what);
    });
}
