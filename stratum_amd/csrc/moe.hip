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
// A token belongs to LANES lanes of a wave, lane l holds experts l * VPL .. l * VPL + VPL - 1. No barrier: what a token has
// in LDS is its wave's. One expert is taken per round: the maximum over a lane's keys, over the lanes (DPP), the lowest
// index that holds it. Bound by instructions: with 8 values a lane the steps over the lanes, and the exponentials of
// the weights, serve two to four tokens at a time (8192 tokens of 128 in bf16, top 8, us: 64 lanes of 2 values 7.4, 16 of 8
// 4.3).
//
// Keys are compared as what they stand for, the lowest index first among equal ones; an expert that cannot be chosen
// has none (-inf; as an unsigned integer 0). Without a bias and without sums over groups the scores are in the order of
// the logits, which are compared as they are (integers in their order, NaN above all; of 16-bit types the low 10 bits,
// which are free, hold the index, so that no two are equal and one maximum finds both). Otherwise the keys are those of
// score + bias in 64 bits: two experts whose keys differ by less than an fp32 rounding are still told apart, and the same
// ones are found as by any other program that computes them so. They are computed in 32 bits first, with a bound on what that
// may be off. Where experts that follow each other are nearer than the bound, the keys of those taken are computed in
// 64 bits, by a lane each; where groups are (or a value is not finite), all of them (16383 tokens of 256, sigmoid, bias, 8
// groups, us: always 43, so 29; 22 if no token needed them).
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

__device__ __forceinline__ float value_of(uint32_t k) {
    return k == ~0u ? __builtin_nanf("") : __uint_as_float(k >> 31 ? k & ~(1u << 31) : ~k);
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

// A lane's N values of a row (of the n that are left), `fill` behind its end; whole ones in one access at any address.
template <typename Tr, int N>
struct Few {
    typedef typename Eight<Tr>::elem elem;
    typedef elem vec __attribute__((ext_vector_type(N)));
    typedef vec loose __attribute__((aligned(sizeof(elem))));

    static __device__ __forceinline__ void load(const void* base, int64_t at, int n, float fill, float (&f)[N]) {
        const elem* p = static_cast<const elem*>(base) + at;
        if (n >= N) {
            const vec v = *reinterpret_cast<const loose*>(p);
#pragma unroll
            for (int i = 0; i < N; ++i) f[i] = Tr::to_f32(v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) f[i] = i < n ? Tr::to_f32(p[i]) : fill;
        }
    }
    static __device__ __forceinline__ void store(void* base, int64_t at, int n, const float (&f)[N]) {
        elem* p = static_cast<elem*>(base) + at;
        if (n >= N) {
            vec v;
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = Tr::from_f32(f[i]);
            *reinterpret_cast<loose*>(p) = v;
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (i < n) p[i] = Tr::from_f32(f[i]);
        }
    }
};

// What the wave wrote to LDS before is there for all its lanes (they execute in order; this holds the compiler to it).
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <typename Key>
__device__ __forceinline__ Key none() {
    return std::is_same_v<Key, float> ? (Key)-INFINITY : (Key)0;
}

template <typename Key>
__device__ __forceinline__ Key larger(Key a, Key b) {
    if constexpr (std::is_same_v<Key, float>)
        return fmaxf(a, b);
    else
        return a > b ? a : b;
}

__device__ __forceinline__ float value_of(float k) { return k; }

__device__ __forceinline__ uint32_t other_lane(uint32_t v, int step) {  // step is uniform
    return step == 1 ? across<1>(v) : step == 2 ? across<2>(v) : step == 4 ? across<4>(v) : step == 8 ? across<8>(v) :
           step == 16 ? across<16>(v) : across<32>(v);
}

__device__ __forceinline__ uint64_t other_lane(uint64_t v, int step) {
    return (uint64_t)other_lane((uint32_t)(v >> 32), step) << 32 | other_lane((uint32_t)v, step);
}

__device__ __forceinline__ float other_lane(float v, int step) {
    return __uint_as_float(other_lane(__float_as_uint(v), step));
}

// What decides between a token's groups.
struct Border {
    float least, next;  // the smallest value of an eligible group, the largest of the others (-inf: none)
    float size;         // the largest sum of the magnitudes that make a value
};

// Takes away the keys of the groups that are not eligible. A group belongs to `share` lanes (a power of two), which read
// its keys back from LDS, `mine` [LANES * VPL]. key: the experts' keys for this; out: those to take away from.
template <int LANES, int VPL, typename Key, typename Out>
__device__ __forceinline__ void keep_groups(const Route& a, const Key (&key)[VPL], Out (&out)[VPL], Key* mine, Border* border) {
    typedef std::conditional_t<LANES <= 32, uint32_t, uint64_t> Bits;
    const int l = threadIdx.x % LANES, size = a.E / a.groups;
    wave_sync();
#pragma unroll
    for (int i = 0; i < VPL; ++i) mine[l * VPL + i] = key[i];
    wave_sync();
    const int bits = 31 - __clz(LANES / a.groups), share = 1 << bits, group = l >> bits;
    Key best = none<Key>(), second = none<Key>();
    if (group < a.groups)
        for (int i = l & (share - 1); i < size; i += share) {
            const Key k = mine[group * size + i];
            second = larger(second, k > best ? best : k);
            best = larger(best, k);
        }
    for (int step = 1; step < share; step <<= 1) {
        const Key b = other_lane(best, step), s = other_lane(second, step);
        second = larger(larger(second, s), b > best ? best : b);
        best = larger(best, b);
    }
    border->size = 0.0f;
    if (a.sums && second > none<Key>()) {
        const auto v = value_of(best), w = value_of(second);
        border->size = fabsf((float)v) + fabsf((float)w);
        if constexpr (std::is_same_v<Key, float>)
            best = v + w;
        else
            best = (Key)key_of(v + w);
    }
    border->size = lanes_max<LANES>(border->size);
    Bits kept = 0;
    Key least = none<Key>();
    for (int j = 0; j < a.top_groups; ++j) {
        least = lanes_max<LANES>(best);
        const uint32_t g = lanes_min<LANES>(best == least ? (uint32_t)group : 63u);
        if (least > none<Key>()) kept |= (Bits)1 << g;
        if ((uint32_t)group == g) best = none<Key>();
    }
    const Key next = lanes_max<LANES>(best);
    border->least = (float)value_of(least);
    border->next = next > none<Key>() ? (float)value_of(next) : -INFINITY;
    int g = l * VPL / size, left = (g + 1) * size - l * VPL;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        if (g < a.groups && !(kept >> g & 1)) out[i] = none<Out>();
        if (--left == 0) ++g, left = size;
    }
}

// The largest of a token's keys.
template <int LANES, int VPL, typename Key>
__device__ __forceinline__ Key largest(const Key (&key)[VPL]) {
    Key top = key[0];
#pragma unroll
    for (int i = 1; i < VPL; ++i) top = larger(top, key[i]);
    return lanes_max<LANES>(top);
}

// Takes it away and says whose it is. PACKED: a key's low 10 bits are 1023 - its expert.
template <int LANES, int VPL, bool PACKED, typename Key>
__device__ __forceinline__ int take(Key (&key)[VPL], Key top) {
    const int l = threadIdx.x % LANES;
    if constexpr (PACKED) {
#pragma unroll
        for (int i = 0; i < VPL; ++i)
            if (key[i] == top) key[i] = 0;
        return 1023 - (int)(top & 1023);
    } else {
        uint32_t at = 1u << 20;
#pragma unroll
        for (int i = VPL - 1; i >= 0; --i)
            if (key[i] == top) at = i;
        const int e = (int)lanes_min<LANES>(at + l * VPL), mine = e - l * VPL;
#pragma unroll
        for (int i = 0; i < VPL; ++i)
            if (mine == i) key[i] = none<Key>();
        return e;
    }
}

// Lane j gets the token's j-th expert (or -1) and its key.
template <int LANES, int VPL, bool PACKED, typename Key>
__device__ __forceinline__ int best_experts(const Route& a, Key (&key)[VPL], Key* of) {
    int chosen = -1;
    *of = none<Key>();
    for (int j = 0; j < a.top_k; ++j) {
        const Key top = largest<LANES, VPL>(key);
        const int e = take<LANES, VPL, PACKED>(key, top);
        if ((int)(threadIdx.x % LANES) == j && top > none<Key>()) chosen = e, *of = top;
    }
    return chosen;
}

// SCORES: with a bias, or sums over groups.
template <typename Tr, int LANES, int VPL, bool SCORES>
__global__ __launch_bounds__(256) void k_route(Route a) {
    typedef std::conditional_t<SCORES, uint64_t, uint32_t> Key;
    constexpr int TOKENS = 256 / LANES;
    __shared__ Key grouped[256 * VPL];
    const int l = threadIdx.x % LANES, left = a.E - l * VPL;
    Key* mine = grouped + (threadIdx.x / LANES) * LANES * VPL;
    float bias[VPL];
    if constexpr (SCORES)
        if (a.bias) Few<F32, VPL>::load(a.bias, l * VPL, left, 0.0f, bias);
    for (int64_t first = (int64_t)blockIdx.x * TOKENS; first < a.tokens; first += (int64_t)gridDim.x * TOKENS) {
        const int64_t token = first + threadIdx.x / LANES;
        const bool on = token < a.tokens && !(a.mask && !a.mask[token]);
        const int64_t row = token * a.E;
        float x[VPL];
        Few<Tr, VPL>::load(a.logits, row + l * VPL, on ? left : 0, -INFINITY, x);
        float top = x[0];
#pragma unroll
        for (int i = 1; i < VPL; ++i) top = fmaxf(top, x[i]);
        top = lanes_max<LANES>(top);
        Border border;
        int chosen;
        float c;  // the chosen expert's logit
        bool spoiled = false;  // no score of the token is a number
        if constexpr (!SCORES) {
            constexpr bool PACKED = sizeof(typename Eight<Tr>::elem) == 2;
            uint32_t key[VPL], of;
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                key[i] = key_of(x[i]);
                if (PACKED && key[i]) key[i] = (key[i] & ~1023u) | (1023 - (l * VPL + i));
            }
            if (a.groups > 1) keep_groups<LANES>(a, key, key, mine, &border);
            chosen = best_experts<LANES, VPL, PACKED>(a, key, &of);
            if constexpr (PACKED) {
                if (of >> 10 == ~0u >> 10) c = __builtin_nanf("");
                else c = __uint_as_float((of >> 31 ? of & ~(1u << 31) : ~of) & ~1023u);
            } else {
                c = value_of(of);
            }
            if (chosen < 0) c = -INFINITY;
        } else {
            // In units of u = 2^-24 a score is off by at most, where the exponential is 2^(x log2 e) with a relative error
            // of 3 |x| + 2 and a reciprocal has 2: sigmoid, e = exp(-|x|), by the exponential ((3 |x| + 2) e, at most 4),
            // 1 + e (1), the reciprocal (2) and the product with e (1): 8 u; softmax, by the exponential (with d = top - x
            // (3 d + 2) exp(-d), at most 4), the sum of at most 16 values a lane over 64 lanes (22) of terms that are off by
            // 3 d + 2 (on average d is at most ln 1024 = 7: 23), the reciprocal and the product (3): 52 u of the largest
            // score. `off` takes 10 and 56. Adding the bias is off by u of the key; a group's sum by its keys' and u of itself.
            constexpr float u = 0x1p-24f;
            float key[VPL], order[VPL], total = 0.0f, off = 10.0f * u;
            bool close = false;
            constexpr float log2e = 1.44269504088896340736f;
            if (a.sigmoid) {
#pragma unroll
                for (int i = 0; i < VPL; ++i) {
                    const float e = __builtin_amdgcn_exp2f(-log2e * fabsf(x[i])), r = __builtin_amdgcn_rcpf(1.0f + e);
                    key[i] = x[i] < 0.0f ? e * r : r;
                }
            } else {
#pragma unroll
                for (int i = 0; i < VPL; ++i) {
                    key[i] = x[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(log2e * (x[i] - top));
                    total += key[i];
                }
                const float r = __builtin_amdgcn_rcpf(lanes_sum<LANES>(total));
                off = 56.0f * u * r;
#pragma unroll
                for (int i = 0; i < VPL; ++i) key[i] *= r;
            }
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                key[i] = x[i] == -INFINITY ? -INFINITY : a.bias ? key[i] + bias[i] : key[i];
                close |= !(key[i] < INFINITY && x[i] < INFINITY);
                order[i] = a.bias ? key[i] : x[i];
            }
            if (a.groups > 1) {
                keep_groups<LANES>(a, key, order, reinterpret_cast<float*>(mine), &border);
                const float err = (a.sums ? 2.0f * off + u * border.size : off) +
                                  u * (fabsf(border.least) + fabsf(border.next));
                close |= border.next > -INFINITY && !(border.least - border.next > 2.0f * err);
            }
            // Without a bias the scores are in the order of the logits, and equal where the logits are. Different logits have
            // scores that are certainly apart in 64 bits too (`parted`, of the larger and the smaller) unless they are less
            // than u apart or where the scores end (a sigmoid beyond 16 is 1 - exp(-x): u exp(-16) is 2^-47; exp(-700) is
            // still normal). Equal logits are in the right order by themselves, but not if one of them may have the score of a
            // logit outside: of a larger one (`linked`), or of a smaller one with a lower index.
            // Lane j takes the j-th key, beyond top_k until the next one is smaller for certain.
            const auto parted = [&](float more, float less) {
                return more - less > u && (a.sigmoid ? more <= 16.0f && less > -700.0f : top - less < 700.0f);
            };
            bool mixed = false, linked = false;
            float before = 0.0f;
            int taken = 0;
            chosen = -1;
            for (;; ++taken) {
                const float k = largest<LANES, VPL>(order);
                bool apart = true, ends = false;  // ends: the choice among equal logits, if no smaller one has their score
                if (taken && k > -INFINITY) {
                    if (a.bias) {
                        apart = before - k > 2.0f * (off + u * (fabsf(before) + fabsf(k)));
                    } else if (before == k) {
                        apart = !linked;
                        ends = apart && taken >= a.top_k;
                    } else {
                        apart = parted(before, k);
                        linked = !apart;
                    }
                }
                if (!a.bias && __any(ends)) {
                    float below = -INFINITY;
#pragma unroll
                    for (int i = 0; i < VPL; ++i) below = fmaxf(below, order[i] < k ? order[i] : -INFINITY);
                    below = lanes_max<LANES>(below);
                    if (ends && below > -INFINITY) apart = parted(k, below);
                }
                mixed |= !apart;
                if (taken >= a.top_k && !__any(!apart)) break;
                if (taken == LANES) {
                    close |= !apart;
                    break;
                }
                const int e = take<LANES, VPL, false>(order, k);
                if (l == taken && k > -INFINITY) chosen = e;
                before = k;
            }
            // the softmax' sum in 64 bits
            auto sum64 = [&]() {
                double sum = 0.0;
#pragma unroll 1
                for (int i = 0; i < VPL; ++i) {
                    const double v = on && i < left ? logit<Tr>(a.logits, row + l * VPL + i) : -INFINITY;
                    sum += v == -INFINITY ? 0.0 : exp(v - (double)top);
                }
                return lanes_sum<LANES>(sum);
            };
            auto key64 = [&](double v, double sum, int e) -> Key {
                if (v == -INFINITY) return 0;
                const double t = a.sigmoid ? 1.0 / (1.0 + exp(-v)) : exp(v - (double)top) / sum;
                return key_of(a.bias ? t + (double)a.bias[e] : t);
            };
            if (!__any(close)) {
                if (__any(mixed)) {  // those that were taken, put in order by their keys in 64 bits
                    const double sum = a.sigmoid ? 1.0 : sum64();
                    const Key k = chosen >= 0 ? key64(logit<Tr>(a.logits, row + chosen), sum, chosen) : 0;
                    int rank = 0;
                    for (int i = 0; i < taken; ++i) {
                        const Key other = __shfl((unsigned long long)k, i, LANES);
                        const int e = __shfl(chosen, i, LANES);
                        rank += other > k || (other == k && e < chosen);
                    }
                    int* place = reinterpret_cast<int*>(mine);
                    wave_sync();
                    place[l] = -1;
                    wave_sync();
                    if (chosen >= 0) place[rank] = chosen;
                    wave_sync();
                    chosen = place[l];
                }
                if (l >= a.top_k) chosen = -1;
            } else {
                Key wide[VPL], of64, *own = mine + l * VPL;
                const double sum = a.sigmoid ? 1.0 : sum64();
                spoiled = sum != sum;
                wave_sync();
#pragma unroll 1
                for (int i = 0; i < VPL; ++i) {
                    const double v = on && i < left ? logit<Tr>(a.logits, row + l * VPL + i) : -INFINITY;
                    own[i] = key64(v, sum, l * VPL + i);
                }
                wave_sync();
#pragma unroll
                for (int i = 0; i < VPL; ++i) wide[i] = own[i];
                if (a.groups > 1) keep_groups<LANES>(a, wide, wide, mine, &border);
                chosen = best_experts<LANES, VPL, false>(a, wide, &of64);
            }
            c = chosen >= 0 ? logit<Tr>(a.logits, row + chosen) : -INFINITY;
        }
        // the weights, each lane one
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
    const int l = threadIdx.x % LANES, left = a.E - l * VPL;
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
            Few<Tr, VPL>::load(a.logits, row + l * VPL, any ? left : 0, -INFINITY, s);
#pragma unroll
            for (int i = 0; i < VPL; ++i) top = fmaxf(top, s[i]);
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
        wave_sync();
#pragma unroll
        for (int i = 0; i < VPL; ++i) mine[l * VPL + i] = 0.0f;
        wave_sync();
        if (chosen >= 0) mine[chosen] = g;
        wave_sync();
        float v[VPL];
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            v[i] = mine[l * VPL + i];
            if (whole) v[i] = s[i] * (v[i] - dot);
        }
        Few<Tr, VPL>::store(a.dlogits, row + l * VPL, on ? left : 0, v);
    }
}

// ------------------------------------------------------------ sort
// A counting sort by expert that keeps the slots' order (so equal inputs give equal outputs): a work-group takes a
// stretch of slots, each of its 8 waves an eighth of it in order, 64 slots at a time. Counts first; where there is more
// than one work-group they go to memory, and a second launch sums those of the work-groups before its own.
// Every work-group sums the counts of all, so there are at most 64 (us for 64 / 128 / 256: 131072 slots of 8 experts
// 9.7 / 8.0 / 8.0, of 128 10.7 / 9.7 / 9.7, of 1024 22 / 27 / 27; 327680 16 / 11 / 9, 18 / 13 / 13, 30 / 31 / 39; up to 65536
// the same).
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
    __shared__ int total[kSortExperts + 1], sums[2][kSortExperts];  // sums: parts * E <= max(kSortThreads, E)
    const int lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    count_slots(a, cnt);
    // per expert: all rows, and those before this work-group's. The work-groups' counts of an expert are split between
    // the threads that there are, which ask for 16 at a time (65536 slots, 128 experts: one thread an expert, one count at
    // a time 19.5 us, so 6.6).
    int parts = 1;
    if (a.groups > 1) {
        while (2 * parts * a.E <= kSortThreads) parts *= 2;
        for (int i = threadIdx.x; i < parts * a.E; i += kSortThreads) {
            const int part = i / a.E, e = i - part * a.E;
            int before = 0, all = 0;
            for (int g0 = part; g0 < a.groups; g0 += 16 * parts) {
                int c[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    const int g = g0 + k * parts;
                    c[k] = g < a.groups ? a.counts[(int64_t)g * a.E + e] : 0;
                }
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    before += g0 + k * parts < (int)blockIdx.x ? c[k] : 0;
                    all += c[k];
                }
            }
            sums[0][i] = before, sums[1][i] = all;
        }
        __syncthreads();
    }
    for (int e = threadIdx.x; e < a.E; e += kSortThreads) {
        int before = 0, all = 0;
        if (a.groups == 1) {
            for (int w = 0; w < kSortWaves; ++w) all += cnt[w][e];
        } else {
            for (int part = 0; part < parts; ++part) before += sums[0][part * a.E + e], all += sums[1][part * a.E + e];
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
// A wave takes 512 columns of a token, 8 a lane: a work-group of four waves the same columns of four tokens, its x the
// columns. The token's positions and weights are uniform.
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

enum class Far { none, loads, both };  // accesses of the gradient to the experts' rows that pass the caches by

constexpr unsigned kMostColumnGroups = 1u << 15, kMostTokenGroups = 1u << 15;

dim3 row_grid(int64_t tokens, int64_t hidden) {
    const int64_t x = (hidden + 511) / 512, y = (tokens + 3) / 4;
    return dim3((unsigned)(x < kMostColumnGroups ? x : kMostColumnGroups), (unsigned)(y < kMostTokenGroups ? y : kMostTokenGroups));
}

// f(token, column, how many of the 8 are there) for what the wave takes.
template <typename F>
__device__ __forceinline__ void each_part(const Rows& a, F f) {
    const int w4 = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int64_t token = (int64_t)blockIdx.y * 4 + w4; token < a.tokens; token += (int64_t)gridDim.y * 4)
        for (int64_t c0 = (int64_t)blockIdx.x * 512; c0 < a.hidden; c0 += (int64_t)gridDim.x * 512) {
            const int64_t c = c0 + 8 * (threadIdx.x & 63), left = a.hidden - c;
            f(token, c, left < 8 ? (int)left : 8);
        }
}

// Rows from `live` = offsets[E] on belong to no slot: zeros. Called by all waves, `wave` of `waves`.
template <typename Tr>
__device__ __forceinline__ void clear_tail(const Rows& a, void* out, int64_t live, int64_t wave, int64_t waves) {
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

// FAR: the stores of the experts' rows pass the caches by; in k_combine the loads.
template <typename Tr, bool FAR>
__global__ __launch_bounds__(256) void k_gather(Rows a) {
    const int64_t live = a.offsets[a.E];
    each_part(a, [&](int64_t token, int64_t c, int n) {
        Eight<Tr> v;
        v.load(a.in, token * a.hidden + c, n);
        for (int j = 0; j < a.top_k; ++j) {
            const int64_t p = a.positions[token * a.top_k + j];
            if (p >= 0 && p < a.rows) v.template store<FAR>(a.out, p * a.hidden + c, n);
        }
    });
    const int64_t group = (int64_t)blockIdx.y * gridDim.x + blockIdx.x, groups = (int64_t)gridDim.x * gridDim.y;
    clear_tail<Tr>(a, a.out, live, group * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), groups * 4);
}

// J of the token's rows are asked for before the first is used.
template <typename Tr, int J, bool FAR>
__global__ __launch_bounds__(256) void k_combine(Rows a) {
    each_part(a, [&](int64_t token, int64_t c, int n) {
        float s[8] = {};
        if (a.other) load_stream<Tr>(a.other, a.wide, token * a.hidden + c, n, s);
        for (int j0 = 0; j0 < a.top_k; j0 += J) {
            Eight<Tr> y[J];
            float w[J];
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const int64_t slot = token * a.top_k + (j0 + j < a.top_k ? j0 + j : 0);
                const int64_t p = j0 + j < a.top_k ? a.positions[slot] : -1;
                const bool live = p >= 0 && p < a.rows;  // (what is not adds 1 * 0: its weight may be anything)
                w[j] = live && a.weights ? a.weights[slot] : 1.0f;
                y[j].template load<FAR>(a.in, p * a.hidden + c, live ? n : 0);
            }
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
                for (int k = 0; k < 8; ++k) s[k] = __builtin_fmaf(w[j], y[j].get(k), s[k]);
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
    });
}

// A work-group takes 4 / W tokens, W waves each, which walk its columns; their sums meet in LDS. J slots at a time, whose
// rows are asked for before the first is used.
template <typename Tr, int J, int W, Far FAR>
__global__ __launch_bounds__(256) void k_combine_bwd(Rows a) {
    constexpr int TOKENS = 4 / W;
    __shared__ float part[4][J];
    const int lane = threadIdx.x & 63, w4 = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t live = a.out ? a.offsets[a.E] : 0;
    for (int64_t first = (int64_t)blockIdx.x * TOKENS; first < a.tokens; first += (int64_t)gridDim.x * TOKENS) {
        const int64_t token = first + w4 / W;
        const bool on = token < a.tokens;
        for (int j0 = 0; j0 < a.top_k; j0 += J) {
            int64_t p[J];
            float w[J], dot[J] = {};
#pragma unroll
            for (int j = 0; j < J; ++j) {
                p[j] = -1, w[j] = 0.0f;
                if (!on || j0 + j >= a.top_k) continue;
                const int64_t slot = token * a.top_k + j0 + j;
                p[j] = a.positions[slot];
                if (p[j] >= a.rows) p[j] = -1;
                if (a.out && p[j] >= 0) w[j] = a.weights[slot];
            }
#pragma unroll 1
            for (int64_t c = 8 * (lane + 64 * (w4 % W)); c < a.hidden && on; c += 512 * W) {
                const int64_t left = a.hidden - c;
                const int n = left < 8 ? (int)left : 8;
                Eight<Tr> y[J];
                float d[8];
                load_stream<Tr>(a.in, a.wide, token * a.hidden + c, n, d);
                if (a.dweights) {
#pragma unroll
                    for (int j = 0; j < J; ++j)
                        y[j].template load<(FAR != Far::none)>(a.other, p[j] * a.hidden + c, p[j] >= 0 ? n : 0);
                }
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    if (p[j] < 0) continue;
                    if (a.dweights) {
#pragma unroll
                        for (int k = 0; k < 8; ++k) dot[j] = __builtin_fmaf(d[k], y[j].get(k), dot[j]);
                    }
                    if (a.out) {
                        float g[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) g[k] = w[j] * d[k];
                        Eight<Tr> o;
                        o.set(g);
                        o.template store<(FAR == Far::both)>(a.out, p[j] * a.hidden + c, n);
                    }
                }
            }
            if (!a.dweights) continue;
#pragma unroll
            for (int j = 0; j < J; ++j) {
                dot[j] = lanes_sum<64>(dot[j]);
                if (W > 1 && lane == 0) part[w4][j] = dot[j];
            }
            if constexpr (W > 1) __syncthreads();
            if (w4 % W == 0) {
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    float s = dot[j];
                    if constexpr (W > 1) {
                        s = part[w4][j];
#pragma unroll
                        for (int k = 1; k < W; ++k) s += part[w4 + k][j];
                    }
                    if (lane == j && on && j0 + j < a.top_k) a.dweights[token * a.top_k + j0 + j] = s;
                }
            }
            if constexpr (W > 1) __syncthreads();
        }
    }
    if (a.out) clear_tail<Tr>(a, a.out, live, (int64_t)blockIdx.x * 4 + w4, (int64_t)gridDim.x * 4);
}

bool known(int dtype) { return dtype == STM_F16 || dtype == STM_BF16 || dtype == STM_F32; }
bool lies(const void* p, int dtype) { return aligned(p, dtype == STM_F32 ? 4 : 2); }

// f(type, lanes, values a lane) of the form that holds a token's experts; its lanes hold one chosen expert and one group
// each. Twice the values on half the lanes, us: 16383 tokens of 256 in bf16 9.8 -> 8.6, with bias and groups 29 -> 37, one
// token 3.8 -> 5.1.
template <typename Tr, typename F>
int each_form(int E, int least, F f) {
    using std::integral_constant;
    if (E <= 16 && least <= 16) return f(Tr{}, integral_constant<int, 16>{}, integral_constant<int, 1>{});
    if (E <= 32 && least <= 16) return f(Tr{}, integral_constant<int, 16>{}, integral_constant<int, 2>{});
    if (E <= 64 && least <= 16) return f(Tr{}, integral_constant<int, 16>{}, integral_constant<int, 4>{});
    if (E <= 128 && least <= 16) return f(Tr{}, integral_constant<int, 16>{}, integral_constant<int, 8>{});
    if (E <= 256 && least <= 32) return f(Tr{}, integral_constant<int, 32>{}, integral_constant<int, 8>{});
    if (E <= 512) return f(Tr{}, integral_constant<int, 64>{}, integral_constant<int, 8>{});
    return f(Tr{}, integral_constant<int, 64>{}, integral_constant<int, 16>{});
}

template <typename F>
int each_route(int dtype, int E, int least, F f) {
    if (dtype == STM_BF16) return each_form<BF16>(E, least, f);
    if (dtype == STM_F16) return each_form<F16>(E, least, f);
    return each_form<F32>(E, least, f);
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

// f(slots at a time) for a token's top_k.
template <typename F>
int each_chunk(int top_k, F f) {
    using std::integral_constant;
    if (top_k <= 1) return f(integral_constant<int, 1>{});
    if (top_k <= 2) return f(integral_constant<int, 2>{});
    if (top_k <= 4) return f(integral_constant<int, 4>{});
    return f(integral_constant<int, 8>{});
}

// Which accesses to the experts' rows pass the caches by. Read once, rows of a good part of the 256 MB memory-side cache
// leave it to what is read again; written, rows that do not fit it gain from passing it by, smaller ones are there for the
// product that takes them. Stores that do so have to fill their 128-byte lines, as those of whole 16-bit chunks do (fp32,
// two halves of a line apart: gather of 256 MiB 64 / 130). bf16, 8 slots a token of 2048 columns, us, nothing / loads / both:
//   MiB                                            62            128            188            256            512
//   combination                                    14 / 15       32 / 29        45 / 42        65 / 56        129 / 106
//   gather, its rows read by a combination         27 / 27 / 30  59 / 50 / 57   80 / 81 / 82   135 / 109 / 108  263 / 226 / 229
//   gather alone                                   13 / 13 / 15  30 / 30 / 28   44 / 44 / 40   59 / 59 / 51   117 / 117 / 104
//   combination and its gradient                   52 / 46 / 48  101 / 95 / 87  145 / 136 / 126  193 / 182 / 162  376 / 360 / 338
// Other rows gain less and lose as often, nothing / loads: fp32 of 125 MiB, combination 31 / 33, after a gather 60 / 55, with
// its gradient 95 / 100; of 512 MiB 134 / 121, 292 / 261 and 371 / 374. bf16 of 1001 columns, 122 MiB 39 / 38, 73 / 74 and
// 131 / 147; 244 MiB 77 / 74, 153 / 144 and 262 / 282.
int64_t row_bytes(int64_t rows, int64_t hidden, int dtype) { return rows * hidden * (dtype == STM_F32 ? 4 : 2); }

bool far_loads(int64_t rows, int64_t hidden, int dtype) { return row_bytes(rows, hidden, dtype) >= 96ll << 20; }

bool far_stores(int64_t rows, int64_t hidden, int dtype) {
    return row_bytes(rows, hidden, dtype) >= 256ll << 20 && dtype != STM_F32 && hidden % 64 == 0;
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
    return each_route(dtype, num_experts, top_k > groups ? top_k : groups, [&](auto tr, auto lanes, auto vpl) {
        const dim3 grid(groups_for(tokens, 256 / lanes.value)), block(256);
        if (bias || sums)
            hipLaunchKernelGGL((k_route<decltype(tr), lanes.value, vpl.value, true>), grid, block, 0,
                               (hipStream_t)stream, a);
        else
            hipLaunchKernelGGL((k_route<decltype(tr), lanes.value, vpl.value, false>), grid, block, 0,
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
    return each_route(dtype, num_experts, top_k, [&](auto tr, auto lanes, auto vpl) {
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
        const auto run = [&](auto far) {
            hipLaunchKernelGGL((k_gather<decltype(tr), far.value>), row_grid(tokens, hidden), dim3(256), 0, (hipStream_t)stream,
                               a);
            return check_launch(what);
        };
        if constexpr (!std::is_same_v<decltype(tr), F32>)
            if (far_stores(tokens * top_k, hidden, dtype)) return run(std::true_type{});
        return run(std::false_type{});
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
        return each_chunk(top_k, [&](auto j) {
            const auto run = [&](auto far) {
                hipLaunchKernelGGL((k_combine<decltype(tr), j.value, far.value>), row_grid(tokens, hidden), dim3(256), 0,
                                   (hipStream_t)stream, a);
                return check_launch(what);
            };
            return far_loads(y_rows, hidden, dtype) ? run(std::true_type{}) : run(std::false_type{});
        });
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
    if (y_rows == 0 || hidden == 0) dy = nullptr;  // nothing of it
    if (tokens == 0 || top_k == 0 || (!dy && !dweights)) return STM_OK;
    if (!positions || (hidden && (!dout || (y_rows && ((dweights && !y) || (dy && (!weights || !offsets)))))))
        return set_error(STM_ERR_INVALID, "%s: null pointer", what);
    if (!lies(dout, dout_dtype) || !lies(y, dtype) || !lies(dy, dtype) || !aligned(positions, 4) || !aligned(weights, 4) ||
        !aligned(offsets, 4) || !aligned(dweights, 4))
        return set_error(STM_ERR_INVALID, "%s: pointers must be aligned to their elements", what);
    const Rows a{dout, y, weights, positions, offsets, dy, dweights, tokens, hidden, y_rows, top_k, num_experts,
                 dout_dtype == STM_F32};
    return each_type(dtype, [&](auto tr) {
        const auto run = [&](auto w) {
            const int64_t groups = (tokens + 4 / w.value - 1) / (4 / w.value);
            const dim3 grid((unsigned)(groups < (1 << 22) ? groups : 1 << 22));
            return each_chunk(top_k, [&](auto j) {
                const auto launch = [&](auto far) {
                    hipLaunchKernelGGL((k_combine_bwd<decltype(tr), j.value, w.value, far.value>), grid, dim3(256), 0,
                                       (hipStream_t)stream, a);
                    return check_launch(what);
                };
                if constexpr (!std::is_same_v<decltype(tr), F32>)
                    if (far_stores(y_rows, hidden, dtype)) return launch(std::integral_constant<Far, Far::both>{});
                if (far_loads(y_rows, hidden, dtype)) return launch(std::integral_constant<Far, Far::loads>{});
                return launch(std::integral_constant<Far, Far::none>{});
            });
        };
        if (hidden <= 512) return run(std::integral_constant<int, 1>{});
        if (hidden <= 1024) return run(std::integral_constant<int, 2>{});
        return run(std::integral_constant<int, 4>{});
    });
}
