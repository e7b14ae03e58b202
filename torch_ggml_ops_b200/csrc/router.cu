// The router of a mixture-of-experts layer and its balance loss, forward and gradient.
//
// A token's scores are x[0..E).  On a logarithmic scale they are u = x ("softmax") or
// u = log sigmoid(x) = min(x, 0) - log1p(exp(-|x|)) ("sigmoid", slope du/dx = sigmoid(-x)); both
// kinds of share are then a softmax of u, which no large score overflows and no small one empties:
//   weights    exp(u_i) / sum over the chosen of exp(u), or, not normalised, exp(u_i) / sum over all
//              (softmax) and exp(u_i) (sigmoid);
//   balance    E * sum_e f_e * P_e,  f_e = pairs of e / all pairs,  P_e = mean over tokens of
//              p_e = exp(u_e) / sum over all of exp(u).
// Gradients, with g the cotangent of the weights and s = sum_i g_i w_i over the chosen:
//   weights    w_i (g_i - s) slope_i at the chosen experts (and, not normalised: softmax -p_j s at the
//              others; sigmoid w_i g_i slope_i at the chosen, nothing elsewhere);
//   balance    p_e (c_e - sum_j c_j p_j) slope_e,  c_e = E f_e / tokens * cotangent; f is a count.
//
// One warp per token, the row in its registers: lane l holds chunks of consecutive experts, so that a
// row is read once, in full lines.
//
// Measured on one B200, GPU time in a graph (us), 256 experts, top 8, bf16 (floor: scores in or out at 6.4 TB/s, 5.2 us for 65536 tokens):
//   router      16 tokens 2.3, 65536 29.4;  gradient 65536 12.3 (normalised)
//   balance     65536 24;  gradient 65536 22 (floor 10.4);  1000 experts, softmax / sigmoid: bf16 89 / 153, gradient 174 / 298 (floors 20.4, 40.8),
//               fp32 50 / 118, gradient 92 / 209 (floors 40.8, 81.5), whose 192 to 241 registers leave
//               one block of 8 warps per SM
//   fp32: router 8200 tokens 6.8, gradient of the plain probabilities 3.7;  1291 tokens of 1000 experts, top 4, 4.6
// What bounds the router: instructions (345 per token, 69 % of the issue slots): keys 40, eight choices 50, the scores put in
// after them 50, softmax and result 60; 40 to 64 warps per SM instead of 32 gain nothing.  Choosing by (score, expert) with two reductions and a search of the registers
// took 61 us, two cached scores per lane with a refill 36.  The balance loss has some 8 us that do not shrink with the
// tokens (clearing the sums, adding them across blocks, the last block's work) and 160 instructions per token.
#include "../../include/tgo_mmq.h"

#include <atomic>
#include <type_traits>

#include "aligned.h"
#include "scores.cuh"

namespace tgo {

int route_fail(int code, const char* msg);  // tgo_api.cu

constexpr int kRouterMaxExperts = 1024;
constexpr int kRouterMaxTopK = 32;   // one lane per chosen expert
constexpr int kRouterWarps = 8;

// Register v of lane l holds expert ((v / CH) * 32 + l) * CH + v % CH.
template <typename T, int VPL>
struct RowLayout {
    static constexpr int CH = VPL < 16 / static_cast<int>(sizeof(T)) ? VPL : 16 / static_cast<int>(sizeof(T));
    __device__ static __forceinline__ int expert(int v, int lane) { return ((v / CH) * 32 + lane) * CH + v % CH; }
    // whether every chunk of every row starts at a multiple of its size and ends inside the row
    static bool whole_chunks(const void* base, int64_t experts, int64_t stride) {
        return experts % CH == 0 && stride % CH == 0 && reinterpret_cast<uintptr_t>(base) % (CH * sizeof(T)) == 0;
    }
};

// A lane's part of a row as it lies in memory, so that the next row can be under way while one is worked on
template <typename T, int VPL>
struct RawRow {
    using L = RowLayout<T, VPL>;
    Pack<T, L::CH> p[VPL / L::CH];
    // -inf beyond the last expert
    __device__ __forceinline__ void load(const T* __restrict__ row, int experts, bool chunks, int lane) {
        const T none = from_f32<T>(-INFINITY);
#pragma unroll
        for (int c = 0; c < VPL / L::CH; ++c) {
            const int e = L::expert(c * L::CH, lane);
#pragma unroll
            for (int j = 0; j < L::CH; ++j) p[c].v[j] = none;
            if (chunks) {
                if (e < experts) p[c] = *reinterpret_cast<const Pack<T, L::CH>*>(row + e);
            } else {
#pragma unroll
                for (int j = 0; j < L::CH; ++j)
                    if (e + j < experts) p[c].v[j] = row[e + j];
            }
        }
    }
    __device__ __forceinline__ void widen(float (&x)[VPL]) const {
#pragma unroll
        for (int v = 0; v < VPL; ++v) x[v] = to_f32(p[v / L::CH].v[v % L::CH]);
    }
};
template <typename T, int VPL>
__device__ __forceinline__ void load_row(const T* __restrict__ row, int experts, bool chunks, int lane, float (&x)[VPL]) {
    RawRow<T, VPL> raw;
    raw.load(row, experts, chunks, lane);
    raw.widen(x);
}
template <typename T, int VPL>
__device__ __forceinline__ void store_row(T* __restrict__ row, int experts, bool chunks, int lane, const float (&x)[VPL]) {
    using L = RowLayout<T, VPL>;
    if (chunks) {
#pragma unroll
        for (int c = 0; c < VPL / L::CH; ++c) {
            const int e = L::expert(c * L::CH, lane);
            Pack<T, L::CH> p;
#pragma unroll
            for (int j = 0; j < L::CH; ++j) p.v[j] = from_f32<T>(x[c * L::CH + j]);
            if (e < experts) *reinterpret_cast<Pack<T, L::CH>*>(row + e) = p;
        }
    } else {
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
            const int e = L::expert(v, lane);
            if (e < experts) row[e] = from_f32<T>(x[v]);
        }
    }
}

template <typename T, int VPL>
__device__ __forceinline__ void copy_row(T* __restrict__ row, const T* from, int experts, bool chunks, int lane) {
    using L = RowLayout<T, VPL>;
    if (chunks) {
#pragma unroll
        for (int c = 0; c < VPL / L::CH; ++c) {
            const int e = L::expert(c * L::CH, lane);
            if (e < experts) *reinterpret_cast<Pack<T, L::CH>*>(row + e) = *reinterpret_cast<const Pack<T, L::CH>*>(from + e);
        }
    } else {
        for (int e = lane; e < experts; e += 32) row[e] = from[e];
    }
}

__device__ __forceinline__ float log_sigmoid(float x) { return fminf(x, 0.0f) - log1pf(expf(-fabsf(x))); }
__device__ __forceinline__ float sigmoid_of_minus(float x) {
    const float far = expf(-fabsf(x));
    return (x > 0.0f ? far : 1.0f) / (1.0f + far);
}
template <bool SIGMOID>
__device__ __forceinline__ float log_score(float x) { return SIGMOID ? log_sigmoid(x) : x; }

// largest value of a warp's registers that is no NaN
template <int VPL>
__device__ __forceinline__ float warp_max(const float (&x)[VPL]) {
    float m = x[0];
#pragma unroll
    for (int v = 1; v < VPL; ++v) m = fmaxf(m, x[v]);
    asm volatile("redux.sync.max.f32 %0, %0, 0xffffffff;" : "+f"(m));
    return m;
}

// exp(d) of a difference d <= 0 for the sums over all experts, in three instructions where expf takes eight: off by
// 4 U + 1.3 |d| U of itself (U = 2^-24): little where it is large, and where it is small it adds little to a sum;
// below 2^-126 it is 0.
__device__ __forceinline__ float exp_below(float d) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d * 1.4426950408889634f));
    return r;
}

// u -> exp(u - the largest); returns 1 / their sum, 0 for a row of -inf.  With a NaN or +inf in the row the products
// with it are all NaN.
template <int VPL>
__device__ __forceinline__ float exponentials(float (&u)[VPL]) {
    float m = warp_max(u);
    if (m == -INFINITY) m = 0.0f;
    float s = 0.0f;
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
        u[v] = exp_below(u[v] - m);
        s += u[v];
    }
    s = warp_sum(s);
    float inv;   // of a sum of 1 at least
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
    return s == 0.0f ? 0.0f : inv;
}

struct RouterArgs {
    const void* logits;
    int64_t tokens, stride;
    int experts, top_k;
    bool normalize, chunks;
    const uint8_t* mask;   // null: every token counts
};

// The top_k largest scores in order, lane s the s-th: (score, expert); of equal scores the lower expert
// first.  -inf and NaN are never chosen: expert -1 where nothing is left.
template <typename T, int VPL>
__device__ __noinline__ void choose_exactly(const float (&x)[VPL], int top_k, int lane, float& score, int& expert) {
    using L = RowLayout<T, VPL>;
    uint32_t key[VPL];   // 0: not to be chosen (any more)
#pragma unroll
    for (int v = 0; v < VPL; ++v) key[v] = x[v] > -INFINITY ? order_of(x[v]) : 0u;
    score = -INFINITY;
    expert = -1;
    for (int s = 0; s < top_k; ++s) {
        uint32_t best = 0;
        int at = 0;
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
            if (key[v] > best) {
                best = key[v];
                at = L::expert(v, lane);
            }
        }
        const uint32_t top = __reduce_max_sync(kAllLanes, best);
        if (top == 0) break;
        const int first = static_cast<int>(__reduce_min_sync(kAllLanes, best == top ? static_cast<uint32_t>(at) : 0xFFFFFFFFu));
        if (lane == s) {
            score = value_of(top);
            expert = first;
        }
#pragma unroll
        for (int v = 0; v < VPL; ++v)
            if (L::expert(v, lane) == first) key[v] = 0;
    }
}

template <int VPL>
__device__ __forceinline__ uint32_t largest(const uint32_t (&k)[VPL]) {
    uint32_t m = k[0];
#pragma unroll
    for (int v = 1; v + 1 < VPL; v += 2) m = __vimax3_u32(m, k[v], k[v + 1]);
    return VPL % 2 == 0 ? max(m, k[VPL - 1]) : m;
}

// the largest of a lane's keys that is below `last`, one of them; 0 if there is none.  Keys below last wrap around
// to the largest differences.
template <int VPL>
__device__ __forceinline__ uint32_t next_below(const uint32_t (&key)[VPL], uint32_t last) {
    uint32_t d[VPL];
#pragma unroll
    for (int v = 0; v < VPL; ++v) d[v] = key[v] - last;
    const uint32_t m = largest(d) + last;
    return m < last ? m : 0u;
}

// The same with one reduction per choice and no search for the expert: a key holds the upper 22 bits of a score's
// order and, below, the expert (the lower expert the larger number), so that no two are equal.  That is all of a
// 16-bit score.  Of two different fp32 scores that agree in the 22 bits the exact comparison decides: a row where such
// are among the best (1 in 70 of 256 normal scores) goes through choose_exactly.
// First the best top_k of the lanes' best, in order, by way of `slot` in shared memory; lane s holds the s-th.  Scores of
// the same lanes that belong among them (one or two in a row as a rule) are then put in one by one.
// bad: the row holds a NaN (its order, like any NaN's after the addition of 0, is above all).
constexpr uint32_t kExpertBits = 1023;
template <typename T, int VPL>
__device__ __forceinline__ void choose(const float (&x)[VPL], const T* __restrict__ row, int top_k, int lane, uint32_t* slot, float& score, int& expert, bool& bad) {
    using L = RowLayout<T, VPL>;
    constexpr bool kWide = sizeof(T) == 4;
    constexpr uint32_t kLeast = 0x00800000u;     // order of the lowest finite fp32 (fp16's and bf16's are no lower): -inf is below
    constexpr uint32_t kInfinite = 0xFF800000u;  // order of +inf
    uint32_t key[VPL];
#pragma unroll
    for (int v = 0; v < VPL; ++v) key[v] = (order_of(x[v]) & ~kExpertBits) | (kExpertBits - L::expert(v, lane));
    const uint32_t first = largest(key);
    uint32_t low = 0, left = first;
    const int slots = kWide && top_k < 32 ? top_k + 1 : top_k;   // fp32: whether the next one is as large has to be seen
    slot[lane] = 0;
    __syncwarp();
#pragma unroll 8
    for (int s = 0; s < slots; ++s) {
        low = __reduce_max_sync(kAllLanes, left);
        if (left == low) {
            slot[s] = low;
            left = 0;
        }
    }
    __syncwarp();
    uint32_t mine = slot[lane];
    __syncwarp();
    bad = __shfl_sync(kAllLanes, mine, 0) > (kInfinite | kExpertBits);
    if (VPL > 1) {
        // `low` is the least that is in; a lane whose best is out has nothing that is better
        uint32_t next = first >= low ? next_below(key, first) : 0u;
        while (__any_sync(kAllLanes, next > low)) {
            const uint32_t put = __reduce_max_sync(kAllLanes, next);
            const uint32_t above = __shfl_up_sync(kAllLanes, mine, 1);
            mine = max(mine, lane == 0 ? put : min(above, put));
            low = __shfl_sync(kAllLanes, mine, slots - 1);
            if (next == put) next = next_below(key, put);
        }
    }
    bool search = bad;
    if (kWide) {
        const uint32_t above = __shfl_up_sync(kAllLanes, mine, 1);
        const bool alike = lane > 0 && lane < slots && mine >= kLeast && ((mine ^ above) & ~kExpertBits) == 0;
        if (__any_sync(kAllLanes, alike) || top_k == 32) {   // the last of 32 has no slot behind it
            // Equal numbers are in order already (fp32 scores that were rounded to bf16 often are equal): those in the slots are compared
            // with the one above, the others that are like the last slot's with it.
            const float x0 = lane < slots && mine >= kLeast ? to_f32(row[kExpertBits - (mine & kExpertBits)]) : 0.0f;
            const float x1 = __shfl_up_sync(kAllLanes, x0, 1);
            bool differ = alike && x0 != x1;
            const uint32_t last = order_of(__shfl_sync(kAllLanes, x0, slots - 1));
#pragma unroll
            for (int v = 0; v < VPL; ++v) differ |= low >= kLeast && ((key[v] ^ low) & ~kExpertBits) == 0 && order_of(x[v]) != last;
            search |= __any_sync(kAllLanes, differ);
        }
    }
    if (search) {
        choose_exactly<T, VPL>(x, top_k, lane, score, expert);
        return;
    }
    const bool got = mine >= kLeast && lane < top_k;
    expert = got ? static_cast<int>(kExpertBits - (mine & kExpertBits)) : -1;
    if (kWide) score = got ? to_f32(row[expert]) : -INFINITY;
    else score = got ? value_of(mine < 0x80000000u ? mine | kExpertBits : mine & ~kExpertBits) : -INFINITY;
}

template <typename T, int VPL, bool SIGMOID>
__global__ void __launch_bounds__(kRouterWarps * 32) router_kernel(RouterArgs a, float* __restrict__ weights, int32_t* __restrict__ ids) {
    __shared__ uint32_t slots[kRouterWarps][32];
    const int lane = threadIdx.x & 31;
    const int64_t step = static_cast<int64_t>(gridDim.x) * kRouterWarps;
    int64_t token = static_cast<int64_t>(blockIdx.x) * kRouterWarps + (threadIdx.x >> 5);
    const T* row = static_cast<const T*>(a.logits) + token * a.stride;
    for (; token < a.tokens; token += step, row += step * a.stride) {
        float w = 0.0f;
        int expert = -1;
        if (a.mask == nullptr || a.mask[token] != 0) {
            float x[VPL];
            load_row<T, VPL>(row, a.experts, a.chunks, lane, x);
            bool bad;
            float score;
            choose<T, VPL>(x, row, a.top_k, lane, slots[threadIdx.x >> 5], score, expert, bad);
            const float u = expert >= 0 ? log_score<SIGMOID>(score) : -INFINITY;
            if (a.normalize || !SIGMOID) {
                const float top = __shfl_sync(kAllLanes, u, 0);   // the largest; u rises with the score
                const float m = top == -INFINITY ? 0.0f : top;
                const float e = expf(u - m);
                float s = 0.0f;
                if (a.normalize) {
                    s = e;
                } else {
#pragma unroll
                    for (int v = 0; v < VPL; ++v) s += exp_below(x[v] - m);
                }
                s = warp_sum(s);
                w = expert >= 0 ? e / s : 0.0f;
            } else {
                w = expf(u);
            }
            if (bad) w = NAN;
        }
        if (lane < a.top_k) {
            weights[token * a.top_k + lane] = w;
            ids[token * a.top_k + lane] = expert;
        }
    }
}

// ids and weights are router_kernel's; d: the cotangent of the weights
template <typename T, int VPL, bool SIGMOID>
__global__ void __launch_bounds__(kRouterWarps * 32) router_grad_kernel(RouterArgs a, const int32_t* __restrict__ ids, const float* __restrict__ weights,
                                                                       const float* __restrict__ d, T* __restrict__ dlogits, bool out_chunks) {
    const int lane = threadIdx.x & 31;
    const int64_t token = static_cast<int64_t>(blockIdx.x) * kRouterWarps + (threadIdx.x >> 5);
    if (token >= a.tokens) return;
    int expert = -1;
    float w = 0.0f, g = 0.0f;
    if (lane < a.top_k) {
        expert = ids[token * a.top_k + lane];
        if (expert >= a.experts) expert = -1;
    }
    if (expert >= 0) {
        w = weights[token * a.top_k + lane];
        g = d[token * a.top_k + lane];
    }
    const bool any = __any_sync(kAllLanes, expert >= 0);
    const T* row = static_cast<const T*>(a.logits) + token * a.stride;
    const float s = warp_sum(expert >= 0 ? g * w : 0.0f);
    float mine = a.normalize || !SIGMOID ? w * (g - s) : w * g;
    if (SIGMOID && expert >= 0) mine *= sigmoid_of_minus(to_f32(row[expert]));
    T* out = dlogits + token * a.experts;
    // the row is put together in shared memory, so that it leaves in full lines
    __shared__ __align__(16) T put[kRouterWarps][VPL * 32];
    T* mem = put[threadIdx.x >> 5];
    float x[VPL];
    if (!SIGMOID && !a.normalize && any) {
        load_row<T, VPL>(row, a.experts, a.chunks, lane, x);
        const float inv = exponentials(x);
#pragma unroll
        for (int v = 0; v < VPL; ++v) x[v] *= inv * -s;
    } else {
#pragma unroll
        for (int v = 0; v < VPL; ++v) x[v] = 0.0f;
    }
    store_row<T, VPL>(mem, VPL * 32, true, lane, x);
    __syncwarp();
    if (expert >= 0) mem[expert] = from_f32<T>(mine);
    __syncwarp();
    copy_row<T, VPL>(out, mem, a.experts, out_chunks, lane);
}

// ------------------------------------------------------------------ balance loss
// A warp's tokens one after another, the next one's ids and scores under way.  A token that names no expert is not
// read (its scores may be anything).
struct BalanceArgs {
    const void* logits;
    int64_t tokens, stride;
    int experts, top_k;
    bool chunks;
    const int32_t* ids;
};
template <typename T, int VPL>
struct TokenWalk {
    const BalanceArgs& a;
    const int lane;
    const int64_t step;
    int64_t token;
    int expert;      // the lane's, of the token; -1: none
    bool live;
    RawRow<T, VPL> raw;
    __device__ __forceinline__ TokenWalk(const BalanceArgs& args, int l)
        : a(args), lane(l), step(static_cast<int64_t>(gridDim.x) * kRouterWarps),
          token(static_cast<int64_t>(blockIdx.x) * kRouterWarps + (threadIdx.x >> 5) - step) {
        next_id = fetch_id();
        advance();
    }
    __device__ __forceinline__ bool done() const { return token >= a.tokens; }
    __device__ __forceinline__ void advance() {
        token += step;
        expert = next_id;
        live = __any_sync(kAllLanes, expert >= 0);
        if (live) raw.load(static_cast<const T*>(a.logits) + token * a.stride, a.experts, a.chunks, lane);
        next_id = fetch_id();
    }

  private:
    int next_id;
    __device__ __forceinline__ int fetch_id() const {
        const int64_t t = token + step;
        const int e = t < a.tokens && lane < a.top_k ? a.ids[t * a.top_k + lane] : -1;
        return e < a.experts ? e : -1;
    }
};

// What the blocks add up.  Probabilities are added as whole numbers of 2^-shift: whole numbers give the same sum in
// every order, and with shift = 62 - log2(tokens) a sum is off by less than 2^-50 of its largest.
struct BalanceSums {
    unsigned long long* p;   // [experts]
    int32_t* pairs;          // [experts], then the tokens that count, the blocks that are done, whether a share was NaN
    int shift;
};

// Every block adds its tokens' probabilities and pairs; the last one done makes the loss, the counts and
// coef[e] = E f_e / tokens of the sums.
template <typename T, int VPL, bool SIGMOID>
__global__ void __launch_bounds__(kRouterWarps * 32) balance_kernel(BalanceArgs a, BalanceSums sums, float* __restrict__ loss, int32_t* __restrict__ counts,
                                                                   float* __restrict__ coef) {
    using L = RowLayout<T, VPL>;
    extern __shared__ float smem[];
    int32_t* pairs = reinterpret_cast<int32_t*>(smem);                       // [experts], then the tokens that count
    float* warp_p = smem + a.experts + 1;                                    // [warps][experts]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int e = threadIdx.x; e <= a.experts; e += blockDim.x) pairs[e] = 0;
    __syncthreads();
    float acc[VPL];
#pragma unroll
    for (int v = 0; v < VPL; ++v) acc[v] = 0.0f;
    int tokens = 0;
    TokenWalk<T, VPL> walk(a, lane);
    while (!walk.done()) {
        const bool live = walk.live;
        const int expert = walk.expert;
        float x[VPL];
        walk.raw.widen(x);
        walk.advance();
        if (!live) continue;
        if (expert >= 0) atomicAdd(&pairs[expert], 1);
        ++tokens;
        if (SIGMOID) {
#pragma unroll
            for (int v = 0; v < VPL; ++v) x[v] = log_sigmoid(x[v]);
        }
        const float inv = exponentials(x);
#pragma unroll
        for (int v = 0; v < VPL; ++v) acc[v] = fmaf(x[v], inv, acc[v]);
    }
    if (lane == 0 && tokens != 0) atomicAdd(&pairs[a.experts], tokens);
#pragma unroll
    for (int v = 0; v < VPL; ++v)
        if (L::expert(v, lane) < a.experts) warp_p[warp * a.experts + L::expert(v, lane)] = acc[v];
    __syncthreads();
    const float unit = ldexpf(1.0f, sums.shift);
    for (int e = threadIdx.x; e < a.experts; e += blockDim.x) {
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < kRouterWarps; ++w) s += warp_p[w * a.experts + e];
        if (isnan(s)) atomicOr(&sums.pairs[a.experts + 2], 1);
        else if (s != 0.0f) atomicAdd(&sums.p[e], __float2ull_rn(s * unit));
        if (pairs[e] != 0) atomicAdd(&sums.pairs[e], pairs[e]);
    }
    __threadfence();
    __syncthreads();
    __shared__ bool last;
    if (threadIdx.x == 0) {
        if (pairs[a.experts] != 0) atomicAdd(&sums.pairs[a.experts], pairs[a.experts]);
        __threadfence();
        last = atomicAdd(&sums.pairs[a.experts + 1], 1) == static_cast<int32_t>(gridDim.x) - 1;
    }
    __syncthreads();
    if (!last) return;

    __threadfence();
    __shared__ long long warp_n[kRouterWarps];
    __shared__ double warp_s[kRouterWarps];
    long long all_pairs = 0;
    for (int e = threadIdx.x; e < a.experts; e += blockDim.x) {
        const int32_t n = __ldcg(&sums.pairs[e]);
        counts[e] = n;
        all_pairs += n;
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) all_pairs += __shfl_xor_sync(kAllLanes, all_pairs, d);
    if (lane == 0) warp_n[warp] = all_pairs;
    __syncthreads();
    all_pairs = 0;
#pragma unroll
    for (int w = 0; w < kRouterWarps; ++w) all_pairs += warp_n[w];
    const int32_t live = __ldcg(&sums.pairs[a.experts]);
    const float per_token = live > 0 ? static_cast<float>(a.experts) / static_cast<float>(live) : 0.0f;
    double total = 0.0;
    for (int e = threadIdx.x; e < a.experts; e += blockDim.x) {
        const float f = all_pairs > 0 ? static_cast<float>(__ldcg(&sums.pairs[e])) / static_cast<float>(all_pairs) : 0.0f;
        coef[e] = f * per_token;
        total += f * static_cast<double>(__ldcg(&sums.p[e]));
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) total += __shfl_xor_sync(kAllLanes, total, d);
    if (lane == 0) warp_s[warp] = total;
    __syncthreads();
    if (threadIdx.x == 0) {
        total = 0.0;
        for (int w = 0; w < kRouterWarps; ++w) total += warp_s[w];
        *loss = __ldcg(&sums.pairs[a.experts + 2]) != 0 ? NAN : static_cast<float>(ldexp(total, -sums.shift)) * per_token;
    }
}

template <typename T, int VPL, bool SIGMOID>
__global__ void __launch_bounds__(kRouterWarps * 32) balance_grad_kernel(BalanceArgs a, const float* __restrict__ coef, const float* __restrict__ dloss,
                                                                        T* __restrict__ dlogits, bool out_chunks) {
    using L = RowLayout<T, VPL>;
    const int lane = threadIdx.x & 31;
    const float g = *dloss;
    float c[VPL];
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
        const int e = L::expert(v, lane);
        c[v] = e < a.experts ? coef[e] * g : 0.0f;
    }
    TokenWalk<T, VPL> walk(a, lane);
    while (!walk.done()) {
        const bool live = walk.live;
        const int64_t token = walk.token;
        float x[VPL], p[VPL];
        walk.raw.widen(x);
        walk.advance();
        if (live) {
#pragma unroll
            for (int v = 0; v < VPL; ++v) p[v] = log_score<SIGMOID>(x[v]);
            const float inv = exponentials(p);
            float inner = 0.0f;
#pragma unroll
            for (int v = 0; v < VPL; ++v) inner = fmaf(c[v], p[v], inner);
            inner = warp_sum(inner) * inv;
#pragma unroll
            for (int v = 0; v < VPL; ++v) {
                p[v] *= (c[v] - inner) * inv;
                if (SIGMOID) p[v] *= sigmoid_of_minus(x[v]);
            }
        } else {
#pragma unroll
            for (int v = 0; v < VPL; ++v) p[v] = 0.0f;
        }
        store_row<T, VPL>(dlogits + token * a.experts, a.experts, out_chunks, lane, p);
    }
}

// ------------------------------------------------------------------ launches
// f(type, registers per lane): the kernels' template arguments for a type code and an expert count
template <typename F>
static int with_layout(int dtype, int64_t experts, F f) {
    auto typed = [&](auto t) {
        if (experts <= 32) return f(t, std::integral_constant<int, 1>());
        if (experts <= 64) return f(t, std::integral_constant<int, 2>());
        if (experts <= 128) return f(t, std::integral_constant<int, 4>());
        if (experts <= 256) return f(t, std::integral_constant<int, 8>());
        if (experts <= 512) return f(t, std::integral_constant<int, 16>());
        return f(t, std::integral_constant<int, 32>());
    };
    if (dtype == TGO_BF16) return typed(__nv_bfloat16());
    if (dtype == TGO_FP16) return typed(__half());
    return typed(float());
}

static int64_t type_bytes(int dtype) { return dtype == TGO_FP32 ? 4 : 2; }
static int check_scores(const void* logits, int dtype, int64_t tokens, int64_t experts, int64_t stride, int64_t top_k, int scoring) {
    if (logits == nullptr) return route_fail(TGO_E_ARG, "null pointer");
    if (dtype != TGO_BF16 && dtype != TGO_FP16 && dtype != TGO_FP32) return route_fail(TGO_E_ARG, "unsupported type of the logits");
    if (tokens <= 0) return route_fail(TGO_E_ARG, "zero-row inputs are not supported");
    if (experts <= 0 || experts > kRouterMaxExperts) return route_fail(TGO_E_ARG, "num_experts must be in 1..1024");
    if (top_k <= 0 || top_k > kRouterMaxTopK || top_k > experts) return route_fail(TGO_E_ARG, "top_k must be in 1..32 and at most num_experts");
    if (tokens > INT32_MAX / top_k) return route_fail(TGO_E_ARG, "tokens * top_k must be below 2^31");
    if (stride < experts && tokens > 1) return route_fail(TGO_E_ARG, "rows of logits overlap");
    if (!aligned_to(type_bytes(dtype), logits)) return route_fail(TGO_E_ARG, "logits are not aligned to their type");
    if (scoring != TGO_SCORING_SOFTMAX && scoring != TGO_SCORING_SIGMOID) return route_fail(TGO_E_ARG, "unknown scoring");
    return TGO_OK;
}
static int launched(const char* what) { return cudaGetLastError() == cudaSuccess ? TGO_OK : route_fail(TGO_E_CUDA, what); }
static unsigned token_blocks(int64_t tokens) { return static_cast<unsigned>((tokens + kRouterWarps - 1) / kRouterWarps); }
// for kernels whose warps take one token after another: as many blocks as run at once.  SMEM: the most shared memory that the kernel is ever
// given, so that a grid, and with it the order of a sum, depends on the call alone and not on the calls before it.
template <auto KERNEL, size_t SMEM = 0>
static unsigned resident_blocks(int64_t tokens) {
    static std::atomic<int> per_sm{0};
    int n = per_sm.load(std::memory_order_relaxed);
    if (n == 0) {
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, KERNEL, kRouterWarps * 32, SMEM) != cudaSuccess || n < 1) n = 1;
        per_sm.store(n, std::memory_order_relaxed);
    }
    const unsigned b = token_blocks(tokens);
    return b < 148u * n ? b : 148u * n;
}
// balance_kernel's blocks: rounds of those that run at once, so many that no warp adds up more than kBalanceRun tokens in fp32 before the sum joins the whole
// numbers.  Each token of a run may put a sum off by U / 2, and tokens that are all alike round the same way: in one round 2^28 of 3
// experts were 3.5e-4 off, so 1.3e-6.
constexpr int64_t kBalanceRun = 256;
template <auto KERNEL, size_t SMEM>
static unsigned balance_blocks(int64_t tokens) {
    const int64_t at_once = resident_blocks<KERNEL, SMEM>(tokens), run = at_once * kRouterWarps * kBalanceRun;
    return static_cast<unsigned>((tokens + run - 1) / run * at_once);
}
// its shared memory: pairs of every expert, the tokens, the warps' sums
static constexpr size_t balance_smem(int64_t experts) { return ((kRouterWarps + 1) * experts + 1) * 4; }

// log2(tokens), rounded up
static int bits_of(int64_t tokens) {
    int b = 0;
    while ((1LL << b) < tokens) ++b;
    return b;
}

}  // namespace tgo

using namespace tgo;

extern "C" {

int tgo_moe_router(const void* logits, int dtype, int64_t tokens, int64_t experts, int64_t row_stride, int64_t top_k, int scoring, int normalize,
                   const uint8_t* token_mask, float* weights, int32_t* expert_ids, void* stream) {
    if (weights == nullptr || expert_ids == nullptr) return route_fail(TGO_E_ARG, "null pointer");
    if (!aligned_to(4, weights, expert_ids)) return route_fail(TGO_E_ARG, kMisaligned);
    const int rc = check_scores(logits, dtype, tokens, experts, row_stride, top_k, scoring);
    if (rc != TGO_OK) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return with_layout(dtype, experts, [&](auto t, auto vpl) {
        using T = decltype(t);
        constexpr int VPL = decltype(vpl)::value;
        const RouterArgs a = {logits, tokens, row_stride, static_cast<int>(experts), static_cast<int>(top_k), normalize != 0,
                              RowLayout<T, VPL>::whole_chunks(logits, experts, row_stride), token_mask};
        if (scoring == TGO_SCORING_SIGMOID) router_kernel<T, VPL, true><<<resident_blocks<router_kernel<T, VPL, true>>(tokens), kRouterWarps * 32, 0, st>>>(a, weights, expert_ids);
        else router_kernel<T, VPL, false><<<resident_blocks<router_kernel<T, VPL, false>>(tokens), kRouterWarps * 32, 0, st>>>(a, weights, expert_ids);
        return launched("router_kernel launch failed");
    });
}

int tgo_moe_router_grad(const void* logits, int dtype, int64_t tokens, int64_t experts, int64_t row_stride, const int32_t* expert_ids,
                        const float* weights, const float* d_weights, int64_t top_k, int scoring, int normalize, void* d_logits, void* stream) {
    if (weights == nullptr || expert_ids == nullptr || d_weights == nullptr || d_logits == nullptr) return route_fail(TGO_E_ARG, "null pointer");
    const int rc = check_scores(logits, dtype, tokens, experts, row_stride, top_k, scoring);
    if (rc != TGO_OK) return rc;
    if (!aligned_to(4, weights, expert_ids, d_weights) || !aligned_to(type_bytes(dtype), d_logits)) return route_fail(TGO_E_ARG, kMisaligned);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return with_layout(dtype, experts, [&](auto t, auto vpl) {
        using T = decltype(t);
        constexpr int VPL = decltype(vpl)::value;
        const RouterArgs a = {logits, tokens, row_stride, static_cast<int>(experts), static_cast<int>(top_k), normalize != 0,
                              RowLayout<T, VPL>::whole_chunks(logits, experts, row_stride), nullptr};
        const bool out_chunks = RowLayout<T, VPL>::whole_chunks(d_logits, experts, experts);
        T* out = static_cast<T*>(d_logits);
        if (scoring == TGO_SCORING_SIGMOID)
            router_grad_kernel<T, VPL, true><<<token_blocks(tokens), kRouterWarps * 32, 0, st>>>(a, expert_ids, weights, d_weights, out, out_chunks);
        else
            router_grad_kernel<T, VPL, false><<<token_blocks(tokens), kRouterWarps * 32, 0, st>>>(a, expert_ids, weights, d_weights, out, out_chunks);
        return launched("router_grad_kernel launch failed");
    });
}

int64_t tgo_moe_balance_workspace_bytes(int64_t tokens, int64_t experts) {
    if (tokens <= 0 || experts <= 0 || experts > kRouterMaxExperts) return -1;
    return experts * 12 + 12;
}

int tgo_moe_balance_loss(const void* logits, int dtype, int64_t tokens, int64_t experts, int64_t row_stride, const int32_t* expert_ids,
                         int64_t top_k, int scoring, float* loss, int32_t* counts, float* coef, void* workspace, int64_t workspace_bytes,
                         void* stream) {
    if (expert_ids == nullptr || loss == nullptr || counts == nullptr || coef == nullptr || workspace == nullptr)
        return route_fail(TGO_E_ARG, "null pointer");
    const int rc = check_scores(logits, dtype, tokens, experts, row_stride, top_k, scoring);
    if (rc != TGO_OK) return rc;
    if (!aligned_to(4, expert_ids, loss, counts, coef)) return route_fail(TGO_E_ARG, kMisaligned);
    if (workspace_bytes < tgo_moe_balance_workspace_bytes(tokens, experts)) return route_fail(TGO_E_WORKSPACE, "balance workspace too small");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (reinterpret_cast<uintptr_t>(workspace) % 8 != 0) return route_fail(TGO_E_ARG, "the workspace must be 8-byte aligned");
    const BalanceSums sums = {static_cast<unsigned long long*>(workspace), reinterpret_cast<int32_t*>(static_cast<unsigned long long*>(workspace) + experts),
                              62 - bits_of(tokens)};
    if (cudaMemsetAsync(workspace, 0, static_cast<size_t>(experts) * 12 + 12, st) != cudaSuccess) return route_fail(TGO_E_CUDA, "cudaMemsetAsync failed");
    const size_t smem = balance_smem(experts);
    return with_layout(dtype, experts, [&](auto t, auto vpl) {
        using T = decltype(t);
        constexpr int VPL = decltype(vpl)::value;
        const BalanceArgs a = {logits, tokens, row_stride, static_cast<int>(experts), static_cast<int>(top_k),
                               RowLayout<T, VPL>::whole_chunks(logits, experts, row_stride), expert_ids};
        if (scoring == TGO_SCORING_SIGMOID) balance_kernel<T, VPL, true><<<balance_blocks<balance_kernel<T, VPL, true>, balance_smem(32 * VPL)>(tokens), kRouterWarps * 32, smem, st>>>(a, sums, loss, counts, coef);
        else balance_kernel<T, VPL, false><<<balance_blocks<balance_kernel<T, VPL, false>, balance_smem(32 * VPL)>(tokens), kRouterWarps * 32, smem, st>>>(a, sums, loss, counts, coef);
        return launched("balance_kernel launch failed");
    });
}

int tgo_moe_balance_grad(const void* logits, int dtype, int64_t tokens, int64_t experts, int64_t row_stride, const int32_t* expert_ids,
                         int64_t top_k, int scoring, const float* coef, const float* d_loss, void* d_logits, void* stream) {
    if (expert_ids == nullptr || coef == nullptr || d_loss == nullptr || d_logits == nullptr) return route_fail(TGO_E_ARG, "null pointer");
    const int rc = check_scores(logits, dtype, tokens, experts, row_stride, top_k, scoring);
    if (rc != TGO_OK) return rc;
    if (!aligned_to(4, expert_ids, coef, d_loss) || !aligned_to(type_bytes(dtype), d_logits)) return route_fail(TGO_E_ARG, kMisaligned);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return with_layout(dtype, experts, [&](auto t, auto vpl) {
        using T = decltype(t);
        constexpr int VPL = decltype(vpl)::value;
        const BalanceArgs a = {logits, tokens, row_stride, static_cast<int>(experts), static_cast<int>(top_k),
                               RowLayout<T, VPL>::whole_chunks(logits, experts, row_stride), expert_ids};
        const bool out_chunks = RowLayout<T, VPL>::whole_chunks(d_logits, experts, experts);
        T* out = static_cast<T*>(d_logits);
        if (scoring == TGO_SCORING_SIGMOID)
            balance_grad_kernel<T, VPL, true><<<resident_blocks<balance_grad_kernel<T, VPL, true>>(tokens), kRouterWarps * 32, 0, st>>>(a, coef, d_loss, out, out_chunks);
        else
            balance_grad_kernel<T, VPL, false><<<resident_blocks<balance_grad_kernel<T, VPL, false>>(tokens), kRouterWarps * 32, 0, st>>>(a, coef, d_loss, out, out_chunks);
        return launched("balance_grad_kernel launch failed");
    });
}

}  // extern "C"
