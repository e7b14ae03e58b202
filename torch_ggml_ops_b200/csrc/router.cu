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
#include "../../include/tgo_mmq.h"

#include <type_traits>

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

// x[v] = the row's scores, -inf beyond the last expert
template <typename T, int VPL>
__device__ __forceinline__ void load_row(const T* __restrict__ row, int experts, bool chunks, int lane, float (&x)[VPL]) {
    using L = RowLayout<T, VPL>;
    if (chunks) {
#pragma unroll
        for (int c = 0; c < VPL / L::CH; ++c) {
            const int e = L::expert(c * L::CH, lane);
            Pack<T, L::CH> p;
            if (e < experts) p = *reinterpret_cast<const Pack<T, L::CH>*>(row + e);
#pragma unroll
            for (int j = 0; j < L::CH; ++j) x[c * L::CH + j] = e < experts ? to_f32(p.v[j]) : -INFINITY;
        }
    } else {
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
            const int e = L::expert(v, lane);
            x[v] = e < experts ? to_f32(row[e]) : -INFINITY;
        }
    }
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
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(kAllLanes, m, d));
    return m;
}

// u -> exp(u) / sum of them, 0 everywhere in a row of -inf; a NaN or +inf among them makes all of them NaN
template <int VPL>
__device__ __forceinline__ void shares(float (&u)[VPL]) {
    float m = warp_max(u);
    if (m == -INFINITY) m = 0.0f;
    float s = 0.0f;
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
        u[v] = expf(u[v] - m);
        s += u[v];
    }
    s = warp_sum(s);
    const float inv = s == 0.0f ? 0.0f : 1.0f / s;
#pragma unroll
    for (int v = 0; v < VPL; ++v) u[v] *= inv;
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
__device__ __forceinline__ void choose(const float (&x)[VPL], int top_k, int lane, float& score, int& expert) {
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

template <typename T, int VPL, bool SIGMOID>
__global__ void __launch_bounds__(kRouterWarps * 32) router_kernel(RouterArgs a, float* __restrict__ weights, int32_t* __restrict__ ids) {
    const int lane = threadIdx.x & 31;
    const int64_t token = static_cast<int64_t>(blockIdx.x) * kRouterWarps + (threadIdx.x >> 5);
    if (token >= a.tokens) return;
    float w = 0.0f;
    int expert = -1;
    if (a.mask == nullptr || a.mask[token] != 0) {
        float x[VPL];
        load_row<T, VPL>(static_cast<const T*>(a.logits) + token * a.stride, a.experts, a.chunks, lane, x);
        bool bad = false;
#pragma unroll
        for (int v = 0; v < VPL; ++v) bad |= isnan(x[v]);
        bad = __any_sync(kAllLanes, bad);
        float score;
        choose<T, VPL>(x, a.top_k, lane, score, expert);
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
                for (int v = 0; v < VPL; ++v) s += expf(x[v] - m);
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
    float x[VPL];
    if (!SIGMOID && !a.normalize && any) {
        load_row<T, VPL>(row, a.experts, a.chunks, lane, x);
        shares(x);
#pragma unroll
        for (int v = 0; v < VPL; ++v) x[v] *= -s;
    } else {
#pragma unroll
        for (int v = 0; v < VPL; ++v) x[v] = 0.0f;
    }
    T* out = dlogits + token * a.experts;
    store_row<T, VPL>(out, a.experts, out_chunks, lane, x);
    __syncwarp();   // the chosen experts' values after what they replace
    if (expert >= 0) out[expert] = from_f32<T>(mine);
}

// ------------------------------------------------------------------ balance loss
struct BalanceArgs {
    const void* logits;
    int64_t tokens, stride;
    int experts, top_k;
    bool chunks;
    const int32_t* ids;
};
__device__ __forceinline__ bool named(const BalanceArgs& a, int64_t token, int lane, int& expert) {
    expert = lane < a.top_k ? a.ids[token * a.top_k + lane] : -1;
    if (expert >= a.experts) expert = -1;
    return __any_sync(kAllLanes, expert >= 0);
}

// Sums of a block over its tokens: probabilities and pairs of every expert, tokens that count.
template <typename T, int VPL, bool SIGMOID>
__global__ void __launch_bounds__(kRouterWarps * 32) balance_sums_kernel(BalanceArgs a, float* __restrict__ part_p, int32_t* __restrict__ part_n) {
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
    const int64_t step = static_cast<int64_t>(gridDim.x) * kRouterWarps;
    for (int64_t token = static_cast<int64_t>(blockIdx.x) * kRouterWarps + warp; token < a.tokens; token += step) {
        int expert;
        if (!named(a, token, lane, expert)) continue;
        if (expert >= 0) atomicAdd(&pairs[expert], 1);
        if (lane == 0) atomicAdd(&pairs[a.experts], 1);
        float x[VPL];
        load_row<T, VPL>(static_cast<const T*>(a.logits) + token * a.stride, a.experts, a.chunks, lane, x);
        if (SIGMOID) {
#pragma unroll
            for (int v = 0; v < VPL; ++v) x[v] = log_sigmoid(x[v]);
        }
        shares(x);
#pragma unroll
        for (int v = 0; v < VPL; ++v) acc[v] += x[v];
    }
#pragma unroll
    for (int v = 0; v < VPL; ++v)
        if (L::expert(v, lane) < a.experts) warp_p[warp * a.experts + L::expert(v, lane)] = acc[v];
    __syncthreads();
    for (int e = threadIdx.x; e < a.experts; e += blockDim.x) {
        float s = 0.0f;
        for (int w = 0; w < kRouterWarps; ++w) s += warp_p[w * a.experts + e];
        part_p[static_cast<int64_t>(blockIdx.x) * a.experts + e] = s;
    }
    for (int e = threadIdx.x; e <= a.experts; e += blockDim.x) part_n[static_cast<int64_t>(blockIdx.x) * (a.experts + 1) + e] = pairs[e];
}

// The blocks' sums in their order (the same bits every time) -> counts, loss, coef[e] = E f_e / tokens.
__global__ void __launch_bounds__(1024) balance_loss_kernel(const float* __restrict__ part_p, const int32_t* __restrict__ part_n, int blocks, int experts,
                                                            float* __restrict__ loss, int32_t* __restrict__ counts, float* __restrict__ coef) {
    __shared__ float warp_s[32];
    __shared__ long long warp_n[32];
    __shared__ long long tokens_s;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = threadIdx.x;
    float p = 0.0f;
    int32_t n = 0;
    if (e < experts) {
        for (int b = 0; b < blocks; ++b) {
            p += part_p[static_cast<int64_t>(b) * experts + e];
            n += part_n[static_cast<int64_t>(b) * (experts + 1) + e];
        }
        counts[e] = n;
    }
    long long total = n, tokens = 0;
    if (warp == 0) {
        for (int b = lane; b < blocks; b += 32) tokens += part_n[static_cast<int64_t>(b) * (experts + 1) + experts];
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) tokens += __shfl_xor_sync(kAllLanes, tokens, d);
        if (lane == 0) tokens_s = tokens;
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) total += __shfl_xor_sync(kAllLanes, total, d);
    if (lane == 0) warp_n[warp] = total;
    __syncthreads();
    total = 0;
    for (int w = 0; w < 32; ++w) total += warp_n[w];
    tokens = tokens_s;
    const float f = total > 0 ? static_cast<float>(n) / static_cast<float>(total) : 0.0f;
    const float per_token = tokens > 0 ? static_cast<float>(experts) / static_cast<float>(tokens) : 0.0f;
    if (e < experts) coef[e] = f * per_token;
    const float s = warp_sum(e < experts ? f * p : 0.0f);
    if (lane == 0) warp_s[warp] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        float all = 0.0f;
        for (int w = 0; w < 32; ++w) all += warp_s[w];
        *loss = all * per_token;
    }
}

template <typename T, int VPL, bool SIGMOID>
__global__ void __launch_bounds__(kRouterWarps * 32) balance_grad_kernel(BalanceArgs a, const float* __restrict__ coef, const float* __restrict__ dloss,
                                                                        T* __restrict__ dlogits, bool out_chunks) {
    using L = RowLayout<T, VPL>;
    const int lane = threadIdx.x & 31;
    const int64_t token = static_cast<int64_t>(blockIdx.x) * kRouterWarps + (threadIdx.x >> 5);
    if (token >= a.tokens) return;
    int expert;
    float p[VPL];
    if (named(a, token, lane, expert)) {
        float x[VPL], c[VPL];
        load_row<T, VPL>(static_cast<const T*>(a.logits) + token * a.stride, a.experts, a.chunks, lane, x);
        const float g = *dloss;
        float inner = 0.0f;
#pragma unroll
        for (int v = 0; v < VPL; ++v) p[v] = log_score<SIGMOID>(x[v]);
        shares(p);
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
            const int e = L::expert(v, lane);
            c[v] = e < a.experts ? coef[e] * g : 0.0f;
            inner += c[v] * p[v];
        }
        inner = warp_sum(inner);
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
            p[v] *= c[v] - inner;
            if (SIGMOID) p[v] *= sigmoid_of_minus(x[v]);
        }
    } else {
#pragma unroll
        for (int v = 0; v < VPL; ++v) p[v] = 0.0f;
    }
    store_row<T, VPL>(dlogits + token * a.experts, a.experts, out_chunks, lane, p);
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
    if (reinterpret_cast<uintptr_t>(logits) % type_bytes(dtype) != 0) return route_fail(TGO_E_ARG, "logits are not aligned to their type");
    if (scoring != TGO_SCORING_SOFTMAX && scoring != TGO_SCORING_SIGMOID) return route_fail(TGO_E_ARG, "unknown scoring");
    return TGO_OK;
}
static int launched(const char* what) { return cudaGetLastError() == cudaSuccess ? TGO_OK : route_fail(TGO_E_CUDA, what); }
static unsigned token_blocks(int64_t tokens) { return static_cast<unsigned>((tokens + kRouterWarps - 1) / kRouterWarps); }

constexpr int64_t kBalanceBlocks = 148 * 2;
static int64_t balance_blocks(int64_t tokens) {
    const int64_t b = token_blocks(tokens);
    return b < kBalanceBlocks ? b : kBalanceBlocks;
}

}  // namespace tgo

using namespace tgo;

extern "C" {

int tgo_moe_router(const void* logits, int dtype, int64_t tokens, int64_t experts, int64_t row_stride, int64_t top_k, int scoring, int normalize,
                   const uint8_t* token_mask, float* weights, int32_t* expert_ids, void* stream) {
    if (weights == nullptr || expert_ids == nullptr) return route_fail(TGO_E_ARG, "null pointer");
    const int rc = check_scores(logits, dtype, tokens, experts, row_stride, top_k, scoring);
    if (rc != TGO_OK) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return with_layout(dtype, experts, [&](auto t, auto vpl) {
        using T = decltype(t);
        constexpr int VPL = decltype(vpl)::value;
        const RouterArgs a = {logits, tokens, row_stride, static_cast<int>(experts), static_cast<int>(top_k), normalize != 0,
                              RowLayout<T, VPL>::whole_chunks(logits, experts, row_stride), token_mask};
        if (scoring == TGO_SCORING_SIGMOID) router_kernel<T, VPL, true><<<token_blocks(tokens), kRouterWarps * 32, 0, st>>>(a, weights, expert_ids);
        else router_kernel<T, VPL, false><<<token_blocks(tokens), kRouterWarps * 32, 0, st>>>(a, weights, expert_ids);
        return launched("router_kernel launch failed");
    });
}

int tgo_moe_router_grad(const void* logits, int dtype, int64_t tokens, int64_t experts, int64_t row_stride, const int32_t* expert_ids,
                        const float* weights, const float* d_weights, int64_t top_k, int scoring, int normalize, void* d_logits, void* stream) {
    if (weights == nullptr || expert_ids == nullptr || d_weights == nullptr || d_logits == nullptr) return route_fail(TGO_E_ARG, "null pointer");
    const int rc = check_scores(logits, dtype, tokens, experts, row_stride, top_k, scoring);
    if (rc != TGO_OK) return rc;
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
    return balance_blocks(tokens) * (2 * experts + 1) * 4;
}

int tgo_moe_balance_loss(const void* logits, int dtype, int64_t tokens, int64_t experts, int64_t row_stride, const int32_t* expert_ids,
                         int64_t top_k, int scoring, float* loss, int32_t* counts, float* coef, void* workspace, int64_t workspace_bytes,
                         void* stream) {
    if (expert_ids == nullptr || loss == nullptr || counts == nullptr || coef == nullptr || workspace == nullptr)
        return route_fail(TGO_E_ARG, "null pointer");
    const int rc = check_scores(logits, dtype, tokens, experts, row_stride, top_k, scoring);
    if (rc != TGO_OK) return rc;
    if (workspace_bytes < tgo_moe_balance_workspace_bytes(tokens, experts)) return route_fail(TGO_E_WORKSPACE, "balance workspace too small");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const unsigned blocks = static_cast<unsigned>(balance_blocks(tokens));
    float* part_p = static_cast<float*>(workspace);
    int32_t* part_n = reinterpret_cast<int32_t*>(part_p + static_cast<int64_t>(blocks) * experts);
    const size_t smem = ((kRouterWarps + 1) * experts + 1) * 4;
    return with_layout(dtype, experts, [&](auto t, auto vpl) {
        using T = decltype(t);
        constexpr int VPL = decltype(vpl)::value;
        const BalanceArgs a = {logits, tokens, row_stride, static_cast<int>(experts), static_cast<int>(top_k),
                               RowLayout<T, VPL>::whole_chunks(logits, experts, row_stride), expert_ids};
        if (scoring == TGO_SCORING_SIGMOID) balance_sums_kernel<T, VPL, true><<<blocks, kRouterWarps * 32, smem, st>>>(a, part_p, part_n);
        else balance_sums_kernel<T, VPL, false><<<blocks, kRouterWarps * 32, smem, st>>>(a, part_p, part_n);
        balance_loss_kernel<<<1, 1024, 0, st>>>(part_p, part_n, static_cast<int>(blocks), static_cast<int>(experts), loss, counts, coef);
        return launched("balance kernel launch failed");
    });
}

int tgo_moe_balance_grad(const void* logits, int dtype, int64_t tokens, int64_t experts, int64_t row_stride, const int32_t* expert_ids,
                         int64_t top_k, int scoring, const float* coef, const float* d_loss, void* d_logits, void* stream) {
    if (expert_ids == nullptr || coef == nullptr || d_loss == nullptr || d_logits == nullptr) return route_fail(TGO_E_ARG, "null pointer");
    const int rc = check_scores(logits, dtype, tokens, experts, row_stride, top_k, scoring);
    if (rc != TGO_OK) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return with_layout(dtype, experts, [&](auto t, auto vpl) {
        using T = decltype(t);
        constexpr int VPL = decltype(vpl)::value;
        const BalanceArgs a = {logits, tokens, row_stride, static_cast<int>(experts), static_cast<int>(top_k),
                               RowLayout<T, VPL>::whole_chunks(logits, experts, row_stride), expert_ids};
        const bool out_chunks = RowLayout<T, VPL>::whole_chunks(d_logits, experts, experts);
        T* out = static_cast<T*>(d_logits);
        if (scoring == TGO_SCORING_SIGMOID)
            balance_grad_kernel<T, VPL, true><<<token_blocks(tokens), kRouterWarps * 32, 0, st>>>(a, coef, d_loss, out, out_chunks);
        else
            balance_grad_kernel<T, VPL, false><<<token_blocks(tokens), kRouterWarps * 32, 0, st>>>(a, coef, d_loss, out, out_chunks);
        return launched("balance_grad_kernel launch failed");
    });
}

}  // extern "C"
