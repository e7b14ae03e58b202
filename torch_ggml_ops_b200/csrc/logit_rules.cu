// What a generation step does to a head's logits before it takes a token from them, row by row:
//   x = logit + sum of the biases that name the token
//   c = occurrences of the token in the row's history;  where c > 0:
//       x = (x > 0 ? x / repetition : x * repetition) - (c * frequency + presence)
//   x = -inf where the grammar's mask has no bit for the token
// in fp32, each operation rounded once, then one rounding to the output's type.
//
// One block per slice of a row's vocabulary: it counts the history's tokens that fall into the slice and
// adds up the biases in shared memory, then passes over the slice once.  So a step is one launch, with no
// table of counts in memory; every block reads the whole history of its row (from L2).
#include "../../include/tgo_mmq.h"

#include <atomic>

#include "scores.cuh"

namespace tgo {

int route_fail(int code, const char* msg);  // tgo_api.cu

constexpr int kRulesThreads = 256;
constexpr int kRulesPad = 16;   // a row's first elements, in front of its first 16-byte boundary

struct RulesArgs {
    const void* logits;
    void* out;
    int64_t rows, vocab, in_stride, out_stride;
    const void* history;   // null: nothing to penalise
    const void* lengths;   // null: all of history_len
    int64_t history_len, history_stride;
    const float *repetition, *presence, *frequency;   // per row; null: the values below
    float repetition_all, presence_all, frequency_all;
    const void* bias_ids;   // null: none
    const float* bias_values;
    int64_t n_bias, bias_ids_stride, bias_values_stride;
    const uint32_t* allowed;   // null: every token
    int64_t allowed_stride;
    int slice, slices;
    bool history_wide, lengths_wide, bias_wide, vectors, in_place;
};

__device__ __forceinline__ int64_t id_at(const void* p, bool wide, int64_t i) {
    return wide ? static_cast<const int64_t*>(p)[i] : static_cast<int64_t>(static_cast<const int32_t*>(p)[i]);
}

struct Penalty {
    float repetition, presence, frequency;
};
__device__ __forceinline__ float penalised(float x, uint32_t count, const Penalty& p) {
    x = x > 0.0f ? __fdiv_rn(x, p.repetition) : __fmul_rn(x, p.repetition);
    return __fsub_rn(x, __fadd_rn(__fmul_rn(static_cast<float>(count), p.frequency), p.presence));
}

template <typename T>
__global__ void __launch_bounds__(kRulesThreads) logit_rules_kernel(RulesArgs a) {
    extern __shared__ uint4 smem[];
    constexpr int VEC = 16 / static_cast<int>(sizeof(T));
    const int64_t row = blockIdx.x / static_cast<unsigned>(a.slices);
    const int part = static_cast<int>(blockIdx.x - row * a.slices);
    const T* in = static_cast<const T*>(a.logits) + row * a.in_stride;
    T* out = static_cast<T*>(a.out) + row * a.out_stride;
    // elements in front of the row's first 16-byte boundary; they go with the first slice
    int head = a.vectors ? static_cast<int>((16 - reinterpret_cast<uintptr_t>(in) % 16) % 16 / sizeof(T)) : 0;
    if (head > a.vocab) head = static_cast<int>(a.vocab);
    const int64_t base = head + static_cast<int64_t>(part) * a.slice;   // what shared memory calls token kRulesPad
    const int64_t lo = part == 0 ? 0 : base;
    const int64_t hi = base + a.slice < a.vocab ? base + a.slice : a.vocab;
    if (lo >= hi) return;

    const bool counting = a.history != nullptr, biased = a.bias_ids != nullptr;
    uint32_t* count = reinterpret_cast<uint32_t*>(smem);
    float* bias = reinterpret_cast<float*>(count + (counting ? a.slice + kRulesPad : 0));
    Penalty pen = {1.0f, 0.0f, 0.0f};
    if (counting || biased) {
        const int words = (a.slice + kRulesPad) * ((counting ? 1 : 0) + (biased ? 1 : 0));
        for (int i = threadIdx.x; i < words; i += kRulesThreads) count[i] = 0;
        __syncthreads();
    }
    if (counting) {
        pen.repetition = a.repetition != nullptr ? a.repetition[row] : a.repetition_all;
        pen.presence = a.presence != nullptr ? a.presence[row] : a.presence_all;
        pen.frequency = a.frequency != nullptr ? a.frequency[row] : a.frequency_all;
        int64_t n = a.history_len;
        if (a.lengths != nullptr) {
            const int64_t own = id_at(a.lengths, a.lengths_wide, row);
            n = own < n ? own : n;
        }
        for (int64_t i = threadIdx.x; i < n; i += kRulesThreads) {
            const int64_t t = id_at(a.history, a.history_wide, row * a.history_stride + i);
            if (t >= lo && t < hi) atomicAdd(&count[t - base + kRulesPad], 1u);
        }
    }
    if (biased && threadIdx.x < 32) {
        // one warp, 32 entries at a time, each token's in the order of the list: the same sum every time
        const int lane = threadIdx.x;
        for (int64_t j0 = 0; j0 < a.n_bias; j0 += 32) {
            int64_t t = -1;
            float v = 0.0f;
            if (j0 + lane < a.n_bias) {
                t = id_at(a.bias_ids, a.bias_wide, row * a.bias_ids_stride + j0 + lane);
                if (t < lo || t >= hi) t = -1;
                else v = a.bias_values[row * a.bias_values_stride + j0 + lane];
            }
            const unsigned same = __match_any_sync(kAllLanes, t);
            const bool first = (same & ((1u << lane) - 1u)) == 0;
            float sum = first && t >= 0 ? bias[t - base + kRulesPad] : 0.0f;
            for (int s = 0; s < 32; ++s) {
                const float o = __shfl_sync(kAllLanes, v, s);
                if (same >> s & 1u) sum = __fadd_rn(sum, o);
            }
            if (first && t >= 0) bias[t - base + kRulesPad] = sum;
            __syncwarp();
        }
    }
    if (counting || biased) __syncthreads();

    const uint32_t* words = a.allowed != nullptr ? a.allowed + row * a.allowed_stride : nullptr;
    auto one = [&](int64_t t) {
        const bool on = words == nullptr || (words[t >> 5] >> (t & 31) & 1u) != 0;
        const int i = static_cast<int>(t - base) + kRulesPad;
        const uint32_t c = counting ? count[i] : 0u;
        const float b = biased ? bias[i] : 0.0f;
        if (!on) {
            out[t] = from_f32<T>(-INFINITY);
        } else if (c != 0 || b != 0.0f) {
            float x = to_f32(in[t]);
            if (b != 0.0f) x = __fadd_rn(x, b);
            if (c != 0) x = penalised(x, c, pen);
            out[t] = from_f32<T>(x);
        } else if (!a.in_place) {
            out[t] = in[t];
        }
    };
    if (!a.vectors) {
        for (int64_t t = lo + threadIdx.x; t < hi; t += kRulesThreads) one(t);
        return;
    }
    if (lo + threadIdx.x < base) one(lo + threadIdx.x);   // the head
    const int vecs = static_cast<int>((hi - base) / VEC);
    for (int v = threadIdx.x; v < vecs; v += kRulesThreads) {
        const int64_t t = base + static_cast<int64_t>(v) * VEC;
        uint32_t on = (1u << VEC) - 1u;
        if (words != nullptr) {
            const uint32_t w0 = words[t >> 5], w1 = words[(t + VEC - 1) >> 5];
            on &= __funnelshift_r(w0, w1, static_cast<uint32_t>(t & 31));
        }
        uint32_t changed = 0;
        uint32_t c[VEC];
        float b[VEC];
        const int i = v * VEC + kRulesPad;
#pragma unroll
        for (int j = 0; j < VEC; ++j) c[j] = 0, b[j] = 0.0f;
        if (counting) {
#pragma unroll
            for (int j = 0; j < VEC; j += 4) {
                const uint4 q = *reinterpret_cast<const uint4*>(count + i + j);
                c[j] = q.x, c[j + 1] = q.y, c[j + 2] = q.z, c[j + 3] = q.w;
            }
        }
        if (biased) {
#pragma unroll
            for (int j = 0; j < VEC; j += 4) {
                const float4 q = *reinterpret_cast<const float4*>(bias + i + j);
                b[j] = q.x, b[j + 1] = q.y, b[j + 2] = q.z, b[j + 3] = q.w;
            }
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) changed |= (c[j] != 0 || b[j] != 0.0f ? 1u : 0u) << j;
        changed &= on;
        if (a.in_place && changed == 0 && on == (1u << VEC) - 1u) continue;
        Pack<T, VEC> x = {};
        if (on != 0) x = *reinterpret_cast<const Pack<T, VEC>*>(in + t);
        if (changed != 0) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                if ((changed >> j & 1u) == 0) continue;
                float f = to_f32(x.v[j]);
                if (b[j] != 0.0f) f = __fadd_rn(f, b[j]);
                if (c[j] != 0) f = penalised(f, c[j], pen);
                x.v[j] = from_f32<T>(f);
            }
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            if ((on >> j & 1u) == 0) x.v[j] = from_f32<T>(-INFINITY);
        *reinterpret_cast<Pack<T, VEC>*>(out + t) = x;
    }
    const int64_t rest = base + static_cast<int64_t>(vecs) * VEC;
    if (rest + threadIdx.x < hi) one(rest + threadIdx.x);
}

template <typename T>
static int launch_rules(const RulesArgs& a, size_t smem, cudaStream_t st) {
    static std::atomic<bool> ready[64];   // a kernel may use more than 48 KB only after a call per device has said so
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return route_fail(TGO_E_CUDA, "cudaGetDevice failed");
    if (dev >= 64 || !ready[dev].load(std::memory_order_relaxed)) {
        if (cudaFuncSetAttribute(logit_rules_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024) != cudaSuccess)
            return route_fail(TGO_E_CUDA, "cudaFuncSetAttribute failed");
        if (dev < 64) ready[dev].store(true, std::memory_order_relaxed);
    }
    logit_rules_kernel<T><<<static_cast<unsigned>(a.rows * a.slices), kRulesThreads, smem, st>>>(a);
    return cudaGetLastError() == cudaSuccess ? TGO_OK : route_fail(TGO_E_CUDA, "logit_rules_kernel launch failed");
}

}  // namespace tgo

using namespace tgo;

extern "C" int tgo_logit_rules(const void* logits, void* out, int dtype, int64_t rows, int64_t vocab, int64_t in_stride, int64_t out_stride,
                               const void* history, const void* lengths, int64_t history_len, int64_t history_stride, int history_id_bytes,
                               int length_bytes, const float* repetition, float repetition_all, const float* presence, float presence_all,
                               const float* frequency, float frequency_all, const void* bias_ids, const float* bias_values, int64_t n_bias,
                               int64_t bias_ids_stride, int64_t bias_values_stride, int bias_id_bytes, const uint32_t* allowed,
                               int64_t allowed_stride, void* stream) {
    if (logits == nullptr || out == nullptr) return route_fail(TGO_E_ARG, "null pointer");
    if (dtype != TGO_BF16 && dtype != TGO_FP16 && dtype != TGO_FP32) return route_fail(TGO_E_ARG, "unsupported type of the logits");
    if (rows <= 0) return route_fail(TGO_E_ARG, "zero-row inputs are not supported");
    if (vocab <= 0 || vocab > INT32_MAX) return route_fail(TGO_E_ARG, "the vocabulary must be in 1..2^31-1");
    if (rows > 1 && (in_stride < vocab || out_stride < vocab)) return route_fail(TGO_E_ARG, "rows of logits overlap");
    if (history_len < 0 || n_bias < 0) return route_fail(TGO_E_ARG, "a negative length");
    auto id_size = [](int b) { return b == 4 || b == 8; };
    if (history != nullptr && (!id_size(history_id_bytes) || (lengths != nullptr && !id_size(length_bytes))))
        return route_fail(TGO_E_ARG, "token ids and lengths must have 4 or 8 bytes");
    if (bias_ids != nullptr && (!id_size(bias_id_bytes) || bias_values == nullptr)) return route_fail(TGO_E_ARG, "bias ids need values, and 4 or 8 bytes");
    const int64_t size = dtype == TGO_FP32 ? 4 : 2;
    const uintptr_t i = reinterpret_cast<uintptr_t>(logits), o = reinterpret_cast<uintptr_t>(out);
    if (i % size != 0 || o % size != 0) return route_fail(TGO_E_ARG, "logits are not aligned to their type");
    RulesArgs a = {};
    a.logits = logits, a.out = out, a.rows = rows, a.vocab = vocab, a.in_stride = in_stride, a.out_stride = out_stride;
    if (history_len > 0) a.history = history, a.lengths = lengths, a.history_len = history_len, a.history_stride = history_stride;
    a.history_wide = history_id_bytes == 8, a.lengths_wide = length_bytes == 8;
    a.repetition = repetition, a.presence = presence, a.frequency = frequency;
    a.repetition_all = repetition_all, a.presence_all = presence_all, a.frequency_all = frequency_all;
    if (n_bias > 0) a.bias_ids = bias_ids, a.bias_values = bias_values, a.n_bias = n_bias;
    a.bias_ids_stride = bias_ids_stride, a.bias_values_stride = bias_values_stride, a.bias_wide = bias_id_bytes == 8;
    a.allowed = allowed, a.allowed_stride = allowed_stride;
    a.in_place = logits == out && (rows == 1 || in_stride == out_stride);
    // 16-byte accesses where every row of the result lies to its boundary as the row of logits does
    a.vectors = (i - o) % 16 == 0 && (rows == 1 || (in_stride - out_stride) * size % 16 == 0);
    const int tables = (a.history != nullptr ? 1 : 0) + (a.bias_ids != nullptr ? 1 : 0);
    // slices: some four blocks per SM, no shorter than 1024 tokens, at most 64 KB of shared memory each
    int64_t slices = (148 * 4 + rows - 1) / rows;
    int64_t slice = (vocab + slices - 1) / slices;
    const int64_t most = tables == 2 ? 8192 : 16384;
    slice = slice < 1024 ? 1024 : slice > most ? most : (slice + 127) / 128 * 128;
    slices = (vocab + slice - 1) / slice;
    if (rows > INT32_MAX / slices) return route_fail(TGO_E_ARG, "too many logits");
    a.slice = static_cast<int>(slice), a.slices = static_cast<int>(slices);
    const size_t smem = static_cast<size_t>(tables) * (slice + kRulesPad) * 4;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == TGO_BF16) return launch_rules<__nv_bfloat16>(a, smem, st);
    if (dtype == TGO_FP16) return launch_rules<__half>(a, smem, st);
    return launch_rules<float>(a, smem, st);
}
