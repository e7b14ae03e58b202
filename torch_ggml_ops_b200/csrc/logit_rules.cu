// What a generation step does to a head's logits before it takes a token from them, row by row:
//   x = logit + sum of the biases that name the token
//   c = occurrences of the token in the row's history;  where c > 0:
//       x = (x > 0 ? x / repetition : x * repetition) - (c * frequency + presence)
//   x = -inf where the grammar's mask has no bit for the token
// in fp32, each operation rounded once, then one rounding to the output's type.
//
// One block per slice of a row's vocabulary: it brings the slice's logits to shared memory, counts the history's
// tokens that fall into the slice meanwhile, amends the logits of the tokens that history or biases name and
// writes the slice out under the mask.  One launch, no table of counts in memory; every slice reads all of its row's
// history, from L2, and that is what bounds long ones.  us on one B200 (248320 tokens; in a graph, one call after another):
//   16 rows bf16 (15.9 MB)      logits alone 4.7, mask 4.8, 16 biases 5.8, 512 ids 7.4, 4096 10.7, 16384 16.2;
//                               ragged histories up to 8192, biases and mask 13.8
//   200 rows bf16 (199 MB)      16 ids 42 (4.7 TB/s), 512 50, 4096 65, 16384 108
//   200 rows fp32 (397 MB)      logits alone 63.4 (6.3 TB/s, as a copy), mask 65.1, mask and 1500 ids 89
// In place (without a mask only the vectors that change are written, after a look at each one's counts): 16 rows bf16 of 512 ids 8.3 for 7.2 into
// a new tensor, of 8192 16.5 for 13.9, 200 rows of 16 53.7 for 43.3; 200 rows fp32 of 1500 85.1 for 89.6.
// Tried: a pass under the mask and a second kernel for the named tokens, with a hash table or ranks in a bit table, that starts
// while the first runs (16 rows 14.2 to 26: its phases are latency, and short histories got slower; 200 rows fp32 81 for 89, so that logits beyond
// the L2 would gain by it); clusters of eight blocks that share one reading of the history (faster for the longest alone); the history sorted by
// slices first (a block per row: 5 us and more, as much of a history is in few slices); larger slices with the tables alone in
// shared memory, looked up in the pass vector by vector (16 rows of 8192 ids, biases and mask 16.9 for 13.8, 200 rows of 16 ids 62 for 42);
// the ids of a slice put together by a warp before they are counted (16 rows of 4096 ids 10.1 for 10.7, 200 rows of 16 44 for 42); slices
// whose number fills the last round of blocks (200 rows of 1500 ids 62 for 58).
#include "../../include/tgo_mmq.h"

#include <atomic>

#include "aligned.h"
#include "scores.cuh"

namespace tgo {

int route_fail(int code, const char* msg);  // tgo_api.cu

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
    int slice, slices;   // tokens of a block, blocks of a row
    bool history_wide, lengths_wide, bias_wide, vectors, in_place;
};

__device__ __forceinline__ int64_t id_at(const void* p, bool wide, int64_t i) {
    return wide ? static_cast<const int64_t*>(p)[i] : static_cast<int64_t>(static_cast<const int32_t*>(p)[i]);
}
// An id's distance from token lo; kNone unless it is one of the span tokens from there on
constexpr uint32_t kNone = 0xFFFFFFFFu;
__device__ __forceinline__ uint32_t distance(uint32_t id, uint32_t lo, uint32_t span) { return id - lo < span ? id - lo : kNone; }
__device__ __forceinline__ uint32_t distance(uint2 id, uint32_t lo, uint32_t span) { return id.y == 0 && id.x - lo < span ? id.x - lo : kNone; }

// f(d[kAhead]) for the distances of ids, by the block's whole warps, where a lane has one: several ids are
// under way per thread, so that the loop waits for L2 once in so many.
constexpr int kAhead = 8;
template <int THREADS, typename Id, typename F>
__device__ __forceinline__ void each_id(const Id* __restrict__ ids, int64_t n, uint32_t lo, uint32_t span, F f) {
    const int lane = threadIdx.x & 31;
    ids += threadIdx.x;
    for (int64_t left = n - (threadIdx.x - lane); left > 0; left -= THREADS * kAhead, ids += THREADS * kAhead) {
        Id id[kAhead];
        uint32_t d[kAhead];
        bool any = false;
        if (left >= THREADS * (kAhead - 1) + 32) {
#pragma unroll
            for (int u = 0; u < kAhead; ++u) id[u] = ids[u * THREADS];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                d[u] = distance(id[u], lo, span);
                any |= d[u] != kNone;
            }
        } else {
            const int mine = static_cast<int>(left) - lane;
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
                if (u * THREADS < mine) id[u] = ids[u * THREADS];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                d[u] = u * THREADS < mine ? distance(id[u], lo, span) : kNone;
                any |= d[u] != kNone;
            }
        }
        if (__any_sync(kAllLanes, any)) f(d);
    }
}
struct Penalty {
    float repetition, presence, frequency;
};
__device__ __forceinline__ float penalised(float x, uint32_t count, const Penalty& p) {
    x = x > 0.0f ? __fdiv_rn(x, p.repetition) : __fmul_rn(x, p.repetition);
    return __fsub_rn(x, __fadd_rn(__fmul_rn(static_cast<float>(count), p.frequency), p.presence));
}

// What a block works on, from the row's first 16-byte boundary on in vectors
template <typename T, int THREADS>
struct Slice {
    static constexpr int VEC = 16 / static_cast<int>(sizeof(T));
    static constexpr uint32_t kAll = (1u << VEC) - 1u;
    int64_t row;
    int part;
    const T* in;
    T* out;
    int64_t base, lo, hi;    // tokens lo..hi-1; base: the first at a boundary of `in` (lo is in front of it in a row's first slice)
    const uint32_t* words;   // the row's mask
    __device__ __forceinline__ explicit Slice(const RulesArgs& a) {
        row = blockIdx.x / static_cast<unsigned>(a.slices);
        part = static_cast<int>(blockIdx.x - row * a.slices);
        in = static_cast<const T*>(a.logits) + row * a.in_stride;
        out = static_cast<T*>(a.out) + row * a.out_stride;
        int head = static_cast<int>((16 - reinterpret_cast<uintptr_t>(in) % 16) % 16 / sizeof(T));
        if (head > a.vocab) head = static_cast<int>(a.vocab);
        base = head + static_cast<int64_t>(part) * a.slice;
        lo = part == 0 ? 0 : base;
        hi = base + a.slice < a.vocab ? base + a.slice : a.vocab;
        words = a.allowed != nullptr ? a.allowed + row * a.allowed_stride : nullptr;
    }
    __device__ __forceinline__ int vecs() const { return hi > base ? static_cast<int>((hi - base) / VEC) : 0; }
    // f(token) for the elements that are in no vector, up to VEC - 1 on either side
    template <typename F>
    __device__ __forceinline__ void edges(F f) const {
        if (lo + threadIdx.x < base && lo + threadIdx.x < hi) f(lo + threadIdx.x);
        const int64_t rest = base + static_cast<int64_t>(vecs()) * VEC;
        if (rest + threadIdx.x < hi) f(rest + threadIdx.x);
    }
    // The slice under its mask to memory, several vectors of each thread under way: x(v) is vector v, same(v) whether it may stay as
    // it is in memory, one(token) an element.
    template <typename X, typename S, typename O>
    __device__ __forceinline__ void finish(const RulesArgs& a, X x, S same, O one) const {
        auto put = [&](int64_t t) { out[t] = words == nullptr || (words[t >> 5] >> (t & 31) & 1u) != 0 ? one(t) : from_f32<T>(-INFINITY); };
        if (!a.vectors) {
            for (int64_t t = lo + threadIdx.x; t < hi; t += THREADS) put(t);
            return;
        }
        edges(put);
        const int n = vecs();
        constexpr int kDeep = 4;
        for (int v0 = threadIdx.x; v0 < n; v0 += THREADS * kDeep) {
            Pack<T, VEC> p[kDeep];
            uint32_t bits[kDeep], w[2][kDeep];
            bool skip[kDeep];
#pragma unroll
            for (int u = 0; u < kDeep; ++u) {
                const int64_t t = base + static_cast<int64_t>(v0 + u * THREADS) * VEC;
                w[0][u] = w[1][u] = 0xFFFFFFFFu;
                if (words != nullptr && v0 + u * THREADS < n) w[0][u] = words[t >> 5], w[1][u] = words[(t + VEC - 1) >> 5];
            }
#pragma unroll
            for (int u = 0; u < kDeep; ++u) {
                const int v = v0 + u * THREADS;
                bits[u] = __funnelshift_r(w[0][u], w[1][u], static_cast<uint32_t>((base + static_cast<int64_t>(v) * VEC) & 31)) & kAll;
                skip[u] = v >= n || (bits[u] == kAll && same(v));
                if (!skip[u] && bits[u] != 0) p[u] = x(v);
            }
#pragma unroll
            for (int u = 0; u < kDeep; ++u) {
                if (skip[u]) continue;
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if ((bits[u] >> j & 1u) == 0) p[u].v[j] = from_f32<T>(-INFINITY);
                *reinterpret_cast<Pack<T, VEC>*>(out + base + static_cast<int64_t>(v0 + u * THREADS) * VEC) = p[u];
            }
        }
    }
};

// the mask alone
constexpr int kMaskThreads = 256;
template <typename T>
__global__ void __launch_bounds__(kMaskThreads, 4) logit_mask_kernel(RulesArgs a) {
    const Slice<T, kMaskThreads> s(a);
    using Vec = Pack<T, Slice<T, kMaskThreads>::VEC>;
    s.finish(
        a, [&](int v) { return *reinterpret_cast<const Vec*>(s.in + s.base + static_cast<int64_t>(v) * Slice<T, kMaskThreads>::VEC); }, [&](int) { return a.in_place; },
        [&](int64_t t) { return s.in[t]; });
}

// C: type of a count; 16 bits where no history is longer than they count.  Shared memory: the slice's logits, its
// counts, its biases, each from token base - kRulesPad on; then the tokens that history or biases name, each once, so that the
// arithmetic runs on 32 of them at a time however thinly they lie.
template <typename T, typename C, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) logit_rules_kernel(RulesArgs a) {
    extern __shared__ uint4 smem[];
    __shared__ int n_named;
    const Slice<T, THREADS> s(a);
    constexpr int VEC = Slice<T, THREADS>::VEC;
    const int tokens = a.slice + kRulesPad, lane = threadIdx.x & 31;
    const bool counting = a.history != nullptr, biased = a.bias_ids != nullptr;
    T* x = reinterpret_cast<T*>(smem);
    C* count = reinterpret_cast<C*>(x + tokens);
    float* bias = reinterpret_cast<float*>(counting ? count + tokens : count);   // +0 until a bias has named the token (a sum of 0 is kept as -0)
    uint16_t* named = reinterpret_cast<uint16_t*>(biased ? bias + tokens : bias);

    // the logits on their way while the tables are made
    for (int v = threadIdx.x; v < s.vecs(); v += THREADS)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<unsigned>(__cvta_generic_to_shared(x + kRulesPad + v * VEC))),
                     "l"(s.in + s.base + static_cast<int64_t>(v) * VEC)
                     : "memory");
    Penalty pen = {1.0f, 0.0f, 0.0f};
    int64_t n = 0;   // ids of the row's history
    if (counting) {
        n = a.history_len;
        if (a.lengths != nullptr) {
            const int64_t own = id_at(a.lengths, a.lengths_wide, s.row);
            n = own < n ? own : n;
        }
        pen.repetition = a.repetition != nullptr ? a.repetition[s.row] : a.repetition_all;
        pen.presence = a.presence != nullptr ? a.presence[s.row] : a.presence_all;
        pen.frequency = a.frequency != nullptr ? a.frequency[s.row] : a.frequency_all;
    }
    s.edges([&](int64_t t) { x[t - s.base + kRulesPad] = s.in[t]; });
    {
        uint4* table = reinterpret_cast<uint4*>(count);
        const int chunks = tokens * static_cast<int>((counting ? sizeof(C) : 0) + (biased ? 4 : 0)) / 16;
        for (int i = threadIdx.x; i < chunks; i += THREADS) table[i] = make_uint4(0, 0, 0, 0);
        if (threadIdx.x == 0) n_named = 0;
        __syncthreads();
    }
    const uint32_t span = s.hi > s.lo ? static_cast<uint32_t>(s.hi - s.lo) : 0u;
    const int first = static_cast<int>(s.lo - s.base) + kRulesPad;
    // Counts tokens and lists those that are counted for the first time: a warp joins what its threads give to the list at once.
    auto add = [&](const uint32_t(&d)[kAhead]) {
        uint32_t before[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            before[u] = 1;
            if (d[u] == kNone) continue;
            const unsigned i = d[u] + first;
            unsigned* table = reinterpret_cast<unsigned*>(count);
            if (sizeof(C) == 4) before[u] = atomicAdd(table + i, 1u);
            else before[u] = atomicAdd(table + i / 2, i % 2 ? 0x10000u : 1u) >> (i % 2 * 16) & 0xFFFFu;
        }
        int mine = 0;
#pragma unroll
        for (int u = 0; u < kAhead; ++u) mine += before[u] == 0;
        if (!__any_sync(kAllLanes, mine != 0)) return;
        int upto = mine;
#pragma unroll
        for (int l = 1; l < 32; l <<= 1) {
            const int o = __shfl_up_sync(kAllLanes, upto, l);
            if (lane >= l) upto += o;
        }
        int at = 0;
        if (lane == 31) at = atomicAdd(&n_named, upto);
        at = __shfl_sync(kAllLanes, at, 31) + upto - mine;
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (before[u] == 0) named[at++] = static_cast<uint16_t>(d[u] + first);
    };
    if (counting) {
        const int64_t at = s.row * a.history_stride;
        if (a.history_wide) each_id<THREADS>(static_cast<const uint2*>(a.history) + at, n, static_cast<uint32_t>(s.lo), span, add);
        else each_id<THREADS>(static_cast<const uint32_t*>(a.history) + at, n, static_cast<uint32_t>(s.lo), span, add);
    }
    if (biased) __syncthreads();
    if (biased && threadIdx.x < 32) {
        // one warp, 32 entries at a time, each token's in the order of the list: the same sum every time
        for (int64_t j0 = 0; j0 < a.n_bias; j0 += 32) {
            int64_t t = -1;
            float v = 0.0f;
            if (j0 + lane < a.n_bias) {
                t = id_at(a.bias_ids, a.bias_wide, s.row * a.bias_ids_stride + j0 + lane);
                if (t < s.lo || t >= s.hi) t = -1;
                else v = a.bias_values[s.row * a.bias_values_stride + j0 + lane];
            }
            if (!__any_sync(kAllLanes, t >= 0)) continue;
            const unsigned same = __match_any_sync(kAllLanes, t);
            const bool leads = t >= 0 && (same & ((1u << lane) - 1u)) == 0;
            const int i = static_cast<int>(t - s.base) + kRulesPad;
            const float old = leads ? bias[i] : 0.0f;
            float sum = old;
            for (int l = 0; l < 32; ++l) {
                const float o = __shfl_sync(kAllLanes, v, l);
                if (same >> l & 1u) sum = __fadd_rn(sum, o);
            }
            if (leads) bias[i] = sum == 0.0f ? -0.0f : sum;
            const bool fresh = leads && __float_as_uint(old) == 0u && !(counting && count[i] != 0);
            const unsigned who = __ballot_sync(kAllLanes, fresh);
            if (fresh) named[n_named + __popc(who & ((1u << lane) - 1u))] = static_cast<uint16_t>(i);
            __syncwarp();
            if (lane == 0) n_named += __popc(who);
            __syncwarp();
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();

    for (int j = threadIdx.x; j < n_named; j += THREADS) {
        const int i = named[j];
        const float b = biased ? bias[i] : 0.0f;
        const uint32_t c = counting ? count[i] : 0u;
        if (c == 0 && b == 0.0f) continue;
        float f = to_f32(x[i]);
        if (b != 0.0f) f = __fadd_rn(f, b);
        if (c != 0) f = penalised(f, c, pen);
        x[i] = from_f32<T>(f);
    }
    __syncthreads();
    using Vec = Pack<T, VEC>;
    s.finish(
        a, [&](int v) { return *reinterpret_cast<const Vec*>(x + kRulesPad + v * VEC); },
        [&](int v) {
            if (!a.in_place) return false;
            bool none = true;
            for (int j = kRulesPad + v * VEC; j < kRulesPad + (v + 1) * VEC; ++j) none &= !(counting && count[j] != 0) && !(biased && bias[j] != 0.0f);
            return none;
        },
        [&](int64_t t) { return x[t - s.base + kRulesPad]; });
}

// Whether two matrices [rows][width] of elements of `size` bytes are the same one or no element of one is in the other: memory that does not
// meet, or columns of one wider matrix side by side.
static bool apart_or_same(uintptr_t a, int64_t stride_a, uintptr_t b, int64_t stride_b, int64_t rows, int64_t width, int64_t size) {
    if (rows == 1) stride_a = stride_b = width;
    if (a == b && stride_a == stride_b) return true;
    if (a + ((rows - 1) * stride_a + width) * size <= b || b + ((rows - 1) * stride_b + width) * size <= a) return true;
    if (stride_a != stride_b) return false;
    const int64_t d = static_cast<int64_t>((a > b ? a - b : b - a) % (stride_a * size));
    return d >= width * size && stride_a * size - d >= width * size;
}

// ------------------------------------------------------------------ launches
constexpr int64_t kThreadMemory = 220;   // bytes of shared memory per thread: an SM's for 1024

template <typename T, typename C, int THREADS>
static int launch_slices(const RulesArgs& a, size_t smem, cudaStream_t st) {
    static std::atomic<bool> ready[64];   // a kernel may use more than 48 KB only after a call per device has said so
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return route_fail(TGO_E_CUDA, "cudaGetDevice failed");
    if (dev >= 64 || !ready[dev].load(std::memory_order_relaxed)) {
        if (cudaFuncSetAttribute(logit_rules_kernel<T, C, THREADS>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kThreadMemory * THREADS)) != cudaSuccess)
            return route_fail(TGO_E_CUDA, "cudaFuncSetAttribute failed");
        if (dev < 64) ready[dev].store(true, std::memory_order_relaxed);
    }
    logit_rules_kernel<T, C, THREADS><<<static_cast<unsigned>(a.rows * a.slices), THREADS, smem, st>>>(a);
    return cudaGetLastError() == cudaSuccess ? TGO_OK : route_fail(TGO_E_CUDA, "logit_rules_kernel launch failed");
}

template <typename T>
static int launch_rules(RulesArgs& a, int64_t id_bytes, cudaStream_t st) {
    const bool tables = a.history != nullptr || a.bias_ids != nullptr, narrow = a.history_len <= UINT16_MAX;
    // Every slice reads all of a history, so that of a long one larger slices read less; small ones overlap their phases better
    // (us with 256 / 512 threads, bf16, 248320 tokens: 16 rows of 1024 ids 7.6 / 10.1, of 4096 10.7 / 10.7, of 16384 20.3 / 16.1;
    // 200 rows of 1024 ids 51.5 / 57.7, of 4096 68.7 / 64.9, of 16384 162 / 122; with 512 / 1024: 16 rows of 16384 16.1 / 18.9,
    // 64 rows 43.6 / 37.2, 200 rows 122 / 108, 64 rows of 8192 29.7 / 33.2).
    const int threads = a.history_len < 4096 ? 256 : a.history_len < 16384 || a.rows < 32 ? 512 : 1024;
    const int64_t token_bytes = static_cast<int64_t>(sizeof(T)) + (a.history != nullptr ? (narrow ? 2 : 4) : 0) + (a.bias_ids != nullptr ? 4 : 0);
    // the list of named tokens is as long as history and biases together, or as the slice
    const int64_t all_names = a.history_len + a.n_bias, memory = kThreadMemory * threads;
    int64_t most = 16384;
    if (tables) {
        const int64_t long_list = memory / (token_bytes + 2), short_list = all_names < memory ? (memory - 2 * all_names) / token_bytes : 0;
        most = ((long_list > short_list ? long_list : short_list) - kRulesPad - 1) / 128 * 128;
        if (most > 65536 - 256) most = 65536 - 256;   // the list holds 16 bits of a token
    }
    // some 1024 threads per SM, no slice shorter than 4 tokens per thread, none longer than its shared memory takes
    int64_t slices = (148 * (1024 / threads) + a.rows - 1) / a.rows;
    if (slices > (a.vocab + 4 * threads - 1) / (4 * threads)) slices = (a.vocab + 4 * threads - 1) / (4 * threads);
    if (a.history != nullptr) {
        // Of a long history so few slices that they read no more than twice as much of it as they read and write else, down to a
        // block per SM (us with / without, bf16: 4 rows of 8192 ids 7.2 / 9.1, of 65535 25.8 / 37.0; 16 rows of 16384 16.2 / 17.9).
        const int64_t fair = 4 * a.vocab * static_cast<int64_t>(sizeof(T)) / (a.history_len * id_bytes), fewest = (148 + a.rows - 1) / a.rows;
        if (slices > fair) slices = fair > fewest ? fair : fewest < slices ? fewest : slices;
    }
    if (slices < (a.vocab + most - 1) / most) slices = (a.vocab + most - 1) / most;
    if (a.rows > INT32_MAX / slices) return route_fail(TGO_E_ARG, "too many logits");
    a.slices = static_cast<int>(slices);
    a.slice = static_cast<int>(((a.vocab + slices - 1) / slices + 127) / 128 * 128);
    if (!tables) {
        if (a.in_place && a.allowed == nullptr) return TGO_OK;
        logit_mask_kernel<T><<<static_cast<unsigned>(a.rows * slices), kMaskThreads, 0, st>>>(a);
        return cudaGetLastError() == cudaSuccess ? TGO_OK : route_fail(TGO_E_CUDA, "logit_mask_kernel launch failed");
    }
    const int64_t names = all_names < a.slice + kRulesPad ? all_names : a.slice + kRulesPad;
    const size_t smem = static_cast<size_t>(token_bytes) * (a.slice + kRulesPad) + static_cast<size_t>(names) * 2;
    if (threads == 256) return launch_slices<T, uint16_t, 256>(a, smem, st);
    if (threads == 1024) return narrow ? launch_slices<T, uint16_t, 1024>(a, smem, st) : launch_slices<T, uint32_t, 1024>(a, smem, st);
    return narrow ? launch_slices<T, uint16_t, 512>(a, smem, st) : launch_slices<T, uint32_t, 512>(a, smem, st);
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
    if ((history != nullptr && (!aligned_to(history_id_bytes, history) || (lengths != nullptr && !aligned_to(length_bytes, lengths)))) ||
        (bias_ids != nullptr && !aligned_to(bias_id_bytes, bias_ids)) || !aligned_to(4, repetition, presence, frequency, bias_values, allowed))
        return route_fail(TGO_E_ARG, kMisaligned);
    if (!apart_or_same(i, in_stride, o, out_stride, rows, vocab, size))
        return route_fail(TGO_E_ARG, "out must be the logits themselves or share no memory with them");
    RulesArgs a = {};
    a.logits = logits, a.out = out, a.rows = rows, a.vocab = vocab, a.in_stride = in_stride, a.out_stride = out_stride;
    if (history != nullptr && history_len > 0) a.history = history, a.lengths = lengths, a.history_len = history_len, a.history_stride = history_stride;
    a.history_wide = history_id_bytes == 8, a.lengths_wide = length_bytes == 8;
    a.repetition = repetition, a.presence = presence, a.frequency = frequency;
    a.repetition_all = repetition_all, a.presence_all = presence_all, a.frequency_all = frequency_all;
    if (bias_ids != nullptr && n_bias > 0) a.bias_ids = bias_ids, a.bias_values = bias_values, a.n_bias = n_bias;
    a.bias_ids_stride = bias_ids_stride, a.bias_values_stride = bias_values_stride, a.bias_wide = bias_id_bytes == 8;
    a.allowed = allowed, a.allowed_stride = allowed_stride;
    a.in_place = logits == out;
    // 16-byte accesses where every row of the result lies to its boundary as the row of logits does
    a.vectors = (i - o) % 16 == 0 && (rows == 1 || (in_stride - out_stride) * size % 16 == 0);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == TGO_BF16) return launch_rules<__nv_bfloat16>(a, history_id_bytes, st);
    if (dtype == TGO_FP16) return launch_rules<__half>(a, history_id_bytes, st);
    return launch_rules<float>(a, history_id_bytes, st);
}
