// Tokens to rows sorted by expert and back, with their gradients, for one GPU's mixture-of-experts layer:
//   dispatch   rows[row_of_pair[t, s]] = x[t]
//   combine    y[t] = sum_s w[t, s] rows[row_of_pair[t, s]]
//              drows[row_of_pair[t, s]] = w[t, s] dy[t],  dw[t, s] = <dy[t], rows[row_of_pair[t, s]]>
// The gradient of dispatch is combine without weights.  bf16 rows, sums in fp32, one rounding.
//
// All of it is bound by memory: a token's row is read once and its top_k rows are written (or read) once.  One B200, rows of
// 2048, top 8, GPU time in a graph (bytes that have to move over it):
//   dispatch 16384 tokens 118 us (5.1 TB/s): the sort 13, the rows 105 (5.8 TB/s); its gradient 93.8 (6.4)
//   combine 600 tokens 4.4 us, 8192 48.6 (6.2 TB/s), its gradients 99 (5.8)
// A copy runs at 6.4.
#include "../../include/tgo_mmq.h"

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "aligned.h"

namespace tgo {

int route_fail(int code, const char* msg);  // tgo_api.cu

constexpr int kMoveThreads = 256;

__device__ __forceinline__ void widen(uint4 q, float (&f)[8]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        f[2 * j] = __uint_as_float(w[j] << 16);
        f[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
    }
}
__device__ __forceinline__ uint4 narrow(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
        w[j] = *reinterpret_cast<const uint32_t*>(&b);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// ------------------------------------------------------------------ the order of the pairs
// A stable sort of the pairs by expert gives every pair its row: the pairs of lower experts, then those of the same
// expert that come before it.  Ids outside the experts name none.

// Few pairs: one launch.  A block holds all ids and counts for its own token's pairs what is in front of them, a
// warp per pair; the experts' end rows are counted the same way, an expert per warp.  Rows behind the last
// expert's are zeros, one for each pair that names no expert.  The work grows with the square of the pairs.  us of
// a whole dispatch of 2048-wide rows in one launch / sorted (below), in a graph:
//   256 experts, top 8     1 token 2.6 / 6.2, 16 2.8 / 7.6, 256 4.8 / 9.6, 512 9.2 / 11.5
//   1000 experts, top 4    16 2.6 / 10.2, 512 5.2 / 12.3, 1024 9.9 / 14.5;   4096 experts, top 8    512 11.8 / 22.2
//   256 experts, top 1     256 2.3 / 7.7, 1024 3.5 / 8.9, 2048 6.8 / 10.9, 4096 15.1 / 13.8;   top 32    16 5.8 / 10.3, 128 11.4 / 12.1
//   1024 experts, top 128  8 18.6 / 22.1, 32 36.1 / 23.9;   top 512    1 55.6 / 57.0, 4 87.9 / 58.6;   top 1024    1 130 / 105, 4 257 / 108
// The rule looks at the pairs alone, as a caller asks for the workspace by them; past a top_k of 100 or so it is not the faster side.
constexpr int kFewPairs = 4096;
constexpr int kMoveWarps = kMoveThreads / 32;
__global__ void __launch_bounds__(kMoveThreads) dispatch_few_kernel(const uint4* __restrict__ x, const int32_t* __restrict__ ids, int experts, int tokens, int top_k,
                                                                    uint4* __restrict__ rows, int32_t* __restrict__ row_of_pair,
                                                                    int64_t* __restrict__ expert_indices, int32_t* __restrict__ expert_offsets,
                                                                    int vec_per_row) {
    __shared__ int32_t id[kFewPairs];
    __shared__ int32_t row[1024];   // of the token's pairs; -1 - r: zeros to row r
    const int pairs = tokens * top_k, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int i = threadIdx.x; i < pairs; i += kMoveThreads) {
        const int e = ids[i];
        id[i] = e >= 0 && e < experts ? e : experts;   // those that name none come last
    }
    __syncthreads();
    const int token = blockIdx.x;
    if (token < tokens) {
        for (int s = warp; s < top_k; s += kMoveWarps) {
            const int pair = token * top_k + s, e = id[pair];
            int before = 0;
            for (int j = lane; j < pairs; j += 32) before += id[j] < e || (id[j] == e && j < pair);
            before = __reduce_add_sync(0xFFFFFFFFu, before);
            if (lane == 0) {
                row[s] = e < experts ? before : -1 - before;
                row_of_pair[pair] = e < experts ? before : -1;
            }
        }
    }
    for (int e = blockIdx.x * kMoveWarps + warp; e < experts; e += gridDim.x * kMoveWarps) {
        int upto = 0;
        for (int j = lane; j < pairs; j += 32) upto += id[j] <= e;
        upto = __reduce_add_sync(0xFFFFFFFFu, upto);
        if (lane == 0) {
            expert_offsets[e] = upto;
            expert_indices[e] = e;
        }
    }
    if (token >= tokens) return;
    __syncthreads();
    for (int c = threadIdx.x; c < vec_per_row; c += kMoveThreads) {
        const uint4 val = x[static_cast<long long>(token) * vec_per_row + c];
        for (int s = 0; s < top_k; ++s) {
            const int r = row[s];
            rows[static_cast<long long>(r >= 0 ? r : -1 - r) * vec_per_row + c] = r >= 0 ? val : make_uint4(0, 0, 0, 0);
        }
    }
}

// More pairs: counts per block and expert, their running sums, the rows.  All three use the whole GPU (the sort of
// routing.cu, for 4096 experts, adds up in one block: 131072 pairs, 256 experts, 21.6 us; these 13).
constexpr int kSortExperts = 1024;
constexpr int kSortPairs = kMoveThreads;   // pairs of a block

__global__ void __launch_bounds__(kMoveThreads) pair_count_kernel(const int32_t* __restrict__ ids, int pairs, int experts, int32_t* __restrict__ counts) {
    __shared__ int32_t hist[kSortExperts];
    for (int e = threadIdx.x; e < experts; e += kMoveThreads) hist[e] = 0;
    __syncthreads();
    const unsigned i = blockIdx.x * kSortPairs + threadIdx.x;   // up to 2^31 + 254
    const int e = i < static_cast<unsigned>(pairs) ? ids[i] : -1;
    if (e >= 0 && e < experts) atomicAdd(&hist[e], 1);
    __syncthreads();
    for (int k = threadIdx.x; k < experts; k += kMoveThreads) counts[static_cast<size_t>(blockIdx.x) * experts + k] = hist[k];
}

// counts[b][e] -> pairs of e in the blocks in front of b; totals[e].  A block takes 32 experts, so that its reads are whole
// lines, its warps a run of blocks each.
constexpr int kScanWarps = 32;
__global__ void __launch_bounds__(kScanWarps * 32) pair_scan_kernel(int32_t* __restrict__ counts, int blocks, int experts, int32_t* __restrict__ totals) {
    __shared__ int32_t sums[kScanWarps][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = blockIdx.x * 32 + lane;
    const int run = (blocks + kScanWarps - 1) / kScanWarps, from = warp * run, to = min(from + run, blocks);
    const bool in = e < experts;
    int sum = 0;
#pragma unroll 8
    for (int b = from; b < to; ++b) sum += in ? counts[static_cast<size_t>(b) * experts + e] : 0;
    sums[warp][lane] = sum;
    __syncthreads();
    int before = 0;
    for (int w = 0; w < warp; ++w) before += sums[w][lane];
    if (warp == kScanWarps - 1 && in) totals[e] = before + sum;
    for (int b0 = from; b0 < to; b0 += 8) {
        int v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = in && b0 + u < to ? counts[static_cast<size_t>(b0 + u) * experts + e] : 0;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            if (in && b0 + u < to) counts[static_cast<size_t>(b0 + u) * experts + e] = before;
            before += v[u];
        }
    }
}

__global__ void __launch_bounds__(kMoveThreads) pair_rows_kernel(const int32_t* __restrict__ ids, int pairs, int experts, const int32_t* __restrict__ starts,
                                                                 const int32_t* __restrict__ totals, int32_t* __restrict__ row_of_pair,
                                                                 int64_t* __restrict__ expert_indices, int32_t* __restrict__ expert_offsets) {
    __shared__ __align__(16) uint16_t seen[kMoveWarps][kSortExperts];   // pairs of an expert per warp, then in the warps in front
    __shared__ int32_t first[kSortExperts];               // an expert's first row of this block
    __shared__ int32_t warp_sum[kMoveWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int k = threadIdx.x; k < kMoveWarps * kSortExperts / 8; k += kMoveThreads) reinterpret_cast<uint4*>(seen)[k] = make_uint4(0, 0, 0, 0);
    // first rows: the lower experts' pairs and this expert's in the blocks in front
    int carry = 0;
    for (int k0 = 0; k0 < experts; k0 += kMoveThreads) {
        const int k = k0 + threadIdx.x, own = k < experts ? totals[k] : 0;
        const int here = k < experts ? starts[static_cast<size_t>(blockIdx.x) * experts + k] : 0;
        int upto = own;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xFFFFFFFFu, upto, d);
            if (lane >= d) upto += o;
        }
        if (lane == 31) warp_sum[warp] = upto;
        __syncthreads();
        int all = 0;
        for (int w = 0; w < kMoveWarps; ++w) {
            upto += w < warp ? warp_sum[w] : 0;
            all += warp_sum[w];
        }
        upto += carry;
        carry += all;
        if (k < experts) {
            first[k] = upto - own + here;
            if (blockIdx.x == 0) {
                expert_offsets[k] = upto;
                expert_indices[k] = k;
            }
        }
        __syncthreads();
    }
    const unsigned i = blockIdx.x * kSortPairs + threadIdx.x;   // up to 2^31 + 254
    const bool in = i < static_cast<unsigned>(pairs);
    int e = in ? ids[i] : -1;
    if (e >= experts) e = -1;
    const unsigned same = __match_any_sync(0xFFFFFFFFu, e);
    const int rank = __popc(same & ((1u << lane) - 1u));
    if (e >= 0 && rank == 0) seen[warp][e] = static_cast<uint16_t>(__popc(same));
    __syncthreads();
    int before = rank;
    if (e >= 0)
        for (int w = 0; w < warp; ++w) before += seen[w][e];
    if (in) row_of_pair[i] = e >= 0 ? first[e] + before : -1;
}

// A token's row to the rows of its pairs; zeros to the rows behind the last expert's (those of the pairs that name no expert).
__global__ void __launch_bounds__(kMoveThreads) dispatch_rows_kernel(const uint4* __restrict__ x, const int32_t* __restrict__ row_of_pair,
                                                                     const int32_t* __restrict__ expert_ends, int experts, long long tokens, int top_k,
                                                                     uint4* __restrict__ rows, int vec_per_row) {
    const long long step = static_cast<long long>(kMoveThreads) * gridDim.x, first = blockIdx.x * static_cast<long long>(kMoveThreads) + threadIdx.x;
    for (long long v = first; v < tokens * vec_per_row; v += step) {
        const long long t = v / vec_per_row;
        const int c = static_cast<int>(v - t * vec_per_row);
        const uint4 val = x[v];
        for (int s = 0; s < top_k; ++s) {
            const int row = row_of_pair[t * top_k + s];
            if (row >= 0) rows[static_cast<long long>(row) * vec_per_row + c] = val;
        }
    }
    const long long end = tokens * top_k * vec_per_row;
    for (long long v = static_cast<long long>(expert_ends[experts - 1]) * vec_per_row + first; v < end; v += step) rows[v] = make_uint4(0, 0, 0, 0);
}

__global__ void __launch_bounds__(kMoveThreads) moe_combine_kernel(const uint4* __restrict__ rows, long long n_rows, const int32_t* __restrict__ row_of_pair,
                                                                   const float* __restrict__ weights, uint4* __restrict__ out, long long tokens,
                                                                   int top_k, int vec_per_row) {
    constexpr int kDeep = 4;   // rows under way per thread (8192 tokens, one row / four: 51.8 / 48.6 us)
    const long long step = static_cast<long long>(kMoveThreads) * gridDim.x;
    for (long long v = blockIdx.x * static_cast<long long>(kMoveThreads) + threadIdx.x; v < tokens * vec_per_row; v += step) {
        const long long t = v / vec_per_row;
        const int c = static_cast<int>(v - t * vec_per_row);
        float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        for (int s0 = 0; s0 < top_k; s0 += kDeep) {
            uint4 q[kDeep];
            float w[kDeep];
            bool in[kDeep];
#pragma unroll
            for (int u = 0; u < kDeep; ++u) {
                const int row = s0 + u < top_k ? row_of_pair[t * top_k + s0 + u] : -1;
                in[u] = row >= 0 && row < n_rows;
                if (in[u]) q[u] = rows[static_cast<long long>(row) * vec_per_row + c];
                w[u] = in[u] && weights != nullptr ? weights[t * top_k + s0 + u] : 1.0f;
            }
#pragma unroll
            for (int u = 0; u < kDeep; ++u) {
                if (!in[u]) continue;
                float f[8];
                widen(q[u], f);
#pragma unroll
                for (int j = 0; j < 8; ++j) acc[j] = fmaf(w[u], f[j], acc[j]);
            }
        }
        out[v] = narrow(acc);
    }
}

// How many pairs name each row.  A map that dispatch makes names a row once at most.  Where one is named more often, the last block to be done
// lists the pairs of such rows, sorted by row and, of a row, in their order (a radix sort by one block, 8 bits a pass: linear in the pairs, and
// the maps that are the rule pay no launch for it, but 0.4 to 1.7 us).  Such a row's count becomes -1 - its first place in the list.
// Gradients of rows and weights, rows of 2048, every row named by two pairs / all pairs naming one row: 65536 pairs 0.6 / 14 ms, 524288 6 / 141 ms.
constexpr int kListThreads = 1024, kListWarps = kListThreads / 32;
struct RowLists {
    int32_t* count;        // [n_rows]
    int32_t* state;        // blocks that are done; whether a row is named twice; the list's length
    int32_t *even, *odd;   // [pairs] each: where passes 0, 2 and 1, 3 leave the list
    int passes;            // bytes of a row's number
    __device__ int32_t* after(int pass) const { return pass & 1 ? odd : even; }
};
__global__ void __launch_bounds__(kListThreads) count_rows_kernel(const int32_t* __restrict__ row_of_pair, long long pairs, long long n_rows, RowLists l) {
    const long long i = blockIdx.x * static_cast<long long>(kListThreads) + threadIdx.x;
    bool again = false;
    if (i < pairs) {
        const int row = row_of_pair[i];
        if (row >= 0 && row < n_rows) again = atomicAdd(&l.count[row], 1) != 0;
    }
    again = __syncthreads_or(again);
    __shared__ bool last;
    if (threadIdx.x == 0) {
        if (again) atomicOr(&l.state[1], 1);
        __threadfence();                          // the whole block's counts, which the barrier has put in front of it
        last = atomicAdd(&l.state[0], 1) == static_cast<int32_t>(gridDim.x) - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    if (__ldcg(&l.state[1]) == 0) return;

    __shared__ int32_t next[256];                 // where a digit's next entry goes
    __shared__ uint16_t among[kListWarps][256];   // a step's entries of a digit per warp, then in the warps in front
    __shared__ int32_t total;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long n = pairs;                          // the first pass looks at all pairs and takes those of rows that are named again
    for (int pass = 0; pass < l.passes; ++pass) {
        const int32_t* from = l.after(pass - 1);
        int32_t* to = l.after(pass);
        int digit;                                // of the entry that was looked at last; -1: none
        auto entry = [&](long long k) {
            digit = -1;
            if (k >= n) return -1;
            const int p = pass == 0 ? static_cast<int>(k) : __ldcg(from + k);
            const int row = row_of_pair[p];
            if (pass > 0 || (row >= 0 && row < n_rows && __ldcg(&l.count[row]) > 1)) digit = row >> (8 * pass) & 255;
            return p;
        };
        if (threadIdx.x < 256) next[threadIdx.x] = 0;
        __syncthreads();
        for (long long k = threadIdx.x; k < n; k += kListThreads) {
            entry(k);
            if (digit >= 0) atomicAdd(&next[digit], 1);
        }
        __syncthreads();
        if (warp == 0) {
            int carry = 0;
            for (int d0 = 0; d0 < 256; d0 += 32) {
                const int own = next[d0 + lane];
                int upto = own;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const int o = __shfl_up_sync(0xFFFFFFFFu, upto, d);
                    if (lane >= d) upto += o;
                }
                next[d0 + lane] = carry + upto - own;
                carry += __shfl_sync(0xFFFFFFFFu, upto, 31);
            }
            if (lane == 0) total = carry;
        }
        for (long long k0 = 0; k0 < n; k0 += kListThreads) {
            for (int k = threadIdx.x; k < kListWarps * 256; k += kListThreads) (&among[0][0])[k] = 0;
            const int p = entry(k0 + threadIdx.x);
            __syncthreads();
            const unsigned same = __match_any_sync(0xFFFFFFFFu, digit);
            const int rank = __popc(same & ((1u << lane) - 1u));
            if (digit >= 0 && rank == 0) among[warp][digit] = static_cast<uint16_t>(__popc(same));
            __syncthreads();
            int here = 0;
            if (threadIdx.x < 256) {
                for (int w = 0; w < kListWarps; ++w) {
                    const int c = among[w][threadIdx.x];
                    among[w][threadIdx.x] = static_cast<uint16_t>(here);
                    here += c;
                }
            }
            __syncthreads();
            if (digit >= 0) to[next[digit] + among[warp][digit] + rank] = p;
            __syncthreads();
            if (threadIdx.x < 256) next[threadIdx.x] += here;
        }
        __syncthreads();
        n = total;
    }
    const int32_t* sorted = l.after(l.passes - 1);
    for (long long k = threadIdx.x; k < n; k += kListThreads) {
        const int row = row_of_pair[__ldcg(sorted + k)];
        if (k == 0 || row_of_pair[__ldcg(sorted + k - 1)] != row) l.count[row] = static_cast<int32_t>(-1 - k);
    }
    if (threadIdx.x == 0) l.state[2] = static_cast<int32_t>(n);
}

// One warp per pair.  A row that none names gets zeros from the warp of that number, one that several pairs name the sum over them: its
// columns are divided among the warps of the first 32 of them.
__global__ void __launch_bounds__(kMoveThreads) combine_grad_kernel(const uint4* __restrict__ dy, const uint4* __restrict__ rows, long long n_rows,
                                                                    const int32_t* __restrict__ row_of_pair, const float* __restrict__ weights,
                                                                    RowLists l, uint4* __restrict__ d_rows, float* __restrict__ d_weights,
                                                                    long long pairs, int top_k, int vec_per_row) {
    const int lane = threadIdx.x & 31;
    const long long pair = blockIdx.x * static_cast<long long>(kMoveThreads / 32) + (threadIdx.x >> 5);
    const int32_t* count = l.count;
    if (d_rows != nullptr && pair < n_rows && count[pair] == 0)
        for (int c = lane; c < vec_per_row; c += 32) d_rows[pair * vec_per_row + c] = make_uint4(0, 0, 0, 0);
    if (pair >= pairs) return;
    int row = row_of_pair[pair];
    if (row >= n_rows) row = -1;
    float dot = 0.0f;
    if (row >= 0) {
        const uint4* g = dy + pair / top_k * vec_per_row;
        const uint4* r = rows + static_cast<long long>(row) * vec_per_row;
        const bool alone = d_rows == nullptr || count[row] == 1;
        const float w = weights != nullptr ? weights[pair] : 1.0f;
        constexpr int kDeep = 4;   // chunks under way per lane (gradients of 8192 tokens, 1 / 2 / 4 / 8 chunks: 102 / 109 / 98 / 130 us)
        for (int c0 = lane; c0 < vec_per_row; c0 += 32 * kDeep) {
            uint4 dyv[kDeep], rowv[kDeep];
#pragma unroll
            for (int u = 0; u < kDeep; ++u) {
                const int c = c0 + 32 * u;
                if (c >= vec_per_row) continue;
                dyv[u] = g[c];
                if (d_weights != nullptr) rowv[u] = r[c];
            }
#pragma unroll
            for (int u = 0; u < kDeep; ++u) {
                const int c = c0 + 32 * u;
                if (c >= vec_per_row) continue;
                float f[8];
                widen(dyv[u], f);
                if (d_weights != nullptr) {
                    float h[8];
                    widen(rowv[u], h);
#pragma unroll
                    for (int j = 0; j < 8; ++j) dot = fmaf(f[j], h[j], dot);
                }
                if (d_rows != nullptr && alone) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) f[j] *= w;
                    d_rows[static_cast<long long>(row) * vec_per_row + c] = narrow(f);
                }
            }
        }
        if (!alone) {
            const int32_t* list = l.after(l.passes - 1);
            const long long first = -1 - static_cast<long long>(count[row]), n = l.state[2];
            // entry k of the list, if it is one of this row; -1 else
            auto of_row = [&](long long k) {
                const int p = k < n ? list[k] : -1;
                return p >= 0 && row_of_pair[p] == row ? p : -1;
            };
            const int p0 = of_row(first + lane);
            const int helpers = __popc(__ballot_sync(0xFFFFFFFFu, p0 >= 0));
            const unsigned me = __ballot_sync(0xFFFFFFFFu, p0 == pair);
            for (int c0 = me == 0 ? vec_per_row : 32 * (__ffs(me) - 1); c0 < vec_per_row; c0 += 32 * helpers) {
                const int c = c0 + lane;
                float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                int m = 32;
                for (long long k = first; m == 32; k += 32) {
                    const int p = of_row(k + lane);
                    const float wp = p >= 0 && weights != nullptr ? weights[p] : 1.0f;
                    m = __popc(__ballot_sync(0xFFFFFFFFu, p >= 0));
#pragma unroll 4
                    for (int j = 0; j < m; ++j) {
                        const int q = __shfl_sync(0xFFFFFFFFu, p, j);
                        const float w = __shfl_sync(0xFFFFFFFFu, wp, j);
                        if (c >= vec_per_row) continue;
                        float f[8];
                        widen(dy[static_cast<long long>(q / top_k) * vec_per_row + c], f);
#pragma unroll
                        for (int u = 0; u < 8; ++u) acc[u] = fmaf(w, f[u], acc[u]);
                    }
                }
                if (c < vec_per_row) d_rows[static_cast<long long>(row) * vec_per_row + c] = narrow(acc);
            }
        }
    }
    if (d_weights != nullptr) {
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) dot += __shfl_xor_sync(0xFFFFFFFFu, dot, d);
        if (lane == 0) d_weights[pair] = dot;
    }
}

static int launched(const char* what) { return cudaGetLastError() == cudaSuccess ? TGO_OK : route_fail(TGO_E_CUDA, what); }
static int check_rows(int64_t tokens, int64_t top_k, int64_t width) {
    if (tokens <= 0) return route_fail(TGO_E_ARG, "zero-row inputs are not supported");
    if (top_k <= 0 || top_k > 1024) return route_fail(TGO_E_ARG, "top_k must be in 1..1024");
    if (tokens > INT32_MAX / top_k) return route_fail(TGO_E_ARG, "tokens * top_k must be below 2^31");
    if (width <= 0 || width % 8 != 0 || width > INT32_MAX) return route_fail(TGO_E_ARG, "the row length must be a positive multiple of 8");
    return TGO_OK;
}
static int move_grid(int64_t work_items) {
    int64_t blocks = (work_items + kMoveThreads - 1) / kMoveThreads;
    if (blocks > 148LL * 16) blocks = 148LL * 16;
    return static_cast<int>(blocks < 1 ? 1 : blocks);
}
static int64_t up16(int64_t n) { return (n + 15) & ~static_cast<int64_t>(15); }

}  // namespace tgo

using namespace tgo;

extern "C" {

int64_t tgo_moe_dispatch_workspace_bytes(int64_t n_pairs, int64_t num_experts) {
    if (n_pairs < 0 || num_experts <= 0) return -1;
    if (n_pairs <= kFewPairs) return 0;
    if (num_experts <= kSortExperts) return ((n_pairs + kSortPairs - 1) / kSortPairs + 1) * num_experts * 4;
    return up16(n_pairs * 4) + tgo_route_workspace_bytes(n_pairs, num_experts);
}

int tgo_moe_dispatch(const void* x, const int32_t* expert_ids, int64_t tokens, int64_t top_k, int64_t num_experts, int64_t width, void* rows,
                     int32_t* row_of_pair, int64_t* expert_indices, int32_t* expert_offsets, void* workspace, int64_t workspace_bytes,
                     void* stream) {
    if (x == nullptr || expert_ids == nullptr || rows == nullptr || row_of_pair == nullptr || expert_indices == nullptr || expert_offsets == nullptr)
        return route_fail(TGO_E_ARG, "null pointer");
    int rc = check_rows(tokens, top_k, width);
    if (rc != TGO_OK) return rc;
    if (!aligned_to(16, x, rows)) return route_fail(TGO_E_ARG, "data pointers must be 16-byte aligned");
    if (!aligned_to(4, expert_ids, row_of_pair, expert_offsets) || !aligned_to(8, expert_indices)) return route_fail(TGO_E_ARG, kMisaligned);
    const int64_t pairs = tokens * top_k;
    if (num_experts <= 0 || num_experts > 4096) return route_fail(TGO_E_ARG, "num_experts must be in 1..4096");
    const int64_t need = tgo_moe_dispatch_workspace_bytes(pairs, num_experts);
    if (workspace_bytes < need || (need > 0 && workspace == nullptr)) return route_fail(TGO_E_WORKSPACE, "dispatch workspace too small");
    if (!aligned_to(4, workspace)) return route_fail(TGO_E_ARG, "the workspace must be 4-byte aligned");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int vec = static_cast<int>(width / 8), n = static_cast<int>(pairs), e = static_cast<int>(num_experts);
    if (need == 0) {
        const int64_t for_experts = (num_experts + 2 * kMoveWarps - 1) / (2 * kMoveWarps);   // two experts' end rows per warp
        dispatch_few_kernel<<<static_cast<unsigned>(tokens > for_experts ? tokens : for_experts), kMoveThreads, 0, st>>>(
            static_cast<const uint4*>(x), expert_ids, e, static_cast<int>(tokens), static_cast<int>(top_k), static_cast<uint4*>(rows), row_of_pair,
            expert_indices, expert_offsets, vec);
        return launched("dispatch_few_kernel launch failed");
    }
    if (num_experts <= kSortExperts) {
        const int blocks = static_cast<int>((pairs + kSortPairs - 1) / kSortPairs);
        int32_t* totals = static_cast<int32_t*>(workspace);
        int32_t* counts = totals + num_experts;
        pair_count_kernel<<<blocks, kMoveThreads, 0, st>>>(expert_ids, n, e, counts);
        pair_scan_kernel<<<(e + 31) / 32, kScanWarps * 32, 0, st>>>(counts, blocks, e, totals);
        pair_rows_kernel<<<blocks, kMoveThreads, 0, st>>>(expert_ids, n, e, counts, totals, row_of_pair, expert_indices, expert_offsets);
    } else {
        int32_t* sorted = static_cast<int32_t*>(workspace);
        const int64_t used = up16(pairs * 4);
        rc = tgo_route_sort(expert_ids, pairs, num_experts, sorted, row_of_pair, expert_indices, expert_offsets, nullptr,
                            static_cast<uint8_t*>(workspace) + used, workspace_bytes - used, stream);
        if (rc != TGO_OK) return rc;
    }
    dispatch_rows_kernel<<<move_grid(tokens * vec), kMoveThreads, 0, st>>>(static_cast<const uint4*>(x), row_of_pair, expert_offsets, e, tokens,
                                                                           static_cast<int>(top_k), static_cast<uint4*>(rows), vec);
    return launched("dispatch kernel launch failed");
}

int tgo_moe_combine(const void* rows, int64_t n_rows, const int32_t* row_of_pair, const float* weights, void* out, int64_t tokens, int64_t top_k,
                    int64_t width, void* stream) {
    if (rows == nullptr || row_of_pair == nullptr || out == nullptr) return route_fail(TGO_E_ARG, "null pointer");
    const int rc = check_rows(tokens, top_k, width);
    if (rc != TGO_OK) return rc;
    if (n_rows < 0) return route_fail(TGO_E_ARG, "a negative number of rows");
    if (!aligned_to(16, rows, out)) return route_fail(TGO_E_ARG, "data pointers must be 16-byte aligned");
    if (!aligned_to(4, row_of_pair, weights)) return route_fail(TGO_E_ARG, kMisaligned);
    const int vec = static_cast<int>(width / 8);
    moe_combine_kernel<<<move_grid(tokens * vec), kMoveThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const uint4*>(rows), n_rows, row_of_pair, weights, static_cast<uint4*>(out), tokens, static_cast<int>(top_k), vec);
    return launched("moe_combine_kernel launch failed");
}

int64_t tgo_moe_combine_grad_workspace_bytes(int64_t n_pairs, int64_t n_rows) {
    if (n_pairs < 0 || n_rows < 0) return -1;
    return (n_rows + 3 + 2 * n_pairs) * 4;
}

int tgo_moe_combine_grad(const void* dy, const void* rows, int64_t n_rows, const int32_t* row_of_pair, const float* weights, void* d_rows,
                         float* d_weights, int64_t tokens, int64_t top_k, int64_t width, void* workspace, int64_t workspace_bytes, void* stream) {
    if (dy == nullptr || row_of_pair == nullptr || (d_weights != nullptr && rows == nullptr)) return route_fail(TGO_E_ARG, "null pointer");
    if (d_rows == nullptr && d_weights == nullptr) return route_fail(TGO_E_ARG, "no gradient is asked for");
    const int rc = check_rows(tokens, top_k, width);
    if (rc != TGO_OK) return rc;
    if (n_rows < 0 || n_rows > INT32_MAX) return route_fail(TGO_E_ARG, "the number of rows must be in 0..2^31-1");
    if (!aligned_to(16, dy, rows, d_rows)) return route_fail(TGO_E_ARG, "data pointers must be 16-byte aligned");
    if (!aligned_to(4, row_of_pair, weights, d_weights)) return route_fail(TGO_E_ARG, kMisaligned);
    const int64_t pairs = tokens * top_k;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    RowLists l = {};
    int64_t items = pairs;
    if (d_rows != nullptr) {
        if (!aligned_to(4, workspace)) return route_fail(TGO_E_ARG, "the workspace must be 4-byte aligned");
        if (workspace == nullptr || workspace_bytes < tgo_moe_combine_grad_workspace_bytes(pairs, n_rows))
            return route_fail(TGO_E_WORKSPACE, "combine workspace too small");
        l.count = static_cast<int32_t*>(workspace);
        l.state = l.count + n_rows;
        l.even = l.state + 3;
        l.odd = l.even + pairs;
        for (l.passes = 1; l.passes < 4 && (n_rows - 1) >> (8 * l.passes) > 0;) ++l.passes;
        if (cudaMemsetAsync(l.count, 0, static_cast<size_t>(n_rows + 3) * 4, st) != cudaSuccess) return route_fail(TGO_E_CUDA, "cudaMemsetAsync failed");
        count_rows_kernel<<<static_cast<unsigned>((pairs + kListThreads - 1) / kListThreads), kListThreads, 0, st>>>(row_of_pair, pairs, n_rows, l);
        if (n_rows > items) items = n_rows;
    }
    combine_grad_kernel<<<static_cast<unsigned>((items + kMoveThreads / 32 - 1) / (kMoveThreads / 32)), kMoveThreads, 0, st>>>(
        static_cast<const uint4*>(dy), static_cast<const uint4*>(rows), n_rows, row_of_pair, weights, l, static_cast<uint4*>(d_rows), d_weights,
        pairs, static_cast<int>(top_k), static_cast<int>(width / 8));
    return launched("combine gradient kernel launch failed");
}

}  // extern "C"
