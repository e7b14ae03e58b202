// Tokens to rows sorted by expert and back, with their gradients, for one GPU's mixture-of-experts layer:
//   dispatch   rows[row_of_pair[t, s]] = x[t]
//   combine    y[t] = sum_s w[t, s] rows[row_of_pair[t, s]]
//              drows[row_of_pair[t, s]] = w[t, s] dy[t],  dw[t, s] = <dy[t], rows[row_of_pair[t, s]]>
// The gradient of dispatch is combine without weights.  bf16 rows, sums in fp32, one rounding.
//
// All of it is bound by memory: a token's row is read once and its top_k rows are written (or read) once.
#include "../../include/tgo_mmq.h"

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

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
    const long long step = static_cast<long long>(kMoveThreads) * gridDim.x;
    for (long long v = blockIdx.x * static_cast<long long>(kMoveThreads) + threadIdx.x; v < tokens * vec_per_row; v += step) {
        const long long t = v / vec_per_row;
        const int c = static_cast<int>(v - t * vec_per_row);
        float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < top_k; ++s) {
            const int row = row_of_pair[t * top_k + s];
            if (row < 0 || row >= n_rows) continue;
            const float w = weights != nullptr ? weights[t * top_k + s] : 1.0f;
            float f[8];
            widen(rows[static_cast<long long>(row) * vec_per_row + c], f);
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] = fmaf(w, f[j], acc[j]);
        }
        out[v] = narrow(acc);
    }
}

// how many pairs name each row
__global__ void __launch_bounds__(kMoveThreads) count_rows_kernel(const int32_t* __restrict__ row_of_pair, long long pairs, long long n_rows,
                                                                  int32_t* __restrict__ count) {
    const long long i = blockIdx.x * static_cast<long long>(kMoveThreads) + threadIdx.x;
    if (i >= pairs) return;
    const int row = row_of_pair[i];
    if (row >= 0 && row < n_rows) atomicAdd(&count[row], 1);
}

// One warp per pair.  A row that several pairs name (dispatch gives none such) gets the sum over them from
// the first of them, a row that none names zeros from the warp of that number.
__global__ void __launch_bounds__(kMoveThreads) combine_grad_kernel(const uint4* __restrict__ dy, const uint4* __restrict__ rows, long long n_rows,
                                                                    const int32_t* __restrict__ row_of_pair, const float* __restrict__ weights,
                                                                    const int32_t* __restrict__ count, uint4* __restrict__ d_rows,
                                                                    float* __restrict__ d_weights, long long pairs, int top_k, int vec_per_row) {
    const int lane = threadIdx.x & 31;
    const long long pair = blockIdx.x * static_cast<long long>(kMoveThreads / 32) + (threadIdx.x >> 5);
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
        for (int c = lane; c < vec_per_row; c += 32) {
            float f[8];
            widen(g[c], f);
            if (d_weights != nullptr) {
                float h[8];
                widen(r[c], h);
#pragma unroll
                for (int j = 0; j < 8; ++j) dot = fmaf(f[j], h[j], dot);
            }
            if (d_rows != nullptr && alone) {
#pragma unroll
                for (int j = 0; j < 8; ++j) f[j] *= w;
                d_rows[static_cast<long long>(row) * vec_per_row + c] = narrow(f);
            }
        }
        if (!alone) {
            long long before = 0;
            while (before < pair && row_of_pair[before] != row) ++before;
            for (int c = lane; before == pair && c < vec_per_row; c += 32) {
                float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                for (long long p = pair; p < pairs; ++p) {
                    if (row_of_pair[p] != row) continue;
                    const float wp = weights != nullptr ? weights[p] : 1.0f;
                    float f[8];
                    widen(dy[p / top_k * vec_per_row + c], f);
#pragma unroll
                    for (int j = 0; j < 8; ++j) acc[j] = fmaf(wp, f[j], acc[j]);
                }
                d_rows[static_cast<long long>(row) * vec_per_row + c] = narrow(acc);
            }
        }
    }
    if (d_weights != nullptr) {
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) dot += __shfl_xor_sync(0xFFFFFFFFu, dot, d);
        if (lane == 0) d_weights[pair] = dot;
    }
}

static bool a16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
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
    const int64_t sort = tgo_route_workspace_bytes(n_pairs, num_experts);
    return sort < 0 ? -1 : up16(n_pairs * 4) + sort;
}

int tgo_moe_dispatch(const void* x, const int32_t* expert_ids, int64_t tokens, int64_t top_k, int64_t num_experts, int64_t width, void* rows,
                     int32_t* row_of_pair, int64_t* expert_indices, int32_t* expert_offsets, void* workspace, int64_t workspace_bytes,
                     void* stream) {
    if (x == nullptr || expert_ids == nullptr || rows == nullptr || row_of_pair == nullptr || expert_indices == nullptr ||
        expert_offsets == nullptr || workspace == nullptr)
        return route_fail(TGO_E_ARG, "null pointer");
    int rc = check_rows(tokens, top_k, width);
    if (rc != TGO_OK) return rc;
    if (!a16(x) || !a16(rows)) return route_fail(TGO_E_ARG, "data pointers must be 16-byte aligned");
    const int64_t pairs = tokens * top_k;
    if (num_experts <= 0 || num_experts > 4096) return route_fail(TGO_E_ARG, "num_experts must be in 1..4096");
    if (workspace_bytes < tgo_moe_dispatch_workspace_bytes(pairs, num_experts)) return route_fail(TGO_E_WORKSPACE, "dispatch workspace too small");
    int32_t* sorted = static_cast<int32_t*>(workspace);
    const int64_t used = up16(pairs * 4);
    rc = tgo_route_sort(expert_ids, pairs, num_experts, sorted, row_of_pair, expert_indices, expert_offsets, nullptr,
                        static_cast<uint8_t*>(workspace) + used, workspace_bytes - used, stream);
    if (rc != TGO_OK) return rc;
    const int vec = static_cast<int>(width / 8);
    dispatch_rows_kernel<<<move_grid(tokens * vec), kMoveThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const uint4*>(x), row_of_pair, expert_offsets, static_cast<int>(num_experts), tokens, static_cast<int>(top_k),
        static_cast<uint4*>(rows), vec);
    return launched("dispatch_rows_kernel launch failed");
}

int tgo_moe_combine(const void* rows, int64_t n_rows, const int32_t* row_of_pair, const float* weights, void* out, int64_t tokens, int64_t top_k,
                    int64_t width, void* stream) {
    if (rows == nullptr || row_of_pair == nullptr || out == nullptr) return route_fail(TGO_E_ARG, "null pointer");
    const int rc = check_rows(tokens, top_k, width);
    if (rc != TGO_OK) return rc;
    if (n_rows < 0) return route_fail(TGO_E_ARG, "a negative number of rows");
    if (!a16(rows) || !a16(out)) return route_fail(TGO_E_ARG, "data pointers must be 16-byte aligned");
    const int vec = static_cast<int>(width / 8);
    moe_combine_kernel<<<move_grid(tokens * vec), kMoveThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const uint4*>(rows), n_rows, row_of_pair, weights, static_cast<uint4*>(out), tokens, static_cast<int>(top_k), vec);
    return launched("moe_combine_kernel launch failed");
}

int tgo_moe_combine_grad(const void* dy, const void* rows, int64_t n_rows, const int32_t* row_of_pair, const float* weights, void* d_rows,
                         float* d_weights, int64_t tokens, int64_t top_k, int64_t width, void* workspace, int64_t workspace_bytes, void* stream) {
    if (dy == nullptr || row_of_pair == nullptr || (d_weights != nullptr && rows == nullptr)) return route_fail(TGO_E_ARG, "null pointer");
    if (d_rows == nullptr && d_weights == nullptr) return route_fail(TGO_E_ARG, "no gradient is asked for");
    const int rc = check_rows(tokens, top_k, width);
    if (rc != TGO_OK) return rc;
    if (n_rows < 0 || n_rows > INT32_MAX) return route_fail(TGO_E_ARG, "the number of rows must be in 0..2^31-1");
    if (!a16(dy) || !a16(rows) || !a16(d_rows)) return route_fail(TGO_E_ARG, "data pointers must be 16-byte aligned");
    const int64_t pairs = tokens * top_k;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    int32_t* count = static_cast<int32_t*>(workspace);
    int64_t items = pairs;
    if (d_rows != nullptr) {
        if (workspace == nullptr || workspace_bytes < n_rows * 4) return route_fail(TGO_E_WORKSPACE, "combine workspace is smaller than n_rows * 4 bytes");
        if (cudaMemsetAsync(count, 0, static_cast<size_t>(n_rows) * 4, st) != cudaSuccess) return route_fail(TGO_E_CUDA, "cudaMemsetAsync failed");
        count_rows_kernel<<<static_cast<unsigned>((pairs + kMoveThreads - 1) / kMoveThreads), kMoveThreads, 0, st>>>(row_of_pair, pairs, n_rows, count);
        if (n_rows > items) items = n_rows;
    }
    combine_grad_kernel<<<static_cast<unsigned>((items + kMoveThreads / 32 - 1) / (kMoveThreads / 32)), kMoveThreads, 0, st>>>(
        static_cast<const uint4*>(dy), static_cast<const uint4*>(rows), n_rows, row_of_pair, weights, count, static_cast<uint4*>(d_rows), d_weights,
        pairs, static_cast<int>(top_k), static_cast<int>(width / 8));
    return launched("combine gradient kernel launch failed");
}

}  // extern "C"
