// token_kernels.hip -- tokens sorted by expert and back: the lists of a routing
// (stable by assignment), the rows copied in their order, the weighted sum of the
// experts' rows per token, and its gradients.
#include "qmoe_device.h"
#include "qmoe_internal.h"

namespace qmoe {

// ---------------------------------------------------------------------------
// Lists.  Workgroup e reads every id once for two counts -- the ids below e (its
// offset) and its own -- and once more to write its own assignments in ascending
// order, so no workgroup waits for another and the result does not depend on
// their order.  Workgroup E takes the ids outside [0, E): place -1, and the list's
// tail behind offsets[E] filled with -1.  The waves take contiguous quarters.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(256) void k_sort_tokens(const int32_t* ids, int A, int top_k, int E, int32_t* offsets,
                                                     int32_t* rows, int32_t* tokens, int32_t* place) {
    __shared__ int s_below[4], s_own[4];
    const int e = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int quarter = ((A + 3) / 4 + 255) / 256 * 256;
    const int64_t from = (int64_t)wave * quarter;
    const int begin = from < A ? (int)from : A, end = A - begin < quarter ? A : begin + quarter;
    int below = 0, own = 0;
    for (int a = begin + lane; a < end; a += 64) {
        const int id = ids[a];
        const bool valid = id >= 0 && id < E;
        below += valid && id < e;
        own += e < E ? id == e : !valid;
    }
    below = group_sum_i32<64>(below);
    own = group_sum_i32<64>(own);
    if (lane == 0) s_below[wave] = below, s_own[wave] = own;
    __syncthreads();
    int at = s_below[0] + s_below[1] + s_below[2] + s_below[3];
    if (threadIdx.x == 0) offsets[e] = at;
    for (int w = 0; w < wave; ++w) at += s_own[w];
    for (int a0 = begin; a0 < end; a0 += 64) {
        const int a = a0 + lane;
        const int id = a < end ? ids[a] : 0;
        const bool mine = a < end && (e < E ? id == e : id < 0 || id >= E);
        const uint64_t mask = __ballot(mine);
        if (mine) {
            const int pos = at + __builtin_popcountll(mask & ((1ull << lane) - 1));
            rows[pos] = e < E ? a : -1;
            tokens[pos] = e < E ? a / top_k : -1;
            place[a] = e < E ? pos : -1;
        }
        at += __builtin_popcountll(mask);
    }
}

hipError_t launch_sort_tokens(const int32_t* ids, int n_tokens, int top_k, int E, int32_t* offsets, int32_t* rows,
                              int32_t* tokens, int32_t* place, hipStream_t stream) {
    hipLaunchKernelGGL(k_sort_tokens, dim3(E + 1), dim3(256), 0, stream, ids, n_tokens * top_k, top_k, E, offsets, rows,
                       tokens, place);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Rows to the experts' order: one workgroup per token reads its row once and
// writes it top_k times (reading by sorted row would read it top_k times).  Rows
// behind the last expert's belong to no token: zeros, by the workgroup that owns
// those list indices.  Pieces of 16 bytes (V = u32x4) or single elements.
// ---------------------------------------------------------------------------
template <typename V>
__global__ __launch_bounds__(256) void k_gather_tokens(const V* x, int n, int top_k, int R, const int32_t* total,
                                                       const int32_t* place, V* y) {
    const int t = blockIdx.x;
    const V* xr = x + (uint64_t)t * n;
    const int32_t* pl = place + (int64_t)t * top_k;
    const int last = *total;
    for (int i = threadIdx.x; i < n; i += 256) {
        const V v = xr[i];
        for (int j = 0; j < top_k; ++j) {
            const int p = pl[j];
            if (p >= 0 && p < R) y[(uint64_t)p * n + i] = v;
            const int r = t * top_k + j;
            if (r >= last) y[(uint64_t)r * n + i] = V{};
        }
    }
}

hipError_t launch_gather_tokens(const void* x, int elem, int n_tokens, int n_cols, int top_k, const int32_t* total,
                                const int32_t* place, void* y, hipStream_t stream) {
    if (n_tokens <= 0) return hipSuccess;
    const int R = n_tokens * top_k;
    const int64_t bytes = (int64_t)n_cols * elem;
    const dim3 grid(n_tokens), block(256);
    if (bytes % 16 == 0 && (((uintptr_t)x | (uintptr_t)y) & 15u) == 0)
        hipLaunchKernelGGL(k_gather_tokens<u32x4>, grid, block, 0, stream, (const u32x4*)x, (int)(bytes / 16), top_k, R, total,
                           place, (u32x4*)y);
    else if (elem == 4)
        hipLaunchKernelGGL(k_gather_tokens<uint32_t>, grid, block, 0, stream, (const uint32_t*)x, n_cols, top_k, R, total,
                           place, (uint32_t*)y);
    else if (elem == 2)
        hipLaunchKernelGGL(k_gather_tokens<uint16_t>, grid, block, 0, stream, (const uint16_t*)x, n_cols, top_k, R, total,
                           place, (uint16_t*)y);
    else
        hipLaunchKernelGGL(k_gather_tokens<uint8_t>, grid, block, 0, stream, (const uint8_t*)x, n_cols, top_k, R, total,
                           place, (uint8_t*)y);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// y[t] = residual[t] + sum_j w[t][j] ys[place[t][j]], j in order in f32, rounded
// once (w null: ones, the gather's gradient).  Assignments without a place add nothing.
// ---------------------------------------------------------------------------
template <bool BF16>
__device__ __forceinline__ float load1(const void* x, uint64_t at) {
    return BF16 ? bf16_to_f32(((const uint16_t*)x)[at]) : ((const float*)x)[at];
}
template <bool BF16>
__device__ __forceinline__ void store1(void* y, uint64_t at, float v) {
    if (BF16) ((uint16_t*)y)[at] = (uint16_t)f32_pack_bf16(v, 0.0f);
    else ((float*)y)[at] = v;
}

template <bool BF16>
__global__ __launch_bounds__(256) void k_combine_tokens(const void* ys, int H, int top_k, int R, const int32_t* place,
                                                        const float* w, const void* residual, void* y) {
    const int t = blockIdx.x;
    for (int i = threadIdx.x; i < H; i += 256) {
        float s = 0.0f;
        for (int j = 0; j < top_k; ++j) {
            const int p = place[(int64_t)t * top_k + j];
            if (p < 0 || p >= R) continue;
            const float v = load1<BF16>(ys, (uint64_t)p * H + i);
            s = w ? fmaf(w[(int64_t)t * top_k + j], v, s) : s + v;
        }
        if (residual) s += load1<BF16>(residual, (uint64_t)t * H + i);
        store1<BF16>(y, (uint64_t)t * H + i, s);
    }
}

hipError_t launch_combine_tokens(const void* ys, bool bf16, int n_tokens, int H, int top_k, const int32_t* place,
                                 const float* w, const void* residual, void* y, hipStream_t stream) {
    if (n_tokens <= 0) return hipSuccess;
    if (bf16)
        hipLaunchKernelGGL(k_combine_tokens<true>, dim3(n_tokens), dim3(256), 0, stream, ys, H, top_k, n_tokens * top_k, place,
                           w, residual, y);
    else
        hipLaunchKernelGGL(k_combine_tokens<false>, dim3(n_tokens), dim3(256), 0, stream, ys, H, top_k, n_tokens * top_k, place,
                           w, residual, y);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// The weighted sum's gradients: dys[place[t][j]] = w[t][j] dy[t] and
// dw[t][j] = <dy[t], ys[place[t][j]]>.  One workgroup per token, so no sum is
// shared between workgroups.  Rows behind the last expert's get zeros.
// ---------------------------------------------------------------------------
template <bool BF16>
__global__ __launch_bounds__(256) void k_combine_tokens_bwd(const void* dy, const void* ys, int H, int top_k, int R,
                                                            const int32_t* total, const int32_t* place, const float* w,
                                                            void* dys, float* dw) {
    __shared__ float s_sum[4];
    const int t = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int last = *total;
    for (int j = 0; j < top_k; ++j) {
        const int a = t * top_k + j, p = place[a];
        float dot = 0.0f;
        if (p >= 0 && p < R) {
            const float wj = w[a];
            for (int i = threadIdx.x; i < H; i += 256) {
                const float g = load1<BF16>(dy, (uint64_t)t * H + i);
                dot = fmaf(g, load1<BF16>(ys, (uint64_t)p * H + i), dot);
                store1<BF16>(dys, (uint64_t)p * H + i, wj * g);
            }
        }
        if (a >= last)
            for (int i = threadIdx.x; i < H; i += 256) store1<BF16>(dys, (uint64_t)a * H + i, 0.0f);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) dot += __shfl_xor(dot, o, 64);
        if (lane == 0) s_sum[wave] = dot;
        __syncthreads();
        if (threadIdx.x == 0) dw[a] = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
        __syncthreads();
    }
}

hipError_t launch_combine_tokens_bwd(const void* dy, const void* ys, bool bf16, int n_tokens, int H, int top_k,
                                     const int32_t* total, const int32_t* place, const float* w, void* dys, float* dw,
                                     hipStream_t stream) {
    if (n_tokens <= 0) return hipSuccess;
    if (bf16)
        hipLaunchKernelGGL(k_combine_tokens_bwd<true>, dim3(n_tokens), dim3(256), 0, stream, dy, ys, H, top_k,
                           n_tokens * top_k, total, place, w, dys, dw);
    else
        hipLaunchKernelGGL(k_combine_tokens_bwd<false>, dim3(n_tokens), dim3(256), 0, stream, dy, ys, H, top_k,
                           n_tokens * top_k, total, place, w, dys, dw);
    return hipGetLastError();
}

}  // namespace qmoe
