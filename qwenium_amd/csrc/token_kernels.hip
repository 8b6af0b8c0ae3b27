// token_kernels.hip -- tokens sorted by expert and back: the lists of a routing
// (stable by assignment), the rows copied in their order, the weighted sum of the
// experts' rows per token, and its gradients.
#include "qmoe_device.h"
#include "qmoe_internal.h"

#include <type_traits>

namespace qmoe {

// ---------------------------------------------------------------------------
// Lists of few assignments.  Workgroup e reads every id once for two counts -- the
// ids below e (its offset) and its own -- and once more to write its own assignments
// in ascending order, so no workgroup waits for another and the result does not
// depend on their order.  Workgroup E takes the ids outside [0, E): place -1, and the
// list's tail behind offsets[E] filled with -1.  The waves take contiguous shares, 4
// ids a lane and step, the next step's in flight.  The loops stay small: the
// instruction fetch of unrolled ones, run once, costs more than it saves (80 ids
// 3.8 -> 5.5 us).
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(256) void k_sort_tokens_few(const int32_t* ids, int A, int top_k, int E, bool vec,
                                                         int32_t* offsets, int32_t* rows, int32_t* tokens, int32_t* place) {
    __shared__ int s_below[4], s_own[4];
    const int e = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int share = (A + 256 * 4 - 1) / (256 * 4) * 256;
    const int begin = wave * share < A ? wave * share : A, end = A - begin < share ? A : begin + share;
    auto load4 = [&](int a) {  // this lane's 4 ids from a on; past the end -1
        u32x4 r = {~0u, ~0u, ~0u, ~0u};
        if (vec && a + 4 <= end) {
            r = *(const u32x4*)(ids + a);
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (a + c < end) r[c] = (uint32_t)ids[a + c];
        }
        return r;
    };
    auto own = [&](uint32_t id, int a) { return e < E ? id == (uint32_t)e : id >= (uint32_t)E && a < end; };
    int below = 0, count = 0;
    u32x4 next = load4(begin + 4 * lane);
#pragma unroll 1
    for (int a = begin + 4 * lane; a - 4 * lane < end; a += 256) {
        const u32x4 id = next;
        next = load4(a + 256);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            below += id[c] < (uint32_t)e && id[c] < (uint32_t)E;
            count += own(id[c], a + c);
        }
    }
    below = group_sum_i32<64>(below);
    count = group_sum_i32<64>(count);
    if (lane == 0) s_below[wave] = below, s_own[wave] = count;
    __syncthreads();
    int at = 0;
    for (int w = 0; w < 4; ++w) {
        at += s_below[w];
        if (w < wave) at += s_own[w];
    }
    if (threadIdx.x == 0) offsets[e] = at;  // (wave 0: no own counts in it)
    if (count == 0) return;
    const uint64_t lower = (1ull << lane) - 1;
    next = load4(begin + 4 * lane);
#pragma unroll 1
    for (int a = begin + 4 * lane; a - 4 * lane < end; a += 256) {
        const u32x4 id = next;
        next = load4(a + 256);
        uint32_t mine = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) mine |= (uint32_t)own(id[c], a + c) << c;
        if (__ballot(mine != 0) == 0) continue;
        const uint32_t n = __builtin_popcount(mine);
        const uint64_t n0 = __ballot(n & 1), n1 = __ballot(n & 2), n2 = __ballot(n & 4);
        int pos = at + __builtin_popcountll(n0 & lower) + 2 * __builtin_popcountll(n1 & lower) +
                  4 * __builtin_popcountll(n2 & lower);
        at += __builtin_popcountll(n0) + 2 * __builtin_popcountll(n1) + 4 * __builtin_popcountll(n2);
        while (mine) {
            const int i = a + __builtin_ctz(mine);
            mine &= mine - 1;
            rows[pos] = e < E ? i : -1;
            tokens[pos] = e < E ? i / top_k : -1;
            place[i] = e < E ? pos : -1;
            ++pos;
        }
    }
}

// ---------------------------------------------------------------------------
// Lists of many.  A workgroup places a contiguous chunk of the ids, 1024 a round.
// It counts every expert's ids before its chunk and from it on by itself, in LDS
// (integer sums: any order), so again no workgroup waits for another: the sums'
// prefix over the experts and the counts before the chunk give each expert's next
// row; a thread's place is that, the earlier waves' counts of its expert, and its
// rank among its wave's lanes with the same expert.  Dropped ids are expert E.
// 32768 ids of 256 experts: 7.4 us (14.5 by k_sort_tokens_few), 1024: 4.4 (3.4).
// ---------------------------------------------------------------------------
constexpr int kSortMaxExperts = 1024;
constexpr int kSortFew = 1024;  // ids that k_sort_tokens_few takes
__global__ __launch_bounds__(1024) void k_sort_tokens(const int32_t* ids, int A, int chunk, int top_k, int E, bool vec,
                                                      int32_t* offsets, int32_t* rows, int32_t* tokens, int32_t* place) {
    __shared__ int s_next[kSortMaxExperts + 1], s_rest[kSortMaxExperts + 1];
    __shared__ __attribute__((aligned(16))) uint16_t s_wave[16][kSortMaxExperts + 2];
    __shared__ int s_scan[16];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int start = blockIdx.x * chunk, stop = A - start < chunk ? A : start + chunk;
    for (int i = tid; i <= E; i += 1024) s_next[i] = s_rest[i] = 0;
    __syncthreads();
    auto bucket = [&](int id) { return (uint32_t)id < (uint32_t)E ? id : E; };
    const int whole = vec ? A & ~3 : 0;  // (chunks start at multiples of 1024)
#pragma unroll 2
    for (int a = 4 * tid; a < whole; a += 4096) {
        const u32x4 id = *(const u32x4*)(ids + a);
        int* count = a < start ? s_next : s_rest;
#pragma unroll
        for (int c = 0; c < 4; ++c) atomicAdd(count + bucket((int)id[c]), 1);
    }
    for (int a = whole + tid; a < A; a += 1024) atomicAdd((a < start ? s_next : s_rest) + bucket(ids[a]), 1);
    __syncthreads();
    // the experts' offsets: the prefix of all counts (bucket E is thread 1023's second at most)
    const int before = tid <= E ? s_next[tid] : 0, all = tid <= E ? before + s_rest[tid] : 0;
    const int incl = wave_incl_scan_i32(all);
    if (lane == 63) s_scan[wave] = incl;
    __syncthreads();
    int first = incl - all;
    for (int w = 0; w < wave; ++w) first += s_scan[w];
    if (tid <= E) {
        s_next[tid] = first + before;
        if (blockIdx.x == 0) offsets[tid] = first;
    }
    if (E == 1024 && tid == 1023) {
        s_next[1024] += first + all;
        if (blockIdx.x == 0) offsets[1024] = first + all;
    }
    for (int a0 = start; a0 < stop; a0 += 1024) {
        for (int i = tid; i < 16 * (kSortMaxExperts + 2) / 2; i += 1024) ((uint32_t*)s_wave)[i] = 0;
        __syncthreads();
        const int a = a0 + tid;
        const bool here = a < stop;
        const int b = here ? bucket(ids[a]) : 0;
        uint64_t same = __ballot(here);
#pragma unroll
        for (int bit = 0; bit < 11; ++bit) {
            const uint64_t m = __ballot(b >> bit & 1);
            same &= b >> bit & 1 ? m : ~m;
        }
        const int rank = __builtin_popcountll(same & ((1ull << lane) - 1));
        if (here && rank == 0) s_wave[wave][b] = (uint16_t)__builtin_popcountll(same);
        __syncthreads();
        if (here) {
            int pos = s_next[b] + rank;
            for (int w = 0; w < wave; ++w) pos += s_wave[w][b];
            rows[pos] = b < E ? a : -1;
            tokens[pos] = b < E ? a / top_k : -1;
            place[a] = b < E ? pos : -1;
        }
        __syncthreads();
        if (a0 + 1024 < stop) {
            for (int i = tid; i <= E; i += 1024) {
                int n = 0;
                for (int w = 0; w < 16; ++w) n += s_wave[w][i];
                s_next[i] += n;
            }
            __syncthreads();
        }
    }
}

hipError_t launch_sort_tokens(const int32_t* ids, int n_tokens, int top_k, int E, int32_t* offsets, int32_t* rows,
                              int32_t* tokens, int32_t* place, hipStream_t stream) {
    const int A = n_tokens * top_k;
    const bool vec = ((uintptr_t)ids & 15u) == 0;
    if (E > kSortMaxExperts) return hipErrorInvalidValue;
    if (A <= kSortFew) {
        hipLaunchKernelGGL(k_sort_tokens_few, dim3(E + 1), dim3(256), 0, stream, ids, A, top_k, E, vec, offsets, rows, tokens,
                           place);
        return hipGetLastError();
    }
    // a round of 1024 a workgroup, more where that were over two workgroups per CU
    const int chunk = (A + 512 * 1024 - 1) / (512 * 1024) * 1024;
    hipLaunchKernelGGL(k_sort_tokens, dim3((A + chunk - 1) / chunk), dim3(1024), 0, stream, ids, A, chunk, top_k, E, vec, offsets,
                       rows, tokens, place);
    return hipGetLastError();
}

// A token's row in pieces of 8 elements over threads x workgroups: workgroups of one
// wave where wider ones would leave CUs without any.
static void row_grid(int n_tokens, int64_t pieces, dim3& grid, dim3& block) {
    const int64_t threads = n_tokens * ((pieces + 255) / 256) >= 512 ? 256 : 64;
    grid = dim3((unsigned)n_tokens, (unsigned)((pieces + threads - 1) / threads));
    block = dim3((unsigned)threads);
}

// ---------------------------------------------------------------------------
// Rows to the experts' order: a token's workgroups read its row once and write it
// top_k times (reading by sorted row would read it top_k times).  Rows behind the
// last expert's belong to no token: zeros, by the token with those list indices.
// 4096 rows of 4 KB, 8 times (151 MB): 24 us, 6.3 TB/s.  A thread takes 16 bytes; a
// row's last 16 may overlap the ones before (the same bytes written twice).  V: 16 bytes, or
// single bytes for rows shorter than that.  Written through the caches: past them
// what reads the rows next pays (with a quantization of them, us through / past: 67 MB
// 39 / 42, 134 MB 71 / 78, 268 MB 145 / 155, f32 185 MB 65 / 76).
// ---------------------------------------------------------------------------
typedef uint32_t u32x4a1 __attribute__((ext_vector_type(4), aligned(1)));
template <typename V>
__global__ __launch_bounds__(256) void k_gather_tokens(const uint8_t* x, int bytes, int top_k, int R, const int32_t* total,
                                                       const int32_t* place, uint8_t* y) {
    constexpr int kSize = sizeof(V);
    const int t = blockIdx.x;
    int i = kSize * (int)(blockIdx.y * blockDim.x + threadIdx.x);
    if (i >= bytes) return;
    if (i + kSize > bytes) i = bytes - kSize;
    const V v = *(const V*)(x + (uint64_t)t * bytes + i);
    const int32_t* pl = place + (int64_t)t * top_k;
    const int last = *total;
#pragma unroll 4
    for (int j = 0; j < top_k; ++j) {
        const int p = pl[j];
        if (p >= 0 && p < R) *(V*)(y + (uint64_t)p * bytes + i) = v;
        const int r = t * top_k + j;
        if (r >= last) *(V*)(y + (uint64_t)r * bytes + i) = V{};
    }
}

hipError_t launch_gather_tokens(const void* x, int elem, int n_tokens, int n_cols, int top_k, const int32_t* total,
                                const int32_t* place, void* y, hipStream_t stream) {
    if (n_tokens <= 0) return hipSuccess;
    const int bytes = n_cols * elem;
    dim3 grid, block;
    row_grid(n_tokens, bytes >= 16 ? (bytes + 15) / 16 : bytes, grid, block);
    if (grid.y > 65535) return hipErrorInvalidValue;
#define QMOE_GATHER(V)                                                                                                 \
    hipLaunchKernelGGL((k_gather_tokens<V>), grid, block, 0, stream, (const uint8_t*)x, bytes, top_k,        \
                       n_tokens * top_k, total, place, (uint8_t*)y)
    if (bytes < 16) QMOE_GATHER(uint8_t);
    else QMOE_GATHER(u32x4a1);
#undef QMOE_GATHER
    return hipGetLastError();
}

// 16 bytes of a row, C elements, at the elements' alignment.  A row's last piece starts at
// H - C: the first of its columns are its neighbour's, which alone stores them.
template <bool BF16>
struct Piece {
    static constexpr int C = BF16 ? 8 : 4;
    u32x4a2 r;
    // of H columns from c on; NT: read once (unaligned pieces share lines)
    template <bool WHOLE, bool NT = false>
    __device__ __forceinline__ void load(const void* row, int c, int H) {
        if (WHOLE || H >= C) {
            const u32x4a2* p = (const u32x4a2*)((const uint8_t*)row + (int64_t)c * (16 / C));
            if constexpr (WHOLE && NT) r = __builtin_nontemporal_load(p);
            else r = *p;
        } else {
            float v[C];
#pragma unroll
            for (int i = 0; i < C; ++i) v[i] = i < H ? load1<BF16>(row, i) : 0.0f;
            set(v);
        }
    }
    __device__ __forceinline__ void set(const float (&v)[C]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (BF16) r[i] = f32_pack_bf16(v[2 * i], v[2 * i + 1]);
            else r[i] = __builtin_bit_cast(uint32_t, v[i]);
        }
    }
    // the columns from c + skip on
    template <bool WHOLE>
    __device__ __forceinline__ void store(void* row, int c, int H, int skip) const {
        if (WHOLE || (H >= C && skip == 0)) {
            *(u32x4a2*)((uint8_t*)row + (int64_t)c * (16 / C)) = r;
        } else {
#pragma unroll
            for (int i = 0; i < C; ++i)
                if (i >= skip && c + i < H) store1<BF16>(row, c + i, (*this)[i]);
        }
    }
    __device__ __forceinline__ float operator[](int i) const {
        const uint32_t v = r[BF16 ? i >> 1 : i];
        if constexpr (BF16) return __builtin_bit_cast(float, i & 1 ? v & 0xffff0000u : v << 16);
        else return __builtin_bit_cast(float, v);
    }
};
template <bool BF16>
__device__ __forceinline__ const void* row_at(const void* x, int64_t row, int H) {
    return (const uint8_t*)x + row * H * (BF16 ? 2 : 4);
}
template <bool BF16>
__device__ __forceinline__ void* row_at(void* x, int64_t row, int H) {
    return (uint8_t*)x + row * H * (BF16 ? 2 : 4);
}

// ---------------------------------------------------------------------------
// y[t] = residual[t] + sum_j w[t][j] ys[place[t][j]], j in order in f32, rounded
// once (w null: ones, the gather's gradient).  Assignments without a place add
// nothing.  16 bytes a thread, the rows of 8 assignments in flight, past the caches (a row
// is read once): 4096 x 8 rows of 4 KB and a residual (168 MB), several in turn, 28.5 us,
// 5.9 TB/s (through the caches 33.6; with a branch around each load 38).
// ---------------------------------------------------------------------------
template <bool BF16, bool WHOLE>
__global__ __launch_bounds__(256) void k_combine_tokens(const void* ys, int H, int top_k, int R, const int32_t* place,
                                                        const float* w, const void* residual, void* y) {
    constexpr int C = Piece<BF16>::C;
    const int t = blockIdx.x, c0 = C * (blockIdx.y * blockDim.x + threadIdx.x);
    if (c0 >= H) return;
    const int c = WHOLE || c0 + C <= H || H < C ? c0 : H - C;
    float s[C] = {};
    Piece<BF16> res;
    if (residual) res.template load<WHOLE>(row_at<BF16>(residual, t, H), c, H);
    // 8 assignments' rows at once (FULL: a branch around a load would hold the next one up)
    auto add8 = [&](int j0, auto full_c) {
        constexpr bool FULL = decltype(full_c)::value;
        Piece<BF16> v[8];
        float wj[8];
        int p[8];
        bool has[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int a = t * top_k + (FULL || j0 + j < top_k ? j0 + j : 0);
            p[j] = place[a];
            wj[j] = w ? w[a] : 1.0f;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            has[j] = (FULL || j0 + j < top_k) && p[j] >= 0 && p[j] < R;
            if (FULL || j0 + j < top_k) v[j].template load<WHOLE, true>(row_at<BF16>(ys, has[j] ? p[j] : 0, H), c, H);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (has[j])
#pragma unroll
                for (int i = 0; i < C; ++i) s[i] = fmaf(wj[j], v[j][i], s[i]);
    };
    int j0 = 0;
    for (; j0 + 8 <= top_k; j0 += 8) add8(j0, std::true_type{});
    if (j0 < top_k) add8(j0, std::false_type{});
    if (residual)
#pragma unroll
        for (int i = 0; i < C; ++i) s[i] += res[i];
    Piece<BF16> out;
    out.set(s);
    out.template store<WHOLE>(row_at<BF16>(y, t, H), c, H, c0 - c);
}

hipError_t launch_combine_tokens(const void* ys, bool bf16, int n_tokens, int H, int top_k, const int32_t* place,
                                 const float* w, const void* residual, void* y, hipStream_t stream) {
    if (n_tokens <= 0) return hipSuccess;
    const int C = bf16 ? 8 : 4;
    const bool whole = H % C == 0;
    dim3 grid, block;
    row_grid(n_tokens, ((int64_t)H + C - 1) / C, grid, block);
    if (grid.y > 65535) return hipErrorInvalidValue;
#define QMOE_COMBINE(B, V) \
    hipLaunchKernelGGL((k_combine_tokens<B, V>), grid, block, 0, stream, ys, H, top_k, n_tokens * top_k, place, w, residual, y)
    if (bf16) { if (whole) QMOE_COMBINE(true, true); else QMOE_COMBINE(true, false); }
    else { if (whole) QMOE_COMBINE(false, true); else QMOE_COMBINE(false, false); }
#undef QMOE_COMBINE
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// The weighted sum's gradients: dys[place[t][j]] = w[t][j] dy[t] and
// dw[t][j] = <dy[t], ys[place[t][j]]>.  One workgroup per token, so no sum is
// shared between workgroups: a thread adds its columns' products in turn (16 bytes of 8
// assignments in flight), then the tree over its wave's lanes and the waves in turn.
// Rows behind the last expert's get zeros.  Written through the caches, as the gather's
// (with a quantization of dys, us through / past: 67 MB 56 / 60, 134 MB 98 / 112, f32 185
// MB 105 / 121).  4096 x 8 rows of 4 KB (285 MB) 52 us, 5.5 TB/s; 8192 x 2 of 8 KB 85.
// ---------------------------------------------------------------------------
template <bool BF16, bool WHOLE>
__global__ __launch_bounds__(1024) void k_combine_tokens_bwd(const void* dy, const void* ys, int H, int top_k, int R,
                                                             const int32_t* total, const int32_t* place, const float* w,
                                                             void* dys, float* dw) {
    constexpr int C = Piece<BF16>::C;
    __shared__ float s_sum[8][16];
    const int t = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, nw = blockDim.x >> 6;
    const int last = *total;
    for (int j0 = 0; j0 < top_k; j0 += 8) {
        float dot[8] = {}, wj[8];
        int p[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int a = t * top_k + (j0 + j < top_k ? j0 + j : 0);
            const int at = place[a];
            p[j] = j0 + j < top_k && at >= 0 && at < R ? at : -1;
            wj[j] = w[a];
        }
        for (int c0 = C * threadIdx.x; c0 < H; c0 += C * blockDim.x) {
            const int c = WHOLE || c0 + C <= H || H < C ? c0 : H - C;
            Piece<BF16> dp, v[8];
            dp.template load<WHOLE>(row_at<BF16>(dy, t, H), c, H);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j0 + j < top_k) v[j].template load<WHOLE, true>(row_at<BF16>(ys, p[j] < 0 ? 0 : p[j], H), c, H);
            float g[C];
#pragma unroll
            for (int i = 0; i < C; ++i) g[i] = WHOLE || i >= c0 - c ? dp[i] : 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (j0 + j >= top_k) continue;
                Piece<BF16> out;
                float o[C];
                if (p[j] >= 0) {
#pragma unroll
                    for (int i = 0; i < C; ++i) {
                        dot[j] = fmaf(g[i], WHOLE || i >= c0 - c ? v[j][i] : 0.0f, dot[j]);
                        o[i] = wj[j] * g[i];
                    }
                    out.set(o);
                    out.template store<WHOLE>(row_at<BF16>(dys, p[j], H), c, H, c0 - c);
                }
                const int a = t * top_k + j0 + j;
                if (a >= last) {
#pragma unroll
                    for (int i = 0; i < C; ++i) o[i] = 0.0f;
                    out.set(o);
                    out.template store<WHOLE>(row_at<BF16>(dys, a, H), c, H, c0 - c);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) dot[j] += __shfl_xor(dot[j], o, 64);
            if (lane == 0) s_sum[j][wave] = dot[j];
        }
        __syncthreads();
        if (threadIdx.x < 8 && j0 + (int)threadIdx.x < top_k) {
            float s = 0.0f;
            for (int i = 0; i < nw; ++i) s += s_sum[threadIdx.x][i];
            dw[t * top_k + j0 + (int)threadIdx.x] = s;
        }
        __syncthreads();
    }
}

hipError_t launch_combine_tokens_bwd(const void* dy, const void* ys, bool bf16, int n_tokens, int H, int top_k,
                                     const int32_t* total, const int32_t* place, const float* w, void* dys, float* dw,
                                     hipStream_t stream) {
    if (n_tokens <= 0) return hipSuccess;
    const int C = bf16 ? 8 : 4;
    const bool whole = H % C == 0;
    const int64_t pieces = ((int64_t)H + C - 1) / C;
    const dim3 grid(n_tokens), block((unsigned)(pieces < 1024 ? (pieces + 63) / 64 * 64 : 1024));
#define QMOE_BWD(B, V)                                                                                                 \
    hipLaunchKernelGGL((k_combine_tokens_bwd<B, V>), grid, block, 0, stream, dy, ys, H, top_k, n_tokens * top_k, total, \
                       place, w, dys, dw)
    if (bf16) { if (whole) QMOE_BWD(true, true); else QMOE_BWD(true, false); }
    else { if (whole) QMOE_BWD(false, true); else QMOE_BWD(false, false); }
#undef QMOE_BWD
    return hipGetLastError();
}

}  // namespace qmoe
