// fp8_kernels.hip -- 8-bit float (OCP e4m3) operands with an f32 scale per block
// of 128: rows quantized in blocks of 128 columns, and the products of such rows
// with weights scaled per block of 128 x 128, dense or grouped by expert.
#include "qmoe_device.h"
#include "qmoe_internal.h"

namespace qmoe {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));

// ---------------------------------------------------------------------------
// Quantization.  Block b of a row: m = max(|v|, kFp8Tiny) over its 128 columns
// (NaN counts as the largest, so a block with a NaN has a NaN scale),
//   scale = m / 448,  q = e4m3(f32(v * f32(448 / m))), nearest, ties to even.
// 448 is e4m3's largest value: the products stay within 448 (1 + 2^-22), which
// rounds to it.  kFp8Tiny keeps 448 / m finite; a block of zeros has zeros.
// 16 lanes take a block, 8 columns each (one or two 16-byte loads), so a wave
// covers 512 columns; no LDS, no barrier.
// ---------------------------------------------------------------------------
__device__ __forceinline__ float fp8_act(int act, float g, float u) {
    if (act == kFp8ActNone) return g;
    // gelu's tanh form is g sigmoid(2 z) with z = sqrt(2/pi) (g + 0.044715 g^3)
    const float z = act == kFp8ActSwiglu ? g : 1.5957691216057308f * (g + 0.044715f * g * g * g);
    return g / (1.0f + expf(-z)) * u;
}

template <bool BF16, bool VEC>
__device__ __forceinline__ void load8(const void* x, uint64_t at, int n, float (&v)[8]) {
    if constexpr (VEC && BF16) {
        const u16x8 r = *(const u16x8*)((const uint16_t*)x + at);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = bf16_to_f32(r[i]);
    } else if constexpr (VEC) {
        const f32x4 r = *(const f32x4*)((const float*)x + at), s = *(const f32x4*)((const float*)x + at + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = r[i], v[4 + i] = s[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = i >= n ? 0.0f : BF16 ? bf16_to_f32(((const uint16_t*)x)[at + i]) : ((const float*)x)[at + i];
    }
}

// VEC: the columns are a multiple of 8 and every row starts 16-byte aligned
template <bool BF16, bool VEC>
__global__ __launch_bounds__(256) void k_fp8_quantize(const void* x, uint32_t n_blocks, int cols, int act, uint8_t* q,
                                                      float* scale) {
    const uint32_t per_row = (uint32_t)(cols + kFp8Block - 1) / kFp8Block;
    const uint32_t id = blockIdx.x * 16u + threadIdx.x / 16u;
    if (id >= n_blocks) return;
    const uint32_t row = id / per_row;
    const int c0 = (int)(id - row * per_row) * kFp8Block + 8 * ((int)threadIdx.x & 15);
    const int n = cols - c0;  // columns from c0 on: none or some of this lane's 8 may exist
    float v[8] = {};
    if (n > 0) {
        if (act == kFp8ActNone) {
            load8<BF16, VEC>(x, (uint64_t)row * cols + c0, n, v);
        } else {
            float u[8];
            load8<BF16, VEC>(x, (uint64_t)row * 2 * cols + c0, n, v);
            load8<BF16, VEC>(x, (uint64_t)row * 2 * cols + cols + c0, n, u);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = fp8_act(act, v[i], u[i]);
        }
    }
    float inv;
    const float m = fp8_block_max(v, inv);
    uint32_t o[2];
    fp8_pack8(v, inv, o);
    if (n > 0) {
        uint8_t* qp = q + (uint64_t)row * cols + c0;
        if (VEC) {
            *(uint2*)qp = make_uint2(o[0], o[1]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < n) qp[i] = (uint8_t)(o[i >> 2] >> (8 * (i & 3)));
        }
    }
    if ((threadIdx.x & 15) == 0) scale[id] = m / kFp8Max;
}

hipError_t launch_fp8_quantize(const void* x, bool bf16, int64_t rows, int cols, int act, uint8_t* q, float* scale,
                               hipStream_t stream) {
    const int64_t blocks = rows * ((cols + kFp8Block - 1) / kFp8Block);
    if (blocks <= 0) return hipSuccess;
    if (blocks > 0xffffffffll) return hipErrorInvalidValue;
    const bool vec = cols % 8 == 0 && (((uintptr_t)x | (uintptr_t)q) & 15u) == 0;
    const dim3 grid((unsigned)((blocks + 15) / 16));
#define QMOE_Q8(B, V) hipLaunchKernelGGL((k_fp8_quantize<B, V>), grid, dim3(256), 0, stream, x, (uint32_t)blocks, cols, act, q, scale)
    if (bf16) { if (vec) QMOE_Q8(true, true); else QMOE_Q8(true, false); }
    else { if (vec) QMOE_Q8(false, true); else QMOE_Q8(false, false); }
#undef QMOE_Q8
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Products:  y[r][n] = sum_b sa[r][b] sw[n / 128][b] sum_{k in b} a[r][k] w[n][k].
// A block's 128 products start from zero and their sum is scaled into the f32
// accumulators.  The e4m3 MFMA (v_mfma_f32_16x16x128_f8f6f4) aligns the products
// of each group of 8 columns to the largest before it adds them: beside a product
// of 2^16 one of 2^3 counts and one of 2^2 is lost (measured; between groups, and
// in the f16 MFMA, all 24 bits are kept).  So the operands go to f16, which holds
// every e4m3 value, and to v_mfma_f32_16x16x32_f16: exact products, f32 sums.
// The weights are the MFMA's rows and the activations its columns: a lane then
// holds four consecutive n of one row r, whose scale is one value per lane, and
// stores them together.  (Both operands take the same permutation of a block's
// columns, which leaves its sum as it is: lane group g reads 16-byte pieces g and
// g + 4.)
// ---------------------------------------------------------------------------
__device__ __forceinline__ int clampi(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }

// Tile g of the list "experts in order, each with ceil(rows / tile) tiles" (a wave
// finds it by itself, 256 experts a step).  Offsets outside [0, R] are taken as its ends.
__device__ __forceinline__ bool fp8_find_tile(const Fp8Product& p, int tile, int g, int& expert, int& row0, int& end) {
    if (!p.offsets) {
        expert = 0;
        row0 = g * tile;
        end = p.R;
        return row0 < p.R;
    }
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (int c = 0; c < p.E; c += 256) {
        int lo[4], hi[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int e = c + 64 * j + lane;
            lo[j] = p.offsets[e < p.E ? e : p.E];
            hi[j] = p.offsets[e < p.E ? e + 1 : p.E];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int l = clampi(lo[j], 0, p.R), h = clampi(hi[j], 0, p.R);
            const int t = h > l ? (h - l + tile - 1) / tile : 0;
            const int incl = wave_incl_scan_i32(t);
            const int total = __builtin_amdgcn_readlane(incl, 63);
            if (g < base + total) {
                const int at = __builtin_ctzll(__ballot(base + incl > g));
                expert = c + 64 * j + at;
                row0 = __builtin_amdgcn_readlane(l, at) + (g - base - __builtin_amdgcn_readlane(incl - t, at)) * tile;
                end = __builtin_amdgcn_readlane(h, at);
                return true;
            }
            base += total;
        }
    }
    return false;
}

// The activation row behind product row r (-1: none, its products are zeros).
__device__ __forceinline__ int fp8_source_row(const Fp8Product& p, int r) {
    if (!p.rows) return r;
    const int s = p.rows[r];
    return s >= 0 && s < p.a_rows ? s : -1;
}

template <bool BF16>
__device__ __forceinline__ void fp8_store4(const Fp8Product& p, int r, int n, const float (&v)[4]) {
    const uint64_t at = (uint64_t)r * p.N + n;
    if (p.vec_out && n + 4 <= p.N) {
        if (BF16)
            *(uint2*)((uint16_t*)p.y + at) = make_uint2(f32_pack_bf16(v[0], v[1]), f32_pack_bf16(v[2], v[3]));
        else
            *(f32x4*)((float*)p.y + at) = f32x4{v[0], v[1], v[2], v[3]};
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < p.N) {
                if (BF16) ((uint16_t*)p.y)[at + i] = (uint16_t)f32_pack_bf16(v[i], 0.0f);
                else ((float*)p.y)[at + i] = v[i];
            }
    }
}

// 8 e4m3 values as f16 (exact, a NaN stays one).
__device__ __forceinline__ f16x8 fp8_to_f16(int a, int b) {
    const f16x2 p = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false);
    const f16x2 q = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true);
    const f16x2 r = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false);
    const f16x2 s = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true);
    return f16x8{p[0], p[1], q[0], q[1], r[0], r[1], s[0], s[1]};
}

// Few rows: a workgroup makes 16 columns of 16 MT rows.  Its four waves take the
// k blocks in turn, straight from memory into the MFMA operands, U blocks in flight;
// their sums are joined in LDS in wave order.
template <int MT, int U, bool BF16>
__global__ __launch_bounds__(256) void k_fp8_stream(Fp8Product p) {
    __shared__ float s_part[4][16 * MT][20];
    const int nt = (p.N + 15) >> 4;
    const int tile = blockIdx.x / nt, n0 = (blockIdx.x - tile * nt) * 16;
    int e, row0, end;
    if (!fp8_find_tile(p, 16 * MT, tile, e, row0, end)) return;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4;
    const int KB = p.KB;
    const int n = n0 + (lane & 15);
    const uint8_t* wr = p.w + ((uint64_t)e * p.N + (n < p.N ? n : p.N - 1)) * p.K;
    const float* sw = p.sw + ((uint64_t)e * p.NB + (n0 >> 7)) * KB;
    const uint8_t* ar[MT];
    const float* sa[MT];
    int src[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int r = row0 + 16 * i + (lane & 15);
        src[i] = fp8_source_row(p, r < end ? r : end - 1);
        const uint64_t at = src[i] < 0 ? 0 : src[i];
        ar[i] = p.a + at * p.K;
        sa[i] = p.sa + at * KB;
    }
    f32x4 acc[MT] = {};
    for (int b0 = wave; b0 < KB; b0 += 4 * U) {
        i32x4 wv[U][2], av[U][MT][2];
        float ws[U], as[U][MT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            // past the end: the last block again, scaled by zero
            const int b = b0 + 4 * u < KB ? b0 + 4 * u : KB - 1;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int c = b * kFp8Block + 16 * (g + 4 * h);
                const int at = c < p.K ? c : p.K - 16;
                wv[u][h] = *(const i32x4*)(wr + at);
#pragma unroll
                for (int i = 0; i < MT; ++i) av[u][i][h] = *(const i32x4*)(ar[i] + at);
            }
            ws[u] = sw[b];
#pragma unroll
            for (int i = 0; i < MT; ++i) as[u][i] = sa[i][b];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int b = b0 + 4 * u;
            if (b * kFp8Block + kFp8Block > p.K) {  // columns past K: zero weights
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (b * kFp8Block + 16 * (g + 4 * h) >= p.K) wv[u][h] = i32x4{};
            }
            f16x8 wf[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) wf[q] = fp8_to_f16(wv[u][q >> 1][2 * (q & 1)], wv[u][q >> 1][2 * (q & 1) + 1]);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                f32x4 t = {};
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    t = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                        wf[q], fp8_to_f16(av[u][i][q >> 1][2 * (q & 1)], av[u][i][q >> 1][2 * (q & 1) + 1]), t, 0, 0, 0);
                const float s = b < KB ? ws[u] * as[u][i] : 0.0f;
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[i][c] = fmaf(s, t[c], acc[i][c]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        if (src[i] < 0) acc[i] = f32x4{};
        *(f32x4*)&s_part[wave][16 * i + (lane & 15)][4 * g] = acc[i];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * MT; i += 256) {
        const int m = i >> 2, q = 4 * (i & 3);
        float v[4];
#pragma unroll
        for (int c = 0; c < 4; ++c)
            v[c] = (s_part[0][m][q + c] + s_part[1][m][q + c]) + (s_part[2][m][q + c] + s_part[3][m][q + c]);
        if (row0 + m < end && n0 + q < p.N) fp8_store4<BF16>(p, row0 + m, n0 + q, v);
    }
}

// Tiles that the rows of a product fill at most, whatever their split over experts.
static int64_t fp8_max_tiles(const Fp8Product& p, int tile) {
    if (!p.offsets) return (p.R + tile - 1) / tile;
    const int64_t active = p.R < p.E ? p.R : p.E;
    return active + (p.R - active) / tile;
}

template <int MT, int U>
static hipError_t launch_stream(const Fp8Product& p, bool bf16, hipStream_t stream) {
    const int64_t blocks = fp8_max_tiles(p, 16 * MT) * ((p.N + 15) / 16);
    if (blocks > 0x7fffffffll) return hipErrorInvalidValue;
    if (bf16) hipLaunchKernelGGL((k_fp8_stream<MT, U, true>), dim3((unsigned)blocks), dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((k_fp8_stream<MT, U, false>), dim3((unsigned)blocks), dim3(256), 0, stream, p);
    return hipGetLastError();
}

hipError_t launch_fp8_matmul(Fp8Product p, bool bf16, hipStream_t stream) {
    if (p.R <= 0) return hipSuccess;
    p.KB = (p.K + kFp8Block - 1) / kFp8Block;
    p.NB = (p.N + kFp8Block - 1) / kFp8Block;
    p.vec_out = p.N % 4 == 0 && ((uintptr_t)p.y & 15u) == 0;
    const int64_t mean = p.offsets ? p.R / p.E : p.R;  // rows per weight matrix
    if (mean >= 32) return launch_stream<4, 1>(p, bf16, stream);
    if (mean >= 12) return launch_stream<2, 2>(p, bf16, stream);
    return launch_stream<1, 4>(p, bf16, stream);
}

}  // namespace qmoe
