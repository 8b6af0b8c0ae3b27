// fp8_kernels.hip -- 8-bit float (OCP e4m3) operands with an f32 scale per block
// of 128: rows quantized in blocks of 128 columns, and the products of such rows
// with weights scaled per block of 128 x 128, dense or grouped by expert.
#include "qmoe_device.h"
#include "qmoe_internal.h"

#include <type_traits>

namespace qmoe {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------------------
// Quantization.  Block b of a row: m = max(|v|, kFp8Tiny) over its 128 columns
// (NaN counts as the largest, so a block with a NaN has a NaN scale),
//   scale = m / 448,  q = e4m3(v * 448 / m), nearest, ties to even.
// 448 is e4m3's largest value.  kFp8Tiny keeps 448 / m finite; a block of zeros has
// zeros.
// q of an activation is the formula's number rounded once too: where f32's errors in v and m
// could put a quotient on the other side of the middle of two e4m3 numbers (a block in some
// 300), the block is made again in f64.  Its scale is m / 448 of the f32 m.
// 16 lanes take a block, 8 columns each (one or two 16-byte loads), so a wave
// covers 512 columns; no LDS, no barrier.  Bound by memory: 4096 x 2048 f32 (42 MB) 8.2
// us, 5.1 TB/s (0.5 of it for the exact quotients); 32768 x 512 SwiGLU of bf16 (84 MB)
// 18.5-19.9 us, 4.4 TB/s, level with its arithmetic (2 more with expf; 0.5 of it for the
// blocks in f64, whose registers are kept within eight waves a SIMD); GeGLU 22.6-24, of
// gates four times as wide 27-28, its values' own error bounds 0.8-1 of it.
// ---------------------------------------------------------------------------
// v = g sigmoid(z) u and a bound of its relative error.  sigmoid_product is off by up to 5 2^-24 (the hardware's 2^t 2, its
// remainder 1, the quotient 1/2, the product 1).  SwiGLU's z is g; gelu's tanh form has z = 2 sqrt(2/pi) (g + 0.044715 g^3),
// which carries up to 6 2^-24 of itself (its constants, two products of the cubic part, the sum, the last product), and
// these count |z| e^-z / (1 + e^-z) times in v: |z| times below zero, at most 0.28 times above.
constexpr float kU32 = 0x1p-24f;  // half a step of f32
template <int ACT>
__device__ __forceinline__ float fp8_act(float g, float u, float& off) {
    const float z = ACT == kFp8ActSwiglu ? g : 1.5957691216057308f * fmaf(0.044715f * g * g, g, g);
    off = ACT == kFp8ActSwiglu ? 5 * kU32 : fmaf(-6 * kU32, __builtin_fminf(__builtin_fmaxf(z, -1e6f), 0.0f), 7 * kU32);
    return sigmoid_product(g, z, u);
}
template <int ACT>
__device__ __forceinline__ double fp8_act_exact(double g, double u) {
    const double z = ACT == kFp8ActSwiglu ? g : 1.5957691216057308 * (g + 0.044715 * g * g * g);
    return u * g * (1.0 / (1.0 + exp(-z)));
}
// f64 to f32 for one more rounding to a type of fewer bits: cut off, the last bit set if anything was.
__device__ __forceinline__ float f32_odd(double v) {
    uint32_t b = __builtin_bit_cast(uint32_t, (float)v);
    if (__builtin_fabs((double)__builtin_bit_cast(float, b)) > __builtin_fabs(v)) b -= 1;
    if ((double)__builtin_bit_cast(float, b) != v) b |= 1;
    return __builtin_bit_cast(float, b);
}
// Block id's q in f64, by the whole wave: two columns a lane.
template <bool BF16, int ACT>
__device__ __forceinline__ void fp8_act_block(const void* x, uint32_t row, int c0, int cols, uint8_t* q) {
    const int c = c0 + 2 * ((int)threadIdx.x & 63);
    const uint64_t at = (uint64_t)row * 2 * cols + c;
    double v[2] = {}, m = kFp8Tiny;
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (c + i < cols) v[i] = fp8_act_exact<ACT>(load1<BF16>(x, at + i), load1<BF16>(x, at + cols + i));
    m = __builtin_fmax(m, __builtin_fmax(__builtin_fabs(v[0]), __builtin_fabs(v[1])));
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = __builtin_fmax(m, __shfl_xor(m, o, 64));
    m *= 1.0 / kFp8Max;
    const uint32_t o = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f32_odd(v[0] / m), f32_odd(v[1] / m), 0, false);
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (c + i < cols) q[(uint64_t)row * cols + c + i] = (uint8_t)(o >> (8 * i));
}

template <bool BF16, bool WHOLE, int ACT>
__global__ __launch_bounds__(256, 8) void k_fp8_quantize(const void* x, uint32_t n_blocks, int cols, uint8_t* q, float* scale,
                                                      bool nt) {
    const uint32_t per_row = (uint32_t)(cols + kFp8Block - 1) / kFp8Block;
    const uint32_t id = blockIdx.x * 16u + threadIdx.x / 16u;
    const uint32_t row = id / per_row;
    const int c0 = (int)(id - row * per_row) * kFp8Block + 8 * ((int)threadIdx.x & 15);
    const int n = id < n_blocks ? cols - c0 : 0;  // columns from c0 on: none or some of this lane's 8 may exist
    float v[8] = {}, off[8] = {};
    if (n > 0) {
        if constexpr (ACT == kFp8ActNone) {
            load8<BF16, WHOLE>(x, (uint64_t)row * cols + c0, n, v);
        } else {
            float u[8];
            load8<BF16, WHOLE>(x, (uint64_t)row * 2 * cols + c0, n, v);
            load8<BF16, WHOLE>(x, (uint64_t)row * 2 * cols + cols + c0, n, u);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = fp8_act<ACT>(v[i], u[i], off[i]);
        }
    }
    const float m = fp8_block_max(v);
    uint32_t o[2];
    if constexpr (ACT == kFp8ActNone) {
        fp8_pack8(v, m, o);
        if (n > 0) store8_fp8(q + (uint64_t)row * cols + c0, n, o, nt);
    } else {
        // the quotients' own roundings (448 / m, its two neighbours, the two products), and m's error: the largest of
        // |v| (1 + off) lies as far above the exact maximum's least value as that above m's
        float near = 12 * kU32;
        if constexpr (ACT == kFp8ActGeglu) {
            float above[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) above[i] = fmaf(__builtin_fabsf(v[i]), off[i], __builtin_fabsf(v[i]));
            const float top = fp8_block_max(above);
            if (m < __builtin_huge_valf()) near = fmaf(1.0f / m, top - m, 7 * kU32);
        }
        uint64_t open = __ballot(!fp8_pack8_near(v, off, m, near, o));
        if (n > 0 && (open >> (threadIdx.x & 48) & 0xffff) == 0) store8_fp8(q + (uint64_t)row * cols + c0, n, o, nt);
        while (open) {
            const int first = __builtin_ctzll(open) & 48;  // the block's first lane
            open &= ~(0xffffull << first);
            fp8_act_block<BF16, ACT>(x, (uint32_t)__builtin_amdgcn_readlane((int)row, first),
                                __builtin_amdgcn_readlane(c0, first), cols, q);
        }
    }
    if (n > 0 && (threadIdx.x & 15) == 0) scale[id] = m / kFp8Max;
}

hipError_t launch_fp8_quantize(const void* x, bool bf16, int64_t rows, int cols, int act, uint8_t* q, float* scale,
                               hipStream_t stream) {
    const int64_t blocks = rows * ((cols + kFp8Block - 1) / kFp8Block);
    if (blocks <= 0) return hipSuccess;
    if (blocks > (1ll << 28) - 16) return hipErrorInvalidValue;  // (16 threads each in whole workgroups of 256, below 2^32 a launch)
    // nt: rows of whole lines past the caches where they are more than an L2 holds and fewer than eight do (32768 x 512 SwiGLU
    // bf16 21.7 -> 20.0 us, f32 without 9.6 -> 9.2).  With the product that reads them next the two are level, us through /
    // past: 8 MB 91.5 / 91.4, 101 / 100, 12 MB 147 / 146, 17 MB 130 / 131, 128 / 127, 119 / 119 (once 108 / 114); beyond,
    // 34 MB 229 / 231, 232 / 236.
    const int64_t bytes = rows * cols;
    const bool whole = cols % 8 == 0, nt = cols % kFp8Block == 0 && bytes > kL2Bytes && bytes < 8 * kL2Bytes;
    const dim3 grid((unsigned)((blocks + 15) / 16));
#define QMOE_Q8A(B, V, A) \
    hipLaunchKernelGGL((k_fp8_quantize<B, V, A>), grid, dim3(256), 0, stream, x, (uint32_t)blocks, cols, q, scale, nt)
#define QMOE_Q8(B, V)                                              \
    do {                                                           \
        if (act == kFp8ActNone) QMOE_Q8A(B, V, kFp8ActNone);       \
        else if (act == kFp8ActSwiglu) QMOE_Q8A(B, V, kFp8ActSwiglu); \
        else QMOE_Q8A(B, V, kFp8ActGeglu);                         \
    } while (0)
    if (bf16) { if (whole) QMOE_Q8(true, true); else QMOE_Q8(true, false); }
    else { if (whole) QMOE_Q8(false, true); else QMOE_Q8(false, false); }
#undef QMOE_Q8
#undef QMOE_Q8A
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Products:  y[r][n] = sum_b sa[r][b] sw[n / 128][b] sum_{k in b} a[r][k] w[n][k].
// A block's 128 products start from zero and their sum is scaled into the f32
// accumulators (one fma per output and block).  The operands are converted to f16, which
// holds every e4m3 value, for v_mfma_f32_16x16x32_f16: exact products, sums with f32's 24
// bits.  The e4m3 instructions are not used: they align the products of each group of 8
// columns to the largest, P, before they add them, and drop what lies below 2^-13 P
// (measured, 16x16x128_f8f6f4 and 16x16x32_fp8_fp8 alike: beside P = 2^16 a product of
// 2^3 counts and one of 2^2 is lost), so that a sum whose large terms cancel is lost
// whole.  16x16x128_f8f6f4 has twice the f16 rate (in registers 4.4 and 2.1-2.4 PFLOP/s;
// 8192 x 4096 x 4096 took 125 us by it); 16x16x32_fp8_fp8 has the f16 rate.
// The weights are the MFMA's rows and the activations its columns: a lane then
// holds four consecutive n of one row r, whose scale is one value per lane, and
// stores them together.  (Both operands take the same permutation of a block's
// columns, which leaves its sum as it is: lane group g reads 16-byte pieces g and
// g + 4.)
//   Where the time goes (us): 8192 x 4096 x 4096 208-232 (1.2-1.3 PFLOP/s, the rate of a
// library's bf16 product), f32 results 218-236: the matrix instructions are busy in 53% of
// the cycles, and the conversions to f16 and the scales' fmas, 66000 vector instructions a
// SIMD of 4 cycles each, take as many again beside them; 256 experts of 1024 x 2048: 80 rows
// 26-28 (147 MB: 5.4 TB/s), 4096 rows 89 (6.0 TB/s), 32768 rows 182-200 (0.7 PFLOP/s).
// ---------------------------------------------------------------------------
__device__ __forceinline__ int clampi(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }

// Tile g of the list "experts in order, each with ceil(rows / tile) tiles" (a wave
// finds it by itself, 256 experts a step); once: its expert has no other.  Offsets
// outside [0, R] are taken as its ends, so that whatever they hold a tile's rows lie
// within [0, R).
__device__ __forceinline__ bool fp8_find_tile(const Fp8Product& p, int tile, int g, int& expert, int& row0, int& end,
                                              bool& once) {
    if (!p.offsets) {
        expert = 0;
        row0 = g * tile;
        end = p.R;
        once = false;
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
                once = __builtin_amdgcn_readlane(t, at) == 1;
                return row0 >= __builtin_amdgcn_readlane(l, at) && row0 < end;  // (offsets that fall can overflow the sums)
            }
            base += total;
        }
    }
    return false;
}

// The row and column tile of a workgroup.  Workgroups are dealt to the 8 XCDs in turn.
// Grouped: XCD x takes every eighth row tile with all its column tiles, so that a tile's
// rows stay in one L2.  One matrix: each XCD a contiguous run of the order "bands of 8 row
// tiles, column by column", whose workgroups in flight share few rows and columns.
__device__ __forceinline__ void fp8_place(const Fp8Product& p, int bm, int nt, int& tile, int& col) {
    const int x = blockIdx.x & 7, j = blockIdx.x >> 3;
    if (p.offsets) {
        tile = (j / nt) * 8 + x;
        col = j % nt;
        return;
    }
    const int mt = (p.R + bm - 1) / bm;
    const int at = x * (int)(gridDim.x >> 3) + j;
    const int band = at / (8 * nt), in = at - band * 8 * nt;
    const int high = mt - 8 * band < 8 ? mt - 8 * band : 8;  // (none past the last tile)
    tile = high > 0 && in / high < nt ? 8 * band + in % high : mt;
    col = high > 0 ? in / high : 0;
}

// The activation row behind product row r (-1: none, its products are zeros).
__device__ __forceinline__ int fp8_source_row(const Fp8Product& p, int r) {
    if (!p.rows) return r;
    const int s = p.rows[r];
    return s >= 0 && s < p.a_rows ? s : -1;
}

template <bool BF16>
__device__ __forceinline__ uint32_t fp8_bits(float a, float b) {  // two bf16 or one f32
    return BF16 ? f32_pack_bf16(a, b) : __builtin_bit_cast(uint32_t, a);
}
// C consecutive columns (4 or 8) of a row from column n on, up to 16 bytes at the elements'
// alignment; those past N are left out.
template <bool BF16, int C>
__device__ __forceinline__ void fp8_store(const Fp8Product& p, int r, int n, const float (&v)[C]) {
    static_assert(C == 4 || (C == 8 && BF16), "up to 16 bytes");
    const uint64_t at = (uint64_t)r * p.N + n;
    if (n + C <= p.N) {
        if constexpr (!BF16) {
            put((float*)p.y + at, f32x4a4{v[0], v[1], v[2], v[3]}, p.stream_out);
        } else if constexpr (C == 4) {
            put((uint16_t*)p.y + at, u32x2a2{f32_pack_bf16(v[0], v[1]), f32_pack_bf16(v[2], v[3])}, p.stream_out);
        } else {
            put((uint16_t*)p.y + at, u32x4a2{f32_pack_bf16(v[0], v[1]), f32_pack_bf16(v[2], v[3]),
                                             f32_pack_bf16(v[4], v[5]), f32_pack_bf16(v[6], v[7])}, p.stream_out);
        }
    } else {
#pragma unroll
        for (int i = 0; i < C; ++i)
            if (n + i < p.N) store1<BF16>(p.y, at + i, v[i]);
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

// Few rows (MT 1 or 2): a workgroup makes 16 columns of 16 MT rows.  Its four waves take the
// k blocks in turn, straight from memory into the MFMA operands, U blocks in flight;
// their sums are joined in LDS in wave order.  Bound by its chain of dependent loads:
// 8 rows on 8 experts of 1024 x 2048 (17 MB) 6.6 us.
template <int MT, int U, bool BF16>
__global__ __launch_bounds__(256) void k_fp8_stream(Fp8Product p) {
    __shared__ float s_part[4][16 * MT][20];
    const int nt = (p.N + 15) >> 4;
    const int tile = blockIdx.x / nt, n0 = (blockIdx.x - tile * nt) * 16;
    int e, row0, end;
    bool once;
    if (!fp8_find_tile(p, 16 * MT, tile, e, row0, end, once)) return;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4;
    const int KB = p.KB;
    const int n = n0 + (lane & 15);
    const uint8_t* wr = p.w + ((uint64_t)e * p.N + (n < p.N ? n : p.N - 1)) * p.K;
    const float* sw = p.sw + ((uint64_t)e * p.NB + (n0 >> 7)) * KB;
    // past the end: the last block again, scaled by zero
    auto block = [&](int b0, int u) { return b0 + 4 * u < KB ? b0 + 4 * u : KB - 1; };
    auto piece = [&](int b, int h) {
        const int c = b * kFp8Block + 16 * (g + 4 * h);
        return c < p.K ? c : p.K - 16;
    };
    i32x4 wv[U][2];
    float ws[U];
    auto load_w = [&](int b0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int h = 0; h < 2; ++h) wv[u][h] = *(const i32x4*)(wr + piece(block(b0, u), h));
            ws[u] = sw[block(b0, u)];
        }
    };
    load_w(wave < KB ? wave : KB - 1);  // the first weights are on their way while the rows' indices come
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
        i32x4 av[U][MT][2];
        float as[U][MT];
        if (b0 != wave) load_w(b0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int b = block(b0, u);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
#pragma unroll
                for (int h = 0; h < 2; ++h) av[u][i][h] = *(const i32x4*)(ar[i] + piece(b, h));
                as[u][i] = sa[i][b];
            }
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
        if (row0 + m < end && n0 + q < p.N) fp8_store<BF16, 4>(p, row0 + m, n0 + q, v);
    }
}

// A wave-uniform read-only value through the scalar cache: no vector memory load, whose
// wait would be one for all direct loads before it.
__device__ __forceinline__ float scalar_load(const float* p) {
    return *(const __attribute__((address_space(4))) float*)(uintptr_t)p;
}
// s_waitcnt's operand for at most n vector memory operations in flight
constexpr int vm_wait(int n) { return (n & 15) | ((n >> 4) << 14) | 0x0F70; }
// A workgroup barrier after this wave's own LDS accesses; direct loads stay in flight.
__device__ __forceinline__ void lds_barrier() {
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
}
template <int WM, int WN, int MS, int NS, int ST, bool BF16>
struct Fp8Tile {
    static constexpr int kWaves = WM * WN, kBM = 16 * MS * WM, kBN = 16 * NS * WN;
    static constexpr int kScaleLoads = (kBM + 63) / 64;
    static constexpr int kStage = (kBM + kBN) * kFp8Block;  // rows, weights
    static constexpr int kScales = 1024 * kScaleLoads;      // row scales of four steps: two buffers behind the stages
    static constexpr int kLds = ST * kStage + 2 * kScales + 64 * kScaleLoads;
    // Columns that a lane stores together: 16 bytes.  Of 4 kCols columns, 4 a + c of P = kCols / 4 subtiles each,
    // weight row 4 P a + 4 n + c is the MFMA's row 4 a + c of subtile n, so that lane group a holds 4 P consecutive
    // columns and a wave's four groups 64 bytes of a row.  The row's pieces lie at slots piece ^ slot_w(row): the
    // eight rows that a quarter of a wave reads (a = 0, 1 or 2, 3; c = 0..3) have eight slots.
    static constexpr int P = BF16 && NS > 1 ? 2 : 1, kCols = 4 * P;
    static_assert(NS % P == 0, "whole groups of subtiles");
    static __host__ __device__ constexpr int slot_w(int row) { return (row & 3) | (row / kCols & 1) << 2; }
    static constexpr int kGroupsA = (kBM / 8 + kWaves - 1) / kWaves;
    static constexpr int kLoads = kGroupsA + kBN / 8 / kWaves;  // of one wave, a step, without scales
    static_assert(kBM % 16 == 0 && kBN % (8 * kWaves) == 0, "whole loads per wave");
    static_assert(16 * NS <= kFp8Block, "a wave's columns share one scale");
};

// Many rows: a workgroup of WM x WN waves makes a tile of 16 MS WM rows and 16 NS WN
// columns.  Each step of 128 columns of K comes straight to LDS (ST buffers): rows of 128
// bytes, whose eight 16-byte pieces lie at slots piece ^ (row & 7), so that the 16 rows of a
// fragment meet all banks.  (What conflicts there are come from the row scales, 4 bytes read
// at steps of 16: two cycles a read, 8192 of a CU's in 8192 x 4096 x 4096.)  The 16-row
// subtiles go to the WM waves in turn and those without rows are left out (MI: how many).
template <int WM, int WN, int MS, int NS, int ST, bool BF16>
__global__ __launch_bounds__(64 * WM * WN) void k_fp8_tile(Fp8Product p) {
    using T = Fp8Tile<WM, WN, MS, NS, ST, BF16>;
    extern __shared__ uint8_t s_dyn[];
    const int nt = (p.N + T::kBN - 1) / T::kBN;
    int tile, n0, e, row0, end;
    bool once;
    fp8_place(p, T::kBM, nt, tile, n0);
    n0 *= T::kBN;
    if (!fp8_find_tile(p, T::kBM, tile, e, row0, end, once)) return;
    // Weights that this row tile alone reads, in whole 128-byte lines, go past the caches.  256 experts of
    // 1024 x 2048, several layers' weights in turn, us without and with: 80 rows 28.8 / 27.2, 1024 rows 90 / 80, 4096
    // 95 / 91, 32768 190 / 185; with two tiles an expert (80000 rows) 384 / 410; with 5.5 lines a row (128 of 2816 x
    // 704, 1688 rows) 58 / 63, 4000 rows 65 / 70.
    once = once && p.K % kFp8Block == 0;
    const int nrows = end - row0 < T::kBM ? end - row0 : T::kBM;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int wm = wave % WM, wn = wave / WM;
    const int KB = p.KB;

    // this lane's share of the loads: groups of 8 rows, 8 lanes a row
    constexpr int kGA = T::kGroupsA, kGW = T::kBN / 8 / T::kWaves;
    const int piece = 16 * ((lane & 7) ^ (lane >> 3));
    const int piece_w = 16 * ((lane & 7) ^ T::slot_w(8 * wave + (lane >> 3)));
    static_assert(T::slot_w(8 * T::kWaves) == 0, "the same slots in every group of a wave");
    // (a tile whose row groups do not divide among the waves: the last ones load some again)
    auto group_a = [&](int i) {
        return (wave + T::kWaves * i) % (T::kBM / 8);
    };
    const uint8_t* ga[kGA];
#pragma unroll
    for (int i = 0; i < kGA; ++i) {
        const int r = 8 * group_a(i) + (lane >> 3);
        const int s = fp8_source_row(p, row0 + (r < nrows ? r : nrows - 1));
        ga[i] = p.a + (uint64_t)(s < 0 ? 0 : s) * p.K;
    }
    const uint8_t* const wt = p.w + ((uint64_t)e * p.N + n0) * p.K;  // the tile's weights, offsets below 2^32
    uint32_t gw[kGW];
#pragma unroll
    for (int i = 0; i < kGW; ++i) {
        const int n = 8 * (wave + T::kWaves * i) + (lane >> 3);
        gw[i] = (uint32_t)(n < p.N - n0 ? n : p.N - n0 - 1) * (uint32_t)p.K;
    }
    const float* gs = nullptr;
    uint8_t* s_none = s_dyn + ST * T::kStage + 2 * T::kScales;  // rows without a source (read after the loop's barriers)
    if (wave < T::kScaleLoads) {
        const int r = 64 * wave + lane;
        const int s = fp8_source_row(p, row0 + (r < nrows ? r : nrows - 1));
        gs = p.sa + (uint64_t)(s < 0 ? 0 : s) * KB;
        s_none[r] = s < 0;
    }
    // The row scales of steps b .. b + 3, by the waves 0 .. kScaleLoads - 1: 64 rows each, 16 bytes a row
    // (a row's scales lie KB apart: one 64-row load of single scales costs as much).  Where KB is no
    // multiple of 4, four loads of one step each.
    const bool quads = KB % 4 == 0 && ((uintptr_t)p.sa & 15) == 0;
    auto load_scales = [&](int b) {
        if (wave >= T::kScaleLoads) return;
        const uint32_t base = lds_addr(s_dyn) + ST * T::kStage + (b >> 2 & 1) * T::kScales + 1024 * wave;
        if (quads) {
            dma_lds16_at(gs + b, base);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) dma_lds4_at(gs + (b + i < KB ? b + i : KB - 1), base + 256 * i);
        }
    };
    // This wave's loads [from, to) of step b into buffer buf, of kLoads: the rows' groups (the row scales of four steps
    // first), then the weights'.
    const uint32_t lds0 = lds_addr(s_dyn);
    auto load = [&](int b, int buf, int from, int to) {
        if (from == 0 && b % 4 == 0) load_scales(b);
        // past K: any valid piece, its weights are zeroed below
        auto column = [&](int piece) { const int c = b * kFp8Block + piece; return c < p.K ? c : p.K - 16; };
        const uint32_t base = lds0 + buf * T::kStage;
        const int ca = column(piece), cw = column(piece_w);
#pragma unroll
        for (int i = 0; i < kGA; ++i)
            if (i >= from && i < to) dma_lds16_at(ga[i] + ca, base + 1024 * group_a(i));
        auto weights = [&](auto nt_c) {
#pragma unroll
            for (int i = 0; i < kGW; ++i)
                if (kGA + i >= from && kGA + i < to)
                    dma_lds16<decltype(nt_c)::value>(wt, gw[i] + (uint32_t)cw,
                                                     base + T::kBM * kFp8Block + 1024 * (wave + T::kWaves * i));
        };
        if (once) weights(std::true_type{});
        else weights(std::false_type{});
    };
    const int scale_row = quads ? 16 : 4, scale_step = quads ? 4 : 256;  // LDS distances

    const int nw0 = n0 + 16 * NS * wn;  // this wave's columns
    const float* sw = p.sw + ((uint64_t)e * p.NB + (nw0 < p.N ? nw0 >> 7 : 0)) * KB;
    const int fr = lane & 15, fg = lane >> 4;
    const int piece0 = fr * kFp8Block + 16 * (fg ^ (fr & 7)), piece1 = piece0 ^ 64;  // (fg + 4) ^ .. = (fg ^ ..) ^ 4
    const int fw = T::kCols * (fr >> 2) + (fr & 3);  // this lane's weight row of subtile 0
    const int wpiece0 = fw * kFp8Block + 16 * (fg ^ T::slot_w(fw)), wpiece1 = wpiece0 ^ 64;
    f32x4 acc[MS][NS] = {};
    // A step's weight fragments, and its first row fragment, are read while the step before it makes its last products.
    auto run = [&](auto mi_c) {
        constexpr int MI = decltype(mi_c)::value;
        constexpr int kLate = MI >= 4 ? 2 : 1;  // subtiles whose products come after the step's last row fragment is read
        // Eight waves load half of a stage after the barrier, half in the next step: all at once they hold each other up
        // (8192 x 4096 x 4096 bf16 220 us, in halves 214; tiles of four waves lose 1-2% by it).
        constexpr int kFirst = T::kWaves == 8 && MI >= 4 ? (T::kLoads + 1) / 2 : T::kLoads;
        int buf = 0;
        float ws_next = scalar_load(sw);
        i32x8 av[3], wv[NS];  // (whole operands: halves carried apart would be copied together)
        float rs[3];
        auto join = [](i32x4 lo, i32x4 hi) { return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7); };
        // subtile 0 has fragment registers of its own
        auto slot = [](int i) { return i == 0 ? 2 : (i - 1) & 1; };
        auto rows = [&](int i, int b, int at) {
            const uint8_t* st = s_dyn + at * T::kStage;
            const uint8_t* scales = s_dyn + ST * T::kStage + (b >> 2 & 1) * T::kScales + (b & 3) * scale_step + fr * scale_row;
            const int sub = WM * i + wm, x = slot(i);
            av[x] = join(*(const i32x4*)(st + 16 * sub * kFp8Block + piece0), *(const i32x4*)(st + 16 * sub * kFp8Block + piece1));
            // (subtile sub is rows 16 (sub % 4) .. of load sub / 4)
            rs[x] = *(const float*)(scales + 1024 * (sub >> 2) + 16 * (sub & 3) * scale_row);
        };
        auto weights = [&](int n, int at) {
            const uint8_t* w = s_dyn + at * T::kStage +
                               (T::kBM + 16 * NS * wn + 4 * T::kCols * (n / T::P) + 4 * (n % T::P)) * kFp8Block;
            wv[n] = join(*(const i32x4*)(w + wpiece0), *(const i32x4*)(w + wpiece1));
        };
        // LAST: no step follows, and K may end inside its block
        auto step = [&](int b, auto last_c) {
            constexpr bool LAST = decltype(last_c)::value;
            const float ws = ws_next;
            ws_next = scalar_load(sw + (b + 1 < KB ? b + 1 : b));
            const int after = buf + 1 == ST ? 0 : buf + 1;
            f16x8 wf[NS][4];
#pragma unroll
            for (int n = 0; n < NS; ++n) {
                if (LAST) {
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        if (16 * (fg + (c & 4)) >= p.K - b * kFp8Block) wv[n][c] = 0;
                }
#pragma unroll
                for (int q = 0; q < 4; ++q) wf[n][q] = fp8_to_f16(wv[n][2 * q], wv[n][2 * q + 1]);
            }
            f16x8 af[kLate][4];
            auto convert = [&](int i, int to) {
#pragma unroll
                for (int q = 0; q < 4; ++q) af[to][q] = fp8_to_f16(av[slot(i)][2 * q], av[slot(i)][2 * q + 1]);
            };
            auto product = [&](int n, int from) {
                f32x4 t = {};
#pragma unroll
                for (int q = 0; q < 4; ++q) t = __builtin_amdgcn_mfma_f32_16x16x32_f16(wf[n][q], af[from][q], t, 0, 0, 0);
                return t;
            };
            auto add = [&](int i, int n, float s, f32x4 t) {
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[i][n][c] = fmaf(s, t[c], acc[i][n][c]);
            };
#pragma unroll
            for (int i = 0; i < MI - kLate; ++i) {
                rows(i + 1, b, buf);
                if (i == 0 && !LAST && kFirst < T::kLoads && b > 0 && b - 1 + ST < KB)
                    load(b - 1 + ST, buf ? buf - 1 : ST - 1, kFirst, T::kLoads);
                const float s = ws * rs[slot(i)];
                convert(i, 0);
                f32x4 t[NS];
#pragma unroll
                for (int n = 0; n < NS; ++n) t[n] = product(n, 0);
#pragma unroll
                for (int n = 0; n < NS; ++n) add(i, n, s, t[n]);
                __builtin_amdgcn_sched_barrier(0);  // (loads moved up from the next subtile would spill)
            }
            if (kLate == 2) rows(MI - 1, b, buf);
            if (!LAST) {
                // step b + 1 has landed (at most the ST - 2 after it are in flight; a wave's scale loads come before its
                // stage's) ...
#pragma unroll
                for (int i = 0; i < MI - kLate; ++i)
#pragma unroll
                    for (int n = 0; n < NS; ++n) asm volatile("" : "+v"(acc[i][n]));  // (sums sunk past the barrier would spill)
                __builtin_amdgcn_sched_barrier(0);
                if (b + ST - 1 < KB) __builtin_amdgcn_s_waitcnt(vm_wait((ST - 2) * T::kLoads));
                else __builtin_amdgcn_s_waitcnt(vm_wait(0));
                lds_barrier();  // ... for every wave, and step b's buffer is no longer read
                __builtin_amdgcn_sched_barrier(0);
                if (b + ST < KB) load(b + ST, buf, 0, kFirst);
                if (MI > 1) rows(0, b + 1, after);
            }
            float s[kLate];
#pragma unroll
            for (int j = 0; j < kLate; ++j) {
                s[j] = ws * rs[slot(MI - kLate + j)];
                convert(MI - kLate + j, j);
            }
#pragma unroll
            for (int n = 0; n < NS; ++n) {
                f32x4 t[kLate];
#pragma unroll
                for (int j = 0; j < kLate; ++j) t[j] = product(n, j);
                if (!LAST) weights(n, after);
#pragma unroll
                for (int j = 0; j < kLate; ++j) add(MI - kLate + j, n, s[j], t[j]);
            }
            if (!LAST && MI == 1) rows(0, b + 1, after);
            buf = after;
        };
        // step 0
        if (ST < KB) __builtin_amdgcn_s_waitcnt(vm_wait((ST - 1) * T::kLoads));
        else __builtin_amdgcn_s_waitcnt(vm_wait(0));
        lds_barrier();
        rows(0, 0, 0);
#pragma unroll
        for (int n = 0; n < NS; ++n) weights(n, 0);
        for (int b = 0; b + 1 < KB; ++b) step(b, std::false_type{});
        step(KB - 1, std::true_type{});
    };
#pragma unroll
    for (int b = 0; b < ST; ++b)
        if (b < KB) load(b, b, 0, T::kLoads);
    const int subs = (nrows + 15) >> 4;                     // subtiles with rows
    const int mine = subs > wm ? (subs - wm + WM - 1) / WM : 0;  // ... of this wave
    constexpr int kHalf = MS / 2 > 1 ? MS / 2 : 1, kQuarter = MS / 4 > 1 ? MS / 4 : 1;
    if (mine > kHalf) run(std::integral_constant<int, MS>{});
    else if (mine > kQuarter) run(std::integral_constant<int, kHalf>{});
    else run(std::integral_constant<int, kQuarter>{});

    // Two 64-byte pieces of a row's columns: lanes of rows 8 apart swap one of theirs, so that a store covers whole
    // 128-byte lines (256 experts x 32768 rows: 67 MB written for 93).
    constexpr bool kLines = NS / T::P % 2 == 0;
    const bool lines = kLines && nw0 + 16 * NS <= p.N;
#pragma unroll
    for (int i = 0; i < MS; ++i) {
        const int m0 = 16 * (WM * i + wm), m = m0 + fr;
        if (m0 >= nrows) continue;
        const bool none = s_none[m];
        auto value = [&](int n, int c) { return none ? 0.0f : acc[i][n + (c >> 2)][c & 3]; };
        if (lines) {
            if constexpr (kLines) {
                const bool high = fr & 8;
                const int ra = m0 + (fr & 7);
#pragma unroll
                for (int n = 0; n < NS; n += 2 * T::P) {
                    uint32_t x[4], y[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const uint32_t v0 = fp8_bits<BF16>(value(n, BF16 ? 2 * c : c), BF16 ? value(n, 2 * c + 1) : 0.0f);
                        const uint32_t v1 = fp8_bits<BF16>(value(n + T::P, BF16 ? 2 * c : c), BF16 ? value(n + T::P, 2 * c + 1) : 0.0f);
                        const uint32_t got = __builtin_amdgcn_update_dpp(0, high ? v0 : v1, 0x128, 0xf, 0xf, false);
                        x[c] = high ? got : v0;
                        y[c] = high ? v1 : got;
                    }
                    const int col = nw0 + 16 * (high ? n + T::P : n) + T::kCols * fg;
                    uint8_t* const to = (uint8_t*)p.y + ((uint64_t)(row0 + ra) * p.N + col) * (BF16 ? 2 : 4);
                    if (ra < nrows) put(to, u32x4a2{x[0], x[1], x[2], x[3]}, p.stream_out);
                    if (ra + 8 < nrows) put(to + (uint64_t)8 * p.N * (BF16 ? 2 : 4), u32x4a2{y[0], y[1], y[2], y[3]}, p.stream_out);
                }
            }
        } else if (m < nrows) {
#pragma unroll
            for (int n = 0; n < NS; n += T::P) {
                const int col = nw0 + 16 * n + T::kCols * fg;
                float v[T::kCols];
#pragma unroll
                for (int c = 0; c < T::kCols; ++c) v[c] = value(n, c);
                if (col < p.N) fp8_store<BF16, T::kCols>(p, row0 + m, col, v);
            }
        }
    }
}

constexpr int64_t kFp8Cus = 256;  // CUs of the MI355X

// Tiles that the rows of a product fill at most, whatever their split over experts.
static int64_t fp8_max_tiles(const Fp8Product& p, int tile) {
    if (!p.offsets) return (p.R + tile - 1) / tile;
    const int64_t active = p.R < p.E ? p.R : p.E;
    return active + (p.R - active) / tile;
}

template <int MT, int U>
static hipError_t launch_stream(const Fp8Product& p, bool bf16, hipStream_t stream) {
    const int64_t blocks = fp8_max_tiles(p, 16 * MT) * ((p.N + 15) / 16);
    if (blocks >= 1ll << 24) return hipErrorInvalidConfiguration;  // (below 2^32 threads)
    if (bf16) hipLaunchKernelGGL((k_fp8_stream<MT, U, true>), dim3((unsigned)blocks), dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((k_fp8_stream<MT, U, false>), dim3((unsigned)blocks), dim3(256), 0, stream, p);
    return hipGetLastError();
}

template <int WM, int WN, int MS, int NS, int ST, bool BF16>
static hipError_t launch_tile_as(const Fp8Product& p, hipStream_t stream) {
    using T = Fp8Tile<WM, WN, MS, NS, ST, BF16>;
    const int64_t tiles = fp8_max_tiles(p, T::kBM), nt = (p.N + T::kBN - 1) / T::kBN;
    const int64_t blocks = p.offsets ? (tiles + 7) / 8 * 8 * nt : (tiles * nt + 7) / 8 * 8;
    if (blocks * (64 * T::kWaves) >= 1ll << 32) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL((k_fp8_tile<WM, WN, MS, NS, ST, BF16>), dim3((unsigned)blocks), dim3(64 * T::kWaves), T::kLds, stream, p);
    return hipGetLastError();
}
template <int WM, int WN, int MS, int NS, int ST>
static hipError_t launch_tile(const Fp8Product& p, bool bf16, hipStream_t stream) {
    return bf16 ? launch_tile_as<WM, WN, MS, NS, ST, true>(p, stream) : launch_tile_as<WM, WN, MS, NS, ST, false>(p, stream);
}

hipError_t launch_fp8_matmul(Fp8Product p, bool bf16, hipStream_t stream) {
    if (p.R <= 0) return hipSuccess;
    p.KB = (p.K + kFp8Block - 1) / kFp8Block;
    p.NB = (p.N + kFp8Block - 1) / kFp8Block;
    // Workgroups of rows x cols tiles (grouped: at most).
    auto wgs = [&](int rows, int cols) { return fp8_max_tiles(p, rows) * ((p.N + cols - 1) / cols); };
    // Results of experts past the caches where they are larger than an L2 (4 MB) and below 64 MB, in whole lines or bf16 of
    // few rows an expert: the product and what reads it next (the block's quantization or weighted sum), us through /
    // past; 256 experts of 1024 x 2048 and 2048 x 512 bf16, 8 MB 95 / 93, 17 MB 111 / 105, 34 MB 67 / 63, 67 MB 203 / 205
    // and 94 / 93, 134 MB 132 / 136; f32 17 MB 101 / 95, 34 MB 64 / 60, 49 MB 133 / 127, 98 MB 86 / 88, 185 MB 159 / 165;
    // rows that share lines (992 columns) 16 MB 111 / 105, 33 MB 139 / 135.  One matrix: 34 MB 118 / 118, 67 MB 232 / 234.
    const int elem = bf16 ? 2 : 4;
    const int64_t out_bytes = (int64_t)p.R * p.N * elem;
    const bool whole_lines = p.N * elem % 128 == 0 && (uintptr_t)p.y % 128 == 0;
    p.stream_out = p.offsets && out_bytes > kL2Bytes && out_bytes < 16 * kL2Bytes && (whole_lines || (bf16 && p.R / p.E <= 256));
    // A grid of at most two workgroups per CU that streams its operands once: latency.
    if (wgs(p.offsets ? 16 : 32, 16) <= 2 * kFp8Cus)
        return p.offsets || p.R <= 16 ? launch_stream<1, 4>(p, bf16, stream) : launch_stream<2, 2>(p, bf16, stream);
    if (!p.offsets) {
        // The largest tile that gives every CU a workgroup.  Rows x 4096 x 4096, bf16, us with tiles of
        // 256x256 / 128x256 / 64x128 / 32x128: 4096 rows 106 / 121 / 148, 2048 97 / 62 / 76, 1024 95 / 58 / 41, 512 95 /
        // 57 / 28, 256 94 / 56 / 27 / 21.
        if (wgs(256, 256) >= kFp8Cus) return launch_tile<2, 4, 8, 4, 2>(p, bf16, stream);
        if (wgs(128, 256) >= kFp8Cus) return launch_tile<2, 4, 4, 4, 3>(p, bf16, stream);
        if (wgs(64, 128) >= kFp8Cus) return launch_tile<1, 4, 4, 2, 3>(p, bf16, stream);
        return launch_tile<1, 4, 2, 2, 3>(p, bf16, stream);
    }
    const int64_t mean = p.R / p.E;
    // By the rows an expert has on average: the tile that holds most experts' rows with few rows to spare.  Several
    // layers' weights in turn, us with 256x256 / 160x128 / 128x256 / 128x128 / 64x128; 256 experts of 1024 x 2048, bf16:
    // 32 rows 116 / 101 / 102 / 98 / 96, 64 rows 144 / 138 / 136 / 126 / 137, 93 rows 161 / 173 / 159 / 154 / 187, 128 rows
    // 218 / 185 / 203 / 198 / 227, 156 rows 246 / 220 / 242 / 237 / 267, 187 rows 254 / 274 / 281 / 271 / 302; f32: 64 rows
    // 150 / 138 / 136 / 129 / 142, 128 rows 222 / 189 / 210 / 206 / 233, 187 rows 269 / 285 / 292 / 279 / 314; 128 of 1408 x
    // 2816, 125 rows 221 / 176 / 201 / 184 / 210; 128 of 2816 x 704, 62 rows 93 / 85 / 92 / 81 / 86, f32 97 / 91 / 96 / 87 /
    // 93; 64 of 1536 x 1536, 281 rows 131 / 105 / 121 / 114 / 134, 562 rows 201 / 187 / 208 / 201 / 241; 500 rows of 8 of
    // 4096 x 1024 57 / 45 / 55 / 46 / 55, of 256 of 1024 x 1024 306 / 331 / 337 / 327 / 407; 8 of 2048 x 2048, 2000 rows 125 /
    // 133 / 134 / 130 / 160.
    if (mean >= 110) {
        if (((mean > 160 && mean <= 256) || mean >= 1024) && wgs(256, 256) >= kFp8Cus)
            return launch_tile<2, 4, 8, 4, 2>(p, bf16, stream);
        if (wgs(160, 128) >= kFp8Cus) return launch_tile<2, 2, 5, 4, 2>(p, bf16, stream);
    } else if (mean >= 56 && wgs(128, 128) >= kFp8Cus) {
        return launch_tile<2, 2, 4, 4, 2>(p, bf16, stream);
    }
    // Weights streamed for few rows: small tiles, many loads in flight, unless K is soon over; up to 20 rows also where
    // there would be few large tiles.  Us with 32x64 in four buffers / in three / 64x128 in three / in two, bf16 (f32 within
    // 3%): 256 experts of 1024 x 2048, 2 tokens 10.5 / 11.7 / 13.8 / 16.6, 10 tokens 28 / 29 / 32 / 29, 256 84 / 84 / 86 / 90,
    // 512 95 / 94 / 91 / 93; 32 of 2048 x 4096, 100 tokens 54 / 57 / 61 / 64; 128 of 2816 x 704, 30 tokens 48 / 46 / 48 / 47,
    // 64 55 / 52 / 55 / 53, 211 60 / 57 / 57 / 54, 500 82 / 78 / 63 / 63; 256 of 2048 x 768, 64 65 / 58 / 61 / 59, 211 80 / 73
    // / 74 / 71; 64 of 3584 x 896, 100 39 / 37 / 38 / 40; 256 of 2048 x 512, 64 tokens 49 / 44 / 47 / 42, 211 61 / 54 / 56 / 51.
    if ((mean < 12 || (mean < 20 && wgs(64, 128) < 4 * kFp8Cus)) && p.KB >= 8)
        return launch_tile<1, 4, 2, 1, 4>(p, bf16, stream);
    if (mean < 16 && p.KB > 4 && p.KB < 8) return launch_tile<1, 4, 2, 1, 3>(p, bf16, stream);
    if (wgs(64, 128) >= kFp8Cus)
        return p.KB <= 4 ? launch_tile<1, 4, 4, 2, 2>(p, bf16, stream) : launch_tile<1, 4, 4, 2, 3>(p, bf16, stream);
    return launch_tile<1, 4, 2, 2, 3>(p, bf16, stream);
}

}  // namespace qmoe
