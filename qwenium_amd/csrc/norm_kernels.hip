// norm_kernels.hip -- the norms between two blocks with the gate, the residual
// scale and the residual add in one pass over the rows.
#include "qmoe_device.h"
#include "qmoe_internal.h"

namespace qmoe {

// ---------------------------------------------------------------------------
//   u  = y / sqrt(mean(y^2) + eps) * post_w        (post_w: a norm after the block)
//   u  = u * sigmoid(gate) | u * silu(gate)        (gate)
//   x' = x + scale * u                             (scale: one value or one per column)
//   h  = x' / sqrt(mean(x'^2) + eps) * w           (the next block's norm)
//   (q, q_scale) = h in e4m3, blocks of 128        (q)
// One workgroup per row, 8 columns a thread (a second 8 above 8192 columns), so
// that the row stays in registers between the loads and the stores: each operand
// is read once, and 16 neighbouring threads hold a block of 128 columns.  The sums
// of squares are f64 of the f32 squares (a thread's in turn, the tree over a wave's
// lanes, the waves in turn), as rms_norm's but for rows whose squares leave f32's range.
// h and q come from the f32 x', not from its rounding to the rows' type.  Bound by memory: 4096 x 2816 bf16 with both norms, gate and a
// scale per column (115 MB) 24.4 us, 4.7 TB/s (26.1 with its outputs through
// the caches, 28.0 with expf and a division too; inputs out of memory 29.3); f32 5.3 TB/s.
// ---------------------------------------------------------------------------
__device__ __forceinline__ double block_sum_f64(double v, double* s) {
    v = dpp_sum_f64<64>(v);
    if ((threadIdx.x & 63) == 63) s[threadIdx.x >> 6] = v;
    __syncthreads();
    double t = 0.0;
    for (int i = 0; i < (int)blockDim.x >> 6; ++i) t += s[i];
    return t;
}

// The row's r = 1 / sqrt(mean(v^2) + eps).  Where squares may leave f32 (the largest above 2^126, or the mean with eps below
// 2^-110, beside which a square's error below 2^-126, 2^-150, would count), v is scaled by a power of two and r is that
// of the scaled row: v r is as it was.
template <int NP>
__device__ __forceinline__ float norm_row(float (&v)[NP][8], int H, float eps, double* s_sum) {
    auto ssq = [&](double* sums) {
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < NP; ++i)
#pragma unroll
            for (int c = 0; c < 8; ++c) s += (double)(v[i][c] * v[i][c]);  // (columns past H are zeros)
        return block_sum_f64(s, sums);
    };
    float r = rms_scale_from_ssq(ssq(s_sum), H, eps);
    if (!(r >= 0x1p-63f && r <= 0x1p55f)) {
        const float by = r > 0x1p55f ? 0x1p100f : 0x1p-66f;
#pragma unroll
        for (int i = 0; i < NP; ++i)
#pragma unroll
            for (int c = 0; c < 8; ++c) v[i][c] *= by;
        r = rms_scale_from_ssq(ssq(s_sum + 16), H, eps * by * by);
    }
    return r;
}

template <bool BF16, bool WHOLE, int NP>
__global__ __launch_bounds__(1024) void k_residual_norm(ResidualNorm p) {
    __shared__ double s_sum[4][16];
    const uint64_t row = (uint64_t)blockIdx.x * p.H;
    const int H = p.H;
    float v[NP][8] = {}, u[NP][8] = {}, g[NP][8] = {};
    int c0[NP], n[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        c0[i] = 8 * ((int)threadIdx.x + i * (int)blockDim.x);
        n[i] = H - c0[i];  // columns from c0 on: none or some of the 8 may exist
        if (n[i] <= 0) continue;
        load8<BF16, WHOLE>(p.x, row + c0[i], n[i], v[i]);
        if (p.y) load8<BF16, WHOLE>(p.y, row + c0[i], n[i], u[i]);
        if (p.gate) load8<BF16, WHOLE>(p.gate, row + c0[i], n[i], g[i]);
    }
    if (p.y) {
        float post = 1.0f;
        if (p.post_w) post = norm_row(u, H, p.eps, s_sum[0]);
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            if (n[i] <= 0) continue;
            if (p.post_w) {
                float w[8];
                load8<false, WHOLE>(p.post_w, c0[i], n[i], w);
#pragma unroll
                for (int c = 0; c < 8; ++c) u[i][c] = u[i][c] * post * w[c];
            }
            if (p.gate) {
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    u[i][c] = sigmoid_product(u[i][c], g[i][c], p.gate_act == kGateSilu ? g[i][c] : 1.0f);
            }
            float sc[8];
            if (p.scale_v) {
                load8<false, WHOLE>(p.scale_v, c0[i], n[i], sc);
            } else {
#pragma unroll
                for (int c = 0; c < 8; ++c) sc[c] = p.scale;
            }
#pragma unroll
            for (int c = 0; c < 8; ++c) v[i][c] += sc[c] * u[i][c];
            store8<BF16, WHOLE>(p.x_out, row + c0[i], n[i], v[i], p.stream_out);
        }
    }
    float w[NP][8];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
#pragma unroll
        for (int c = 0; c < 8; ++c) w[i][c] = 1.0f;
        if (p.w && n[i] > 0) load8<false, WHOLE>(p.w, c0[i], n[i], w[i]);
    }
    const float r = norm_row(v, H, p.eps, s_sum[2]);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
#pragma unroll
        for (int c = 0; c < 8; ++c) v[i][c] = v[i][c] * r * w[i][c];
        if (n[i] > 0) store8<BF16, WHOLE>(p.h, row + c0[i], n[i], v[i], p.stream_out);
        if (p.q) {
            const float m = fp8_block_max(v[i]);
            uint32_t o[2];
            fp8_pack8(v[i], m, o);
            if (n[i] > 0) {
                store8_fp8(p.q + row + c0[i], n[i], o, p.stream_out);
                const int nb = (H + kFp8Block - 1) / kFp8Block;
                if ((threadIdx.x & 15) == 0) p.q_scale[(uint64_t)blockIdx.x * nb + c0[i] / kFp8Block] = m / kFp8Max;
            }
        }
    }
}

template <bool BF16, bool WHOLE>
static void launch_norm(const ResidualNorm& p, int n_tokens, hipStream_t stream) {
    const int pieces = (p.H + 7) / 8, np = pieces > 1024 ? 2 : 1;
    const dim3 grid(n_tokens), block((unsigned)(((pieces + np - 1) / np + 63) / 64 * 64));
    if (np == 2) hipLaunchKernelGGL((k_residual_norm<BF16, WHOLE, 2>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((k_residual_norm<BF16, WHOLE, 1>), grid, block, 0, stream, p);
}

hipError_t launch_residual_norm(ResidualNorm p, bool bf16, int n_tokens, hipStream_t stream) {
    if (n_tokens <= 0) return hipSuccess;
    if (p.H > 16384) return hipErrorInvalidValue;
    const bool whole = p.H % 8 == 0;
    // Rows of whole lines past the caches where they are more than an L2 holds and fewer than eight do (of two bytes a
    // column; 4096 x 2816 bf16 25.4 -> 24.2 us).  With the product that reads them next, us through / past: 2048 x 2048 bf16
    // 138 / 134, 4096 201 / 199, 2048 x 4096 99 / 97, 1500 x 2048 f32 129 / 126; beyond, 8192 x 2048 343 / 347, with a norm 38 / 39.
    const int64_t bytes = (int64_t)n_tokens * p.H * 2;
    p.stream_out = p.H % kFp8Block == 0 && bytes > kL2Bytes && bytes < 8 * kL2Bytes;
    if (bf16) { if (whole) launch_norm<true, true>(p, n_tokens, stream); else launch_norm<true, false>(p, n_tokens, stream); }
    else { if (whole) launch_norm<false, true>(p, n_tokens, stream); else launch_norm<false, false>(p, n_tokens, stream); }
    return hipGetLastError();
}

}  // namespace qmoe
