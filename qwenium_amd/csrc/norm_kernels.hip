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
// One workgroup per row; the row's x' stays in LDS as f32 between its two
// passes.  The sums of squares are f64 of the f32 squares.  h and q come from the
// f32 x', not from its rounding to the rows' type.
// ---------------------------------------------------------------------------
__device__ __forceinline__ double block_sum_f64(double v, double* s, int nw) {
    v = dpp_sum_f64<64>(v);
    __syncthreads();  // s is free again
    if ((threadIdx.x & 63) == 63) s[threadIdx.x >> 6] = v;
    __syncthreads();
    double t = 0.0;
    for (int i = 0; i < nw; ++i) t += s[i];
    return t;
}

template <bool BF16>
__global__ __launch_bounds__(256) void k_residual_norm(ResidualNorm p) {
    extern __shared__ float s_row[];
    __shared__ double s_sum[4];
    const uint64_t row = (uint64_t)blockIdx.x * p.H;
    const int H = p.H;
    auto at = [&](const void* m, int i) {
        return BF16 ? bf16_to_f32(((const uint16_t*)m)[row + i]) : ((const float*)m)[row + i];
    };
    auto put = [&](void* m, int i, float v) {
        if (BF16) ((uint16_t*)m)[row + i] = (uint16_t)f32_pack_bf16(v, 0.0f);
        else ((float*)m)[row + i] = v;
    };
    float post = 1.0f;
    if (p.y && p.post_w) {
        double s = 0.0;
        for (int i = threadIdx.x; i < H; i += 256) {
            const float v = at(p.y, i);
            s += (double)(v * v);
        }
        post = rms_scale_from_ssq(block_sum_f64(s, s_sum, 4), H, p.eps);
    }
    double s = 0.0;
    for (int i = threadIdx.x; i < H; i += 256) {
        float v = at(p.x, i);
        if (p.y) {
            float u = at(p.y, i);
            if (p.post_w) u = u * post * p.post_w[i];
            if (p.gate) {
                const float g = at(p.gate, i);
                u = u / (1.0f + expf(-g));
                if (p.gate_act == kGateSilu) u *= g;
            }
            v += (p.scale_v ? p.scale_v[i] : p.scale) * u;
            put(p.x_out, i, v);
        }
        s_row[i] = v;
        s += (double)(v * v);
    }
    const float r = rms_scale_from_ssq(block_sum_f64(s, s_sum, 4), H, p.eps);
    for (int i = threadIdx.x; i < H; i += 256) {
        float v = s_row[i] * r;
        if (p.w) v *= p.w[i];
        s_row[i] = v;
        put(p.h, i, v);
    }
    if (!p.q) return;
    __syncthreads();
    const int nb = (H + kFp8Block - 1) / kFp8Block;
    for (int b = threadIdx.x >> 4; b < nb; b += 16) {
        const int c0 = b * kFp8Block + 8 * ((int)threadIdx.x & 15);
        float v[8], inv;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c0 + i < H ? s_row[c0 + i] : 0.0f;
        const float m = fp8_block_max(v, inv);
        uint32_t o[2];
        fp8_pack8(v, inv, o);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c0 + i < H) p.q[row + c0 + i] = (uint8_t)(o[i >> 2] >> (8 * (i & 3)));
        if ((threadIdx.x & 15) == 0) p.q_scale[(uint64_t)blockIdx.x * nb + b] = m / kFp8Max;
    }
}

hipError_t launch_residual_norm(const ResidualNorm& p, bool bf16, int n_tokens, hipStream_t stream) {
    if (n_tokens <= 0) return hipSuccess;
    const size_t lds = (size_t)p.H * sizeof(float);
    if (bf16) hipLaunchKernelGGL(k_residual_norm<true>, dim3(n_tokens), dim3(256), lds, stream, p);
    else hipLaunchKernelGGL(k_residual_norm<false>, dim3(n_tokens), dim3(256), lds, stream, p);
    return hipGetLastError();
}

}  // namespace qmoe
