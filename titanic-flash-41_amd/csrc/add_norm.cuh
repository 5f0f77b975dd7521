// The boundary between two sublayers of a residual stream: the sublayer's output joins the residual, the sum is normalized and
// quantized for the next product, in one pass over the row.
//   r      = bf16(x + residual)                                       (residual == null: r = x)
//   normed = bf16((r * (1 / sqrt(sum(r^2) / cols + eps))) * weight)     sum in FP32 (of a scaled row where FP32 does not hold it), division
//                                                                       and root correctly rounded
//   codes / scales (zero block: scale byte 0) and codes_min / scales_min (amax floored at 1e-4): the MXFP8 flavours of the normalized row,
//   as ca_ffn_norm_quant has them
// The statistics are those of the BF16 residual that the next boundary reads, so that they do not depend on who forms them.
#pragma once
#include "common.cuh"

struct AddNormArgs {
    const uint16_t *x, *residual, *weight;
    uint16_t *residual_out, *normed;
    uint8_t *codes, *scales, *codes_min, *scales_min;
    long long x_stride, residual_stride, residual_out_stride;        // values
    int rows, cols, act_block;
    float eps;
};

// WAVES waves a row (1: four rows a workgroup; else one), PIECES 8-value pieces a lane.
template <int WAVES, int PIECES>
__global__ void __launch_bounds__(WAVES == 1 ? 256 : WAVES * 64) tf_add_norm_quant(const AddNormArgs p) {
    constexpr int LANES = WAVES * 64;
    __shared__ float s_wave[WAVES];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int row = WAVES == 1 ? blockIdx.x * 4 + wave : blockIdx.x;
    if (row >= p.rows) return;                             // a whole wave (WAVES 1: no barrier below) or nobody
    const int t = WAVES == 1 ? lane : threadIdx.x, per_row = p.cols >> 3, group_bits = p.act_block == 128 ? 4 : 2, group_lanes = 1 << group_bits;
    const u4v* x = reinterpret_cast<const u4v*>(p.x + (long long)row * p.x_stride);
    const u4v* res = reinterpret_cast<const u4v*>(p.residual + (long long)row * p.residual_stride);
    const u4v* weight = reinterpret_cast<const u4v*>(p.weight);
    u4v* res_out = reinterpret_cast<u4v*>(p.residual_out + (long long)row * p.residual_out_stride);
    // Everything the row reads is requested before anything waits: with the loads inside `q < per_row` every piece was a round trip of its own.
    u4v r[PIECES], b[PIECES], w[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) r[i] = x[min(i * LANES + t, per_row - 1)];
    if (p.residual != nullptr)
#pragma unroll
        for (int i = 0; i < PIECES; ++i) b[i] = res[min(i * LANES + t, per_row - 1)];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) w[i] = weight[min(i * LANES + t, per_row - 1)];
    if (p.residual != nullptr)
#pragma unroll
        for (int i = 0; i < PIECES; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                r[i][j] = tf_pack_bf16(__fadd_rn(tf_bf16_lo(r[i][j]), tf_bf16_lo(b[i][j])), __fadd_rn(tf_bf16_hi(r[i][j]), tf_bf16_hi(b[i][j])));
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int q = i * LANES + t;
        if (q >= per_row) r[i] = u4v{0, 0, 0, 0};
        else if (p.residual_out != nullptr) res_out[q] = r[i];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            ss = __fmaf_rn(tf_bf16_lo(r[i][j]), tf_bf16_lo(r[i][j]), ss);
            ss = __fmaf_rn(tf_bf16_hi(r[i][j]), tf_bf16_hi(r[i][j]), ss);
        }
    }
    auto row_sum = [&](float v) {
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) v = __fadd_rn(v, __shfl_xor(v, o));
        if constexpr (WAVES > 1) {
            if (lane == 0) s_wave[wave] = v;
            __syncthreads();
            v = s_wave[0];
#pragma unroll
            for (int i = 1; i < WAVES; ++i) v = __fadd_rn(v, s_wave[i]);
        }
        return v;
    };
    ss = row_sum(ss);
    const float mean = __fadd_rn(ss / (float)p.cols, p.eps);
    float inverse = 1.0f / __builtin_sqrtf(mean);
    // Squares of BF16 values reach 2^256 and 2^-266.  Where their sum passes FP32's range, or is so small that squares of the row vanished in it, the
    // row's statistics are formed again with the row scaled by a power of two: 2^-80 (its largest square is then 2^96) or 2^80 (the
    // sum was below 2^-83, so the largest is 2^77, the least 2^-106).  1 / root is as small as 2^-128 for large rows, a subnormal: 2^8 of it goes to the row.
    if (__builtin_expect(!(mean >= 0x1p-96f && mean < __builtin_inff()), 0)) {      // the whole row's lanes alike; NaN too, and comes out as NaN
        const bool small = mean < 1.f;
        const float scale = small ? 0x1p80f : 0x1p-80f, share = small ? 0x1p80f : 0x1p-8f;
        ss = 0.f;
#pragma unroll
        for (int i = 0; i < PIECES; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float lo = tf_bf16_lo(r[i][j]), hi = tf_bf16_hi(r[i][j]), a = __fmul_rn(lo, scale), b = __fmul_rn(hi, scale);
                ss = __fmaf_rn(a, a, ss);
                ss = __fmaf_rn(b, b, ss);
                r[i][j] = tf_pack_bf16(__fmul_rn(lo, share), __fmul_rn(hi, share));      // exact, or so small that its result is zero
            }
        if constexpr (WAVES > 1) __syncthreads();                                        // s_wave has been read
        ss = row_sum(ss);
        inverse = 1.0f / __builtin_sqrtf(__fadd_rn(ss / (float)p.cols, __fmul_rn(__fmul_rn(p.eps, scale), scale)));
        if (!small) inverse = __fmul_rn(inverse, 0x1p-72f);
    }
    const int groups = per_row >> group_bits;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int q = i * LANES + t;
        const bool on = q < per_row;                       // whole groups of lanes together: per_row is a multiple of group_lanes
        float v[8];
        u4v o;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            o[j] = tf_pack_bf16(__fmul_rn(__fmul_rn(tf_bf16_lo(r[i][j]), inverse), tf_bf16_lo(w[i][j])),
                                __fmul_rn(__fmul_rn(tf_bf16_hi(r[i][j]), inverse), tf_bf16_hi(w[i][j])));
#pragma unroll
        for (int j = 0; j < 4; ++j) { v[2 * j] = tf_bf16_lo(o[j]); v[2 * j + 1] = tf_bf16_hi(o[j]); }
        const float amax = tf_group_amax(v, group_lanes);
        if (!on) continue;
        const size_t at = (size_t)row * per_row + q;
        const size_t group = (size_t)row * groups + (q >> group_bits);
        if (p.normed != nullptr) reinterpret_cast<u4v*>(p.normed)[at] = o;
        if (p.codes != nullptr) {
            const Quant8 c = tf_quant8(v, amax, 0.f);
            reinterpret_cast<u2v*>(p.codes)[at] = u2v{c.lo, c.hi};
            if ((q & (group_lanes - 1)) == 0) p.scales[group] = (uint8_t)c.exponent;
        }
        if (p.codes_min != nullptr) {
            const Quant8 c = tf_quant8(v, amax, 1e-4f);
            reinterpret_cast<u2v*>(p.codes_min)[at] = u2v{c.lo, c.hi};
            if ((q & (group_lanes - 1)) == 0) p.scales_min[group] = (uint8_t)c.exponent;
        }
    }
}
// Up to two rows a CU the latency of the row's own loads, sums and exchange is the time, so a lane takes one piece (4 rows x 1,024: 2.7 us against 3.3
// of one wave with two pieces, x 4,096: 2.9 against 3.5 of four waves, x 8,192: 4.6 against 5.8; 512 rows x 4,096: 5.5 against 5.9).  Beyond, HBM
// is: fewer waves that meet at a barrier and more loads in flight a lane (2,048 rows x 4,096: 14.2 of eight waves against 13.1, 16,384 x 5,120: 144
// against 132 us = 5.7 TB/s of the 9 bytes a value that the row moves; 16,384 x 1,024: four waves 28, one 23.5; 16,384 x 4,096 with a wave a row
// 117 against 106).  The order of the sum of squares follows the variant.
inline void tf_launch_add_norm(const AddNormArgs& p, int cus, hipStream_t s) {
    const int quarter = (p.rows + 3) / 4;
    if (p.cols <= 512) tf_add_norm_quant<1, 1><<<quarter, 256, 0, s>>>(p);
    else if (p.rows <= 2 * cus) {
        if (p.cols <= 1024) tf_add_norm_quant<2, 1><<<p.rows, 128, 0, s>>>(p);
        else if (p.cols <= 2048) tf_add_norm_quant<4, 1><<<p.rows, 256, 0, s>>>(p);
        else if (p.cols <= 4096) tf_add_norm_quant<8, 1><<<p.rows, 512, 0, s>>>(p);
        else tf_add_norm_quant<16, 1><<<p.rows, 1024, 0, s>>>(p);
    } else {
        if (p.cols <= 1024) tf_add_norm_quant<1, 2><<<quarter, 256, 0, s>>>(p);
        else if (p.cols <= 2048) tf_add_norm_quant<4, 1><<<p.rows, 256, 0, s>>>(p);
        else if (p.cols <= 4096) tf_add_norm_quant<4, 2><<<p.rows, 256, 0, s>>>(p);
        else tf_add_norm_quant<4, 4><<<p.rows, 256, 0, s>>>(p);
    }
}
