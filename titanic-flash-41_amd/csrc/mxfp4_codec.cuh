// Microscaled FP4 (OCP MXFP4): a block of 32 consecutive columns of a row is 32 E2M1 codes (low nibble = even column) and one
// UE8M0 scale byte e, value = code * 2^(e - 127).
//   e = clamp(floor(log2(amax)) - 2 + 127, 1, 247)          amax: the block's largest magnitude
//   code = the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6 to x * 2^(127 - e), ties to the even code, magnitudes past 6 saturate
// A block whose amax is zero or subnormal in FP32 has zero codes and e = 127; one that holds a NaN or an infinity has zero
// codes and e = 255, the scale format's NaN (every value of the block reads back as NaN).
#pragma once
#include "common.cuh"

typedef _Float16 tf_f16x2 __attribute__((ext_vector_type(2)));

#define TF_TYPE_BF16 0
#define TF_TYPE_FP16 1
#define TF_TYPE_FP32 2

// Eight consecutive values (16 bytes of BF16 / FP16, 32 of FP32) as FP32.
template <int TYPE>
__device__ __forceinline__ void tf_load8(const void* p, float (&v)[8]) {
    const u4v a = reinterpret_cast<const u4v*>(p)[0];
    if constexpr (TYPE == TF_TYPE_FP32) {
        const u4v b = reinterpret_cast<const u4v*>(p)[1];
#pragma unroll
        for (int j = 0; j < 4; ++j) { v[j] = __uint_as_float(a[j]); v[4 + j] = __uint_as_float(b[j]); }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (TYPE == TF_TYPE_BF16) { v[2 * j] = tf_bf16_lo(a[j]); v[2 * j + 1] = tf_bf16_hi(a[j]); }
            else { const uint32_t pair = a[j]; const tf_f16x2 h = __builtin_bit_cast(tf_f16x2, pair); v[2 * j] = (float)h[0]; v[2 * j + 1] = (float)h[1]; }
        }
    }
}
// Bits of the largest magnitude of the eight: as whole numbers, so that infinities and NaNs order above every finite value.
__device__ __forceinline__ uint32_t tf_amax_bits8(const float (&v)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
    return m;
}
// Maximum over the four lanes of a quad, in every lane.
__device__ __forceinline__ uint32_t tf_quad_max_bits(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xb1, 0xf, 0xf, true));       // quad_perm [1,0,3,2]
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4e, 0xf, 0xf, true));    // quad_perm [2,3,0,1]
}
__device__ __forceinline__ uint32_t tf_mxfp4_scale(uint32_t amax_bits) {
    const int e = (int)(amax_bits >> 23);              // floor(log2(amax)) + 127; 0: zero or subnormal, 255: infinity or NaN
    return e == 255 ? 255u : e == 0 ? 127u : (uint32_t)min(max(e - 2, 1), 247);
}
// 2^(127 - e), 0 where the block's codes are zero whatever its values.
__device__ __forceinline__ float tf_mxfp4_inverse(uint32_t amax_bits, uint32_t e) {
    return amax_bits >= 0x7f800000u || amax_bits < 0x00800000u ? 0.f : __uint_as_float((254u - e) << 23);
}
// Codes of eight values, the first in the lowest nibble.  The hardware conversion rounds to the nearest, ties to the even code,
// and saturates; its scale operand is 1 (the product with the power of two before it is exact).  0 * infinity and 0 * NaN are
// replaced by zeros: those blocks' codes are zero.
__device__ __forceinline__ uint32_t tf_mxfp4_codes8(const float (&v)[8], float inverse) {
    uint32_t w = 0;
    float s[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = inverse != 0.f ? __fmul_rn(v[j], inverse) : 0.f;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, s[0], s[1], 1.0f, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, s[2], s[3], 1.0f, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, s[4], s[5], 1.0f, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, s[6], s[7], 1.0f, 3);
    return w;
}
// 2^(e - 127) in FP32: exact for every byte (0 is the subnormal 2^-127), NaN for 255.
__device__ __forceinline__ float tf_e8m0(uint32_t e) {
    return e == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(e ? e << 23 : 0x00400000u);
}

// Row and place in the row of item q, q / per_row by its reciprocal (inverse = 2^32 / per_row rounded down, per_row > 1): the estimate is at
// most one short for q < 2^31.
__device__ __forceinline__ void tf_item_place(uint32_t q, uint32_t per_row, uint32_t inverse, uint32_t& row, uint32_t& at) {
    row = __umulhi(q, inverse);
    at = q - row * per_row;
    if (at >= per_row) { ++row; at -= per_row; }
}
// x [rows][cols] (row pitch `stride` bytes) -> words [rows][cols / 2], scales [rows][cols / 32].  One item of eight values a lane, so that four
// adjacent lanes hold a block.  HBM-bound byte work: 2 (4) bytes read, 17/32 written a value, 16,384 x 8,192 of BF16 in 58 us (5.9 TB/s), of FP32 in
// 105 (5.8); back in 65 and 114 (5.3).  Several items a thread in flight gain nothing at full occupancy: four of them 60, 114, 62 and
// 149 us, and 5.7 against 5.0 for 2,304 x 5,120 of BF16, whose workgroups are then few.
template <int TYPE>
__global__ void __launch_bounds__(256) tf_mxfp4_quant(const uint8_t* __restrict__ x, long long stride, uint32_t* __restrict__ words,
                                                      uint8_t* __restrict__ scales, uint32_t items, uint32_t per_row, uint32_t inverse) {
    constexpr int BYTES = TYPE == TF_TYPE_FP32 ? 32 : 16;
    const uint32_t q = blockIdx.x * 256 + threadIdx.x;
    if (q >= items) return;                                // (items is a multiple of four: the quads stay whole)
    uint32_t row, at;
    tf_item_place(q, per_row, inverse, row, at);
    float v[8];
    tf_load8<TYPE>(x + (long long)row * stride + (long long)at * BYTES, v);
    const uint32_t amax = tf_quad_max_bits(tf_amax_bits8(v)), e = tf_mxfp4_scale(amax);
    words[q] = tf_mxfp4_codes8(v, tf_mxfp4_inverse(amax, e));
    if ((q & 3) == 0) scales[q >> 2] = (uint8_t)e;
}
// The values of the codes, rounded once to the output's type (exact wherever it holds them).
template <int TYPE>
__global__ void __launch_bounds__(256) tf_mxfp4_dequant(const uint32_t* __restrict__ words, const uint8_t* __restrict__ scales, uint8_t* __restrict__ out,
                                                        long long stride, uint32_t items, uint32_t per_row, uint32_t inverse) {
    constexpr int BYTES = TYPE == TF_TYPE_FP32 ? 32 : 16;
    const uint32_t q = blockIdx.x * 256 + threadIdx.x;
    if (q >= items) return;
    const uint32_t w = words[q];
    const float s = tf_e8m0(scales[q >> 2]);
    uint32_t row, at;
    tf_item_place(q, per_row, inverse, row, at);
    float v[8];
#define TF_PAIR(i) { const tf_f32x2 t = __builtin_bit_cast(tf_f32x2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, i)); v[2 * i] = __fmul_rn(t[0], s); v[2 * i + 1] = __fmul_rn(t[1], s); }
    TF_PAIR(0) TF_PAIR(1) TF_PAIR(2) TF_PAIR(3)
#undef TF_PAIR
    u4v* to = reinterpret_cast<u4v*>(out + (long long)row * stride + (long long)at * BYTES);
    if constexpr (TYPE == TF_TYPE_FP32) {
        to[0] = u4v{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
        to[1] = u4v{__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])};
    } else {
        u4v o;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (TYPE == TF_TYPE_BF16) o[j] = tf_pack_bf16(v[2 * j], v[2 * j + 1]);
            else o[j] = __builtin_bit_cast(uint32_t, (tf_f16x2){(_Float16)v[2 * j], (_Float16)v[2 * j + 1]});
        }
        to[0] = o;
    }
}

// Canonical words [n][k / 2] and scales [n][k / 32] -> the order in which a wave's lanes load them for the matrix instruction, the
// layout of the layer's prepared experts, padded: words [ceil(n/16)][ceil(k/128)][lane 64][16 B], lane 16 g + r of tile (nt, ks) = row
// 16 nt + r, columns 128 ks + 32 g ..; scales [ceil(n/16)][ceil(k/512)][lane 64][4 B], byte q = the scale of row 16 nt + r, block
// 4 (4 kq + q) + g.  What lies past n or k is zero (a zero code with scale byte 0).
__global__ void __launch_bounds__(256) tf_mxfp4_prepare_words(const u4v* __restrict__ source, u4v* __restrict__ out, int n, int k, long long chunks) {
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= chunks) return;
    const int lane = (int)(i & 63), ksteps = (k + 127) / 128;
    const long long tile = i >> 6;
    const int ks = (int)(tile % ksteps), block = 4 * ks + (lane >> 4);
    const long long row = tile / ksteps * 16 + (lane & 15);
    out[i] = row < n && block < k / 32 ? source[row * (k / 32) + block] : u4v{0, 0, 0, 0};
}
__global__ void __launch_bounds__(256) tf_mxfp4_prepare_scales(const uint8_t* __restrict__ source, uint32_t* __restrict__ out, int n, int k, long long words) {
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= words) return;
    const int lane = (int)(i & 63), rounds = (k + 511) / 512;
    const long long tile = i >> 6;
    const int kq = (int)(tile % rounds);
    const long long row = tile / rounds * 16 + (lane & 15);
    uint32_t w = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int block = 4 * (4 * kq + q) + (lane >> 4);
        if (row < n && block < k / 32) w |= (uint32_t)source[row * (k / 32) + block] << (8 * q);
    }
    out[i] = w;
}
