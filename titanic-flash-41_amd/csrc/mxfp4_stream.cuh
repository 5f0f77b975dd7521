// Products with prepared MXFP4 weights for few rows: the weights are streamed once, straight into the matrix instruction.
//   y[m][n]  = bf16(sum over k of A[m][k] W[n][k])
//   gated:     h = bf16(g * logistic(g) * u), g = min(A Gate^T, limit), u = clamp(A Up^T, -limit, limit), and its codes
// A: rows of E4M3 codes with scales of 32 or 128 columns (MXFP8), or of E2M1 words with scales of 32 (MXFP4).  One
// v_mfma_scale_f32_16x16x128_f8f6f4 takes 16 weight rows (first operand) and 16 token rows over 128 columns; both formats
// are decoded and both scales applied in the matrix core, sums are FP32.
#pragma once
#include "mxfp4_codec.cuh"

struct MxArgs {
    const uint8_t *a, *a_scales;
    const u4v *w, *w2;                   // prepared words (gated: w = up, w2 = gate)
    const uint32_t *ws, *ws2;
    int rows, n, k;                      // n: output columns (gated: of the activation)
    int block_shift;                     // log2 of the columns an A scale spans: 5 or 7
    // product
    uint16_t* out;
    long long out_stride;
    int wide;                            // stores of 8 bytes (1) or of 16 too (2) to a row's multiples of four (eight) columns are aligned
    // gated product
    uint16_t* act;
    uint8_t *codes, *scales;
    int out_block, out_fp4;              // columns a scale of the codes spans; E2M1 instead of E4M3
    float limit;
};

// The byte of lane group g at k-step ks of a row's 16-byte pieces.  Columns past k (the last step of a k that is no multiple of
// 128) meet zero weights; the lane then reads its row's last piece again, so that nothing outside the row is touched and a
// NaN can enter the sum only from the row itself, whose result it is anyway.
template <bool FP4A>
__device__ __forceinline__ v8i tf_mx_row_fragment(const uint8_t* row, int ks, int g, int k) {
    if constexpr (FP4A) {
        const u4v a = *reinterpret_cast<const u4v*>(row + min(ks * 64 + g * 16, (k >> 1) - 16));
        return v8i{(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
    } else {
        const u4v a = *reinterpret_cast<const u4v*>(row + min(ks * 128 + g * 16, k - 16));
        const u4v b = *reinterpret_cast<const u4v*>(row + min(ks * 128 + 64 + g * 16, k - 16));
        return v8i{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
    }
}
template <bool FP4A, int Q>
__device__ __forceinline__ v4f tf_mx_product(const u4v& w, const v8i& a, const v4f& c, uint32_t scale_w, uint32_t scale_a) {
    const v8i wv = v8i{(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wv, a, c, 4, FP4A ? 4 : 0, Q, (int)scale_w, 0, (int)scale_a);
}
// The activation of one pair of sums.  Comparisons, not minima: a NaN stays one.
__device__ __forceinline__ float tf_mx_swiglu(float up, float gate, float limit) {
    const float g = gate > limit ? limit : gate;
    const float u = up > limit ? limit : up < -limit ? -limit : up;
    return __fmul_rn(__fmul_rn(g, tf_logistic_fast(g)), u);
}
// Eight consecutive columns of the activation (BF16) per lane: the BF16 copy, the codes and the block's scale byte.  All lanes of
// the wave call; `on`: the lane's columns exist.  Adjacent lanes hold adjacent columns, a block's lanes start at a multiple of their count.
__device__ __forceinline__ void tf_mx_store_activation(const MxArgs& p, const u4v& o, size_t row, int col, bool on) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v[2 * j] = tf_bf16_lo(o[j]);
        v[2 * j + 1] = tf_bf16_hi(o[j]);
    }
    if (p.act != nullptr && on) *reinterpret_cast<u4v*>(p.act + row * p.n + col) = o;
    if (p.codes == nullptr) return;
    if (p.out_fp4) {
        const uint32_t amax = tf_quad_max_bits(tf_amax_bits8(v)), e = tf_mxfp4_scale(amax);
        if (!on) return;
        *reinterpret_cast<uint32_t*>(p.codes + row * (p.n >> 1) + (col >> 1)) = tf_mxfp4_codes8(v, tf_mxfp4_inverse(amax, e));
        if ((col & 31) == 0) p.scales[row * (p.n >> 5) + (col >> 5)] = (uint8_t)e;
    } else {
        const float amax = tf_group_amax(v, p.out_block >> 3);
        if (!on) return;
        const Quant8 c = tf_quant8(v, amax, 0.f);
        *reinterpret_cast<u2v*>(p.codes + row * p.n + col) = u2v{c.lo, c.hi};
        if ((col & (p.out_block - 1)) == 0) p.scales[row * (p.n / p.out_block) + col / p.out_block] = (uint8_t)c.exponent;
    }
}

// A workgroup: NW column groups of CT 16-column tiles (gated: of both matrices) x MT 16-row tiles; its waves share out the column
// groups and, within one, the rounds of four k-steps (wave kw takes rounds kw, kw + KW, ..).  Partial sums meet in LDS and are
// added in the order of the waves.
template <bool FP4A, bool GATED, int CT, int MT, int NW>
__global__ void __launch_bounds__(NW == 1 ? 512 : 1024) tf_mx_stream(const MxArgs p) {
    constexpr int T = GATED ? 2 * CT : CT, COLS = NW * CT * 16;
    extern __shared__ __attribute__((aligned(16))) uint8_t s_dynamic[];
    v4f* s_part = reinterpret_cast<v4f*>(s_dynamic);                            // [wave][T][64]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int nw = wave % NW, kw = wave / NW, KW = waves / NW, g = lane >> 4, r16 = lane & 15;
    float* s_h = reinterpret_cast<float*>(s_part + waves * T * 64);              // gated: [16][COLS + 4]
    const int KS = (p.k + 127) >> 7, KQ = (p.k + 511) >> 9, tiles = (p.n + 15) >> 4;
    const int tile0 = (blockIdx.x * NW + nw) * CT, row0 = blockIdx.y * (16 * MT);
    const int a_pitch = FP4A ? p.k >> 1 : p.k, s_pitch = p.k >> p.block_shift;

    const u4v* w[T];
    const uint32_t* ws[T];
#pragma unroll
    for (int t = 0; t < T; ++t) {
        const bool second = GATED && t >= CT;
        const size_t tile = min(tile0 + (second ? t - CT : t), tiles - 1);       // past the last tile: its bytes again, never stored
        w[t] = (second ? p.w2 : p.w) + tile * KS * 64 + lane;
        ws[t] = (second ? p.ws2 : p.ws) + tile * KQ * 64 + lane;
    }
    const uint8_t *a[MT], *as[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const size_t row = min(row0 + 16 * m + r16, p.rows - 1);                  // past the last row: that row again, never stored
        a[m] = p.a + row * a_pitch;
        as[m] = p.a_scales + row * s_pitch;
    }
    v4f acc[MT][T];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int t = 0; t < T; ++t) acc[m][t] = v4f{0.f, 0.f, 0.f, 0.f};
    for (int kq = kw; kq < KQ; kq += KW) {
        uint32_t sw[T];
#pragma unroll
        for (int t = 0; t < T; ++t) sw[t] = ws[t][kq * 64];
        auto step = [&](auto q_constant) {
            constexpr int Q = decltype(q_constant)::value;
            const int ks = 4 * kq + Q;
            if (ks >= KS) return;
            u4v wv[T];
#pragma unroll
            for (int t = 0; t < T; ++t) wv[t] = w[t][ks * 64];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const v8i av = tf_mx_row_fragment<FP4A>(a[m], ks, g, p.k);
                const uint32_t sa = as[m][min((ks * 128 + g * 32) >> p.block_shift, s_pitch - 1)];
#pragma unroll
                for (int t = 0; t < T; ++t) acc[m][t] = tf_mx_product<FP4A, Q>(wv[t], av, acc[m][t], sw[t], sa);
            }
        };
        step(std::integral_constant<int, 0>{});
        step(std::integral_constant<int, 1>{});
        step(std::integral_constant<int, 2>{});
        step(std::integral_constant<int, 3>{});
    }
    // lane (g, r16) of acc[m][t]: columns 16 tile + 4 g .. + 3 of token row 16 m + r16
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        if (row0 + 16 * m >= p.rows) break;
        if (m > 0) __syncthreads();
#pragma unroll
        for (int t = 0; t < T; ++t) s_part[(wave * T + t) * 64 + lane] = acc[m][t];
        __syncthreads();
        auto total = [&](int t) {
            v4f s = s_part[(nw * T + t) * 64 + lane];
            for (int i = 1; i < KW; ++i) {
                const v4f v = s_part[((i * NW + nw) * T + t) * 64 + lane];
#pragma unroll
                for (int j = 0; j < 4; ++j) s[j] = __fadd_rn(s[j], v[j]);
            }
            return s;
        };
        const int row = row0 + 16 * m + r16;
        for (int c = kw; c < CT; c += KW) {
            if constexpr (GATED) {
                const v4f u = total(c), gt = total(CT + c);
                float* to = s_h + r16 * (COLS + 4) + (nw * CT + c) * 16 + 4 * g;
#pragma unroll
                for (int j = 0; j < 4; ++j) to[j] = tf_mx_swiglu(u[j], gt[j], p.limit);
            } else {
                const v4f s = total(c);
                const int col = (tile0 + c) * 16 + 4 * g;
                if (row < p.rows && col < p.n) {
                    uint16_t* to = p.out + (size_t)row * p.out_stride + col;
                    const u2v o = {tf_pack_bf16(s[0], s[1]), tf_pack_bf16(s[2], s[3])};
                    if (p.wide && col + 4 <= p.n) *reinterpret_cast<u2v*>(to) = o;
                    else
#pragma unroll
                        for (int j = 0; j < 4; ++j) if (col + j < p.n) to[j] = (uint16_t)(o[j >> 1] >> (16 * (j & 1)));
                }
            }
        }
        if constexpr (GATED) {
            __syncthreads();
            constexpr int PIECES = COLS / 8;
            for (int i = threadIdx.x; i < 16 * PIECES; i += blockDim.x) {
                const int r = i / PIECES, piece = i % PIECES, at = row0 + 16 * m + r, col = blockIdx.x * COLS + piece * 8;
                const float* from = s_h + r * (COLS + 4) + piece * 8;
                u4v h;
#pragma unroll
                for (int j = 0; j < 4; ++j) h[j] = tf_pack_bf16(from[2 * j], from[2 * j + 1]);
                tf_mx_store_activation(p, h, (size_t)at, col, at < p.rows && col < p.n);
            }
        }
    }
}
template <bool FP4A, bool GATED, int CT, int MT, int NW>
inline int tf_mx_stream_go(const MxArgs& p, int kw, hipStream_t s) {
    constexpr int T = GATED ? 2 * CT : CT, COLS = NW * CT * 16;
    const int waves = kw * NW;
    const size_t lds = (size_t)waves * T * 1024 + (GATED ? 16 * (COLS + 4) * 4 : 0);
    const dim3 grid((p.n + COLS - 1) / COLS, (p.rows + 16 * MT - 1) / (16 * MT));
    tf_mx_stream<FP4A, GATED, CT, MT, NW><<<grid, waves * 64, lds, s>>>(p);
    return (int)hipGetLastError();
}
template <bool FP4A, bool GATED, int CT, int NW>
inline int tf_mx_stream_rows(const MxArgs& p, int most, hipStream_t s) {
    const int rounds = (p.k + 511) / 512, kw = rounds < most ? rounds : most;
    if (p.rows <= 16) return tf_mx_stream_go<FP4A, GATED, CT, 1, NW>(p, kw, s);
    if (p.rows <= 32) return tf_mx_stream_go<FP4A, GATED, CT, 2, NW>(p, kw, s);
    return tf_mx_stream_go<FP4A, GATED, CT, 4, NW>(p, kw, s);
}
template <bool FP4A>
inline int tf_launch_mx_stream(const MxArgs& p, bool gated, hipStream_t s) {
    if (!gated) return tf_mx_stream_rows<FP4A, false, 2, 1>(p, 8, s);
    // a workgroup's columns hold whole blocks of the activation's codes
    if (p.out_block == 128) return tf_mx_stream_rows<FP4A, true, 2, 4>(p, 4, s);
    return tf_mx_stream_rows<FP4A, true, 2, 1>(p, 8, s);
}
