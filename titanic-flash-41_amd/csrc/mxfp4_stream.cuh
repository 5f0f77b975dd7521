// Products with prepared MXFP4 weights for few rows: the weights are streamed once, straight into the matrix instruction.
//   y[m][n]  = bf16(sum over k of A[m][k] W[n][k])
//   gated:     h = bf16(g * logistic(g) * u), g = min(A Gate^T, limit), u = clamp(A Up^T, -limit, limit), and its codes
// A: rows of E4M3 codes with scales of 32 or 128 columns (MXFP8), or of E2M1 words with scales of 32 (MXFP4).  One
// v_mfma_scale_f32_16x16x128_f8f6f4 takes 16 weight rows (first operand) and 16 token rows over 128 columns; both formats
// are decoded and both scales applied in the matrix core, sums are FP32.
#pragma once
#include "mxfp4_choice.hpp"
#include "mxfp4_codec.cuh"
#include <type_traits>

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

template <bool FP4A, int Q>
__device__ __forceinline__ v4f tf_mx_product(const u4v& w, const v8i& a, const v4f& c, uint32_t scale_w, uint32_t scale_a) {
    const v8i wv = v8i{(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wv, a, c, 4, FP4A ? 4 : 0, Q, (int)scale_w, 0, (int)scale_a);
}
// The activation of one pair of sums.  (The minimum and maximum that keep a NaN.)
__device__ __forceinline__ float tf_mx_swiglu(float up, float gate, float limit) {
    const float g = __builtin_elementwise_minimum(gate, limit);
    const float u = __builtin_elementwise_maximum(__builtin_elementwise_minimum(up, limit), -limit);
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

// Units a batch: what 128 (16 waves) or 256 (8 waves) registers a lane and 160 KiB of LDS hold.
constexpr int tf_mx_units(bool gated) { return gated ? 1 : 2; }
// A workgroup: NW column groups of CT 16-column tiles (gated: of both matrices) x MT 16-row tiles; its waves share out the column
// groups and, within one, the units of two k-steps (wave kw takes units kw, kw + KW, ..), UNITS of them at a time, all of whose loads are
// in flight before the first product.  Partial sums meet in LDS and are added in the order of the waves.
//
// Token rows pass through LDS (a region a wave, so no barrier): the lanes that load a row's 128 bytes of a k-step are neighbours, eight rows
// (E2M1: sixteen) an instruction.  Loaded straight in the matrix instruction's order, sixteen neighbouring lanes want sixteen different
// rows, each 16-byte piece is a cache look-up of its own, and 16 rows of 4,096 columns cost a launch 3 us.  A row's scales come as one word a
// k-step, lane group g holding that of the batch's k-step g.
template <bool FP4A, bool GATED, int CT, int MT, int NW, int WAVES>
__global__ void __launch_bounds__(WAVES * 64) tf_mx_stream(const MxArgs p) {
    constexpr int T = GATED ? 2 * CT : CT, COLS = NW * CT * 16, UNITS = tf_mx_units(GATED);
    constexpr int ROWB = FP4A ? 64 : 128, LOADS = ROWB / 64, LANES_ROW = ROWB / 16, OWN = UNITS * 2 * MT * 16 * ROWB;
    extern __shared__ __attribute__((aligned(16))) uint8_t s_dynamic[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int nw = wave % NW, kw = wave / NW, KW = waves / NW, g = lane >> 4, r16 = lane & 15;
    uint8_t* s_a = s_dynamic + wave * OWN;                                       // [unit][k-step][MT][16 rows][ROWB], the wave's own
    v4f* s_part = reinterpret_cast<v4f*>(s_dynamic);                             // [wave][T][64]: behind the last product
    float* s_h = reinterpret_cast<float*>(s_part + waves * T * 64);              // gated: [16][COLS + 4]
    const int KS = (p.k + 127) >> 7, KQ = (p.k + 511) >> 9, KU = (KS + 1) >> 1, tiles = (p.n + 15) >> 4;
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
    // loads of token rows: lane l takes 16 bytes (l % LANES_ROW) of row l / LANES_ROW; in LDS a row's pieces are permuted by the row (banks)
    auto swizzle = [](int r) { return FP4A ? ((r >> 1) & 3) ^ (r >> 3) : (r & 7) ^ (r >> 3); };
    const uint8_t *a[MT][LOADS], *as[MT];
    const uint32_t a_col = (uint32_t)(lane % LANES_ROW) * 16;
    uint32_t to_lds[LOADS];
#pragma unroll
    for (int c = 0; c < LOADS; ++c) {
        const int r = c * (64 / LANES_ROW) + lane / LANES_ROW;
        to_lds[c] = (uint32_t)(r * ROWB + (((lane % LANES_ROW) ^ swizzle(r)) << 4));
#pragma unroll
        for (int m = 0; m < MT; ++m) a[m][c] = p.a + (size_t)min(row0 + 16 * m + r, p.rows - 1) * a_pitch;   // past the last row: that row again, never stored
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) as[m] = p.a_scales + (size_t)min(row0 + 16 * m + r16, p.rows - 1) * s_pitch;
    const uint32_t from_lds = (uint32_t)(r16 * ROWB + ((g ^ swizzle(r16)) << 4));
    const bool words = p.block_shift == 5 && p.k % 128 == 0 && ((size_t)p.a_scales & 3) == 0;
    v4f acc[MT][T];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int t = 0; t < T; ++t) acc[m][t] = v4f{0.f, 0.f, 0.f, 0.f};
    // U units from unit u on, KW apart, of two k-steps each (the last one of an odd k alone: `odd`)
    auto units = [&](auto count, auto steps, int u) {
        constexpr int U = decltype(count)::value, S = decltype(steps)::value;
        u4v wv[U][S][T], ar[U][S][MT][LOADS];
        uint32_t sw[U][T], sr[MT];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int unit = u + i * KW;
#pragma unroll
            for (int t = 0; t < T; ++t) sw[i][t] = ws[t][(unit >> 1) * 64];
#pragma unroll
            for (int q = 0; q < S; ++q) {
                const int ks = 2 * unit + q;
#pragma unroll
                for (int t = 0; t < T; ++t) wv[i][q][t] = w[t][ks * 64];
                // Columns past k (the last step of a k that is no multiple of 128) meet zero weights; the lane then reads its row's last piece
                // again, so that nothing outside the row is touched and a NaN can enter the sum only from the row itself.
                const uint32_t at = min((uint32_t)ks * ROWB + a_col, (uint32_t)a_pitch - 16);
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int c = 0; c < LOADS; ++c) ar[i][q][m][c] = *reinterpret_cast<const u4v*>(a[m][c] + at);
            }
        }
        const int mine = min(2 * (u + (U == 2 ? (g >> 1) * KW : 0)) + (g & 1), KS - 1);      // the k-step whose scales this lane group loads
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            if (words) sr[m] = *reinterpret_cast<const uint32_t*>(as[m] + mine * 4);
            else {
                sr[m] = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) sr[m] |= (uint32_t)as[m][min((mine * 128 + j * 32) >> p.block_shift, s_pitch - 1)] << (8 * j);
            }
        }
        asm volatile("" ::: "memory");               // the previous batch's reads of the wave's LDS region come before these writes, theirs after them
#pragma unroll
        for (int i = 0; i < U; ++i)
#pragma unroll
            for (int q = 0; q < S; ++q)
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int c = 0; c < LOADS; ++c) *reinterpret_cast<u4v*>(s_a + ((i * 2 + q) * MT + m) * (16 * ROWB) + to_lds[c]) = ar[i][q][m][c];
        asm volatile("" ::: "memory");
        auto fragment = [&](int i, int q, int m) {
            const uint8_t* at = s_a + ((i * 2 + q) * MT + m) * (16 * ROWB);
            const u4v lo = *reinterpret_cast<const u4v*>(at + from_lds);
            if constexpr (FP4A) return v8i{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], 0, 0, 0, 0};
            else {
                const u4v hi = *reinterpret_cast<const u4v*>(at + (from_lds ^ 64));
                return v8i{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
            }
        };
        auto scale = [&](int i, int q, int m) { return (uint32_t)__shfl((int)sr[m], (i * 2 + q) * 16 + r16) >> (8 * g); };
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int shift = ((u + i * KW) & 1) * 16;                           // the unit's two bytes of its round's four
            uint32_t sh[T];
#pragma unroll
            for (int t = 0; t < T; ++t) sh[t] = sw[i][t] >> shift;
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const v8i av = fragment(i, 0, m);
                const uint32_t sa = scale(i, 0, m);
#pragma unroll
                for (int t = 0; t < T; ++t) acc[m][t] = tf_mx_product<FP4A, 0>(wv[i][0][t], av, acc[m][t], sh[t], sa);
            }
            if constexpr (S == 2)
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const v8i av = fragment(i, 1, m);
                    const uint32_t sa = scale(i, 1, m);
#pragma unroll
                    for (int t = 0; t < T; ++t) acc[m][t] = tf_mx_product<FP4A, 1>(wv[i][1][t], av, acc[m][t], sh[t], sa);
                }
        }
    };
    const std::integral_constant<int, 1> one;
    const std::integral_constant<int, 2> two;
    const int whole = KS >> 1;                                                   // units of two k-steps
    int u = kw;
    if constexpr (UNITS == 2)
        for (; u + KW < whole; u += 2 * KW) units(two, two, u);
    for (; u < whole; u += KW) units(one, two, u);
    if (u < KU) units(one, one, u);
    __syncthreads();                                                             // the regions of the rows become those of the sums
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
            for (int i = threadIdx.x; i < 16 * PIECES; i += blockDim.x) {        // (16 columns: half a wave, no codes)
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
template <bool FP4A, bool GATED, int CT, int MT, int NW, int WAVES>
inline int tf_mx_stream_go(const MxArgs& p, hipStream_t s) {
    constexpr int T = GATED ? 2 * CT : CT, COLS = NW * CT * 16;
    const int units = ((p.k + 127) / 128 + 1) / 2, most = WAVES / NW, waves = (units < most ? units : most) * NW;
    constexpr int UNITS = tf_mx_units(GATED), OWN = UNITS * 2 * MT * 16 * (FP4A ? 64 : 128);
    const size_t sums = (size_t)waves * T * 1024 + (GATED ? 16 * (COLS + 4) * 4 : 0), rows = (size_t)waves * OWN, lds = sums > rows ? sums : rows;
    const dim3 grid((p.n + COLS - 1) / COLS, (p.rows + 16 * MT - 1) / (16 * MT));
    tf_mx_stream<FP4A, GATED, CT, MT, NW, WAVES><<<grid, waves * 64, lds, s>>>(p);
    return (int)hipGetLastError();
}
// Codes of an activation that is in memory: 8 columns a lane.
__global__ void __launch_bounds__(256) tf_mx_codes(MxArgs p, uint32_t items) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x, per_row = (uint32_t)p.n >> 3;
    const bool on = i < items;
    const uint32_t at = on ? i : 0, row = at / per_row, piece = at - row * per_row;
    const u4v h = reinterpret_cast<const u4v*>(p.act)[at];
    p.act = nullptr;
    tf_mx_store_activation(p, h, row, (int)piece * 8, on);
}
inline int tf_launch_mx_codes(const MxArgs& p, hipStream_t s) {
    const uint32_t items = (uint32_t)p.rows * ((uint32_t)p.n >> 3);
    tf_mx_codes<<<(items + 255) / 256, 256, 0, s>>>(p, items);
    return (int)hipGetLastError();
}
template <bool FP4A, bool GATED>
inline int tf_mx_stream_launch(const MxArgs& p, int kernel, hipStream_t s) {
    if constexpr (GATED) {
        if (kernel == MX_FEW_128) return tf_mx_stream_go<FP4A, true, 2, 1, 4, 16>(p, s);
        return kernel == MX_FEW_32 ? tf_mx_stream_go<FP4A, true, 2, 1, 1, 16>(p, s) : tf_mx_stream_go<FP4A, true, 1, 1, 1, 16>(p, s);
    } else {
        if (p.rows <= 16) return kernel == MX_FEW_32 ? tf_mx_stream_go<FP4A, false, 2, 1, 1, 16>(p, s) : tf_mx_stream_go<FP4A, false, 1, 1, 1, 16>(p, s);
        return kernel == MX_FEW_32 ? tf_mx_stream_go<FP4A, false, 2, 2, 1, 8>(p, s) : tf_mx_stream_go<FP4A, false, 1, 2, 1, 8>(p, s);
    }
}
