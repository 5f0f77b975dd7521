// Products with prepared MXFP4 weights for many rows: tiles of 256 rows x 256 weight rows on the matrix cores.
//
// A workgroup of WM x WN waves (one a SIMD); a wave holds 16 FM token rows x 16 FT weight rows in 4 FM FT accumulator registers a lane.
// A k-step is 128 columns: FM FT instructions of 16 x 16 x 128 a wave.  Both operands come into LDS by global_load_lds in a ring of NS
// stages, requested NS k-steps ahead.  In k-step s the wave multiplies from registers (one set), reads k-step s + 1 from LDS into
// the other set between its products, and requests k-step s + NS into the stage that k-step s lay in; one barrier a k-step, at its
// top: behind it stage s + 1 is whole (every wave has waited for its share) and stage s is free (every wave's reads of it, made
// during k-step s - 1, have returned).  So neither LDS nor memory latency lies between the products.
//
// The requests are inline assembly that the compiler's wait insertion does not know; the kernel counts them (they complete in
// order): a wait lets the requests of the NS - 2 younger stages stay in flight.
//
// Token rows in LDS: row-major, a row's 16-byte pieces (4 of E2M1, 8 of E4M3) permuted by a function of the row, so that the lanes
// that copy a row read one contiguous piece of memory and the sixteen rows of a fragment fall into different banks.  Weights: as
// prepared, 1 KiB a 16-row tile and k-step in fragment order.  Scales come once a round of four k-steps, a byte of a register a k-step.
#pragma once
#include "mxfp4_stream.cuh"

// Lane l of the wave copies 16 (4) bytes from global address base + offset to LDS byte address lds_base + 16 l (4 l).
__device__ __forceinline__ void tf_mx_dma16(const uint8_t* base, uint32_t offset, uint32_t lds_base) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "s"(lds_base) : "memory", "m0");
}
__device__ __forceinline__ void tf_mx_dma4(const uint8_t* base, uint32_t offset, uint32_t lds_base) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(offset), "s"(base), "s"(lds_base) : "memory", "m0");
}
template <int N>
__device__ __forceinline__ void tf_mx_wait() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void tf_mx_barrier() {                  // LDS accesses done, then everyone's
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ uint32_t tf_mx_lds(const void* p) { return (uint32_t)(size_t)(const __attribute__((address_space(3))) uint8_t*)p; }
template <bool FP4A> struct MxFragment { typedef v8i type; };
template <> struct MxFragment<true> { typedef u4v type; };
// acc += weights x tokens, the sums held in place in the accumulator registers (256 of them leave the ordinary ones to the operands).
// Lane (g, r) of the result: weight rows 4 g .. 4 g + 3 of the tile for token row r.  Read only behind tf_mx_settle().
template <int SW, int ST>
__device__ __forceinline__ void tf_mx_mfma(v4f& acc, const u4v& w, const v8i& a, uint32_t sw, uint32_t sa) {
    asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%5,%6,0] op_sel_hi:[%7,%8,0] cbsz:4"
                 : "+a"(acc) : "v"(w), "v"(a), "v"(sw), "v"(sa), "n"(SW & 1), "n"(ST & 1), "n"(SW >> 1), "n"(ST >> 1));
}
template <int SW, int ST>
__device__ __forceinline__ void tf_mx_mfma(v4f& acc, const u4v& w, const u4v& a, uint32_t sw, uint32_t sa) {
    asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%5,%6,0] op_sel_hi:[%7,%8,0] cbsz:4 blgp:4"
                 : "+a"(acc) : "v"(w), "v"(a), "v"(sw), "v"(sa), "n"(SW & 1), "n"(ST & 1), "n"(SW >> 1), "n"(ST >> 1));
}
// The last results have reached the registers (the longest product takes 8 passes of 4 cycles), and the compiler reads none of these before.
template <int FM, int FT>
__device__ __forceinline__ void tf_mx_settle(v4f (&acc)[FM][FT]) {
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
    for (int f = 0; f < FM; ++f)
#pragma unroll
        for (int t = 0; t < FT; t += 4) asm volatile("" : "+a"(acc[f][t]), "+a"(acc[f][t + 1]), "+a"(acc[f][t + 2]), "+a"(acc[f][t + 3]));
}

// How a row's scales reach the lanes (all end as one register a fragment and round, byte q = k-step q of the round):
enum { MX_SCALES_32 = 0,      // blocks of 32, k a multiple of 512: 16 bytes a row and round, copied by the memory system
       MX_SCALES_128 = 1,     // blocks of 128, k a multiple of 512: 4 bytes a row and round, likewise
       MX_SCALES_ANY = 2 };   // any k: a thread reads its row's bytes one by one a round ahead and writes them to LDS

// What the k-steps of the last round past the end of k multiply by: zero codes (a round is four k-steps whatever k is; the loop body then
// has no branch, which its 256 accumulators would not survive in registers).
static __device__ const u4v tf_mx_zeros[64] = {};

template <bool FP4A, bool GATED, int SC, int FM, int FT, int WM, int WN, int NS>
__global__ void __launch_bounds__(WM * WN * 64, 1) tf_mx_gemm(const MxArgs p, int tiles_m, int tiles_n) {
    constexpr int WAVES = WM * WN, BM = 16 * FM * WM, TILES = FT * WN, ROWB = FP4A ? 64 : 128;
    constexpr int A_STAGE = BM * ROWB, B_STAGE = TILES * 1024, STAGE = A_STAGE + B_STAGE;
    constexpr int NA = A_STAGE / 1024 / WAVES, NB = TILES / WAVES, DATA = NA + NB, MORE = SC == MX_SCALES_ANY ? 1 : 2;
    constexpr int COLS = (GATED ? TILES / 2 : TILES) * 16, LANES_ROW = ROWB / 16, ROWS_REQ = 64 / LANES_ROW;
    static_assert(NA * WAVES * 1024 == A_STAGE && NB * WAVES == TILES && TILES == 4 * WAVES && BM <= WAVES * 64 && (SC != MX_SCALES_ANY || BM == WAVES * 64), "whole requests a wave");
    typedef typename MxFragment<FP4A>::type Fragment;
    __shared__ __attribute__((aligned(1024))) uint8_t s_ring[NS * STAGE];
    __shared__ __attribute__((aligned(1024))) uint32_t s_wsc[TILES * 64];
    __shared__ __attribute__((aligned(1024))) uint32_t s_asc[SC == MX_SCALES_128 ? BM : BM * 4];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN, g = lane >> 4, r16 = lane & 15;
    const int KS = (p.k + 127) >> 7, KQ = (p.k + 511) >> 9, n_tiles = (p.n + 15) >> 4;
    const int a_pitch = FP4A ? p.k >> 1 : p.k, s_pitch = p.k >> p.block_shift;

    // Workgroup b runs on XCD b % 8.  An XCD takes a contiguous run of the tiles, eight row tiles side by side and column after column, so that the
    // tiles at work on it at once share their rows and weights in its L2.
    const int total = tiles_m * tiles_n, chunk = (total + 7) >> 3;
    const int id = (blockIdx.x & 7) * chunk + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= chunk || id >= total) return;
    const int band = id / (8 * tiles_n), in_band = id - band * 8 * tiles_n, band_m = min(8, tiles_m - band * 8);
    const int tile_m = band * 8 + in_band % band_m, tile_n = in_band / band_m;
    const int row0 = tile_m * BM, rows = min(BM, p.rows - row0);

    // ---- requests ----------------------------------------------------------------------------------------------------
    const uint32_t lds_ring = tf_mx_lds(s_ring), lds_wsc = tf_mx_lds(s_wsc), lds_asc = tf_mx_lds(s_asc);
    const uint8_t* a_base = p.a + (size_t)row0 * a_pitch;
    uint32_t a_row[NA], a_col[NA];
#pragma unroll
    for (int c = 0; c < NA; ++c) {
        const int row = (wave * NA + c) * ROWS_REQ + lane / LANES_ROW, r = row & 15;
        const int swz = FP4A ? ((r >> 1) & 3) ^ (r >> 3) : (r & 7) ^ (r >> 3);
        a_row[c] = (uint32_t)min(row, rows - 1) * (uint32_t)a_pitch;        // past the last row: that row again, never stored
        a_col[c] = (uint32_t)((lane % LANES_ROW) ^ swz) * 16;
    }
    // weight tile T of the workgroup (gated: a wave's FT tiles are FT / 2 of `up`, then the same columns' of `gate`)
    auto weight_tile = [&](int T, bool& second) {
        const int w = T / FT, t = T - w * FT;
        second = GATED && t >= FT / 2;
        const int tile = GATED ? tile_n * (TILES / 2) + w * (FT / 2) + (second ? t - FT / 2 : t) : tile_n * TILES + T;
        return min(tile, n_tiles - 1);                                       // past the last tile: that tile again, never stored
    };
    const uint8_t* b_base[NB];
#pragma unroll
    for (int c = 0; c < NB; ++c) {
        bool second;
        const int tile = weight_tile(wave * NB + c, second);
        b_base[c] = reinterpret_cast<const uint8_t*>(second ? p.w2 : p.w) + (size_t)tile * KS * 1024;
    }
    // weight scales: a wave requests four tiles' 256 bytes of the round at once, 16 lanes a tile
    const uint8_t* wsc_base;
    {
        bool second;
        const int tile = weight_tile(wave * 4 + (lane >> 4), second);
        wsc_base = reinterpret_cast<const uint8_t*>(second ? p.ws2 : p.ws) + (size_t)tile * KQ * 256 + (lane & 15) * 16;
    }
    const uint8_t* asc_row = p.a_scales + (size_t)(row0 + min(tid & (BM - 1), rows - 1)) * s_pitch;
    const uint8_t* zeros = reinterpret_cast<const uint8_t*>(tf_mx_zeros);
    const uint32_t lane16 = lane * 16;
    auto issue = [&](int op, int ks, int stage) {                            // request `op` of k-step ks into ring stage `stage`
        if (op < NA) tf_mx_dma16(a_base, a_row[op] + min((uint32_t)ks * ROWB + a_col[op], (uint32_t)a_pitch - 16), lds_ring + stage * STAGE + (wave * NA + op) * 1024);
        else tf_mx_dma16(ks < KS ? b_base[op - NA] + (size_t)ks * 1024 : zeros, lane16, lds_ring + stage * STAGE + A_STAGE + (wave * NB + op - NA) * 1024);
    };
    auto copy16 = [&](const uint8_t* from, uint32_t lds) {                   // a lane's own 64-bit address
        asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(lds) : "memory", "m0");
    };
    auto copy4 = [&](const uint8_t* from, uint32_t lds) {
        asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(from), "s"(lds) : "memory", "m0");
    };
    const int asc_wave = wave & (BM / 64 - 1);                               // waves past the tile's rows repeat the first ones' request
    auto issue_scales = [&](int kq) {                                        // the MORE requests of a round (kq clamped: the count stays)
        kq = min(kq, KQ - 1);
        copy16(wsc_base + (size_t)kq * 256, lds_wsc + wave * 1024);
        if constexpr (SC == MX_SCALES_32) copy16(asc_row + kq * 16, lds_asc + asc_wave * 1024);
        if constexpr (SC == MX_SCALES_128) copy4(asc_row + kq * 4, lds_asc + asc_wave * 256);
    };
    uint32_t any[16];
    auto read_scales = [&](int kq) {                                         // MX_SCALES_ANY: this thread's row, one byte a block of 32
#pragma unroll
        for (int j = 0; j < 16; ++j) any[j] = asc_row[min((kq * 512 + j * 32) >> p.block_shift, s_pitch - 1)];
    };
    auto write_scales = [&]() {
        u4v w;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = any[4 * j] | (any[4 * j + 1] << 8) | (any[4 * j + 2] << 16) | (any[4 * j + 3] << 24);
        *reinterpret_cast<u4v*>(s_asc + tid * 4) = w;
    };

    // ---- fragments ---------------------------------------------------------------------------------------------------
    const int swz = FP4A ? ((r16 >> 1) & 3) ^ (r16 >> 3) : (r16 & 7) ^ (r16 >> 3);
    const int a_at = (wm * 16 * FM + r16) * ROWB + ((g ^ swz) << 4), b_at = A_STAGE + wn * FT * 1024 + lane16;
    v4f acc[FM][FT];
#pragma unroll
    for (int f = 0; f < FM; ++f)
#pragma unroll
        for (int t = 0; t < FT; ++t) acc[f][t] = v4f{0.f, 0.f, 0.f, 0.f};
    Fragment av[2][FM];
    u4v wv[2][FT];
    uint32_t sa[2][FM], sw[2][FT];
    auto read_a = [&](Fragment& to, int f, int stage) {
        const uint8_t* at = s_ring + stage * STAGE + f * 16 * ROWB;
        if constexpr (FP4A) to = *reinterpret_cast<const u4v*>(at + a_at);
        else {
            const u4v l = *reinterpret_cast<const u4v*>(at + a_at), h = *reinterpret_cast<const u4v*>(at + (a_at ^ 64));
            to = v8i{(int)l[0], (int)l[1], (int)l[2], (int)l[3], (int)h[0], (int)h[1], (int)h[2], (int)h[3]};
        }
    };
    auto read_w = [&](u4v& to, int t, int stage) { to = *reinterpret_cast<const u4v*>(s_ring + stage * STAGE + b_at + t * 1024); };
    auto read_sa = [&](uint32_t& to, int f) {
        const int row = wm * 16 * FM + 16 * f + r16;
        if constexpr (SC == MX_SCALES_128) to = s_asc[row];
        else {                                                                // byte g of each k-step's word
            const u4v w = *reinterpret_cast<const u4v*>(s_asc + row * 4);
            const uint32_t pick = (uint32_t)g | ((uint32_t)(4 + g) << 8);     // bytes g of the second and the first operand
            const uint32_t lo = __builtin_amdgcn_perm(w[1], w[0], pick), hi = __builtin_amdgcn_perm(w[3], w[2], pick);
            to = (lo & 0xffffu) | (hi << 16);
        }
    };
    auto read_sw = [&](uint32_t& to, int t) { to = s_wsc[(wn * FT + t) * 64 + lane]; };

    // ---- the first k-steps ---------------------------------------------------------------------------------------------
    if constexpr (SC == MX_SCALES_ANY) { read_scales(0); write_scales(); }
    issue_scales(0);
#pragma unroll
    for (int d = 0; d < NS; ++d)
#pragma unroll
        for (int op = 0; op < DATA; ++op) issue(op, d, d);
    tf_mx_wait<(NS - 1) * DATA>();
    tf_mx_barrier();
#pragma unroll
    for (int t = 0; t < FT; ++t) { read_w(wv[0][t], t, 0); read_sw(sw[0][t], t); }
#pragma unroll
    for (int f = 0; f < FM; ++f) { read_a(av[0][f], f, 0); read_sa(sa[0][f], f); }

    int stage = 0;                                                           // of k-step ks
    // requests that may be in flight at the top of k-step Q of a round: those of the NS - 2 k-steps before it
    auto behind = [](int q) constexpr {
        int n = 0;
        for (int j = 1; j < NS - 1; ++j) n += DATA + (((q - j) & 3) == 0 ? MORE : 0);
        return n;
    };
    auto k_step = [&](auto q_constant, int ks) {
        constexpr int Q = decltype(q_constant)::value, X = Q & 1, Y = X ^ 1;
        const int next = NS == 4 ? (Q + 1) & 3 : (stage + 1 == NS ? 0 : stage + 1), now = NS == 4 ? Q : stage;
        tf_mx_wait<behind(Q)>();
        tf_mx_barrier();
        if constexpr (Q == 0) {
            issue_scales((ks >> 2) + 1);
            if constexpr (SC == MX_SCALES_ANY) read_scales(min((ks >> 2) + 1, KQ - 1));
        }
        if constexpr (Q == 2 && SC == MX_SCALES_ANY) write_scales();
        const int ahead = min(ks + NS, 4 * KQ - 1);                          // behind the last: that one again, never read
#pragma unroll
        for (int f = 0; f < FM; ++f) {
            // fragment f's products, beside them what the next k-step needs from LDS and a share of the requests
            read_a(av[Y][f], f, next);
#pragma unroll
            for (int t = f * FT / FM; t < (f + 1) * FT / FM; ++t) read_w(wv[Y][t], t, next);
            if constexpr (Q == 3) {
                read_sa(sa[1][f], f);
#pragma unroll
                for (int t = f * FT / FM; t < (f + 1) * FT / FM; ++t) read_sw(sw[1][t], t);
            }
#pragma unroll
            for (int t = 0; t < FT; ++t) tf_mx_mfma<Q, Q>(acc[f][t], wv[X][t], av[X][f], sw[0][t], sa[0][f]);
#pragma unroll
            for (int op = f * DATA / FM; op < (f + 1) * DATA / FM; ++op) issue(op, ahead, now);
            __builtin_amdgcn_sched_barrier(0);
        }
        stage = next;
    };
    for (int kq = 0; kq < KQ; ++kq) {
        k_step(std::integral_constant<int, 0>{}, 4 * kq);
        k_step(std::integral_constant<int, 1>{}, 4 * kq + 1);
        k_step(std::integral_constant<int, 2>{}, 4 * kq + 2);
        k_step(std::integral_constant<int, 3>{}, 4 * kq + 3);
#pragma unroll
        for (int f = 0; f < FM; ++f) sa[0][f] = sa[1][f];
#pragma unroll
        for (int t = 0; t < FT; ++t) sw[0][t] = sw[1][t];
    }
    tf_mx_wait<0>();                                                         // nothing writes LDS any more
    tf_mx_settle(acc);

    // ---- results: lane (g, r16) of acc[f][t] holds columns 4 g .. 4 g + 3 of tile t for token row 16 f + r16 of the wave -----------
    const int first_row = wm * 16 * FM + r16;
    if constexpr (!GATED) {
#pragma unroll
        for (int f = 0; f < FM; ++f) {
            const int row = first_row + 16 * f;
            __builtin_amdgcn_sched_barrier(0);
            if (row < rows) {
                uint16_t* to = p.out + (size_t)(row0 + row) * p.out_stride;
#pragma unroll
                for (int t = 0; t < FT; ++t) {
                    const int col = tile_n * COLS + (wn * FT + t) * 16 + 4 * g;
                    const u2v o = {tf_pack_bf16(acc[f][t][0], acc[f][t][1]), tf_pack_bf16(acc[f][t][2], acc[f][t][3])};
                    if (p.wide && col + 4 <= p.n) *reinterpret_cast<u2v*>(to + col) = o;
                    else
#pragma unroll
                        for (int j = 0; j < 4; ++j) if (col + j < p.n) to[col + j] = (uint16_t)(o[j >> 1] >> (16 * (j & 1)));
                }
            }
        }
    } else {
        constexpr int HT = FT / 2;                                           // activation tiles of the wave
        static_assert(HT % 2 == 0, "whole blocks of 32 columns a wave");
        float* s_max = reinterpret_cast<float*>(s_ring);                     // [WN][BM]: row maxima of the waves' columns (blocks of 128)
        tf_mx_barrier();                                                     // every wave has read its last stage
        u2v h[FM][HT];
        float amax[FM][HT / 2];
#pragma unroll
        for (int f = 0; f < FM; ++f) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int t = 0; t < HT; ++t) {
                float v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = tf_mx_swiglu(acc[f][t][i], acc[f][HT + t][i], p.limit);
                h[f][t] = u2v{tf_pack_bf16(v[0], v[1]), tf_pack_bf16(v[2], v[3])};
            }
#pragma unroll
            for (int b = 0; b < HT / 2; ++b) {
                // bits of the magnitudes: a NaN orders above everything (E2M1); the E4M3 scale leaves NaNs out, as the row quantizers do
                uint32_t m = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t w = h[f][2 * b + (j >> 1)][j & 1], lo = w & 0x7fffu, hi = (w >> 16) & 0x7fffu;
                    m = max(m, p.out_fp4 || lo <= 0x7f80u ? lo : 0u);
                    m = max(m, p.out_fp4 || hi <= 0x7f80u ? hi : 0u);
                }
                m = max(m, (uint32_t)__shfl_xor((int)m, 16));
                m = max(m, (uint32_t)__shfl_xor((int)m, 32));
                amax[f][b] = __uint_as_float(m << 16);
            }
        }
        if (p.codes != nullptr && p.out_block == 128) {                      // the 128 columns lie in WN / (COLS / 128) waves
            constexpr int SHARE = 128 / (HT * 16);                           // waves a block
#pragma unroll
            for (int f = 0; f < FM; ++f) {
                float m = amax[f][0];
#pragma unroll
                for (int b = 1; b < HT / 2; ++b) m = fmaxf(m, amax[f][b]);
                if (g == 0) s_max[wn * BM + first_row + 16 * f] = m;
            }
            tf_mx_barrier();
#pragma unroll
            for (int f = 0; f < FM; ++f) {
                float m = 0.f;
#pragma unroll
                for (int i = 0; i < SHARE; ++i) m = fmaxf(m, s_max[(wn / SHARE * SHARE + i) * BM + first_row + 16 * f]);
#pragma unroll
                for (int b = 0; b < HT / 2; ++b) amax[f][b] = m;
            }
        }
#pragma unroll
        for (int f = 0; f < FM; ++f) {
            const int row = first_row + 16 * f;
            if (row >= rows) continue;
            const size_t at = (size_t)(row0 + row);
#pragma unroll
            for (int b = 0; b < HT / 2; ++b) {
                const int block_col = tile_n * COLS + wn * HT * 16 + b * 32;
                if (block_col >= p.n) continue;                              // n is a multiple of 32
                const uint32_t bits = __float_as_uint(amax[f][b]);
                const uint32_t e = p.out_fp4 ? tf_mxfp4_scale(bits) : tf_block_exponent(amax[f][b]);
                const float inverse = p.out_fp4 ? tf_mxfp4_inverse(bits, e) : tf_block_inverse(e);
#pragma unroll
                for (int t = 2 * b; t < 2 * b + 2; ++t) {
                    const int col = block_col + (t - 2 * b) * 16 + 4 * g;
                    if (p.act != nullptr) *reinterpret_cast<u2v*>(p.act + at * p.n + col) = h[f][t];
                    if (p.codes != nullptr) {
                        const float v[4] = {tf_bf16_lo(h[f][t][0]), tf_bf16_hi(h[f][t][0]), tf_bf16_lo(h[f][t][1]), tf_bf16_hi(h[f][t][1])};
                        if (p.out_fp4) {
                            const float v8[8] = {v[0], v[1], v[2], v[3], 0.f, 0.f, 0.f, 0.f};
                            *reinterpret_cast<uint16_t*>(p.codes + at * (p.n >> 1) + (col >> 1)) = (uint16_t)tf_mxfp4_codes8(v8, inverse);
                        } else {
                            *reinterpret_cast<uint32_t*>(p.codes + at * p.n + col) =
                                tf_pack_e4m3(__fmul_rn(v[0], inverse), __fmul_rn(v[1], inverse), __fmul_rn(v[2], inverse), __fmul_rn(v[3], inverse));
                        }
                    }
                }
                if (p.codes != nullptr && g == 0 && (p.out_block == 32 || (block_col & 127) == 0))
                    p.scales[at * (p.n / p.out_block) + block_col / p.out_block] = (uint8_t)e;
            }
        }
    }
}

template <bool FP4A, bool GATED, int SC>
inline int tf_mx_gemm_go(const MxArgs& p, hipStream_t s) {
    constexpr int NS = FP4A ? 4 : 3;
    const int tiles_m = (p.rows + 255) / 256, cols = GATED ? 128 : 256, tiles_n = (p.n + cols - 1) / cols;
    const long long total = (long long)tiles_m * tiles_n;
    tf_mx_gemm<FP4A, GATED, SC, 8, 8, 2, 2, NS><<<(unsigned)((total + 7) / 8 * 8), 256, 0, s>>>(p, tiles_m, tiles_n);
    return (int)hipGetLastError();
}
template <bool FP4A, bool GATED>
inline int tf_launch_mx_gemm(const MxArgs& p, hipStream_t s) {
    if (p.k % 512 == 0 && p.block_shift == 5 && (size_t)p.a_scales % 16 == 0) return tf_mx_gemm_go<FP4A, GATED, MX_SCALES_32>(p, s);
    if constexpr (!FP4A)
        if (p.k % 512 == 0 && p.block_shift == 7 && (size_t)p.a_scales % 4 == 0) return tf_mx_gemm_go<FP4A, GATED, MX_SCALES_128>(p, s);
    return tf_mx_gemm_go<FP4A, GATED, MX_SCALES_ANY>(p, s);
}
// Both regimes of the products.
inline int tf_launch_mx(const MxArgs& p, bool gated, bool fp4_rows, hipStream_t s) {
    if (p.rows <= 64) return fp4_rows ? tf_launch_mx_stream<true>(p, gated, s) : tf_launch_mx_stream<false>(p, gated, s);
    if (gated) return fp4_rows ? tf_launch_mx_gemm<true, true>(p, s) : tf_launch_mx_gemm<false, true>(p, s);
    return fp4_rows ? tf_launch_mx_gemm<true, false>(p, s) : tf_launch_mx_gemm<false, false>(p, s);
}
