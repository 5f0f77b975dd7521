// Products with prepared MXFP4 weights for many rows: tiles of 256 (128, 64) rows x as many weight rows, or 32 x 64, on the matrix cores.
//
// A workgroup of WM x WN = 4 waves (one a SIMD); a wave holds 16 FM token rows x 16 FT weight rows in 4 FM FT accumulator registers a lane.
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
// that copy a row read one contiguous piece of memory and the sixteen rows of a fragment, 256 bytes a piece, cover the banks once.  (The
// counters report 30 to 38 % of the cycles with LDS at work as conflicts all the same; which accesses they are is not known.)  Weights: as
// prepared, 1 KiB a 16-row tile and k-step in fragment order.  Scales come once a round of four k-steps, a byte of a register a k-step.
#pragma once
#include "mxfp4_stream.cuh"
#include <utility>

// Requests: lane l copies 16 (4) bytes from its address to LDS byte address m0 + OFFSET + 16 l (4 l); OFFSET is added to the memory
// address too.  m0 is set apart from them, once for several requests, and nothing else in the kernel writes it.
__device__ __forceinline__ void tf_mx_m0(uint32_t lds_base) { asm volatile("s_mov_b32 m0, %0\n\ts_nop 0" ::"s"(lds_base) : "memory"); }
template <int OFFSET>
__device__ __forceinline__ void tf_mx_dma16(const uint8_t* base, uint32_t offset) {
    asm volatile("global_load_lds_dwordx4 %0, %1 offset:%2" ::"v"(offset), "s"(base), "n"(OFFSET) : "memory");
}
__device__ __forceinline__ void tf_mx_dma16(const uint8_t* from) { asm volatile("global_load_lds_dwordx4 %0, off" ::"v"(from) : "memory"); }
__device__ __forceinline__ void tf_mx_dma4(const uint8_t* from) { asm volatile("global_load_lds_dword %0, off" ::"v"(from) : "memory"); }
// One byte a lane, as a word in LDS (only its low byte is used).
__device__ __forceinline__ void tf_mx_dma1(const uint8_t* from) { asm volatile("global_load_lds_ubyte %0, off" ::"v"(from) : "memory"); }
template <class F, int... I>
__device__ __forceinline__ void tf_static_for(F&& f, std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>{}), ...); }
template <int N, class F>
__device__ __forceinline__ void tf_static_for(F&& f) { tf_static_for(f, std::make_integer_sequence<int, N>{}); }
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
// Lane (g, r) of the result: weight rows 4 g .. 4 g + 3 of the tile for token row r.  The compiler does not know that these registers are
// written late (12 wait states behind the instruction): wherever it may copy them, which is at the ends of its blocks, they have to be done.
// So a k-step's LAST product waits 16 in the same statement, under the barrier that follows it.  The build reads the machine code and fails where it
// touches a sum, an operand, a request's base or the count of requests in a way that these statements do not allow for (listing.py).
#define TF_MX_MFMA(FORMATS, WAIT) \
    asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%5,%6,0] op_sel_hi:[%7,%8,0] " FORMATS WAIT \
                 : "+a"(acc) : "v"(w), "v"(a), "v"(sw), "v"(sa), "n"(Q & 1), "n"(Q & 1), "n"(Q >> 1), "n"(Q >> 1))
template <int Q, bool LAST>
__device__ __forceinline__ void tf_mx_mfma(v4f& acc, const u4v& w, const v8i& a, uint32_t sw, uint32_t sa) {
    if constexpr (LAST) TF_MX_MFMA("cbsz:4", "\n\ts_nop 15");
    else TF_MX_MFMA("cbsz:4", "");
}
template <int Q, bool LAST>
__device__ __forceinline__ void tf_mx_mfma(v4f& acc, const u4v& w, const u4v& a, uint32_t sw, uint32_t sa) {
    if constexpr (LAST) TF_MX_MFMA("cbsz:4 blgp:4", "\n\ts_nop 15");
    else TF_MX_MFMA("cbsz:4 blgp:4", "");
}
#undef TF_MX_MFMA
// What the k-steps of the last round past the end of k multiply by: zero codes (a round is four k-steps whatever k is; the loop body then
// has no branch, which its 256 accumulators would not survive in registers).
static __device__ const u4v tf_mx_zeros[64] = {};

// LDS of a workgroup: the ring, the weights' scales of a round, the rows' (a word a row and block where SC is MX_SCALES_ANY).
constexpr int tf_mx_scale_rows(int fm, int wm) { return 16 * fm * wm < 64 ? 64 : 16 * fm * wm; }
constexpr int tf_mx_scale_words(int sc, int rows) { return sc == MX_SCALES_128 ? rows : sc == MX_SCALES_ANY ? rows * 16 : rows * 4; }
constexpr int tf_mx_lds_bytes(bool fp4_rows, int sc, int fm, int ft, int wm, int wn, int stages) {
    return stages * (16 * fm * wm * (fp4_rows ? 64 : 128) + ft * wn * 1024) + ft * wn * 256 + tf_mx_scale_words(sc, tf_mx_scale_rows(fm, wm)) * 4;
}
// Workgroups a CU: as many as leave registers for the sums (the largest tiles 1, 64 sums a lane 2, else 3) and fit into its 160 KiB.  With 64 sums
// it is 1 for the MX_SCALES_ANY tiles of 128 x 128 E4M3 rows (83,968 bytes) and for the gated 64 x 128 tiles of E2M1 rows (87,040 to 90,112).
constexpr int tf_mx_resident(bool fp4_rows, int sc, int fm, int ft, int wm, int wn, int stages) {
    const int registers = fm * ft >= 64 ? 1 : fm * ft >= 16 ? 2 : 3, lds = 160 * 1024 / tf_mx_lds_bytes(fp4_rows, sc, fm, ft, wm, wn, stages);
    return registers < lds ? registers : lds;
}

template <bool FP4A, bool GATED, int SC, int FM, int FT, int WM, int WN, int NS>
__global__ void __launch_bounds__(WM * WN * 64, tf_mx_resident(FP4A, SC, FM, FT, WM, WN, NS)) tf_mx_gemm(const MxArgs p, int tiles_m, int tiles_n) {
    constexpr int WAVES = WM * WN, BM = 16 * FM * WM, TILES = FT * WN, ROWB = FP4A ? 64 : 128;
    constexpr int A_STAGE = BM * ROWB, B_STAGE = TILES * 1024, STAGE = A_STAGE + B_STAGE;
    constexpr int NA = A_STAGE / 1024 / WAVES > 0 ? A_STAGE / 1024 / WAVES : 1, NB = TILES / WAVES, DATA = NA + NB, SROWS = tf_mx_scale_rows(FM, WM);
    constexpr int A_WAVES = A_STAGE / 1024 / NA;                               // waves past them repeat the first ones' requests of token rows
    constexpr int MORE = SC == MX_SCALES_ANY ? 1 + SROWS / 4 / WAVES : SC >= MX_SCALES_STEP_32 ? 5 : 2;
    constexpr int COLS = (GATED ? TILES / 2 : TILES) * 16, LANES_ROW = ROWB / 16, ROWS_REQ = 64 / LANES_ROW;
    static_assert(NA * A_WAVES * 1024 == A_STAGE && (A_WAVES & (A_WAVES - 1)) == 0 && A_WAVES <= WAVES && NB * WAVES == TILES && TILES % 4 == 0 && TILES <= 4 * WAVES &&
                  SROWS % 64 == 0 && SROWS <= WAVES * 64, "whole requests a wave");
    typedef typename MxFragment<FP4A>::type Fragment;
    __shared__ __attribute__((aligned(1024))) uint8_t s_ring[NS * STAGE];
    __shared__ __attribute__((aligned(1024))) uint32_t s_wsc[TILES * 64];
    __shared__ __attribute__((aligned(1024))) uint32_t s_asc[tf_mx_scale_words(SC, SROWS)];
    static_assert(sizeof(s_ring) + sizeof(s_wsc) + sizeof(s_asc) == tf_mx_lds_bytes(FP4A, SC, FM, FT, WM, WN, NS), "the LDS that the occupancy was counted with");

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN, g = lane >> 4, r16 = lane & 15;
    const int KS = (p.k + 127) >> 7, KQ = (p.k + 511) >> 9, n_tiles = (p.n + 15) >> 4;
    const int a_pitch = FP4A ? p.k >> 1 : p.k, s_pitch = p.k >> p.block_shift;

    // Workgroup b runs on XCD b % 8.  An XCD takes a contiguous run of the tiles, eight row tiles side by side and column after column, so that the
    // tiles at work on it at once share their rows and weights in its L2.
    constexpr bool PERSIST = tf_mx_persistent(FP4A, GATED, FM * FT);
    const int total = tiles_m * tiles_n, chunk = (total + 7) >> 3, first_id = (blockIdx.x & 7) * chunk, last_id = min(first_id + chunk, total);
    int id = first_id + (int)(blockIdx.x >> 3);
    if (id >= last_id) return;
    struct Tile { int row0, rows, n; };
    auto tile_of = [&](int i) {
        const int band = i / (8 * tiles_n), in_band = i - band * 8 * tiles_n, band_m = min(8, tiles_m - band * 8);
        const int row0 = (band * 8 + in_band % band_m) * BM;
        return Tile{row0, min(BM, p.rows - row0), in_band / band_m};
    };
    Tile cur = tile_of(id);

    // ---- requests ----------------------------------------------------------------------------------------------------
    const uint32_t lds_ring = tf_mx_lds(s_ring), lds_wsc = tf_mx_lds(s_wsc), lds_asc = tf_mx_lds(s_asc);
    // Every request is a scalar base that moves on with the k-step plus the lane's own offset; four requests share an m0, so a request's
    // offset holds 1,024 bytes for every one before it in its four less (and the bases point 4,096 bytes before their data).
    constexpr bool ROUNDS = SC <= MX_SCALES_128, STEPS = SC != MX_SCALES_ANY;   // k is whole rounds / k-steps: no request / no lane needs a bound
    const uint32_t lane16 = lane * 16;
    uint32_t a_col[NA];
    const int a_wave = wave & (A_WAVES - 1);
#pragma unroll
    for (int c = 0; c < NA; ++c) {
        const int r = ((a_wave * NA + c) * ROWS_REQ + lane / LANES_ROW) & 15;
        const int swz = FP4A ? ((r >> 1) & 3) ^ (r >> 3) : (r & 7) ^ (r >> 3);
        a_col[c] = (uint32_t)((lane % LANES_ROW) ^ swz) * 16;
    }
    // the tiles a wave requests are of one matrix (gated: NB <= FT / 2), or half of them of either (NB == FT)
    constexpr bool BOTH = GATED && NB == FT;
    static_assert(!GATED || BOTH || FT / 2 % NB == 0, "whole halves");
    // weight scales: a wave requests four tiles' 256 bytes of the round at once, 16 lanes a tile; waves past the tiles repeat the first ones' request
    const int wsc_wave = wave & (TILES / 4 - 1);
    struct Source {                                                          // where a tile's requests come from
        int row0, rows;
        const uint8_t *a, *b[2], *wsc, *asc;                                 // (wsc, asc: the lane's own)
        uint32_t a_off[NA], b_off[NB];
    };
    auto source_of = [&](const Tile& tile) {
        Source s;
        s.row0 = tile.row0; s.rows = tile.rows;
        s.a = p.a + (size_t)tile.row0 * a_pitch - 4096;
#pragma unroll
        for (int c = 0; c < NA; ++c) {
            const int row = (a_wave * NA + c) * ROWS_REQ + lane / LANES_ROW;
            // past the last row: that row again, never stored
            s.a_off[c] = (uint32_t)min(row, tile.rows - 1) * (uint32_t)a_pitch + 4096 - 1024 * (c & 3) + (STEPS ? a_col[c] : 0);
        }
        // weight tile T of the workgroup (gated: a wave's FT tiles are FT / 2 of `up`, then the same columns' of `gate`)
        auto weight_tile = [&](int T, bool& second) {
            const int w = T / FT, t = T - w * FT;
            second = GATED && t >= FT / 2;
            const int at = GATED ? tile.n * (TILES / 2) + w * (FT / 2) + (second ? t - FT / 2 : t) : tile.n * TILES + T;
            return min(at, n_tiles - 1);                                     // past the last tile: that tile again, never stored
        };
        bool second;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int first = weight_tile(wave * NB + (BOTH ? half * (NB / 2) : 0), second);
            s.b[half] = reinterpret_cast<const uint8_t*>(second ? p.w2 : p.w) + (size_t)first * KS * 1024 - 4096;
#pragma unroll
            for (int c = half * NB / 2; c < (half + 1) * NB / 2 || (NB == 1 && c == 0); ++c)
                s.b_off[c] = (uint32_t)(weight_tile(wave * NB + c, second) - first) * (uint32_t)KS * 1024 + lane16 + 4096 - 1024 * (c & 3);
        }
        const int scale_tile = weight_tile(wsc_wave * 4 + (lane >> 4), second);
        s.wsc = reinterpret_cast<const uint8_t*>(second ? p.ws2 : p.ws) + (size_t)scale_tile * KQ * 256 + (lane & 15) * 16;
        s.asc = p.a_scales + (size_t)(tile.row0 + min(tid & (SROWS - 1), tile.rows - 1)) * s_pitch;
        return s;
    };
    Source from = source_of(cur);
    const uint8_t* zeros = reinterpret_cast<const uint8_t*>(tf_mx_zeros) - 4096;
    // Request OP of k-step ks into the ring stage at lds_stage; the first of four sets m0.
    auto issue = [&](auto op_constant, int ks, uint32_t lds_stage) {
        constexpr int OP = decltype(op_constant)::value;
        if constexpr (OP < NA) {
            if constexpr (OP % 4 == 0) tf_mx_m0(lds_stage + (a_wave * NA + OP) * 1024);
            if constexpr (STEPS) tf_mx_dma16<1024 * (OP & 3)>(from.a + (size_t)(ROUNDS ? ks : min(ks, KS - 1)) * ROWB, from.a_off[OP]);
            else tf_mx_dma16<1024 * (OP & 3)>(from.a, from.a_off[OP] + min((uint32_t)ks * ROWB + a_col[OP], (uint32_t)a_pitch - 16));
        } else {
            constexpr int C = OP - NA, H = BOTH && C >= NB / 2 ? 1 : 0;
            if constexpr (C % 4 == 0) tf_mx_m0(lds_stage + A_STAGE + (wave * NB + C) * 1024);
            if constexpr (ROUNDS) tf_mx_dma16<1024 * (C & 3)>(from.b[H] + (size_t)ks * 1024, from.b_off[C]);
            else tf_mx_dma16<1024 * (C & 3)>(ks < KS ? from.b[H] + (size_t)ks * 1024 : zeros, ks < KS ? from.b_off[C] : lane16 + 4096 - 1024 * (C & 3));
        }
    };
    const int asc_wave = wave & (SROWS / 64 - 1);                               // waves past the tile's rows repeat the first ones' request
    auto issue_scales = [&](int kq) {                                        // the MORE requests of a round
        tf_mx_m0(lds_wsc + wsc_wave * 1024);
        tf_mx_dma16(from.wsc + (size_t)kq * 256);
        if constexpr (SC == MX_SCALES_32) { tf_mx_m0(lds_asc + asc_wave * 1024); tf_mx_dma16(from.asc + kq * 16); }
        if constexpr (SC == MX_SCALES_128) { tf_mx_m0(lds_asc + asc_wave * 256); tf_mx_dma4(from.asc + kq * 4); }
        if constexpr (SC == MX_SCALES_STEP_32 || SC == MX_SCALES_STEP_128) {     // [k-step][row]
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int ks = min(4 * kq + q, KS - 1);
                tf_mx_m0(lds_asc + q * (SROWS * 4) + asc_wave * 256);
                if constexpr (SC == MX_SCALES_STEP_32) tf_mx_dma4(from.asc + ks * 4);
                else tf_mx_dma1(from.asc + ks);
            }
        }
        if constexpr (SC == MX_SCALES_ANY) {                                 // [block of the round][row]; request i of the wave's: block i / (SROWS / 64), 64 rows
#pragma unroll
            for (int i = 0; i < MORE - 1; ++i) {
                const int request = wave * (MORE - 1) + i, block = request / (SROWS / 64), row = request % (SROWS / 64) * 64;
                tf_mx_m0(lds_asc + (block * SROWS + row) * 4);
                tf_mx_dma1(p.a_scales + (size_t)(from.row0 + min(row + lane, from.rows - 1)) * s_pitch + min(16 * kq + block, s_pitch - 1));
            }
        }
    };

    // ---- fragments ---------------------------------------------------------------------------------------------------
    const int swz = FP4A ? ((r16 >> 1) & 3) ^ (r16 >> 3) : (r16 & 7) ^ (r16 >> 3);
    const int a_at = (wm * 16 * FM + r16) * ROWB + ((g ^ swz) << 4), b_at = A_STAGE + wn * FT * 1024 + lane16;
    v4f acc[FM][FT];
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
            u4v w;
            if constexpr (SC == MX_SCALES_ANY) w = u4v{s_asc[g * SROWS + row], s_asc[(4 + g) * SROWS + row], s_asc[(8 + g) * SROWS + row], s_asc[(12 + g) * SROWS + row]};
            else if constexpr (SC == MX_SCALES_STEP_32 || SC == MX_SCALES_STEP_128) w = u4v{s_asc[row], s_asc[SROWS + row], s_asc[2 * SROWS + row], s_asc[3 * SROWS + row]};
            else w = *reinterpret_cast<const u4v*>(s_asc + row * 4);
            const uint32_t byte = SC >= MX_SCALES_STEP_128 ? 0 : (uint32_t)g, pick = byte | ((4 + byte) << 8);       // of the second and the first operand
            const uint32_t lo = __builtin_amdgcn_perm(w[1], w[0], pick), hi = __builtin_amdgcn_perm(w[3], w[2], pick);
            to = (lo & 0xffffu) | (hi << 16);
        }
    };
    auto read_sw = [&](uint32_t& to, int t) { to = s_wsc[(wn * FT + t) * 64 + lane]; };

    // ---- the first k-steps ---------------------------------------------------------------------------------------------
    issue_scales(0);
#pragma unroll
    for (int d = 0; d < NS; ++d) tf_static_for<DATA>([&](auto op) { issue(op, d, lds_ring + d * STAGE); });
    tf_mx_wait<(NS - 1) * DATA>();
    tf_mx_barrier();
#pragma unroll
    for (int t = 0; t < FT; ++t) { read_w(wv[0][t], t, 0); read_sw(sw[0][t], t); }
#pragma unroll
    for (int f = 0; f < FM; ++f) { read_a(av[0][f], f, 0); read_sa(sa[0][f], f); }

    int stage = 0;                                                           // of k-step ks
    // The k-step of a round that requests the next round's scales: the first from whose own requests on a persistent workgroup's last round asks
    // for the next tile (k-step + NS lies past the round).
    constexpr int SWITCH = 4 - NS;
    // requests that may be in flight at the top of k-step Q of a round: those of the NS - 2 k-steps before it
    auto behind = [](int q) constexpr {
        int n = 0;
        for (int j = 1; j < NS - 1; ++j) n += DATA + (((q - j) & 3) == SWITCH ? MORE : 0);
        return n;
    };
    Tile next = cur;
    bool stored = false;                                                     // the tile before has stored: younger than the first k-steps' requests
    auto k_step = [&](auto q_constant, int kq) {
        constexpr int Q = decltype(q_constant)::value, X = Q & 1, Y = X ^ 1;
        const int next_stage = NS == 4 ? (Q + 1) & 3 : (stage + 1 == NS ? 0 : stage + 1), now = NS == 4 ? Q : stage;
        constexpr int STORES = FM * FT / 2;
        static_assert(!PERSIST || behind(0) + STORES <= 63, "the counter's six bits");
        if (PERSIST && Q < NS - 1 && kq == 0 && stored) tf_mx_wait<(PERSIST ? behind(Q) + STORES : 0)>();
        else tf_mx_wait<behind(Q)>();
        tf_mx_barrier();
        const bool last = kq == KQ - 1;
        if constexpr (Q == SWITCH) {
            if (PERSIST && last) from = source_of(next);
            issue_scales(PERSIST ? (last ? 0 : kq + 1) : min(kq + 1, KQ - 1));       // (not persistent: the last round's again, never read)
        }
        int ahead = 4 * kq + Q + NS;                                         // behind the last k-step: the next tile's, or the last one again, never read
        if constexpr (PERSIST) ahead = Q >= SWITCH && last ? Q - SWITCH : ahead;
        else ahead = min(ahead, 4 * KQ - 1);
        const uint32_t lds_now = lds_ring + now * STAGE;
        // Product i (fragment i / FT, tile i % FT); behind it, spread over the step, what the next k-step needs from LDS (weights first) and the
        // requests, one instruction between two products where it fits: the wave is alone on its SIMD, and what does not issue under a
        // product leaves the matrix pipeline idle.
        constexpr int P = FM * FT, READS = FT + FM, SCALES = Q == 3 ? FT + FM : 0, ALL = READS + SCALES;
        tf_static_for<P>([&](auto i_constant) {
            constexpr int I = decltype(i_constant)::value, F = I / FT, T = I % FT;
            tf_mx_mfma<Q, I == P - 1>(acc[F][T], wv[X][T], av[X][F], sw[0][T], sa[0][F]);
            // reads within the first three quarters
            constexpr int R = I * ALL * 4 / (P * 3) < ALL ? I * ALL * 4 / (P * 3) : ALL, R_NEXT = (I + 1) * ALL * 4 / (P * 3) < ALL ? (I + 1) * ALL * 4 / (P * 3) : ALL;
            tf_static_for<R_NEXT - R>([&](auto j_constant) {
                constexpr int J = R + decltype(j_constant)::value;
                if constexpr (J < FT) read_w(wv[Y][J], J, next_stage);
                else if constexpr (J < READS) read_a(av[Y][J - FT], J - FT, next_stage);
                else if constexpr (J < READS + FT) read_sw(sw[1][J - READS], J - READS);
                else read_sa(sa[1][J - READS - FT], J - READS - FT);
            });
            constexpr int D = (I * DATA + P - 1) / P, D_NEXT = ((I + 1) * DATA + P - 1) / P;
            tf_static_for<D_NEXT - D>([&](auto j_constant) { issue(std::integral_constant<int, D + decltype(j_constant)::value>{}, ahead, lds_now); });
            __builtin_amdgcn_sched_barrier(0);
        });
        stage = next_stage;
    };
    auto all_steps = [&]() {
#pragma unroll
        for (int f = 0; f < FM; ++f)
#pragma unroll
            for (int t = 0; t < FT; ++t) acc[f][t] = v4f{0.f, 0.f, 0.f, 0.f};
        for (int kq = 0; kq < KQ; ++kq) {
            k_step(std::integral_constant<int, 0>{}, kq);
            k_step(std::integral_constant<int, 1>{}, kq);
            k_step(std::integral_constant<int, 2>{}, kq);
            k_step(std::integral_constant<int, 3>{}, kq);
#pragma unroll
            for (int f = 0; f < FM; ++f) sa[0][f] = sa[1][f];
#pragma unroll
            for (int t = 0; t < FT; ++t) sw[0][t] = sw[1][t];
        }
    };

    if constexpr (PERSIST) {
        // ---- tile after tile: while a tile's results are formed and stored, without LDS, the next one's first k-steps arrive in the ring ----------
        const int per_xcd = gridDim.x >> 3;
        for (;;) {
            id += per_xcd;
            const bool more = id < last_id;
            if (more) next = tile_of(id);                                    // (else: the last tile's first k-steps again, never read)
            all_steps();
            // Two tiles' columns of a token row as BF16, eight consecutive ones a lane: lane group g takes tile t + g / 2, columns 8 (g % 2) ..; two
            // swaps of lane rows a register pair instead of a way through LDS.
            auto pieces = [](const v4f& first, const v4f& second) {
                auto swapped = [](uint32_t a, uint32_t b) {
                    const auto far = __builtin_amdgcn_permlane32_swap(a, b, false, false);
                    return __builtin_amdgcn_permlane16_swap(far[0], far[1], false, false);
                };
                const auto lo = swapped(tf_pack_bf16(first[0], first[1]), tf_pack_bf16(second[0], second[1]));
                const auto hi = swapped(tf_pack_bf16(first[2], first[3]), tf_pack_bf16(second[2], second[3]));
                return u4v{(uint32_t)lo[0], (uint32_t)hi[0], (uint32_t)lo[1], (uint32_t)hi[1]};
            };
            // Every lane stores every time (a skipped store would make the count of the waits too high): what lies outside the tile goes to an
            // offset past the descriptor's bytes, which the hardware drops.
            constexpr uint32_t OUTSIDE = 0x80000000u;
            auto bytes_at = [](void* base, size_t offset, size_t bytes) { return __builtin_amdgcn_make_buffer_rsrc((uint8_t*)base + offset, 0, (int)bytes, 0x00027000); };
            const int first_row = wm * 16 * FM + r16, lane_col = (g >> 1) * 16 + (g & 1) * 8;
            const auto to = bytes_at(p.out, (size_t)cur.row0 * p.out_stride * 2, ((size_t)(cur.rows - 1) * p.out_stride + p.n) * 2);
            const int col0 = cur.n * COLS + wn * FT * 16 + lane_col;
#pragma unroll
            for (int f = 0; f < FM; ++f) {
                const int row = first_row + 16 * f;
                const uint32_t at = (uint32_t)(row * (int)p.out_stride + col0) * 2;
#pragma unroll
                for (int t = 0; t < FT; t += 2) {
                    __builtin_amdgcn_sched_barrier(0);
                    const u4v o = pieces(acc[f][t], acc[f][t + 1]);
                    __builtin_amdgcn_raw_buffer_store_b128(o, to, row < cur.rows && col0 + t * 16 < p.n ? at + t * 32 : OUTSIDE, 0, 0);
                }
            }
            stored = true;
            if (!more) break;
            cur = next;
        }
        tf_mx_wait<0>();                                                     // nothing is on its way into LDS any more
        return;
    }
    all_steps();
    tf_mx_wait<0>();                                                         // nothing writes LDS any more
    const int row0 = cur.row0, rows = cur.rows, tile_n = cur.n;

    // ---- results ---------------------------------------------------------------------------------------------------------
    // Lane (g, r16) of acc[f][t] holds columns 4 g .. 4 g + 3 of tile t for token row 16 f + r16 of the wave.  They pass through LDS as BF16 rows of
    // the wave (gated: the workgroup) (eight-byte chunks permuted by the row: a row's own lanes would all meet in four banks), so that what follows is one short
    // loop over whole 16-byte pieces of rows: written out for every accumulator, its code alone was 50 KiB and ran at the speed of
    // the instruction cache's misses (17 us a tile).
    tf_mx_barrier();                                                         // every wave has read its last stage
    if constexpr (!GATED) {
        constexpr int RB = FT * 32, PIECES = RB / 16;                        // a wave's own rows of 16 FT columns
        uint8_t* own = s_ring + wave * (16 * FM * RB);
        constexpr int MIX = RB / 8 - 2;                                      // the chunk's bits that the row permutes (pairs of chunks stay together)
        static_assert((RB & (RB - 1)) == 0 && WAVES * 16 * FM * RB <= NS * STAGE, "rows of a power of two of chunks");
#pragma unroll
        for (int f = 0; f < FM; ++f)
#pragma unroll
            for (int t = 0; t < FT; ++t)
                *reinterpret_cast<u2v*>(own + (16 * f + r16) * RB + (((t * 4 + g) ^ ((r16 << 1) & MIX)) << 3)) =
                    u2v{tf_pack_bf16(acc[f][t][0], acc[f][t][1]), tf_pack_bf16(acc[f][t][2], acc[f][t][3])};
        const int piece = lane % PIECES, col = tile_n * COLS + wn * FT * 16 + piece * 8;
#pragma unroll 4
        for (int r = lane / PIECES; r < 16 * FM; r += 64 / PIECES) {
            const u4v o = *reinterpret_cast<const u4v*>(own + r * RB + (((piece << 1) ^ (((r & 15) << 1) & MIX)) << 3));
            const int row = wm * 16 * FM + r;
            if (row < rows && col < p.n) {
                uint16_t* to = p.out + (size_t)(row0 + row) * p.out_stride + col;
                if (p.wide == 2 && col + 8 <= p.n) *reinterpret_cast<u4v*>(to) = o;
                else
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        if (p.wide && col + 4 * half + 4 <= p.n) *reinterpret_cast<u2v*>(to + 4 * half) = u2v{o[2 * half], o[2 * half + 1]};
                        else
#pragma unroll
                            for (int j = 0; j < 4; ++j) if (col + 4 * half + j < p.n) to[4 * half + j] = (uint16_t)(o[2 * half + (j >> 1)] >> (16 * (j & 1)));
                    }
            }
        }
    } else {
        constexpr int HT = FT / 2, RB = COLS * 2, PIECES = RB / 16;          // the workgroup's rows of COLS columns of the activation
        constexpr int MIX = RB / 8 - 2;
        static_assert((RB & (RB - 1)) == 0 && BM * RB <= NS * STAGE, "rows of a power of two of chunks");
#pragma unroll
        for (int f = 0; f < FM; ++f) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int t = 0; t < HT; ++t) {
                float v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = tf_mx_swiglu(acc[f][t][i], acc[f][HT + t][i], p.limit);
                *reinterpret_cast<u2v*>(s_ring + (wm * 16 * FM + 16 * f + r16) * RB + ((((wn * HT + t) * 4 + g) ^ ((r16 << 1) & MIX)) << 3)) =
                    u2v{tf_pack_bf16(v[0], v[1]), tf_pack_bf16(v[2], v[3])};
            }
        }
        tf_mx_barrier();
        const int piece = lane % PIECES, col = tile_n * COLS + piece * 8;
        for (int r = tid / PIECES; r < BM; r += WAVES * 64 / PIECES) {
            const u4v h = *reinterpret_cast<const u4v*>(s_ring + r * RB + (((piece << 1) ^ (((r & 15) << 1) & MIX)) << 3));
            tf_mx_store_activation(p, h, (size_t)(row0 + r), col, r < rows && col < p.n);
        }
    }
}

template <bool FP4A, bool GATED, int SC, int FM, int FT, int WM, int WN, int NS>
inline int tf_mx_gemm_tiles(const MxArgs& p, int cus, hipStream_t s) {
    constexpr int ROWS = 16 * FM * WM, COLS = (GATED ? 8 : 16) * FT * WN;
    const int tiles_m = (p.rows + ROWS - 1) / ROWS, tiles_n = (p.n + COLS - 1) / COLS;
    const long long total = (long long)tiles_m * tiles_n, whole = (total + 7) / 8 * 8, resident = cus / 8 * 8;
    if (total > 0xfffff0ll) return -1;                                      // 2^32 threads a launch
    const long long grid = tf_mx_persistent(FP4A, GATED, FM * FT) && resident > 0 && resident < whole ? resident : whole;      // a workgroup a CU
    tf_mx_gemm<FP4A, GATED, SC, FM, FT, WM, WN, NS><<<(unsigned)grid, 256, 0, s>>>(p, tiles_m, tiles_n);
    return (int)hipGetLastError();
}
template <bool FP4A, bool GATED, int SC>
inline int tf_mx_gemm_go(const MxArgs& p, int tile, int cus, hipStream_t s) {
    constexpr int STAGES = FP4A ? 4 : 3;
    switch (tile) {
    case MX_TILE_32X64: return tf_mx_gemm_tiles<FP4A, GATED, SC, 1, 2, 2, 2, 4>(p, cus, s);
    case MX_TILE_64X64: return tf_mx_gemm_tiles<FP4A, GATED, SC, 1, 4, 4, 1, 4>(p, cus, s);
    case MX_TILE_128X128: return tf_mx_gemm_tiles<FP4A, GATED, SC, 4, 4, 2, 2, STAGES>(p, cus, s);
    case MX_TILE_256X256:
        if constexpr (SC != MX_SCALES_ANY) return tf_mx_gemm_tiles<FP4A, GATED, SC, 8, 8, 2, 2, STAGES>(p, cus, s);
        break;
    case MX_TILE_64X256:                                                     // (a context has one width of MXFP8 blocks: E4M3 rows of 32 have codes of 32)
        if constexpr (GATED && (FP4A || SC == MX_SCALES_128 || SC == MX_SCALES_STEP_128)) return tf_mx_gemm_tiles<FP4A, GATED, SC, 4, 4, 1, 4, STAGES>(p, cus, s);
        break;
    }
    return -1;
}
template <bool FP4A, bool GATED>
inline int tf_mx_gemm_launch(const MxArgs& p, const MxChoice& choice, int cus, hipStream_t s) {
    switch (choice.scales) {
    case MX_SCALES_32: return tf_mx_gemm_go<FP4A, GATED, MX_SCALES_32>(p, choice.kernel, cus, s);
    case MX_SCALES_STEP_32: return tf_mx_gemm_go<FP4A, GATED, MX_SCALES_STEP_32>(p, choice.kernel, cus, s);
    case MX_SCALES_ANY: return tf_mx_gemm_go<FP4A, GATED, MX_SCALES_ANY>(p, choice.kernel, cus, s);
    }
    if constexpr (!FP4A)
        switch (choice.scales) {
        case MX_SCALES_128: return tf_mx_gemm_go<FP4A, GATED, MX_SCALES_128>(p, choice.kernel, cus, s);
        case MX_SCALES_STEP_128: return tf_mx_gemm_go<FP4A, GATED, MX_SCALES_STEP_128>(p, choice.kernel, cus, s);
        }
    return -1;
}
template <bool FP4A, bool GATED>
inline int tf_mx_launch(const MxArgs& p, const MxChoice& choice, int cus, hipStream_t s) {
    return choice.kernel <= MX_FEW_128 ? tf_mx_stream_launch<FP4A, GATED>(p, choice.kernel, s) : tf_mx_gemm_launch<FP4A, GATED>(p, choice, cus, s);
}
inline int tf_launch_mx(const MxArgs& p, bool gated, bool fp4_rows, int cus, hipStream_t s) {
    const MxChoice choice = tf_mx_choose({p.rows, p.n, p.k, cus, fp4_rows, gated, p.block_shift, (size_t)p.a_scales, p.wide, p.out_stride, p.act != nullptr,
                                          p.codes != nullptr, p.out_block});
    MxArgs first = p;
    if (choice.codes_apart) first.codes = first.scales = nullptr;
    const int status = gated ? fp4_rows ? tf_mx_launch<true, true>(first, choice, cus, s) : tf_mx_launch<false, true>(first, choice, cus, s)
                             : fp4_rows ? tf_mx_launch<true, false>(first, choice, cus, s) : tf_mx_launch<false, false>(first, choice, cus, s);
    return status || !choice.codes_apart ? status : tf_launch_mx_codes(p, s);
}
