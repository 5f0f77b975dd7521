// Which kernel a product with prepared MXFP4 weights runs: a rule on its sizes, types and alignment.  Plain C++, so that it can be asked on any machine.
#pragma once
#include <stddef.h>

// How a row's scales reach the lanes of a many-row product (all end as one register a fragment and round, byte q = k-step q of the round):
enum { MX_SCALES_32 = 0,         // blocks of 32, k a multiple of 512: 16 bytes a row and round, copied by the memory system
       MX_SCALES_128 = 1,        // blocks of 128, k a multiple of 512: 4 bytes a row and round, likewise
       MX_SCALES_STEP_32 = 2,    // blocks of 32, k a multiple of 128: 4 bytes a row and k-step
       MX_SCALES_STEP_128 = 3,   // blocks of 128, any k they divide: 1 byte a row and k-step (a word in LDS)
       MX_SCALES_ANY = 4 };      // blocks of 32, k no multiple of 128: 1 byte a row and block, likewise (16 words a row: no room beside 256 x 256 tiles)

// Few rows: columns a workgroup (a gated product's: of the activation).  Many: token rows x weight rows a tile.
enum { MX_FEW_16 = 0, MX_FEW_32, MX_FEW_128, MX_TILE_32X64, MX_TILE_64X64, MX_TILE_128X128, MX_TILE_256X256, MX_TILE_64X256 };

struct MxCall {
    int rows, n, k, cus;
    bool fp4_rows, gated;
    int block_shift;                     // log2 of the columns a scale of the rows spans
    size_t a_scales;                     // their address
    int wide;                            // product: stores of 16 bytes are aligned (2)
    long long out_stride;
    bool act, codes;                     // gated: the outputs asked for, columns a scale of the codes spans
    int out_block;
};
struct MxChoice {
    int kernel;                          // MX_FEW_*, MX_TILE_*
    int scales;                          // MX_SCALES_* (many rows)
    bool codes_apart;                    // the codes are a launch of their own behind the activation's
};

// The largest tiles of a product of E2M1 rows: several a workgroup, one after the other, the next one's first k-steps on their way while the
// last one's results are formed (16,384 x 4,096 x 2,048: 106 -> 87 us, 16,384 x 8,192 x 4,096: 314 -> 294).  E4M3 rows' operands leave too few registers
// for it (4,096 x 4,096 x 4,096: 55 -> 57 us, 16,384 x 8,192 x 4,096: 486 -> 473), and a gated product's results spill beside them (16,384 x 8,192 x
// 4,096: 945 -> 1,140).
constexpr bool tf_mx_persistent(bool fp4_rows, bool gated, int products) { return fp4_rows && !gated && products == 64; }

inline int tf_mx_scales(const MxCall& c) {
    if (c.block_shift == 7) return c.k % 512 == 0 && c.a_scales % 4 == 0 ? MX_SCALES_128 : MX_SCALES_STEP_128;
    return c.k % 512 == 0 && c.a_scales % 16 == 0 ? MX_SCALES_32 : c.k % 128 == 0 && c.a_scales % 4 == 0 ? MX_SCALES_STEP_32 : MX_SCALES_ANY;
}

// The tile's size.  A 256 x 256 tile takes 54 us of a CU at k = 4,096 (E4M3 rows), one of 128 x 128 (two a CU at once) 14.5 us, one of 64 x 64
// 6 us (plus 3 us once): the large ones read LDS and L2 least for a product, the small ones give every CU something to do.
//  - 32 x 64 while they are at most one a CU: 64 rows x 4,096: 6.8 us against 7.4 of 64 x 64, 64 rows x 8,192 x 8,192: 13.1, 15.1; 256 rows (two a CU): 9.4, 8.3
//  - 64 x 64 while they are at most two a CU: 256 rows x 4,096: 8.5 us, against 14.8 (128) and 40 (256); 512 rows: 13.6, 15.8, 41
//  - 256 x 256 where whole rounds of them cost less than whole rounds of 128 x 128, a quarter of the work at 15 / 16 of the time: 4,096 rows x
//    4,096: 54 us against 58; but 2,048 rows (half the CUs without a tile) 46 against 30, 16 x 18 tiles (two rounds for 1.1) 74 against 70
//  - else 128 x 128: 1,024 rows: 18.8 us, against 25.5 (64) and 42 (256)
// All of these were taken with E4M3 rows at a k of 4,096; the rule stands unmeasured for E2M1 rows, gated products and other k.  It is known to be off where k is no
// multiple of 128 with blocks of 32: no 256 x 256 tile has room for the scales, and of E4M3 rows' 128 x 128 one fits a CU instead of two (4,096 x
// 4,096 x 4,128 88 us, x 4,224 57; E2M1 rows 62 and the gated 4,096 x 2,048 x 4,128 94).
inline int tf_mx_tile(const MxCall& c, int scales) {
    auto tiles = [&](int rows, int cols) { return (long long)((c.rows + rows - 1) / rows) * ((c.n * (c.gated ? 2ll : 1ll) + cols - 1) / cols); };
    auto rounds = [&](long long t) { return (t + c.cus - 1) / c.cus; };
    if (tiles(32, 64) <= c.cus) return MX_TILE_32X64;
    if (tiles(64, 64) <= 2 * c.cus) return MX_TILE_64X64;
    // the persistent workgroups store whole 16-byte pieces, at 31-bit offsets from the tile's first row
    const bool storable = !tf_mx_persistent(c.fp4_rows, c.gated, 64) || (c.wide == 2 && c.n % 8 == 0 && c.out_stride <= (1 << 21));
    return scales != MX_SCALES_ANY && storable && 15 * rounds(tiles(256, 256)) <= 4 * rounds(tiles(128, 128)) ? MX_TILE_256X256 : MX_TILE_128X128;
}

// Both regimes of the products.  The streaming kernel reads every weight once for all its rows, but each workgroup reads all the rows: it takes
// up to 32 (4,096 x 4,096: 24 rows 5.2 us against 6.7 of the tiles, 40 rows 7.9 against 6.7), and 16 of a gated product, which has twice
// the weights a column (2,048 x 4,096: 16 rows 6.2 us against 7.2, 24 rows 8.3 against 7.2).
//
// Few rows.  A workgroup fills a CU.  Columns a workgroup: 16 while that is one round of workgroups (4 rows x 4,096 x 4,096: 3.6 us against 4.0 of 32
// columns), else 32 (16 rows x 5,120 x 4,096: 4.4 against 6.6, 32 rows x 8,192 x 8,192: 10.2 against 15.3).  A gated product's hold whole
// blocks of its codes: 32, or 128 of blocks of 128 where the activation itself has nowhere to go.  With the activation in memory those codes
// are a launch of their own behind 16 columns a workgroup (4 rows x 2,048 x 4,096: 16 workgroups 11.8 us, 128 and the second launch 7.2).
//
// Many rows.  Blocks of 128 columns of a gated product's codes need the tile's columns to be whole blocks: 64 rows x 128 columns (256 weight rows) in place
// of the smaller ones, or, where one of the two smallest would be chosen and the activation goes to memory too, its codes in a launch of their
// own behind those (64 rows x 2,048 x 4,096: 15.2 -> 9.0 us).
inline MxChoice tf_mx_choose(const MxCall& c) {
    const bool wide_blocks = c.gated && c.codes && c.out_block == 128;
    if (c.rows <= (c.gated ? 16 : 32)) {
        const int columns = (c.n + 15) / 16 > c.cus ? MX_FEW_32 : MX_FEW_16;
        if (!c.gated || !c.codes) return {columns, 0, false};
        return wide_blocks ? c.act ? MxChoice{columns, 0, true} : MxChoice{MX_FEW_128, 0, false} : MxChoice{MX_FEW_32, 0, false};
    }
    const int scales = tf_mx_scales(c), tile = tf_mx_tile(c, scales);
    if (!wide_blocks || tile == MX_TILE_256X256) return {tile, scales, false};
    return c.act && tile <= MX_TILE_64X64 ? MxChoice{tile, scales, true} : MxChoice{MX_TILE_64X256, scales, false};
}
