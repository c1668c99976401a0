// hx_i8_rule.h — which kernel takes an 8-bit product, by its sizes alone (host code).
#pragma once

#include <cstdint>

namespace hx {

// Outputs of a block: rows by outputs of the few rows' kernel, or the side of a tile of many rows'.
enum class I8Kernel { kRows16x16, kRows32x32, kRows64x32, kTiles128, kTiles256 };

// whole_rows: rows of X start at 16 bytes, less than 2^22 bytes apart.
inline I8Kernel i8_kernel(int64_t M, int64_t N, int64_t K, bool whole_rows) {
    const auto tiles = [&](int64_t side) { return ((M + side - 1) / side) * ((N + side - 1) / side); };
    // Many rows: tiles of 128 where there are enough for half the chip, two blocks to a CU, so that one's outputs are written while the
    // other multiplies; tiles of 256 from K 4096 on. 128 and 256 wide, in us: 8192 x 8192 x 2048 177 and 178, x 4096 361 and
    // 306, 4096 x 4096 x 8192 143 and 118, 13479 x 13976 x 272 to fp32 286 and 357. Tiles of 128 and few rows' kernel: 1024 x 2048 x
    // 2048 14.6 and 15.7 (128 tiles), 512 x 2048 x 2048 14.1 and 10.5 (64 tiles). Over so many outputs that a single row has 256 tiles of 256,
    // tiles of 128 serve from 17 rows on, those of 256 from 129 on, and fewer rows stay with their own kernel: 131072 outputs, K 4096, to
    // fp32, few rows' best kernel, 128 and 256: 1 row 89, 99 and 134; 16 96, 102 and 137; 32 107, 104 and 140; 64 128, 111 and 147; 128 254,
    // 118 and 158; 129 344, 187 and 157; 256 507, 207 and 170.
    if (whole_rows && tiles(128) < (1 << 23)) {
        if (K >= 4096 && tiles(256) >= 256 && M > 16) return M > 128 ? I8Kernel::kTiles256 : I8Kernel::kTiles128;
        if (M > 128 && tiles(128) >= 128) return I8Kernel::kTiles128;
    }
    // Few rows, a block's outputs by rows: 16 x 16 where blocks are wanting, 32 x 32, 32 x 64 where there are more of them than are
    // resident. 16 x 16, 32 x 32 and 32 x 64: 48 x 2048 x 8192 9.4, 8.5 and 12.0; 32 x 2048 x 8192 6.8, 8.1 and 11.8; 48 x 8192 x
    // 2048 8.1, 7.4 and 8.1; 256 x 1024 x 8192 13.9, 9.5 and 12.3; 1024 x 2048 x 2048 23.8, 15.7 and 18.0; 4096 x 4096 x 8192 597,
    // 320 and 267.
    const int64_t outs = (N + 15) / 16;
    if (M <= 16 || (M <= 32 && outs <= 128)) return I8Kernel::kRows16x16;
    return outs * ((M + 63) / 64) < 4096 ? I8Kernel::kRows32x32 : I8Kernel::kRows64x32;
}

}  // namespace hx
