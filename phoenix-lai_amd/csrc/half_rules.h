// Which kernel a product with fp16 or bf16 matrices takes, by its sizes: host code of its own, so that a test can ask it too.
#pragma once
#include <algorithm>
#include <cstdint>

namespace phx {

constexpr int kHalfRows = 32, kHalfNarrow = 128, kHalfTile = 256;  // places a tile: the row kernel's (16 or 32), the tile kernel's two
constexpr int kHalfTerms = 96;  // the tile kernel's where x's rows are two terms

// The tiles of n places in n_mat groups, at most.
inline int most_tiles(int n, int n_mat, int cap) { return n / cap + std::min(n, n_mat); }

// The places a tile of a product over n places with n_mat matrices of rg 32-row groups, which says its kernel, on ncu compute units;
// x_terms: of a row of x.
// Row kernel to 6 places a group, and where its workgroups number under three per compute unit (us, row kernel and tile kernel; 128
// groups of 1408 x 2816: 4 places 120, 131; 6 153, 153; 7 163, 155; 9.7 181, 161; 64 of 4096 x 1408: 5 102, 110; 6.9 115, 115; 9.4 127,
// 121; 32 of 1024 x 1024: 12.5 14.1, 15.0; 25 16.4, 17.5; 50 21.3, 19.3; one of 4096 x 4096: 128 places 17.6, 40; 256 29, 41; 512 51,
// 42; 1024 92, 44).  Its tiles of 16 places to two a group and to 64 in all, else of 32 (one of 4096 x 4096: 64 places 12.7, 16.7; 128
// 20.5, 17.6; 128 groups, 8.8 places 167, 157).  Matrices of up to 32 rows stay on it whatever the places (one of 32 x 4096: 1000
// places 15.6, 41; 8000 16.8, 42; 64000 140, 128).
// Tiles of 256 places, one workgroup a compute unit, past 192 places a group where they number two per compute unit, else of 128, two
// workgroups (us, tiles of 128 and 256; 32 groups of 2816 x 4096, 513 places 393, 381; 128 of 1408 x 2816, 128 places 249, 252; one of
// 4096 x 4096, 2048 places 60, 78; 512 42, 71).
// Rows of two terms in tiles of 96 places, with two workgroups a compute unit: with 128 the loop's registers spill, as the weights
// are held for both terms (us of the whole experts, 96, 128 and 256; 128 experts of 2816 x 704, eight of them for 1024 rows 367, 375, 381;
// 2048 466, 476, 491; 4096 721, 735, 741; four of 64 of 4096 x 1408 for 2048 616, 633, 642; four of 32 of 2816 x 2048 for 4096 749,
// 773, 753).
inline int half_cap(int ncu, int n, int n_mat, int rg, int x_terms)
{
    const int64_t groups = std::min(n, n_mat);
    if (n <= 6 * n_mat || (n / 32 + groups / 2) * (rg / 2) < 3 * ncu) return n <= 64 || n <= 2 * n_mat ? 16 : kHalfRows;
    if (x_terms == 2) return kHalfTerms;
    return n > 192 * n_mat && (int64_t)(n / kHalfTile) * (rg / 8) >= 2 * ncu ? kHalfTile : kHalfNarrow;
}

// Whether the weights, `bytes` in all, pass the caches by: more than the last cache keeps to the next call, and, on the row kernel, hardly a
// group of two tiles (us, through the caches and past them; 96 places in 64 groups of 4096 x 1408 67, 60; 512 in 128 of 1408 x 2816
// 146, 134; 1120 there 179, 179; 192 in 32 of 1408 x 2816 52, 48; 192 in 32 of 1024 x 1024 12.6, 13.9; one group of 16384 x 4096: 12
// places 32, 28; 24 49, 50).  The tile kernel of up to 128 places then sees to the groups of one tile; that of 256 takes no notice.
inline bool half_once(int64_t bytes, int n_mat, int n, int cap)
{
    return bytes > 128000000 && (cap > kHalfRows || n <= std::max(8 * n_mat, 16));
}

}  // namespace phx
