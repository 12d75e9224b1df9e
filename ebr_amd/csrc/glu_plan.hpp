// How the products of the gated projection are cut into tiles and split among workgroups, from types and sizes alone: plain C++,
// for the launches in ebr_glu.hip and for a test without a GPU.
#pragma once
#include <stdint.h>

#include <algorithm>

#include "../../include/ebr_block.h"

namespace ebr_glu {

constexpr int STAGE = 64;  // bytes of k a stage
constexpr int FEW = 32;    // rows, up to which gate and up read the weight straight into registers

static int size_of(int dtype) { return dtype == EBR_DTYPE_F64 ? 8 : dtype == EBR_DTYPE_F32 ? 4 : 2; }

enum { UNSPLIT = 0, MANY_K = 1, FEW_TILES = 2 };

// The tiles that a product is cut into, from its sizes alone.
struct Cut {
    int tile;            // 256, 128 or 64
    int64_t ti, tj;
    int splits = 1;      // of the tiles from ``whole`` on
    int64_t steps, whole;
    int64_t tiles() const { return ti * tj; }
    int64_t part_bytes() const { return splits > 1 ? splits * (tiles() - whole) * tile * tile * 4 : 0; }
    // gated: 0, 1, or 2 for TWO; split: of many k by plan, or FEW_TILES, where the tiles of an unsplit product are few;
    // largest: the largest tile
    Cut(int dtype, int64_t ni, int64_t nj, int64_t nk, int pairs, int gated, int split, int largest = 256) {
        const auto up = [](int64_t n, int64_t by) { return (n + by - 1) / by; };
        const int64_t wide = gated ? 2 * ni : ni, high = gated == 2 ? 2 * nj : nj, all = up(nk, STAGE / size_of(dtype)) * pairs;
        tile = largest;
        if (dtype == EBR_DTYPE_F64) tile = 64;
        else if (dtype == EBR_DTYPE_F32) tile = std::min(largest, 128);
        const auto tiles = [&](int t) { return up(wide, t) * up(high, t); };
        if (dtype != EBR_DTYPE_F64) {
            if (tile == 256 && tiles(256) < (split == MANY_K ? 4 : 200)) tile = 128;
            if (tile == 128 && tiles(128) < (split == MANY_K ? 8 : 200)) tile = 64;
        }
        ti = dtype == EBR_DTYPE_F64 ? up(ni, 64) : up(wide, tile);
        tj = dtype == EBR_DTYPE_F64 ? up(nj, 64) : up(high, tile);
        steps = all;
        whole = ti * tj;
        if (split && dtype != EBR_DTYPE_F64) {
            // As many workgroups as the card holds at once, and not one more: 258 of 62208 x 256 -> 1536 took 165 us, 252 113. Where
            // there are more tiles than that, those of the last round alone are split: 352 of 8192 x 2048 -> 11264 take 357 us, 410 unsplit.
            const int64_t held = tile == 256 ? 256 : 512, last = whole <= held ? whole : tile == 256 ? whole % held : 0;
            const int64_t most = split == FEW_TILES ? all / 8 : whole <= held ? up(all, 4) : all / 64;
            const int64_t want = last && !(split == FEW_TILES && whole >= 128) ? std::min(held / last, most) : 1;
            if (want > 1) {
                steps = up(all, want);
                splits = (int)up(all, steps);
                if (splits > 1) whole -= last;
            }
        }
    }
};

// Whether gate and up go through the kernel of few rows.
static bool is_few(int dtype, int64_t N, int64_t C) { return dtype != EBR_DTYPE_F64 && N <= FEW && C * size_of(dtype) >= 16; }

// Whether a tile's sums reach memory through shared memory, element for element of the type. What a value lacks once rounded is
// written straight from the registers alone: by the smaller tiles, and of few rows.
constexpr bool staged(int bytes, int tile) { return bytes == 2 && tile >= 128; }

// Whether the derivatives' products take what [dg|du] and [gg|gu] lack of their values before rounding as well: of few rows a
// weight's gradient adds up few products, and shows their roundings. Gate and up then go in tiles that write it: of 48 x 4096 ->
// 14336 in bf16 those of 64 take 74 us with the first derivative and 111 with the second (tiles of 128, which leave it, 77 and 94
// for 65 rows; all of that backward 248 and 330).
static bool with_rest(int dtype, int64_t N) { return size_of(dtype) == 2 && N <= 64; }

// The products of gate and up where the rows are not few, in the forward (order 0) or with a derivative behind them.
static Cut gates_cut(int dtype, int order, int64_t N, int64_t C, int64_t I) {
    return Cut(dtype, I, N, C, 1, order == 2 ? 2 : 1, UNSPLIT, order > 0 && with_rest(dtype, N) ? 64 : 256);
}

// dx of [dg|du]. Of few rows it has few tiles, and many k: split among workgroups and joined it takes 9.0 us of 81 x 1536 -> 256
// (10.8 unsplit); a pass of 4 x 1649 -> 2240 in fp32 to second order, which has two of them, went from 545 us to 325 by it.
static Cut input_cut(int dtype, int64_t N, int64_t C, int64_t I, int pairs) { return Cut(dtype, C, N, 2 * I, pairs, 0, FEW_TILES); }

// dw of the rows of all pairs.
static Cut weight_cut(int dtype, int64_t N, int64_t C, int64_t I, int pairs) {
    return Cut(dtype, C, 2 * I, N, pairs, 0, MANY_K);
}

// Widths up to whole 16-byte chunks, in which the products run.
static int64_t padded(int dtype, int64_t width) {
    const int64_t per = dtype == EBR_DTYPE_F64 ? 1 : 16 / size_of(dtype);
    return (width + per - 1) / per * per;
}

// Threads of a workgroup of a product's kernel, gated as in Cut.
constexpr int product_threads(int bytes, int tile, int gated) {
    return bytes == 8 || tile == 128 ? 256 : tile == 256 ? (gated ? 512 : 256) : gated == 2 ? 64 : 128;
}
constexpr int FEW_WAVES = 8;

// Whether every launch of the forward (order 0) or a derivative holds fewer than 2^32 threads, as it has to.
static bool fits(int dtype, int order, int64_t N, int64_t C, int64_t I) {
    const auto holds = [](int64_t groups, int threads) { return groups < ((int64_t)1 << 32) / threads; };
    const auto both = [&](const Cut& c, int gated) {
        const int threads = product_threads(size_of(dtype), c.tile, gated);
        const int64_t split = c.tiles() - c.whole;
        return holds(c.whole, threads) && holds(split * c.splits, threads) && holds(split * (c.tile * c.tile / 1024), 256);
    };
    C = padded(dtype, C), I = padded(dtype, I);
    if (is_few(dtype, N, C) ? !holds((I + 15) / 16, 64 * FEW_WAVES) : !both(gates_cut(dtype, order, N, C, I), order == 2 ? 2 : 1)) return false;
    const int each = with_rest(dtype, N) ? 2 : 1;
    return order == 0 || (both(input_cut(dtype, N, C, I, each), 0) && both(weight_cut(dtype, N, C, I, order * each), 0));
}

static bool known(int d) { return d == EBR_DTYPE_F32 || d == EBR_DTYPE_BF16 || d == EBR_DTYPE_F16 || d == EBR_DTYPE_F64; }

static int check(int dtype, int order, int64_t N, int64_t C, int64_t I) {
    if (!known(dtype)) return EBR_ERR_DTYPE;
    if (N < 1 || C < 1 || I < 1 || N >= ((int64_t)1 << 31) || C > (1 << 20) - 8 || I > (1 << 19) - 8) return EBR_ERR_SHAPE;
    return fits(dtype, order, N, C, I) ? EBR_OK : EBR_ERR_SHAPE;
}

}  // namespace ebr_glu
