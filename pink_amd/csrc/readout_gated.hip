// readout_gated.hip -- the gated feed-forward block of the read-out (pink_hip_readout_gated* of include/pink_hip.h), forward and backward.
#include "readout_handle.h"

#include <type_traits>

#include "readout_tile.inc"
#include "readout_gated.inc"

namespace {

typedef pink_hip_readout_gated_config Shape;

struct GatedLayout {
    uint64_t stride;               // elements between rows of hidden values: whole 16-byte chunks
    size_t row_bytes;              // of one such matrix
};

GatedLayout gated_layout(const pink_hip_readout *r, const Shape &c, uint64_t images)
{
    const uint64_t per = 16 / element_bytes(r);
    GatedLayout l;
    l.stride = (c.hidden + per - 1) / per * per;
    l.row_bytes = align256(images * l.stride * element_bytes(r));
    return l;
}

constexpr uint32_t kLeastM = 16, kSumRows = 512;

size_t parts_bytes(uint64_t count, uint32_t cols) { return align256((count + kSumRows - 1) / kSumRows * cols * 4); }

// Of a call's workspace.  Backward: gradients of both hidden values, sums of them down runs of rows, shares of those, and of the
// products' depth.
struct GatedWork {
    size_t hidden, partial, parts, answer_parts, shares, bytes;
};

constexpr uint32_t kFewRows = 32;

struct Split {
    uint32_t splits, each;
};

constexpr uint32_t kFullTiles = 160, kSplitTiles = 256;    // tiles of 64 x 64: that nearly fill the card; that a product is split into

// Gradients of the weights in tiles of 128 x 128, some hundreds of them over all images: cut so that 512 places come out even, two a compute unit.  A place of the
// axis takes two tiles that share a unit 0.11 us (float32; bfloat16 0.012), runs are joined in 5 us and 8 bytes a value.  Measured (us, a training
// step, rows x features x hidden x outputs, whole / cut): 16000 x 1600 x 3200 x 1600 (650 and 325 tiles) float32 13797 / 12800, bfloat16 2013 / 1934;
// 16000 x 1600 x 1600 x 1600 (325, 169) 7387 / 6769, 1166 / 1099; 4096 x 1024 x 2048 x 1024 (256) stays whole.
constexpr uint32_t kMostRuns = 4, kCutTiles = 256;         // (with fewer tiles split_of takes smaller ones)
constexpr uint32_t kLeastRun = 512;
uint64_t gradient_tiles(uint32_t rows, uint32_t cols) { return (uint64_t)((rows + 127) / 128) * ((cols + 127) / 128); }
template <typename E> bool stays_whole(uint32_t rows, uint32_t cols)
{
    const bool larger = sizeof(E) == 2 && (uint64_t)((rows + 255) / 256) * ((cols + 255) / 256) >= 192;          // (tiles of 256 x 256)
    return larger || gradient_tiles(rows, cols) >= 2048;
}
template <typename E> Split split_of_gradients(uint32_t rows, uint32_t cols, uint32_t depth)
{
    const uint64_t tiles = gradient_tiles(rows, cols);
    if (stays_whole<E>(rows, cols)) return {1, depth};
    double best = 0.0;
    uint32_t splits = 1;
    for (uint32_t s = 1; s <= kMostRuns && depth / s >= kLeastRun; ++s) {
        const uint64_t blocks = s * tiles, more = blocks % 512;
        const double rounds = (double)(blocks / 512) + (more > 256 ? 1.0 : more ? 0.6 : 0.0);
        const double time = rounds / s * depth * (sizeof(E) == 4 ? 0.11 : 0.012) + (s > 1 ? 5.0 + 2e-6 * s * rows * cols : 0.0);
        if (s > 1 && time >= best) continue;
        best = time;
        splits = s;
    }
    const uint32_t each = ((depth + splits - 1) / splits + 127) / 128 * 128;
    return {(depth + each - 1) / each, each};
}

// A product of few results over a long axis is cut into runs, whose sums are float32 and joined afterwards by a launch of its own (4 to 5 us).  Sums over
// rows are cut for two tiles a compute unit, in runs of 256 at least; the others, whose other forms for few tiles are faster up to a depth of 1024 for bfloat16
// and 2048 for float32, for one, in runs of 1024 and 512.  Measured (us, the block's forward pass, float32; whole, in runs of 1024 at least / of
// 512): kDown of 64 rows, 4096 hidden values, 1024 results 43 / 35, 98 x 3000 x 1000 85 / 70, 200 x 2048 x 1024 50 / 42, 256 x 1024 x 784 25 / 32.
// (A training step, rows x features x hidden x outputs, float32 and bfloat16; sums over rows for one tile a unit in runs of 512 at least / for two in runs
// of 256): 6000 x 331 x 331 x 331 355 / 303, 183 / 154; 16000 x 784 x 256 x 784 717 / 673, 217 / 185; 16000 x 100 x 200 x 100 157 / 166, 127 / 116.
template <typename E, int OP> Split split_of(uint32_t rows, uint32_t cols, uint32_t depth)
{
    constexpr bool over_rows = OP == kGradGate || OP == kGradDown;
    if constexpr (over_rows)
        if (gradient_tiles(rows, cols) >= kCutTiles) return split_of_gradients<E>(rows, cols, depth);
    const uint32_t least = over_rows ? 256 : sizeof(E) == 4 && depth >= 2048 ? 512 : 1024;
    const uint64_t tiles = (uint64_t)((rows + 63) / 64) * ((cols + 63) / 64);
    const uint64_t full = over_rows ? 300 : kFullTiles, places = over_rows ? 512 : kSplitTiles;
    const uint64_t splits = tiles >= full ? 1 : std::max<uint64_t>(1, std::min<uint64_t>(places / tiles, depth / least));
    const uint32_t each = (uint32_t)(((depth + splits - 1) / splits + 127) / 128 * 128);
    return {(depth + each - 1) / each, each};
}

// kGate of float32, whose few tiles of 64 x 64 take a compute unit tens of microseconds each: cut so that the card's 512 places, two a compute unit, come out
// even.  A place on the summed axis takes two tiles that share a unit 0.026 us, one that has it for itself 0.6 of that; runs are joined in 3 us and
// 0.004 a tile.  Measured (us, the block's forward pass; in 1 / 2 / 3 / 4 / 6 / 8 runs, * the rule's):
//    160 tiles, depth 2025  55 / 55 / 46* / 49 / 48 / 48        188, 1936  85 / 78 / 85 / 73* / 80 / 81
//    256 tiles, depth 4096  127 / 125* / 132 / 129 / 140 / 134  376, 1936  109 / 100* / 114 / 103 / 113 / 113
// Below a depth of 1536 or 96 tiles smaller tiles are no slower (128 tiles, 1024: 43 / 44 / 49 / 45).
constexpr uint32_t kGateTiles = 1536;                      // of all runs
Split split_of_gate(uint32_t rows, uint32_t cols, uint32_t depth)
{
    const uint64_t tiles = (uint64_t)((rows + 63) / 64) * ((2 * (uint64_t)cols + 63) / 64);
    if (tiles < 96 || tiles > kGateTiles / 2 || depth < 1536) return {1, depth};
    double best = 0.0;
    uint32_t splits = 1;
    for (uint32_t s = 1; s <= 8 && s * tiles <= kGateTiles && depth / s >= 256; ++s) {
        const uint64_t blocks = s * tiles, more = blocks % 512;
        const double rounds = (double)(blocks / 512) + (more > 256 ? 1.0 : more ? 0.6 : 0.0);
        const double time = rounds / s * depth * 0.026 + (s > 1 ? 3.0 + 0.004 * (double)blocks : 0.0);
        if (s > 1 && time >= best) continue;
        best = time;
        splits = s;
    }
    const uint32_t each = ((depth + splits - 1) / splits + 127) / 128 * 128;
    return {(depth + each - 1) / each, each};
}

// What the shares take at most, for any number of images up to this: of split_of and split_of_gate, and of split_of_gradients.
constexpr size_t kMostShares = std::max(kSplitTiles, kGateTiles) * 64 * 64 * 4;
template <typename E> size_t most_shares_of_gradients(uint32_t rows, uint32_t cols, uint64_t images)
{
    const uint64_t runs = std::min<uint64_t>(kMostRuns, images / kLeastRun);
    return runs < 2 || gradient_tiles(rows, cols) < kCutTiles || stays_whole<E>(rows, cols) ? 0 : runs * rows * cols * 4;
}
template <typename E> size_t most_shares(const pink_hip_readout *r, const Shape &c, uint64_t images)
{
    return std::max({kMostShares, most_shares_of_gradients<E>((uint32_t)(2 * gated_layout(r, c, images).stride), c.features, images),
                     most_shares_of_gradients<E>(c.outputs, c.hidden, images)});
}

template <typename E, int OP> size_t shares_bytes(uint32_t rows, uint32_t cols, uint32_t depth)
{
    const Split s = split_of<E, OP>(rows, cols, depth);
    return s.splits > 1 ? align256((size_t)s.splits * rows * cols * 4) : 0;
}

template <typename E> GatedWork gated_work(const pink_hip_readout *r, const Shape &c, uint64_t images, bool backward)
{
    const GatedLayout l = gated_layout(r, c, images);
    GatedWork w = {};
    size_t at = 0;
    const auto take = [&](size_t bytes) {
        const size_t here = at;
        at += align256(bytes);
        return here;
    };
    w.hidden = take(l.row_bytes * 2);                      // (forward: h, and what its rounding leaves)
    size_t shares = shares_bytes<E, kDown>((uint32_t)images, c.outputs, c.hidden);
    if constexpr (sizeof(E) == 4) {
        const Split s = split_of_gate((uint32_t)images, c.hidden, c.features);
        if (s.splits > 1) shares = std::max(shares, (size_t)s.splits * 2 * images * l.stride * 4);
    }
    if (backward) {
        const uint64_t runs = (images + 255) / 256 * (256 / kLeastM);
        w.partial = take(runs * 2 * l.stride * 4);
        w.parts = take(parts_bytes(runs, (uint32_t)(2 * l.stride)));
        w.answer_parts = take(parts_bytes(images, c.outputs));
        shares = std::max({shares, shares_bytes<E, kBackInput>((uint32_t)images, c.features, (uint32_t)(2 * l.stride)),
                           shares_bytes<E, kGradGate>((uint32_t)(2 * l.stride), c.features, (uint32_t)images),
                           shares_bytes<E, kGradDown>(c.outputs, c.hidden, (uint32_t)images)});
    }
    w.shares = take(shares);
    w.bytes = at;
    return w;
}

template <typename E, int OP> bool is_direct(const DenseArgs &g)
{
    constexpr uint32_t per = 16 / sizeof(E);
    const auto whole = [](const void *at, uint64_t stride) { return ((uintptr_t)at & 15) == 0 && stride % per == 0; };
    bool direct = whole(g.p, g.p_stride) && whole(g.q, g.q_stride) && (!g.q2 || whole(g.q2, g.q_stride));
    if (OP == kGate || OP == kDown || OP == kBackGate) direct = direct && g.depth % per == 0;
    if (OP == kBackGate || OP == kBackInput || OP == kGradGate) direct = direct && g.cols % per == 0;
    if (OP == kGradDown) direct = direct && g.rows % per == 0;
    return direct;
}

template <typename E, int OP, int PR, int QC, int PW, int QW, int KW, int M, int DEEP, bool DIRECT>
int dense_of_tile(pink_hip_readout *r, DenseArgs &g, uint32_t *runs)
{
    constexpr uint32_t cols_of_tile = OP == kGate ? QC / 2 : QC;
    const uint32_t over = OP == kGate ? (uint32_t)g.out_stride : OP == kBackGate ? g.half : g.cols;      // (padding is written too)
    g.row_tiles = (g.rows + PR - 1) / PR;
    g.col_tiles = (over + cols_of_tile - 1) / cols_of_tile;
    if (runs) *runs = g.row_tiles * (PR / M);
    const uint64_t blocks = (uint64_t)g.row_tiles * g.col_tiles * g.splits;
    REFUSE(r, too_many(blocks, 64 * PW * QW * KW), "too many images for one call");
    k_dense<E, OP, PR, QC, PW, QW, KW, M, DEEP, DIRECT><<<(uint32_t)blocks, 64 * PW * QW * KW, 0, r->stream>>>(g);
    return launched(r, "k_dense");
}

// k_dense_large's offsets within a tile have 31 bits, and a stage of kBackInput is of one matrix.
template <int OP> bool is_large(const DenseArgs &g)
{
    const uint64_t lines_p = OP == kGradGate || OP == kGradDown ? 64 : 256, lines_q = OP == kGate || OP == kDown ? 256 : 64;
    return (lines_p * g.p_stride + 256) * 2 < 0x80000000u && (lines_q * g.q_stride + 256) * 2 < 0x80000000u && (OP != kBackInput || g.half % 64 == 0);
}

template <int OP> int dense_large(pink_hip_readout *r, DenseArgs &g, uint32_t *runs)
{
    const uint32_t over = OP == kGate ? (uint32_t)g.out_stride : OP == kBackGate ? g.half : g.cols;      // (padding is written too)
    g.row_tiles = (g.rows + 255) / 256;
    g.col_tiles = (over + (OP == kGate ? 127 : 255)) / (OP == kGate ? 128 : 256);
    if (runs) *runs = g.row_tiles * (256 / 32);
    const uint64_t tiles = (uint64_t)g.row_tiles * g.col_tiles;
    REFUSE(r, tiles > 0xffffffffu, "too many images for one call");
    k_dense_large<OP><<<(uint32_t)std::min<uint64_t>(tiles, 256), 512, 0, r->stream>>>(g);              // one a CU
    return launched(r, "k_dense_large");
}

// Tiles as large as there are enough of, to fetch less for each product; of the smallest the four waves share a stage's steps, as there a
// block's way through the depth is what takes time.  Measured (us; tiles of 16 x 32 / 32 x 32 / 64 x 64 / 128 x 128):
//   bfloat16  500 rows, 784 columns, depth 512 (104 tiles of 64 x 64)      8.2 /   6.1 /  7.4 /  14     500 x 512, 784 (64)        6.2 / 7.4 / 11 / 15
//             304 x 2048, 2048 (160)                                       18 /    20 /    17 /  30     1000 x 1024, 1024 (256)     17 /  15 / 12 / 20
//             2000 x 8192, 1024 (4096, of 128 x 128 1024)                 210 /   202 /    81 /  52     1024 x 4096, 2000 (256)    138 /  85 / 37 / 33
//   float32   304 x 2048, 2048 (160)                                       41 /    43 /    45 / 136     2000 x 1024, 784 (512)      56 /  55 / 38 / 60
//             4096 x 4096, 1024 (4096, of 128 x 128 1024)                 459 /   446 /   326 / 308     1024 x 2048, 4096 (128)    248 / 212 / 168 / 299
// and of 256 x 256 as in the header of k_dense_large.
template <typename E, int OP, bool DIRECT> int dense_as(pink_hip_readout *r, DenseArgs &g, uint32_t *runs)
{
    const auto tiles = [&](uint32_t pr, uint32_t qc) { return (uint64_t)((g.rows + pr - 1) / pr) * ((g.cols * (OP == kGate ? 2ull : 1ull) + qc - 1) / qc); };
    if (g.splits > 1 && tiles(128, 128) < 256) return dense_of_tile<E, OP, 64, 64, 2, 2, 1, 16, 2, DIRECT>(r, g, runs);
    if constexpr (sizeof(E) == 2 && DIRECT)
        if (g.splits == 1 && tiles(256, 256) >= 192 && is_large<OP>(g)) return dense_large<OP>(r, g, runs);
    if (tiles(128, 128) >= 256) return dense_of_tile<E, OP, 128, 128, 2, 2, 1, 32, 1, DIRECT>(r, g, runs);
    if (tiles(64, 64) >= (sizeof(E) == 2 ? kFullTiles : 192)) return dense_of_tile<E, OP, 64, 64, 2, 2, 1, 16, 2, DIRECT>(r, g, runs);
    if (tiles(32, 32) >= 384) return dense_of_tile<E, OP, 32, 32, 1, 1, 4, 16, 4, DIRECT>(r, g, runs);
    return dense_of_tile<E, OP, 16, 32, 1, 1, 4, 16, 4, DIRECT>(r, g, runs);
}

template <typename E, int OP> int dense(pink_hip_readout *r, DenseArgs &g, uint32_t *runs = nullptr)
{
    g.splits = 1;
    g.depth_each = g.depth;
    if constexpr (OP == kGate || OP == kDown) {
        if (g.rows <= kFewRows && !g.out2) {
            const uint32_t blocks = (uint32_t)(((OP == kGate ? g.out_stride : g.cols) + 15) / 16);
            const auto run = [&](auto twice) {
                constexpr bool kTwice = decltype(twice)::value;
                if (g.rows <= 16) k_few<E, OP, 1, 8, kTwice><<<blocks, 512, 0, r->stream>>>(g);
                else k_few<E, OP, 2, 8, kTwice><<<blocks, 512, 0, r->stream>>>(g);
                return launched(r, "k_few");
            };
            if constexpr (OP == kDown && sizeof(E) == 2)
                if (g.lower) return run(std::true_type());
            return run(std::false_type());
        }
    }
    if constexpr (OP != kBackGate && (OP != kGate || sizeof(E) == 4)) {
        const Split s = OP == kGate ? split_of_gate(g.rows, g.cols, g.depth) : split_of<E, OP>(g.rows, g.cols, g.depth);
        g.splits = s.splits;
        g.depth_each = s.each;
        if (s.splits == 1) g.shares = nullptr;
    }
    TRY((is_direct<E, OP>(g) ? dense_as<E, OP, true>(r, g, runs) : dense_as<E, OP, false>(r, g, runs)));
    if (g.splits == 1) return PINK_HIP_OK;
    if constexpr (OP == kGate) {
        const uint64_t blocks = (g.rows * (g.out_stride / 4) + 255) / 256;
        REFUSE(r, too_many(blocks, 256), "too many images for one call");
        k_join_gate<E><<<(uint32_t)blocks, 256, 0, r->stream>>>(g);
        return launched(r, "k_join_gate");
    }
    const uint64_t blocks = ((uint64_t)g.rows * g.cols + 255) / 256;
    REFUSE(r, too_many(blocks, 256), "too many images for one call");
    k_join<E><<<(uint32_t)blocks, 256, 0, r->stream>>>(g.shares, g.splits, g.rows, g.cols, OP == kDown ? (const E *)g.bias : nullptr,
                                                       OP == kDown ? (const E *)g.residual : nullptr, g.residual_stride, (E *)g.out, (E *)g.out2, g.out_stride,
                                                       OP == kGradGate ? g.half : 0, g.hidden);
    return launched(r, "k_join");
}

// Some of the last three products of a backward pass.
template <typename E, bool DIRECT> int dense_three_as(pink_hip_readout *r, DenseThree &g, const bool (&wanted)[3], int tile)
{
    DenseArgs *const of[3] = {&g.input, &g.grad_gate, &g.grad_down};
    const auto run = [&](uint32_t pr, uint32_t qc, auto kernel) {
        uint64_t at = 0;
        for (int n = 0; n < 3; ++n) {
            DenseArgs &d = *of[n];
            d.row_tiles = (d.rows + pr - 1) / pr;
            d.col_tiles = (d.cols + qc - 1) / qc;
            g.begin[n] = (uint32_t)at;
            g.blocks[n] = wanted[n] ? d.row_tiles * d.col_tiles : 0;
            at += (g.blocks[n] + 7) / 8 * 8;
        }
        if (!at) return (int)PINK_HIP_OK;
        kernel<<<(uint32_t)at, 256, 0, r->stream>>>(g);
        return launched(r, "k_dense_three");
    };
    if (tile == 64) return run(64, 64, k_dense_three<E, 64, 64, 2, 2, 1, 16, 2, DIRECT>);
    if constexpr (sizeof(E) == 4)
        if (tile == 32) return run(32, 32, k_dense_three<E, 32, 32, 1, 1, 4, 16, 4, DIRECT>);
    return run(16, 32, k_dense_three<E, 16, 32, 1, 1, 4, 16, 4, DIRECT>);
}

// One launch where none of them fills the card with larger tiles, nor has so long an axis that its tiles would be under way long after all others are done, and
// which is then cut into runs.  Tiles as large as all three have enough of.  Measured (us, the whole training step, rows x features x hidden x outputs,
// each alone / together):
//                              float32        bfloat16
//    100 x  331 x  256 x  331      37 /  29       35 /  29     tiles of 16 x 32 (of 32 x 32 float32  31, of 64 x 64 41; bfloat16 29, 32)
//    500 x  784 x  512 x  784      86 /  76       48 /  40     32 x 32 (76 / 80), bfloat16 64 x 64 (50 / 40 of 16 x 32 / 64 x 64)
//   2000 x  784 x  256 x  784     142 / 130       70 /  60     the same
//   1000 x 1024 x 1024 x 1024     226 / 216       84 /  71     64 x 64
//    300 x 2025 x 1000 x  331     172 / 160      106 /  86     64 x 64
//   1000 x  784 x 3000 x  784     608 / 517      173 / 144     64 x 64
//   1000 x   64 x   64 x   16      52 /  32       43 /  29     16 x 32
//   2000 x  331 x  256 x  331     117 /  97       77 /  71     16 x 32
//   3000 x  331 x  256 x  331     144 / 147       84 / 117     not: 3000 rows
//  10813 x  784 x  256 x  784     570 / 737      180 / 186     not: 595 tiles of 128 x 128 in the first
constexpr uint32_t kTogether = 2048;                       // rows that sums over them take in one go
template <typename E> int dense_three(pink_hip_readout *r, DenseThree &g)
{
    const bool input = g.input.out, gate = g.grad_gate.out || g.grad_gate.out2, down = g.grad_down.out;
    const auto tiles_of = [](const DenseArgs &d, uint32_t size) { return (uint64_t)((d.rows + size - 1) / size) * ((d.cols + size - 1) / size); };
    uint64_t tiles = 0, work = 0;
    for (const DenseArgs *const d : {&g.input, &g.grad_gate, &g.grad_down}) {
        tiles += tiles_of(*d, 64);
        work += tiles_of(*d, 64) * d->depth;
    }
    const int tile = sizeof(E) == 2 ? tiles >= 300 ? 64 : 16 : tiles >= 800 ? 64 : tiles >= 200 ? 32 : 16;
    const auto few = [&](const DenseArgs &d, bool whole) { return tiles_of(d, 128) < 512 && (work / 256 >= d.depth || whole); };
    // (by the sizes alone: a gradient has the same bits whichever others are wanted)
    const bool together = few(g.input, split_of<E, kBackInput>(g.input.rows, g.input.cols, g.input.depth).splits == 1) &&
                          few(g.grad_gate, g.grad_gate.depth < kTogether) && few(g.grad_down, g.grad_down.depth < kTogether);
    if (together) {
        for (DenseArgs *const d : {&g.input, &g.grad_gate, &g.grad_down}) {
            d->splits = 1;
            d->depth_each = d->depth;
            d->shares = nullptr;
        }
        const auto run = [&](bool a, bool b, bool c) {
            const bool direct = (!a || is_direct<E, kBackInput>(g.input)) && (!b || is_direct<E, kGradGate>(g.grad_gate)) &&
                                (!c || is_direct<E, kGradDown>(g.grad_down));
            return direct ? dense_three_as<E, true>(r, g, {a, b, c}, tile) : dense_three_as<E, false>(r, g, {a, b, c}, tile);
        };
        // The features' gradients may lie where x or dy does, which the others read.
        const auto apart = [&](const void *from, uint64_t stride, uint64_t rows, uint64_t cols) {
            const uintptr_t to = (uintptr_t)g.input.out, at = (uintptr_t)from;
            return at + ((rows - 1) * stride + cols) * sizeof(E) <= to || to + ((g.input.rows - 1) * g.input.out_stride + g.input.cols) * sizeof(E) <= at;
        };
        if (apart(g.grad_gate.q, g.grad_gate.q_stride, g.grad_gate.depth, g.grad_gate.cols) &&
            apart(g.grad_down.p, g.grad_down.p_stride, g.grad_down.depth, g.grad_down.rows))
            return run(input, gate, down);
        TRY(run(false, gate, down));
        return run(input, false, false);
    }
    if (gate) TRY((dense<E, kGradGate>(r, g.grad_gate)));
    if (down) TRY((dense<E, kGradDown>(r, g.grad_down)));
    return input ? dense<E, kBackInput>(r, g.input) : PINK_HIP_OK;
}

// Sums by column of two matrices at once, by way of shares of 512 rows each where there are more.  A matrix without rows there is none of.
template <typename E, typename V1, typename V2> int sum_columns(pink_hip_readout *r, SumJob first, SumJob second)
{
    const auto blocks = [](const SumJob &g) { return g.count ? (g.cols + 63) / 64 : 0; };
    const auto shares = [](const SumJob &g) { return (uint32_t)(((uint64_t)g.count + kSumRows - 1) / kSumRows); };
    const uint32_t most = std::max(shares(first), shares(second));
    REFUSE(r, most > 65535, "too many images for one call");
    SumJob then[2] = {first, second};
    for (SumJob *const g : {&first, &second}) {
        g->each = kSumRows;
        SumJob &after = then[g == &second];
        if (shares(*g) > 1) {
            after.rows = g->shares;
            after.stride = g->cols;
            after.count = after.each = shares(*g);
        } else {
            g->shares = nullptr;
            after.count = 0;
        }
        after.shares = nullptr;
    }
    k_sum_rows<E, V1, V2><<<dim3(blocks(first) + blocks(second), most), 1024, 0, r->stream>>>(first, blocks(first), second);
    TRY(launched(r, "k_sum_rows"));
    if (most <= 1) return PINK_HIP_OK;
    k_sum_rows<E, float, float><<<blocks(then[0]) + blocks(then[1]), 1024, 0, r->stream>>>(then[0], blocks(then[0]), then[1]);
    return launched(r, "k_sum_rows");
}

template <typename E>
int gated(pink_hip_readout *r, const Shape &c, const void *x, uint32_t images, uint64_t x_stride, const pink_hip_readout_gated_weights &weights,
          const void *residual, uint64_t residual_stride, void *y, uint64_t y_stride, void *keep)
{
    const GatedLayout l = gated_layout(r, c, images);
    const GatedWork w = gated_work<E>(r, c, images, false);
    TRY(grow(r, w.bytes));
    char *const saved = keep ? (char *)keep : (char *)r->work;
    DenseArgs g = {};
    g.activation = c.activation;
    g.rows = images;
    g.p = x;
    g.p_stride = x_stride;
    g.q = weights.gate;
    g.q2 = weights.up;
    g.q_stride = c.features;
    g.cols = c.hidden;
    g.depth = c.features;
    g.bias = weights.gate_bias;
    g.bias2 = weights.up_bias;
    g.out = saved;
    g.out2 = keep ? saved + l.row_bytes : nullptr;
    g.out3 = keep ? saved + 2 * l.row_bytes : nullptr;
    g.lower = (uint16_t *)(saved + 3 * l.row_bytes);       // (bfloat16)
    g.out_stride = l.stride;
    g.shares = sizeof(E) == 4 ? (float *)((char *)r->work + w.shares) : nullptr;
    if (!keep) g.lower = sizeof(E) == 2 && images <= kFewRows ? (uint16_t *)(saved + l.row_bytes) : nullptr;
    TRY((dense<E, kGate>(r, g)));
    if (keep) g.lower = nullptr;                           // (kDown: h is one value)
    g.p = saved;
    g.p_stride = l.stride;
    g.q = weights.down;
    g.q2 = nullptr;
    g.q_stride = c.hidden;
    g.cols = c.outputs;
    g.depth = c.hidden;
    g.bias = weights.down_bias;
    g.residual = residual;
    g.residual_stride = residual_stride;
    g.shares = (float *)((char *)r->work + w.shares);
    g.out = y;
    g.out2 = g.out3 = nullptr;
    g.out_stride = y_stride;
    return dense<E, kDown>(r, g);
}

template <typename E>
int gated_backward(pink_hip_readout *r, const Shape &c, const void *x, uint32_t images, uint64_t x_stride, const pink_hip_readout_gated_weights &weights,
                   const void *keep, const void *dy, uint64_t dy_stride, const pink_hip_readout_gated_gradients &out, uint64_t dx_stride)
{
    const GatedLayout l = gated_layout(r, c, images);
    const GatedWork w = gated_work<E>(r, c, images, true);
    TRY(grow(r, w.bytes));
    char *const work = (char *)r->work;
    const char *const saved = (const char *)keep;
    const uint32_t half = (uint32_t)l.stride;
    const bool biases = out.gate_bias || out.up_bias, matrices = out.gate || out.up;
    SumJob hidden_sums = {}, answer_sums = {};
    if (out.features || matrices || biases) {
        DenseArgs g = {};
        g.rows = images;
        g.p = dy;
        g.p_stride = dy_stride;
        g.q = weights.down;
        g.q_stride = c.hidden;
        g.cols = c.hidden;
        g.depth = c.outputs;
        g.half = half;
        g.hidden = c.hidden;
        g.value = saved + l.row_bytes;
        g.slope = saved + 2 * l.row_bytes;
        g.value_lower = (const uint16_t *)(saved + 3 * l.row_bytes);
        g.out = work + w.hidden;
        g.out_stride = 2 * l.stride;
        g.partial = biases ? (float *)(work + w.partial) : nullptr;
        uint32_t runs = 0;
        TRY((dense<E, kBackGate>(r, g, &runs)));
        if (biases) {
            hidden_sums.rows = g.partial;
            hidden_sums.stride = 2 * l.stride;
            hidden_sums.count = runs;
            hidden_sums.cols = 2 * half;
            hidden_sums.shares = (float *)(work + w.parts);
            hidden_sums.out = out.gate_bias;
            hidden_sums.out2 = out.up_bias;
            hidden_sums.half = half;
            hidden_sums.hidden = c.hidden;
        }
    }
    if (out.down_bias) {
        answer_sums.rows = dy;
        answer_sums.stride = dy_stride;
        answer_sums.count = images;
        answer_sums.cols = c.outputs;
        answer_sums.shares = (float *)(work + w.answer_parts);
        answer_sums.out = out.down_bias;
    }
    if (biases || out.down_bias) TRY((sum_columns<E, float, E>(r, hidden_sums, answer_sums)));
    DenseThree three = {};
    DenseArgs &gate = three.grad_gate, &down = three.grad_down, &input = three.input;
    gate.rows = 2 * half;
    gate.p = work + w.hidden;
    gate.p_stride = 2 * l.stride;
    gate.q = x;
    gate.q_stride = x_stride;
    gate.cols = c.features;
    gate.depth = images;
    gate.half = half;
    gate.hidden = c.hidden;
    gate.out = out.gate;
    gate.out2 = out.up;
    gate.out_stride = c.features;
    down.rows = c.outputs;
    down.p = dy;
    down.p_stride = dy_stride;
    down.q = saved;
    down.q_stride = l.stride;
    down.cols = c.hidden;
    down.depth = images;
    down.out = out.down;
    down.out_stride = c.hidden;
    input.rows = images;
    input.p = work + w.hidden;
    input.p_stride = 2 * l.stride;
    input.q = weights.gate;
    input.q2 = weights.up;
    input.q_stride = c.features;
    input.cols = c.features;
    input.depth = 2 * half;
    input.half = half;
    input.hidden = c.hidden;
    input.out = out.features;
    input.out_stride = dx_stride;
    gate.shares = down.shares = input.shares = (float *)(work + w.shares);
    return dense_three<E>(r, three);
}

int check_shape(pink_hip_readout *r, const Shape *c, uint32_t images)
{
    REFUSE(r, !c, "pink_hip_readout_gated: null argument");
    REFUSE(r, !c->features || !c->hidden || !c->outputs || c->features > kMaxSize || c->hidden > kMaxSize || c->outputs > kMaxSize,
           "pink_hip_readout_gated: features, hidden and outputs must be between 1 and 1048576");
    REFUSE(r, c->activation > PINK_HIP_SILU, "unknown activation");
    REFUSE(r, images > 0x7fffff00u, "too many images for one call");
    return PINK_HIP_OK;
}

}  // namespace

extern "C" {

size_t pink_hip_readout_gated_saved_bytes(pink_hip_readout *r, const pink_hip_readout_gated_config *c, uint32_t images)
{
    return !r || check_shape(r, c, images) != PINK_HIP_OK ? 0 : (element_bytes(r) == 2 ? 4 : 3) * gated_layout(r, *c, images).row_bytes;
}

int pink_hip_readout_gated_reserve(pink_hip_readout *r, const pink_hip_readout_gated_config *c, uint32_t images)
{
    if (!r) return PINK_HIP_EINVAL;
    TRY(check_shape(r, c, images));
    if (images == 0) return PINK_HIP_OK;
    HIP_TRY(r, hipSetDevice(r->cfg.device));
    // (fewer images may be cut into runs where more are not)
    const bool bfloat = element_bytes(r) == 2;
    const size_t before = bfloat ? gated_work<Bfloat>(r, *c, images, true).shares : gated_work<float>(r, *c, images, true).shares;
    return grow(r, before + align256(bfloat ? most_shares<Bfloat>(r, *c, images) : most_shares<float>(r, *c, images)));
}

int pink_hip_readout_gated(pink_hip_readout *r, const pink_hip_readout_gated_config *c, const void *x, uint32_t images, uint64_t x_stride,
                           const pink_hip_readout_gated_weights *weights, const void *residual, uint64_t residual_stride, void *y, uint64_t y_stride,
                           void *saved)
{
    if (!r) return PINK_HIP_EINVAL;
    TRY(check_shape(r, c, images));
    x_stride = x_stride ? x_stride : c->features;
    y_stride = y_stride ? y_stride : c->outputs;
    residual_stride = residual_stride ? residual_stride : c->outputs;
    REFUSE(r, x_stride < c->features || y_stride < c->outputs || residual_stride < c->outputs, "pink_hip_readout_gated: rows overlap");
    // (blocks of kDown write rows that others have yet to read; x has been read by then)
    REFUSE(r, images > 1 && y && y == residual && y_stride != residual_stride, "pink_hip_readout_gated: rows overlap");
    REFUSE(r, (uintptr_t)saved & 255, "pink_hip_readout_gated: saved must be aligned to 256 bytes");
    if (images == 0) return PINK_HIP_OK;
    REFUSE(r, !x || !weights || !weights->gate || !weights->up || !weights->down || !y, "pink_hip_readout_gated: null argument");
    HIP_TRY(r, hipSetDevice(r->cfg.device));
    if (r->cfg.element == PINK_HIP_ELEMENT_BFLOAT) return gated<Bfloat>(r, *c, x, images, x_stride, *weights, residual, residual_stride, y, y_stride, saved);
    return gated<float>(r, *c, x, images, x_stride, *weights, residual, residual_stride, y, y_stride, saved);
}

int pink_hip_readout_gated_backward(pink_hip_readout *r, const pink_hip_readout_gated_config *c, const void *x, uint32_t images, uint64_t x_stride,
                                    const pink_hip_readout_gated_weights *weights, const void *saved, const void *dy, uint64_t dy_stride,
                                    const pink_hip_readout_gated_gradients *out, uint64_t dx_stride)
{
    if (!r) return PINK_HIP_EINVAL;
    TRY(check_shape(r, c, images));
    x_stride = x_stride ? x_stride : c->features;
    dx_stride = dx_stride ? dx_stride : c->features;
    dy_stride = dy_stride ? dy_stride : c->outputs;
    REFUSE(r, x_stride < c->features || dx_stride < c->features || dy_stride < c->outputs, "pink_hip_readout_gated_backward: rows overlap");
    REFUSE(r, (uintptr_t)saved & 255, "pink_hip_readout_gated_backward: saved must be aligned to 256 bytes");
    REFUSE(r, !out, "pink_hip_readout_gated_backward: null argument");
    HIP_TRY(r, hipSetDevice(r->cfg.device));
    if (images == 0) {                                     // sums over nothing
        const size_t e = element_bytes(r);
        const auto clear = [&](void *at, uint64_t n) {
            if (at) k_clear<<<1024, 256, 0, r->stream>>>((uint8_t *)at, n * e);
        };
        clear(out->gate, (uint64_t)c->hidden * c->features);
        clear(out->gate_bias, c->hidden);
        clear(out->up, (uint64_t)c->hidden * c->features);
        clear(out->up_bias, c->hidden);
        clear(out->down, (uint64_t)c->outputs * c->hidden);
        clear(out->down_bias, c->outputs);
        return launched(r, "k_clear");
    }
    REFUSE(r, !x || !weights || !weights->gate || !weights->up || !weights->down || !saved || !dy, "pink_hip_readout_gated_backward: null argument");
    if (r->cfg.element == PINK_HIP_ELEMENT_BFLOAT) return gated_backward<Bfloat>(r, *c, x, images, x_stride, *weights, saved, dy, dy_stride, *out, dx_stride);
    return gated_backward<float>(r, *c, x, images, x_stride, *weights, saved, dy, dy_stride, *out, dx_stride);
}

}  // extern "C"
