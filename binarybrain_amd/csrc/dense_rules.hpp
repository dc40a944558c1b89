// Rules by which the entries of dense layers and of the loss on top of one divide their work, apart from the code that launches: plain C++.
#pragma once

#include <initializer_list>

#include "launch_rules.hpp"

namespace bbhip {

// (31 rows of the largest stride are less than 2^32 bytes: what dense_direct_kernel's 32-bit offsets hold)
constexpr int kDenseNodesMost = 1 << 24, kDenseFramesMost = 1 << 25, kDenseStrideMost = 33 << 20;

// How a product straight from its operands is divided: tiles of 32 x 32, wavefronts that share a tile's k axis (chunks of 32), and workgroups that do.
struct DirectShape { int waves, n_tiles, slabs, slab_chunks; long long tiles; };
inline DirectShape direct_shape(int m, int n, int k, int waves = 0)
{
    DirectShape s;
    int const chunks = ceil_div(k, 32);
    s.n_tiles = ceil_div(n, 32);
    s.tiles = (long long)ceil_div(m, 32) * s.n_tiles;
    s.waves = waves ? waves : chunks > 16 ? (s.tiles <= 64 && chunks <= 64 ? 16 : 8) : chunks > 2 || s.tiles < 2048 ? 4 : 1;
    // two chunks for a wavefront are what a join is worth from six on
    int slabs = 1;
    if (s.tiles < 512 && chunks >= 6 * s.waves) {
        slabs = chunks / (2 * s.waves);
        int const most = (int)(1024 / s.tiles);
        if (slabs > most) { slabs = most; }
    }
    s.slab_chunks = ceil_div(chunks, slabs);
    s.slabs = ceil_div(chunks, s.slab_chunks);
    return s;
}

// Both products of a backward pass: as many wavefronts for either, and so one launch, while the device holds all of them at once or nearly so; beyond that a short k axis leaves most of
// the longer one's wavefronts without work (9932 x 6136 x 25 frames 1143 us, with a launch each 470; 191 x 227 x 56 frames 8.3 and 16.8).
inline void direct_shapes(int m0, int n0, int k0, int m1, int n1, int k1, DirectShape &s0, DirectShape &s1)
{
    s0 = direct_shape(m0, n0, k0);
    s1 = direct_shape(m1, n1, k1);
    if (s0.waves > 8) { s0 = direct_shape(m0, n0, k0, 8); }
    if (s1.waves > 8) { s1 = direct_shape(m1, n1, k1, 8); }
    if (s0.tiles + s1.tiles <= 1024 && s0.waves != s1.waves) {
        int const more = s0.waves > s1.waves ? s0.waves : s1.waves, waves = more < 8 ? more : 8;
        s0 = direct_shape(m0, n0, k0, waves);
        s1 = direct_shape(m1, n1, k1, waves);
    }
}

// Whether a product goes by way of packed halves (two launches at least, and both operands are written once more) instead of straight from its operands.
inline bool product_packed(int m, int n, int k) { return (long long)m * n * k >= 1LL << 29 && m >= 32 && n >= 32 && k >= 32; }

// Tiles of a packed product: 256 x 256 by eight wavefronts, 256 x 128 or 128 x 128 by four (two such workgroups on a compute unit); stages that lie in LDS.
enum PackedTile : int { kTileLarge = 0, kTileMiddle = 1, kTileSmall = 2, kTileSizes = 3 };
constexpr int kTileRows[kTileSizes] = {256, 256, 128}, kTileColumns[kTileSizes] = {256, 128, 128}, kTileThreads[kTileSizes] = {512, 256, 256};
constexpr int kTileBuffers[kTileSizes] = {4, 3, 4}, kTileWaveRows[kTileSizes] = {128, 128, 64}, kTileAtOnce[kTileSizes] = {256, 512, 512};

// How a packed product is divided: tiles, and how many workgroups share a tile's k axis.
struct PackedShape {
    int  size;
    int  m_tiles, n_tiles, k_steps, slabs, slab_stages;
    long long workgroups(void) const { return (long long)m_tiles * n_tiles * slabs; }
    int  tile_rows(void) const { return kTileWaveRows[size]; }         // that a wavefront owns
};

inline int pack_steps(int depth) { return ceil_div(depth, 16); }

inline PackedShape packed_shape(int size, int slabs, int m, int n, int k)
{
    PackedShape s;
    s.size = size;
    s.m_tiles = ceil_div(m, kTileRows[size]); s.n_tiles = ceil_div(n, kTileColumns[size]);
    s.k_steps = pack_steps(k);
    s.slab_stages = ceil_div(s.k_steps, slabs);
    s.slabs = ceil_div(s.k_steps, s.slab_stages);
    return s;
}

// Time of a launch in stages of a small tile on a compute unit (384 cycles of matrix instructions with two halves per operand, 0.16 us).  A large tile's stage is four of them, a middle
// one's two; of the tiles of four wavefronts two are on a compute unit, each at half the speed.  Six stages' worth are a workgroup's beginning and end.
constexpr double kTileStage[kTileSizes] = {4.0 / 0.75, 2 * 2.0 / 0.7, 2 * 1.0 / 0.55};
inline double packed_length(PackedShape const &s, long long workgroups)
{
    // (where each has a compute unit of its own it is not half as fast, though nothing covers what it waits for)
    bool const alone = s.size != kTileLarge && workgroups <= 256;
    return (s.slab_stages + 6) * kTileStage[s.size] * (alone ? 0.65 : 1.0);
}
inline int    packed_at_once(PackedShape const &s) { return kTileAtOnce[s.size]; }

// sums written and read again at about 4 TB/s, and a launch
inline double join_cost(PackedShape const &s, int m, int n) { return s.slabs > 1 ? (double)s.slabs * m * n * 8.0 / 4.0e6 / 0.16 : 0.0; }
constexpr double kJoinLaunch = 25.0;

// Two kinds of workgroups dealt out in order to whoever is free: when the last one ends.
inline double packed_end(PackedShape const &x, PackedShape const &y)
{
    long long const at_once = packed_at_once(x), n1 = x.workgroups(), n2 = y.workgroups();
    double const l1 = packed_length(x, n1 + n2), l2 = packed_length(y, n1 + n2);
    long long const full = n1 / at_once, more = n1 % at_once;           // `more` places are taken once more than the others
    double const free0 = full * l1, free1 = more ? free0 + l1 : free0;
    if (n2 == 0) { return free1; }
    // the places that are free first take `head` workgroups each before the others join in
    long long const head = more ? (long long)(l1 / l2) : 0, first = at_once - more;
    if (n2 <= first * head) { double const end = free0 + (double)((n2 + first - 1) / first) * l2; return end > free1 ? end : free1; }
    long long const left = n2 - first * head;
    return (more ? free1 : free0) + (double)((left + at_once - 1) / at_once) * l2;
}

// The division of one product (n1 = 0) or of two in one launch, tiles of one size: a length of the k axis for all workgroups is tried, halved from the longest on.
inline void best_shapes(int m0, int n0, int k0, int m1, int n1, int k1, PackedShape &s0, PackedShape &s1)
{
    int const longest = pack_steps(k0 > k1 ? k0 : k1);
    double least = -1.0;
    for (int size = 0; size < kTileSizes; ++size) {
        for (int parts : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64}) {
            int const length = ceil_div(longest, parts);
            if (parts > 1 && length < 8) { break; }
            PackedShape const x = packed_shape(size, ceil_div(pack_steps(k0), length), m0, n0, k0);
            PackedShape const y = m1 ? packed_shape(size, ceil_div(pack_steps(k1), length), m1, n1, k1) : PackedShape{size, 0, 0, 0, 1, 0};
            double const join = join_cost(x, m0, n0) + (m1 ? join_cost(y, m1, n1) : 0.0);
            double const cost = packed_end(x, y) + join + (join > 0 ? kJoinLaunch : 0.0);
            if (least < 0 || cost < least) { least = cost; s0 = x; s1 = y; }
        }
    }
}

inline PackedShape best_shape(int m, int n, int k)
{
    PackedShape s{}, none{};
    best_shapes(m, n, k, 0, 0, 0, s, none);
    return s;
}

// The channels of a loss are taken in pieces, so that what is held of the logits does not grow with their number.
constexpr int kLossTile = 32;               // channels per (largest, sum of exponents) of the direct products and of joined sums
struct LossPlan {
    bool packed;
    int piece;                  // channels, a multiple of 256 unless all of them
    int stride;                 // floats from row to row of a piece's logits
    int tile;                   // channels per (largest, sum of exponents)
    int tiles;                  // of all channels
    PackedShape logits;
};

inline LossPlan loss_plan(int inputs, int channels, int frames)
{
    LossPlan p;
    p.packed = product_packed(channels, frames, inputs);
    p.stride = ceil_div(frames, 64) * 64;
    long long const most = (64ll << 20) / p.stride / 256 * 256;
    p.piece = most < 256 ? 256 : (int)(most < (1 << 24) ? most : (1 << 24));
    if (p.piece > channels) { p.piece = channels; }
    p.logits = best_shape(p.piece, frames, inputs);
    p.tile = p.packed && p.logits.slabs == 1 ? p.logits.tile_rows() : kLossTile;
    p.tiles = ceil_div(channels, p.tile);
    return p;
}

}  // namespace bbhip
