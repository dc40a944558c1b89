// Rules by which the entries of dense layers and of the loss on top of one divide their work, apart from the code that launches: plain C++.
#pragma once

#include "launch_rules.hpp"

namespace bbhip {

constexpr int kDenseNodesMost = 1 << 24, kDenseFramesMost = 1 << 26;

// Wavefronts that share the k axis of a tile in dense_direct_kernel.
inline int direct_waves(int depth) { return depth >= 256 ? 8 : 4; }

// Whether a product goes by way of packed halves (two launches at least, and both operands are written once more) instead of straight from its operands.
inline bool product_packed(int m, int n, int k) { return (long long)m * n * k >= 1LL << 26 && m >= 32 && n >= 32 && k >= 32; }

// How a packed product is divided: tiles of 256 x 256 or 128 x 128, and how many workgroups share a tile's k axis.
struct PackedShape {
    bool large;
    int  m_tiles, n_tiles, k_steps, slabs, slab_stages;
    long long workgroups(void) const { return (long long)m_tiles * n_tiles * slabs; }
    int  tile_rows(void) const { return large ? 128 : 64; }         // that a wavefront owns
};

inline int pack_steps(int depth) { return ceil_div(depth, 32) * 2; }

inline PackedShape packed_shape(bool large, int slabs, int m, int n, int k)
{
    PackedShape s;
    int const side = large ? 256 : 128;
    s.large = large;
    s.m_tiles = ceil_div(m, side); s.n_tiles = ceil_div(n, side);
    s.k_steps = pack_steps(k);
    s.slab_stages = ceil_div(s.k_steps / 2, slabs);
    s.slabs = ceil_div(s.k_steps / 2, s.slab_stages);
    return s;
}

// Time of a launch in stages of a small tile on a compute unit (768 cycles of matrix instructions with two halves per operand): a large tile's stage is four of them.  Workgroups of one
// length run in rounds of 256; small tiles two on a compute unit, each at half the speed.
inline double packed_cost(PackedShape const &s, int m, int n)
{
    long long const wgs = s.workgroups();
    double const stage = s.large ? 4.0 / 0.75 : 1.0 / 0.6, at_once = s.large ? 256 : 512;
    double const rounds = (double)((wgs + (long long)at_once - 1) / (long long)at_once) * (s.large ? 1 : 2);
    double cost = (s.slab_stages + 3) * rounds * stage;
    // sums written and read again at about 4 TB/s, and a launch: a unit is 0.32 us
    if (s.slabs > 1) { cost += 10 + (double)s.slabs * m * n * 8.0 / 4.0e6 / 0.32; }
    return cost;
}

inline PackedShape best_shape(int m, int n, int k, bool only_whole = false)
{
    PackedShape best = packed_shape(true, 1, m, n, k);
    for (int large = 0; large < 2; ++large) {
        for (int slabs : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
            if (slabs > 1 && (only_whole || pack_steps(k) / 2 / slabs < 4)) { break; }
            PackedShape const s = packed_shape(large != 0, slabs, m, n, k);
            if (packed_cost(s, m, n) < packed_cost(best, m, n)) { best = s; }
        }
    }
    return best;
}

// Two products in one launch: tiles of one size, each with its own division of the k axis so that the longest workgroup does not outlast the rest.
inline void best_shapes(int m0, int n0, int k0, int m1, int n1, int k1, PackedShape &s0, PackedShape &s1)
{
    double least = -1.0;
    for (int large = 0; large < 2; ++large) {
        for (int a : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
            if (a > 1 && pack_steps(k0) / 2 / a < 4) { break; }
            for (int b : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
                if (b > 1 && pack_steps(k1) / 2 / b < 4) { break; }
                PackedShape const x = packed_shape(large != 0, a, m0, n0, k0), y = packed_shape(large != 0, b, m1, n1, k1);
                double const stage = large ? 4.0 / 0.75 : 1.0 / 0.6;
                double const total = (double)x.workgroups() * (x.slab_stages + 3) + (double)y.workgroups() * (y.slab_stages + 3);
                int const longest = x.slab_stages > y.slab_stages ? x.slab_stages : y.slab_stages;
                double cost = (total / 256 + 0.5 * (longest + 3) * (large ? 1 : 2)) * stage;
                if (cost < (longest + 3) * stage * (large ? 1 : 2)) { cost = (longest + 3) * stage * (large ? 1 : 2); }
                if (x.slabs > 1 || y.slabs > 1) {
                    double const moved = (x.slabs > 1 ? (double)x.slabs * m0 * n0 : 0.0) + (y.slabs > 1 ? (double)y.slabs * m1 * n1 : 0.0);
                    cost += 10 + moved * 8.0 / 4.0e6 / 0.32;
                }
                if (least < 0 || cost < least) { least = cost; s0 = x; s1 = y; }
            }
        }
    }
}

// The channels of a loss are taken in pieces, so that what is held of the logits does not grow with their number.
constexpr int kLossTile = 32;               // channels per (largest, sum of exponents) of the direct products
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
    long long const most = (16ll << 20) / p.stride / 256 * 256;
    p.piece = most < 256 ? 256 : (int)(most < (1 << 24) ? most : (1 << 24));
    if (p.piece > channels) { p.piece = channels; }
    p.logits = best_shape(p.piece, frames, inputs, true);
    p.tile = p.packed ? p.logits.tile_rows() : kLossTile;
    p.tiles = ceil_div(channels, p.tile);
    return p;
}

}  // namespace bbhip
