// Rules by which the entries of dense layers and of the loss on top of one divide their work, apart from the code that launches: plain C++.
#pragma once

#include <initializer_list>

#include "launch_rules.hpp"

namespace bbhip {

// (31 rows of the largest stride are less than 2^32 bytes: what dense_direct_kernel's 32-bit offsets hold)
constexpr int kDenseNodesMost = 1 << 24, kDenseFramesMost = 1 << 25, kDenseStrideMost = 33 << 20;

// How a product straight from its operands is divided: tiles of 32 x 32, wavefronts that share a tile's k axis (chunks of 32), and workgroups that do.
// Wavefronts: 512 x 512 (256 tiles) over 128 inputs take 4.5 us with eight and 5.0 with four, over 512 6.5 and 9.0; 1024 x 600 (608 tiles) over 128 6.8 with four and 7.7 with eight,
// over 512 13.2 and 13.7; 4096 x 1024 over 64 17.1 with one and 19.9 with four, 2048 x 1024 over 64 12.6 and 11.9.  (Sixteen are within 0.3 us of eight.)
// Slabs: a chunk for every wavefront while there is a compute unit for each workgroup, four chunks and twice as many workgroups otherwise.  128 x 128 over 512 inputs 6.3 us whole and 7.3 in
// two, over 1024 9.0 and (in four) 7.2, over 8192 48.5 and (in sixteen) 10.1; 1024 x 64 over 2048 15.0 whole, 9.3 in four, 9.9 in eight; 1024 x 128 over 4096 29.2 whole, 19.9 in four,
// 21.3 in eight; 512 x 512 over 4096 30.1 whole and 30.8 in two.  A slab is whole rounds of the wavefronts' chunks: 1024 x 65 over 6144 takes 23.9 in eight and 27.2 in six.
struct DirectShape { int waves, n_tiles, slabs, slab_chunks; long long tiles; };
inline DirectShape direct_shape(int m, int n, int k, int waves = 0, int shared_from = 24)
{
    DirectShape s;
    int const chunks = ceil_div(k, 32);
    s.n_tiles = ceil_div(n, 32);
    s.tiles = (long long)ceil_div(m, 32) * s.n_tiles;
    s.waves = waves ? waves : s.tiles <= 512 || chunks > 16 ? 8 : chunks > 2 || s.tiles <= 2048 ? 4 : 1;
    int slabs = 1;
    if (s.tiles < 256 && chunks >= shared_from) {
        auto const least = [](int a, long long b) { return a < b ? a : (int)b; };
        int const one = least(chunks / s.waves, 256 / s.tiles), four = least(chunks / (4 * s.waves), 512 / s.tiles);
        slabs = one > four ? one : four;
        slabs = slabs < 1 ? 1 : slabs > 16 ? 16 : slabs;
    }
    s.slab_chunks = slabs > 1 ? ceil_div(ceil_div(chunks, slabs), s.waves) * s.waves : chunks;
    s.slabs = ceil_div(chunks, s.slab_chunks);
    return s;
}

// Logits: the launch that joins slabs is one more of a loss's four, so a longer axis is whole (a loss of ten classes, 1024 inputs, 64 frames takes 20 us whole and 22 shared).
inline DirectShape logits_shape(int channels, int frames, int inputs) { return direct_shape(channels, frames, inputs, 0, 48); }

// Both products of a backward pass: as many wavefronts for either, and so one launch, while the device holds all of them at once or nearly so; beyond that a short k axis leaves most of
// the longer one's wavefronts without work (9932 x 6136 x 25 frames 1143 us, with a launch each 470; 191 x 227 x 56 frames 8.3 and 16.8).  256 x 256 x 256 (136 tiles) 8.1 us with eight and
// 9.4 with four, 1024 x 256 x 64 frames (328) 9.3 and 8.1, 512 x 512 x 512 (528) 20.7 and 18.1; 256 x 256 x 4096 frames (1096) 35.0 with four and 44.6 with a launch each.
inline void direct_shapes(int m0, int n0, int k0, int m1, int n1, int k1, DirectShape &s0, DirectShape &s1)
{
    s0 = direct_shape(m0, n0, k0);
    s1 = direct_shape(m1, n1, k1);
    if (s0.tiles + s1.tiles <= 2048) {
        int const waves = s0.tiles + s1.tiles <= 256 ? 8 : 4;
        s0 = direct_shape(m0, n0, k0, waves);
        s1 = direct_shape(m1, n1, k1, waves);
    }
}

// Whether a product goes by way of packed halves (two launches at least, and both operands are read and written once more) instead of straight from its operands: the products saved
// against the launch and the values packed.  A forward pass, inputs x outputs x frames, us straight and packed: 777 x 1001 x 500 23 and 30, 777 x 1001 x 1000 41 and 32, 64 x 4096 x 4096 53 and
// 41, 128 x 8192 x 1024 46 and 32, 4096 x 4096 x 64 32 and 60 (the weights are all there is to read).  Straight products read rows of a multiple of four weights sixteen bytes at a time, which
// counts up to 1024 inputs: 784 x 1024 x 1024 22 and 32, 1024 x 1024 x 1024 30 and 33, 512 x 2048 x 1024 30 and 31, 784 x 1024 x 2048 40 and 35; 1536 x 1024 x 1024 38 and 37, 2048 x 1024 x 1024 47 and
// 41 (2048 x 1024 x 512 29 and 34).
inline bool long_enough(int a, int b, int c) { return a >= 32 && b >= 32 && c >= 32; }
inline double volume(int a, int b, int c) { return (double)a * b * c; }
inline bool forward_packed(int inputs, int outputs, int frames)
{
    return long_enough(inputs, outputs, frames) && volume(inputs, outputs, frames) >= ((1 << 29) + 80.0 * inputs * ((double)outputs + frames)) * (inputs % 4 == 0 && inputs <= 1024 ? 1.6 : 1.0);
}

// A backward pass, which packs dz as rows and as columns, inputs x outputs x frames: 512 x 512 x 1024 29 and 34, 256 x 1024 x 1024 31 and 31, 777 x 1001 x 500 35 and 39, 384 x 1000 x 1000 35 and 35,
// 784 x 512 x 1024 34 and 38, 256 x 2048 x 1024 51 and 43, 1024 x 1024 x 1024 82 and 41, 96 x 4096 x 1024 43 and 57, 64 x 8192 x 1024 58 and 94, 128 x 8192 x 1024 93 and 102, 4096 x 4096 x 32 70
// and 95, x 64 88 and 101.
inline bool backward_packed(int inputs, int outputs, int frames)
{
    return long_enough(inputs, outputs, frames) &&
           volume(inputs, outputs, frames) >= 2.9e8 + 48.0 * (2.0 * outputs * frames + (double)inputs * frames + (double)inputs * outputs);
}

// A loss, with its gradients or alone (a frame's loss has the same bits either way); packed gradients are triples.  With gradients, inputs x channels x frames, straight and
// packed: 256 x 2048 x 1024 77 us and 82, 1024 x 1001 x 700 87 and 99, 777 x 1001 x 1000 107 and 94, 1024 x 1024 x 1024 118 and 106, 512 x 2048 x 1024 111 and 99, 128 x 8192 x 1024 156 and 157,
// 128 x 2048 x 4096 159 and 128, 64 x 4096 x 4096 187 and 220, 64 x 8192 x 2048 176 and 243, 4096 x 256 x 1024 127 and 109, 4096 x 4096 x 64 127 and 213, x 128 225 and 243, 784 x 1000 x 2048 164
// and 122; over packed bits 1024 x 1024 x 1024 89 and 97, 784 x 1000 x 2048 128 and 114; the loss alone 777 x 1001 x 1000 44 and 33, 1024 x 1024 x 1024 34 and 40.
inline bool loss_packed(int inputs, int channels, int frames)
{
    return long_enough(inputs, channels, frames) &&
           volume(inputs, channels, frames) >= (1 << 29) + 50.0 * channels * frames + 100.0 * inputs * ((double)channels + frames);
}

// Tiles of a packed product: 256 x 256 by eight wavefronts, 256 x 128 or 128 x 128 by four (two such workgroups on a compute unit); stages that lie in LDS.  Large, middle and small tiles, us:
// 4096 x 4096 x 8192 with packed bits 494, 493, 548, its backward pass on real values 1550, 1611, 1737; 784 inputs x 6144 x 1024 82, 61, 56; backward 1024 x 1001 x 1000 55, 51, 44;
// 10007 channels x 513 frames x 1024 bits 78, 62, 55.
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

// Packing keeps the values of a row between finding the largest and splitting, kPackHeld groups of eight per thread, the threads of a workgroup side by side for kPackRows rows; 1024 threads
// instead of 512 where a row of real values is longer than these hold: 6144 inputs x 1024 x 1024 70 us and 74, 16384 x 512 x 512 90 and 95; where they do hold it 92.6 and 88.3 (a backward
// pass over 1024 x 1024 x 4096 frames).
constexpr int kPackRows = 8, kPackHeld = 8;
inline bool pack_is_wide(int depth) { return depth > kPackHeld * 8 * (512 / kPackRows); }

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

// Sums written and read again at about 4 TB/s, and a launch: 1024 outputs x 1024 frames x 2048 inputs take 54 us with no tile shared and 39 with its k axis in three parts, 784 x 6144 x 1024 55
// whole and 79 in two, a backward pass 1024 x 1001 x 1000 40 and 44.
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

// The channels of a loss are taken in pieces, so that what is held of the logits does not grow with their number: 256 MiB of them: 32768 channels x 4096 frames take 3.31 ms
// (64 MiB: 3.72, more launches of fewer tiles).
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
    p.packed = loss_packed(inputs, channels, frames);
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
