// Rules by which the entries of dense layers and of the loss on top of one divide their work, apart from the code that launches: plain C++.
#pragma once

#include "launch_rules.hpp"

namespace bbhip {

constexpr int kDenseNodesMost = 1 << 24, kDenseFramesMost = 1 << 26;

// Wavefronts that share the k axis of a tile in dense_direct_kernel.
inline int direct_waves(int depth) { return depth >= 512 ? 16 : 4; }

// The channels of a loss are taken in pieces, so that what is held of the logits does not grow with their number.
constexpr int kLossTile = 32;               // channels per (largest, sum of exponents)
struct LossPlan {
    int piece;                  // channels
    int stride;                 // floats from row to row of a piece's logits
    int tiles;                  // of all channels
};

inline LossPlan loss_plan(int inputs, int channels, int frames)
{
    (void)inputs;
    LossPlan p;
    p.stride = ceil_div(frames, 64) * 64;
    long long const most = (16ll << 20) / p.stride / 256 * 256;
    p.piece = most < 256 ? 256 : most > channels ? channels : (int)most;
    p.tiles = ceil_div(channels, kLossTile);
    return p;
}

}  // namespace bbhip
