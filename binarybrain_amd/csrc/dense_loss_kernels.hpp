// The cross entropy on top of a dense layer, apart from its products: what the pieces of the channels left per frame becomes the loss and what the gradient needs.
//
//   z = W x + b;   loss[f] = w * (log(sum over c of exp(z_c - top)) - (z_label - top));   dz_c = g * (softmax(z)_c - [c is the label]),  g = w / weight_sum
// Each tile of channels leaves the largest logit and the sum of exponents against it; here a frame's tiles are joined.  A frame that does not count (no label,
// weight 0) gets loss 0 and g 0, whatever its logits are.
#pragma once

#include "dense_operands.hpp"

namespace bbhip {

constexpr int kFinishFrames = 8, kFinishGroups = 64;

struct LossFinishArgs {
    float2 const *partial;          // [tiles][frames]
    float const  *label_logit;
    int const    *label;
    float const  *weight;           // null: 1
    float *loss;
    float *top, *share, *coef;      // null: no gradient
    float  reciprocal_weight_sum;
    int    tiles, frames, channels;
};

// Eight frames per workgroup; 64 threads of a frame take its tiles in turn (neighbouring lanes neighbouring frames) and are joined two by two through LDS (3.9 us for 1001
// channels x 1000 frames, 7.4 for 32768 x 4096: a chain of loads and joins)
__global__ __launch_bounds__(kFinishFrames * kFinishGroups) void dense_loss_finish_kernel(LossFinishArgs a)
{
    __shared__ float2 part[kFinishGroups][kFinishFrames];
    int const group = threadIdx.x / kFinishFrames, at = threadIdx.x % kFinishFrames, f = blockIdx.x * kFinishFrames + at;
    float2 s = make_float2(-INFINITY, 0.0f);
    if (f < a.frames) {
        for (int t = group; t < a.tiles; t += kFinishGroups) { s = joined(s, a.partial[(long long)t * a.frames + f]); }
    }
    part[group][at] = s;
    for (int step = kFinishGroups / 2; step > 0; step /= 2) {
        __syncthreads();
        if (group < step) { s = joined(s, part[group + step][at]); part[group][at] = s; }
    }
    if (group != 0 || f >= a.frames) { return; }
    int const label = a.label[f];
    float const w = a.weight ? a.weight[f] : 1.0f;
    bool const counts = label >= 0 && label < a.channels && w != 0.0f;
    a.loss[f] = counts ? w * (logf(s.y) - (a.label_logit[f] - s.x)) : 0.0f;
    if (a.coef) {
        float const g = counts ? w * a.reciprocal_weight_sum : 0.0f;
        a.coef[f]  = g;
        a.top[f]   = s.x;
        a.share[f] = g / s.y;
    }
}

}  // namespace bbhip
