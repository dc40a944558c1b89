// Products of dense layers straight from the operands as they lie, on the fp32 matrix instructions: small problems, and few frames.
//
// A workgroup owns a tile of 32 x 32 elements; its wavefronts share the k axis (chunks of 32, taken in turn) and add their tiles up through LDS in a fixed order.
// v_mfma_f32_32x32x2_f32 takes one value per lane and operand: lane l holds row l & 31 at the k of its half, l >> 5, so a lane loads 16 consecutive k of one row
// (64 bytes where these are neighbours in memory, 16 times 128 bytes of a half wavefront where rows are) and the 16 instructions of a chunk each take one of them:
// which k meets which in an instruction does not matter as long as both operands agree.  Every product and sum is fp32; no operand is written anywhere.
// One launch, and what it costs is the latency of a chunk's loads and 16 x 64 cycles of matrix instructions per chunk and wavefront.
#pragma once

#include "dense_operands.hpp"

namespace bbhip {

typedef float DenseAcc __attribute__((ext_vector_type(16)));

constexpr int kDirectTile = 32, kDirectChunk = 32;

struct DirectProduct {
    Operand     a, b;
    DenseOutput out;
    int n_tiles;                    // tiles side by side
    int tiles;
};

template <int KA, int KB, int WAVES>
__device__ __forceinline__ void direct_product(DirectProduct const &t, int tile, float *lds)
{
    int const m0 = tile / t.n_tiles * kDirectTile, n0 = (tile % t.n_tiles) * kDirectTile;
    int const lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int const r = lane & 31, half = lane >> 5;
    // (rows behind the last one read the last one: their elements are not stored)
    int const row_a = min(m0 + r, t.a.rows - 1);
    int const row_b = (n0 + r < t.b.rows || n0 + r == t.b.ones) ? n0 + r : t.b.rows - 1;
    int const chunks = (t.a.depth + kDirectChunk - 1) / kDirectChunk;
    DenseAcc acc = {};
    float a[16], b[16];
    if (wave < chunks) {
        load_values<KA, 16>(t.a, row_a, wave * kDirectChunk + half * 16, a);
        load_values<KB, 16>(t.b, row_b, wave * kDirectChunk + half * 16, b);
    }
    for (int c = wave; c < chunks; c += WAVES) {
        float an[16], bn[16];
        if (c + WAVES < chunks) {
            load_values<KA, 16>(t.a, row_a, (c + WAVES) * kDirectChunk + half * 16, an);
            load_values<KB, 16>(t.b, row_b, (c + WAVES) * kDirectChunk + half * 16, bn);
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) { acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], acc, 0, 0, 0); }
#pragma unroll
        for (int j = 0; j < 16; ++j) { a[j] = an[j]; b[j] = bn[j]; }
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) { lds[(wave * 16 + j) * 64 + lane] = acc[j]; }
    __syncthreads();

    DenseOutput const &o = t.out;
    constexpr int kPer = 16 / WAVES;
    float z[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        int const reg = e * WAVES + wave;
        float d = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) { d += lds[(w * 16 + reg) * 64 + lane]; }
        int const m = m0 + acc_row(reg, lane), n = n0 + r;
        bool const inside = m < o.rows && n < o.columns;
        if (o.kind == kOutForward) {
            if (inside) { static_cast<float *>(o.out)[m * o.stride + n] = activated(before_activation(o, d, m, n), o.activation); }
        }
        else if (o.kind == kOutBits) {
            uint64_t const bits = __ballot(inside && before_activation(o, d, m, n) > 0.0f);
            if (r == 0 && m < o.rows) { static_cast<uint32_t *>(o.out)[m * o.stride + (n0 >> 5)] = (uint32_t)(bits >> (half * 32)); }
        }
        else if (o.kind == kOutStore) {
            if (m < o.rows && (n < o.columns || (n == o.columns && o.line))) { store_element(o, d, m, n); }
        }
        else {
            z[e] = inside ? before_activation(o, d, m, n) : 0.0f;
            if (inside) {
                if (o.out) { static_cast<float *>(o.out)[m * o.stride + n] = z[e]; }
                if (o.label[n] == m + o.first_channel) { o.label_logit[n] = z[e]; }
            }
        }
    }
    if (o.kind == kOutLogits) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kPer; ++e) { lds[(e * WAVES + wave) * 64 + lane] = z[e]; }
        __syncthreads();
        int const n = n0 + r;
        if (threadIdx.x < 32 && n < o.columns) {
            int const rows = min(kDirectTile, o.rows - m0);
            float top = -INFINITY, sum = 0.0f;
            for (int i = 0; i < rows; ++i) { top = fmaxf(top, lds[((i & 3) + 4 * (i >> 3)) * 64 + ((i >> 2) & 1) * 32 + r]); }
            for (int i = 0; i < rows; ++i) {
                float const v = lds[((i & 3) + 4 * (i >> 3)) * 64 + ((i >> 2) & 1) * 32 + r];
                sum += v == -INFINITY ? 0.0f : exp_of_nonpositive(v - top);
            }
            o.partial[(long long)(m0 / kDirectTile) * o.columns + n] = make_float2(top, sum);
        }
    }
}

template <int KA, int KB, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void dense_direct_kernel(DirectProduct t)
{
    __shared__ float lds[WAVES * 16 * 64];
    direct_product<KA, KB, WAVES>(t, blockIdx.x, lds);
}

// the weights' gradient (x as KX) and behind it the input's, in one launch
template <int KX, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void dense_direct_backward_kernel(DirectProduct dw, DirectProduct dx)
{
    __shared__ float lds[WAVES * 16 * 64];
    if ((int)blockIdx.x < dw.tiles) { direct_product<kGradRows, KX, WAVES>(dw, blockIdx.x, lds); }
    else                            { direct_product<kColumns, kGradColumns, WAVES>(dx, blockIdx.x - dw.tiles, lds); }
}

// dr = dz: one value per thread
__global__ __launch_bounds__(256) void dense_dz_kernel(Operand o, float *out, long long stride)
{
    int const frame = blockIdx.x * 256 + threadIdx.x, row = blockIdx.y + blockIdx.z * 65535;
    if (frame < o.depth && row < o.rows) { out[row * stride + frame] = operand_at<kGradRows>(o, row, frame); }
}

}  // namespace bbhip
