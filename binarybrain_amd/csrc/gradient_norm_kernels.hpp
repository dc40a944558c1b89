// The norm of a list of gradients as if they were one vector, the list scaled to a norm, and the Adam step that takes the scale on its way.
//
//   norm = sqrt(sum over tensors and elements of g^2);   scale = norm > max_norm ? max_norm / norm : 1
// Sizes and addresses lie in device tables, as the optimizer has them, so the host does not know how much there is: a fixed number of workgroups walks pieces of
// 4096 elements of whatever tensors there are, piece c of the whole list going to workgroup c mod gridDim.  Each workgroup finds its pieces by a running sum of the
// tensors' piece counts, 256 tensors at a time.  Squares are summed in 64 bits: the kernel waits for memory, and a sum in 64 bits neither overflows nor loses small
// gradients beside large ones.  The order of the sums is fixed by the sizes alone.  What bounds it: HBM (4 bytes per element), or the
// latency of two launches: three tensors of 463 thousand values 4.3 + 2.5 us; 2^26 values 80 us, and the Adam step on them 345 (1.9 GB at 5.4 TB/s).
#pragma once

#include "vector_kernels.hpp"

namespace bbhip {

constexpr int kNormBlock = 256, kNormPiece = 4096, kNormGrid = 1024;

// calls f(tensor, first element, count) for every piece of this workgroup
template <bool BACKWARDS, class F>
__device__ __forceinline__ void for_each_piece(int size, int const *size_table, F const &f)
{
    __shared__ int scan[kNormBlock], waves[kNormBlock / 64];            // pieces up to and with each tensor of the batch
    int const batches = (size + kNormBlock - 1) / kNormBlock;
    // (pieces of the batches before; a list of many batches is walked in order, a short one may be walked backwards)
    long long before = 0;
    for (int batch = 0; batch < batches; ++batch) {
        int const t0 = batch * kNormBlock, t = t0 + threadIdx.x;
        int mine = t < size ? (size_table[t] > 0 ? (size_table[t] - 1) / kNormPiece + 1 : 0) : 0;
        // running sum: within the wavefront, then the wavefronts'
        int const lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
        for (int step = 1; step < 64; step *= 2) {
            int const add = __shfl_up(mine, step);
            mine += lane >= step ? add : 0;
        }
        if (lane == 63) { waves[wave] = mine; }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kNormBlock / 64 - 1; ++w) { mine += w < wave ? waves[w] : 0; }
        scan[threadIdx.x] = mine;
        __syncthreads();
        int const total = scan[kNormBlock - 1];
        int const first = (int)((blockIdx.x + gridDim.x - before % gridDim.x) % gridDim.x);
        int const count = first < total ? (total - first - 1) / (int)gridDim.x + 1 : 0;
        for (int i = 0; i < count; ++i) {
            int const c = first + (BACKWARDS ? count - 1 - i : i) * (int)gridDim.x;
            int lo = 0, hi = kNormBlock - 1;            // the first tensor whose running count exceeds c
            while (lo < hi) { int const mid = (lo + hi) / 2; if (scan[mid] > c) { hi = mid; } else { lo = mid + 1; } }
            int const piece = c - (lo > 0 ? scan[lo - 1] : 0);
            int const at = piece * kNormPiece, left = size_table[t0 + lo] - at;
            f(t0 + lo, at, left < kNormPiece ? left : kNormPiece);
        }
        before += total;
        __syncthreads();
    }
}

__device__ __forceinline__ double block_sum(double v)
{
    __shared__ double part[kNormBlock / 64];
#pragma unroll
    for (int step = 32; step > 0; step /= 2) { v += __shfl_xor(v, step); }
    if ((threadIdx.x & 63) == 0) { part[threadIdx.x >> 6] = v; }
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int w = 0; w < kNormBlock / 64; ++w) { v += part[w]; }
    __syncthreads();
    return v;
}

__global__ __launch_bounds__(kNormBlock) void gradient_squares_kernel(int size, int const *size_table, float const *const *grads_table, double *partial)
{
    double sum = 0.0;
    for_each_piece<false>(size, size_table, [&](int tensor, int at, int count) {
        float const *g = grads_table[tensor] + at;
        if (count == kNormPiece && (reinterpret_cast<uintptr_t>(g) & 15) == 0) {
            float4 v[kNormPiece / (4 * kNormBlock)];
#pragma unroll
            for (int j = 0; j < kNormPiece / (4 * kNormBlock); ++j) { v[j] = reinterpret_cast<float4 const *>(g)[j * kNormBlock + threadIdx.x]; }
#pragma unroll
            for (int j = 0; j < kNormPiece / (4 * kNormBlock); ++j) {
                sum = fma((double)v[j].x, (double)v[j].x, sum); sum = fma((double)v[j].y, (double)v[j].y, sum);
                sum = fma((double)v[j].z, (double)v[j].z, sum); sum = fma((double)v[j].w, (double)v[j].w, sum);
            }
        }
        else {
            for (int i = threadIdx.x; i < count; i += kNormBlock) { double const v = g[i]; sum = fma(v, v, sum); }
        }
    });
    sum = block_sum(sum);
    if (threadIdx.x == 0) { partial[blockIdx.x] = sum; }
}

// (norm, scale) from the workgroups' sums; every workgroup that asks gets the same bits
__device__ __forceinline__ float2 norm_and_scale(double const *partial, float max_norm)
{
    double sum = 0.0;
    for (int i = threadIdx.x; i < kNormGrid; i += kNormBlock) { sum += partial[i]; }
    double const norm = sqrt(block_sum(sum));
    return make_float2((float)norm, norm > (double)max_norm ? (float)((double)max_norm / norm) : 1.0f);
}

__global__ __launch_bounds__(kNormBlock) void gradient_norm_kernel(double const *partial, float max_norm, float *norm)
{
    float2 const s = norm_and_scale(partial, max_norm);
    if (threadIdx.x == 0) { norm[0] = s.x; norm[1] = s.y; }
}

// g *= scale.  A scale of 1 leaves every bit as it is, so nothing is read then.
__global__ __launch_bounds__(kNormBlock) void gradient_clip_kernel(int size, int const *size_table, float *const *grads_table, double const *partial, float max_norm, float *norm)
{
    float2 const s = norm_and_scale(partial, max_norm);
    if (blockIdx.x == 0 && threadIdx.x == 0) { norm[0] = s.x; norm[1] = s.y; }
    if (s.y == 1.0f) { return; }
    for_each_piece<true>(size, size_table, [&](int tensor, int at, int count) {
        float *g = grads_table[tensor] + at;
        if (count == kNormPiece && (reinterpret_cast<uintptr_t>(g) & 15) == 0) {
            float4 v[kNormPiece / (4 * kNormBlock)];
#pragma unroll
            for (int j = 0; j < kNormPiece / (4 * kNormBlock); ++j) { v[j] = reinterpret_cast<float4 const *>(g)[j * kNormBlock + threadIdx.x]; }
#pragma unroll
            for (int j = 0; j < kNormPiece / (4 * kNormBlock); ++j) {
                reinterpret_cast<float4 *>(g)[j * kNormBlock + threadIdx.x] = make_float4(v[j].x * s.y, v[j].y * s.y, v[j].z * s.y, v[j].w * s.y);
            }
        }
        else {
            for (int i = threadIdx.x; i < count; i += kNormBlock) { g[i] *= s.y; }
        }
    });
}

// the Adam step with g * scale in the place of g, the gradients left as they are or (ZERO) set to zero
template <bool ZERO>
__global__ __launch_bounds__(kNormBlock) void adam_clipped_kernel(int size, int const *size_table, float *const *params_table, float *const *grads_table,
                                                                  float *const *m_table, float *const *v_table, float lr_t, float nb1, float nb2, double const *partial,
                                                                  float max_norm, float *norm)
{
    float2 const s = norm_and_scale(partial, max_norm);
    if (blockIdx.x == 0 && threadIdx.x == 0) { norm[0] = s.x; norm[1] = s.y; }
    for_each_piece<true>(size, size_table, [&](int tensor, int at, int count) {
        float *__restrict__ p = params_table[tensor] + at;
        float *__restrict__ g = grads_table[tensor] + at;
        float *__restrict__ m = m_table[tensor] + at;
        float *__restrict__ v = v_table[tensor] + at;
        bool const aligned = ((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(g) | reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v)) & 15) == 0;
        int const quads = aligned ? count / 4 : 0;
        for (int q = threadIdx.x; q < quads; q += kNormBlock) {
            float4 pi = reinterpret_cast<float4 *>(p)[q];
            float4 const gi = reinterpret_cast<float4 const *>(g)[q];
            float4 mi = reinterpret_cast<float4 *>(m)[q];
            float4 vi = reinterpret_cast<float4 *>(v)[q];
            adam_update(pi.x, rounded_mul(gi.x, s.y), mi.x, vi.x, lr_t, nb1, nb2);
            adam_update(pi.y, rounded_mul(gi.y, s.y), mi.y, vi.y, lr_t, nb1, nb2);
            adam_update(pi.z, rounded_mul(gi.z, s.y), mi.z, vi.z, lr_t, nb1, nb2);
            adam_update(pi.w, rounded_mul(gi.w, s.y), mi.w, vi.w, lr_t, nb1, nb2);
            reinterpret_cast<float4 *>(p)[q] = pi;
            reinterpret_cast<float4 *>(m)[q] = mi;
            reinterpret_cast<float4 *>(v)[q] = vi;
            if (ZERO) { reinterpret_cast<float4 *>(g)[q] = make_float4(0.0f, 0.0f, 0.0f, 0.0f); }
        }
        for (int i = quads * 4 + threadIdx.x; i < count; i += kNormBlock) {
            float pi = p[i], mi = m[i], vi = v[i];
            adam_update(pi, rounded_mul(g[i], s.y), mi, vi, lr_t, nb1, nb2);
            p[i] = pi; m[i] = mi; v[i] = vi;
            if (ZERO) { g[i] = 0.0f; }
        }
    });
}

}  // namespace bbhip
