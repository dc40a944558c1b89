// Distillation from the logits that a teacher kept.  For every (pixel, frame) with the kept logits z_j of the channels i_j (entries whose channel is
// not one of the layer's are no entries), the student's logits y, the temperature T and the weight w of the place:
//   q_j = exp(z_j / T) / sum_j exp(z_j / T),   p_c = exp(y_c / T) / sum_c exp(y_c / T),
//   loss = w T^2 sum_j q_j (log q_j - log p_{i_j}),   dy_c = w T (p_c - sum_{j : i_j = c} q_j) / weight_sum.
// A place without entries (or whose kept logits are all minus infinity) and one with w = 0 has loss 0 and gradient 0 whatever its logits are.
//
// Two launches.  The first takes, per column and slab of channels, the running maximum m and the sum of exp((y - m) / T) in one pass; workgroups behind
// those read the lists and leave per column the largest z, the reciprocal of their sum and  sum_j q_j ((z_j - z_max) - y_{i_j}) / T - log(sum),  to which the
// second launch adds the student's log-sum-exp to have the loss.  The second launch joins the slabs and writes dy: first p for every channel of its slab, then, behind a
// barrier, the few channels of the lists.  Exponents are taken of differences to the maximum, (y - m) * (log2 e / T): the rounding of the product
// grows with the distance from the maximum and weighs as little as the term itself.
#pragma once

#include "layer_norm_kernels.hpp"

namespace bbhip {

struct DistillArgs {
    ColumnSpace c;                  // rows = channels
    TileDivisor tiles;
    TileDivisor frames;             // of a column index that counts existing frames only
    float const *y, *logit, *weight;
    int const   *index;
    float       *dy, *loss;
    float2      *partial;           // [slabs][units * W]: (m, sum)
    float4      *lists;             // [units * W]: (z_max, 1 / sum, the loss without the student's log-sum-exp, entries or not)
    float scale;                    // log2(e) / T
    float reciprocal_t, t_square, coefficient;      // 1 / T, T^2, T / weight_sum
    int   top_size, pix_size, frame_stride, list_stride;
    int   main_blocks, unit_width;
};

constexpr int kListColumns = kWave;         // columns of a workgroup that reads lists; its wavefronts share the entries

__device__ __forceinline__ float exp_scaled(float d, float scale) { return __builtin_amdgcn_exp2f(d * scale); }
// what sums of exponentials are taken against: a maximum of minus infinity (nothing there yet) is not subtracted
__device__ __forceinline__ float reference_of(float m) { return m == -__builtin_inff() ? 0.0f : m; }

// (m, s) of W columns joined with another's
template <int W>
__device__ __forceinline__ void join_sums(float (&m)[W], float (&s)[W], float const (&om)[W], float const (&os)[W], float scale)
{
#pragma unroll
    for (int j = 0; j < W; ++j) {
        float const top = fmaxf(m[j], om[j]), r = reference_of(top);
        s[j] = s[j] * exp_scaled(m[j] - r, scale) + os[j] * exp_scaled(om[j] - r, scale);
        m[j] = top;
    }
}

// over the lanes and wavefronts of a workgroup that hold the same unit; the result is wavefront 0's.  share: 2 * kColShareMax floats
template <int W>
__device__ __forceinline__ void join_workgroup(float (&m)[W], float (&s)[W], int log_tx, float scale, float *share)
{
    int const lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, tx = lane & ((1 << log_tx) - 1);
    for (int o = 1 << log_tx; o < kWave; o <<= 1) {
        float om[W], os[W];
#pragma unroll
        for (int j = 0; j < W; ++j) { om[j] = lane_xor_any(m[j], o); os[j] = lane_xor_any(s[j], o); }
        join_sums<W>(m, s, om, os, scale);
    }
    float *const s_m = share, *const s_s = share + kColShareMax;
    if (lane < (1 << log_tx)) {
#pragma unroll
        for (int j = 0; j < W; ++j) { s_m[(wave * kWave + tx) * W + j] = m[j]; s_s[(wave * kWave + tx) * W + j] = s[j]; }
    }
    __syncthreads();
    if (wave == 0) {
        for (int w = 1; w < kColWaves; ++w) {
            float om[W], os[W];
#pragma unroll
            for (int j = 0; j < W; ++j) { om[j] = s_m[(w * kWave + tx) * W + j]; os[j] = s_s[(w * kWave + tx) * W + j]; }
            join_sums<W>(m, s, om, os, scale);
        }
    }
}

// the lists of 64 columns: four wavefronts share the entries of each
__device__ __forceinline__ void distillation_lists(DistillArgs const &a, int block, float *share)
{
    int const lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    int const column = block * kListColumns + lane, columns = a.pix_size * a.c.frame_size;
    bool const in = column < columns;
    int pix, f;
    split_tile(in ? column : 0, a.frames, pix, f);
    size_t const at = (size_t)pix * a.list_stride + f, entry = (size_t)a.pix_size * a.list_stride;
    size_t const y_at = (size_t)pix * a.frame_stride + f, channel = (size_t)a.pix_size * a.frame_stride;
    float top = -__builtin_inff();
    int entries = 0;
#pragma unroll 4
    for (int j = wave; j < a.top_size; j += kColWaves) {
        bool const valid = (unsigned)a.index[at + j * entry] < (unsigned)a.c.rows;
        float const z = a.logit[at + j * entry];
        entries += valid && !(z == -__builtin_inff()) ? 1 : 0;
        top = fmaxf(top, valid ? z : top);
    }
    share[wave * kWave + lane] = top;
    share[kColShareMax + wave * kWave + lane] = (float)entries;
    __syncthreads();
    float any = 0.0f;
    for (int w = 0; w < kColWaves; ++w) { top = fmaxf(top, share[w * kWave + lane]); any += share[kColShareMax + w * kWave + lane]; }
    __syncthreads();
    float const r = reference_of(top);
    float sum = 0.0f, part = 0.0f;
#pragma unroll 4
    for (int j = wave; j < a.top_size; j += kColWaves) {
        int const c = a.index[at + j * entry];
        float const z = a.logit[at + j * entry];
        bool const valid = (unsigned)c < (unsigned)a.c.rows;
        float const d = z == top ? 0.0f : z - r, e = valid ? exp_scaled(d, a.scale) : 0.0f;
        if (!(e == 0.0f)) {                                                     // (not a number: counts)
            sum += e;
            part = __builtin_fmaf(e, d - a.y[y_at + c * channel], part);
        }
    }
    share[wave * kWave + lane] = sum;
    share[kColShareMax + wave * kWave + lane] = part;
    __syncthreads();
    if (wave == 0 && in) {
        for (int w = 1; w < kColWaves; ++w) { sum += share[w * kWave + lane]; part += share[kColShareMax + w * kWave + lane]; }
        a.lists[(size_t)pix * a.c.units_per_row.count * a.unit_width + f] =
            any > 0.0f ? make_float4(top, 1.0f / sum, part * a.reciprocal_t / sum - logf(sum), 1.0f) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
}

template <int W>
__global__ __launch_bounds__(kColBlock) void distillation_sums_kernel(DistillArgs a)
{
    __shared__ float share[2 * kColShareMax];
    if ((int)blockIdx.x >= a.main_blocks) { distillation_lists(a, (int)blockIdx.x - a.main_blocks, share); return; }       // workgroup-uniform
    ColumnThread<W> const t(a.c, a.tiles, blockIdx.x, a.main_blocks);
    ColumnUnit<W> const u(a.c, (t.tile << a.c.log_tx) + t.tx);
    constexpr int B = 8;
    size_t const channel = (size_t)a.pix_size * a.frame_stride;
    float const *const y = a.y + (size_t)u.pix * a.frame_stride + u.f0;
    float m[W], s[W] = {};
#pragma unroll
    for (int j = 0; j < W; ++j) { m[j] = -__builtin_inff(); }
    for (int r = t.first; r < t.end; r += B * t.step) {
        float v[B][W];
#pragma unroll
        for (int i = 0; i < B; ++i) {
            int const row = r + i * t.step;
            column_load<W>(y + (size_t)(row < t.end ? row : r) * channel, u.live, v[i]);
            if (row >= t.end) {
#pragma unroll
                for (int j = 0; j < W; ++j) { v[i][j] = -__builtin_inff(); }
            }
        }
#pragma unroll
        for (int j = 0; j < W; ++j) {
            float top = m[j];
#pragma unroll
            for (int i = 0; i < B; ++i) { top = fmaxf(top, v[i][j]); }
            float const ref = reference_of(top);
            s[j] *= exp_scaled(m[j] - ref, a.scale);
            m[j] = top;
#pragma unroll
            for (int i = 0; i < B; ++i) { s[j] += exp_scaled(v[i][j] - ref, a.scale); }
        }
    }
    join_workgroup<W>(m, s, a.c.log_tx, a.scale, share);
    if (threadIdx.x < (1u << a.c.log_tx) && u.live > 0) {
        float2 *const partial = a.partial + (size_t)t.slab * (a.c.units * W) + u.column;
#pragma unroll
        for (int j = 0; j < W; ++j) { partial[j] = make_float2(m[j], s[j]); }
    }
}

template <int W>
__global__ __launch_bounds__(kColBlock) void distillation_gradient_kernel(DistillArgs a)
{
    __shared__ float share[2 * kColShareMax];
    __shared__ float of_m[kWave * W], of_s[kWave * W], of_k[kWave * W];         // per column: reference, 1 / sum, w T / weight_sum (0: nothing to learn)
    ColumnThread<W> const t(a.c, a.tiles, blockIdx.x, gridDim.x);
    ColumnUnit<W> const u(a.c, (t.tile << a.c.log_tx) + t.tx);
    int const part = (int)threadIdx.x >> a.c.log_tx, parts = kColBlock >> a.c.log_tx;
    size_t const channel = (size_t)a.pix_size * a.frame_stride, place = (size_t)u.pix * a.frame_stride + u.f0;
    float m[W], s[W] = {};
#pragma unroll
    for (int j = 0; j < W; ++j) { m[j] = -__builtin_inff(); }
    for (int slab = part; slab < a.c.slabs; slab += parts) {
        float2 const *const p = a.partial + (size_t)slab * (a.c.units * W) + u.column;
        float om[W], os[W];
#pragma unroll
        for (int j = 0; j < W; ++j) { float2 const v = p[j]; om[j] = v.x; os[j] = v.y; }
        join_sums<W>(m, s, om, os, a.scale);
    }
    join_workgroup<W>(m, s, a.c.log_tx, a.scale, share);
    if (threadIdx.x < (1u << a.c.log_tx) && u.live > 0) {
        float loss[W];
#pragma unroll
        for (int j = 0; j < W; ++j) {
            float4 const l = a.lists[u.column + j];
            float const w = j < u.live ? (a.weight != nullptr ? a.weight[place + j] : 1.0f) : 0.0f;
            bool const none = l.w == 0.0f || w == 0.0f;
            loss[j] = none ? 0.0f : w * a.t_square * (l.z + (m[j] * a.reciprocal_t + logf(s[j])));
            of_m[t.tx * W + j] = reference_of(m[j]);
            of_s[t.tx * W + j] = 1.0f / s[j];
            of_k[t.tx * W + j] = none ? 0.0f : w * a.coefficient;
        }
        if (t.slab == 0) { column_store<W>(a.loss + place, u.live, loss); }
    }
    __syncthreads();
    float const *const y = a.y + place;
    float *const dy = a.dy + place;
    float ref[W], gain[W];
    bool learns[W];
#pragma unroll
    for (int j = 0; j < W; ++j) {
        float const k = of_k[t.tx * W + j];
        ref[j] = of_m[t.tx * W + j]; gain[j] = k * of_s[t.tx * W + j]; learns[j] = !(k == 0.0f);
    }
    constexpr int B = 4;
    for (int r = t.first; r < t.end; r += B * t.step) {
        float v[B][W];
#pragma unroll
        for (int i = 0; i < B; ++i) { column_load<W>(y + (size_t)(r + i * t.step < t.end ? r + i * t.step : r) * channel, u.live, v[i]); }
#pragma unroll
        for (int i = 0; i < B; ++i) {
            int const row = r + i * t.step;
            if (row < t.end) {
#pragma unroll
                for (int j = 0; j < W; ++j) { v[i][j] = learns[j] ? exp_scaled(v[i][j] - ref[j], a.scale) * gain[j] : 0.0f; }
                column_store<W>(dy + (size_t)row * channel, u.live, v[i]);
            }
        }
    }
    __syncthreads();                                                            // the slab's p is written; the listed channels follow
    int const log_columns = a.c.log_tx + (W == 4 ? 2 : 0), columns = 1 << log_columns, begin = t.slab * a.c.slab_rows;
    size_t const entry = (size_t)a.pix_size * a.list_stride;
    for (int e = threadIdx.x; e < columns * a.top_size; e += kColBlock) {
        int const col = e & (columns - 1), j = e >> log_columns;
        ColumnUnit<W> const at(a.c, (t.tile << a.c.log_tx) + col / W);
        float const k = of_k[col];
        if (col % W >= at.live || k == 0.0f) { continue; }
        int const *const index = a.index + (size_t)at.pix * a.list_stride + at.f0 + col % W;
        int const c = index[j * entry];
        if (c < begin || c >= t.end) { continue; }
        float const *const logit = a.logit + (size_t)at.pix * a.list_stride + at.f0 + col % W;
        float4 const l = a.lists[at.column + col % W];
        float q = 0.0f;
        bool first = true;
        for (int i = 0; i < a.top_size; ++i) {                                  // a channel that the list names twice has both shares, added in the list's order
            if (index[i * entry] == c) {
                first = first && i >= j;
                float const z = logit[i * entry];
                q += exp_scaled(z == l.x ? 0.0f : z - reference_of(l.x), a.scale);
            }
        }
        if (first) {
            size_t const here = (size_t)at.pix * a.frame_stride + at.f0 + col % W + (size_t)c * channel;
            float const p = exp_scaled(a.y[here] - of_m[col], a.scale) * of_s[col];
            a.dy[here] = k * (p - q * l.y);
        }
    }
}

}  // namespace bbhip
