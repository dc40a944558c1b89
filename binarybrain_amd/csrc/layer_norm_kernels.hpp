// LayerNormalization: every frame is normalised over all nodes of its layer, then each node is mapped by its own gamma and beta:
//   mean = sum_n x / N,  var = sum_n (x - mean)^2 / N,  rstd = 1 / sqrt(var + eps),  y = ((x - mean) rstd) gamma_n + beta_n
// and backward, with xh = (x - mean) rstd and g = dy gamma_n:
//   dgamma_n = sum_f dy xh,  dbeta_n = sum_f dy,  dx = rstd (g - sum_n g / N - xh (sum_n g xh) / N).
// The statistics are sums down the columns of the buffer (column_tiles.hpp), the weights' gradients sums along its rows.
//
// Means and squared deviations are formed over eight rows at a time and merged pairwise with their counts (the update of Chan, Golub and
// LeVeque), so a mean that is large against the deviation costs no digits; packed bits are counted, and their squared deviation is
// ones * zeros / N.  Squares are summed in 32 bits; the square of what float32 holds need not be one itself (values around 1e20 or, with eps 0, deviations of
// 1e-25), and where a frame's sum leaves the range its deviations are read and squared again in 64 bits.  (Squares of 64 bits throughout cost 4 to 9 % of small calls.)
// All sums are taken in a fixed order: the same input gives the same bits on every run.
//
// Columns that a workgroup can hold go in one launch (forward; layer_norm_whole in launch_rules.hpp has both sides).  Any other size goes in two: the sums of a slab of rows per workgroup (forward: mean and squared deviation; backward: the two sums per
// frame and, of the same reading, the two sums per node over the tile's frames), then every workgroup adds up the slabs of its frames and writes.
// 4096 nodes x 8192 frames, inputs not in the caches: forward 57 us = 4.7 TB/s (135 MB read, 135 written; one workgroup per compute unit reads, waits and writes in turn), backward 118 us
// (42 + 64 with what fits in the memory-side cache): 640 MB through the fabric at 6 TB/s, of which 403 would do if x and dy were read once.
#pragma once

#include "column_tiles.hpp"

namespace bbhip {

struct LayerNormArgs {
    ColumnSpace c;
    TileDivisor tiles;              // of one slab
    void const  *x;                 // fp32 frames or packed words
    float const *dy;                // backward
    float       *out;               // y or dx
    float const *gamma, *beta;      // NULL: 1 and 0
    float       *mean, *rstd;       // forward: written unless NULL; backward: read
    float2      *partial;           // [slabs][units * W]: forward (mean, squared deviation; negative: less the root of its mean) or (ones, -), backward (sum g, sum g xh)
    float2      *row_partial;       // [tiles][rows]: (sum dy xh, sum dy)
    float       *dgamma, *dbeta;    // backward
    double inverse_rows;            // forward
    float eps, reciprocal_rows;
    int   x_stride, out_stride;     // (dy has the pitch of dx)
    int   accumulate;               // dgamma, dbeta: added to
    int   main_blocks;              // backward's second launch: workgroups that write dx, behind them those that close the rows' sums
};

// W values of row `r` of a unit
template <int W, bool BIT>
__device__ __forceinline__ void layer_norm_load(void const *__restrict__ x, int stride, int r, int f0, float (&v)[W])
{
    if constexpr (BIT) {
        uint32_t const word = static_cast<uint32_t const *>(x)[(size_t)r * stride + (f0 >> 5)] >> (f0 & 31);
#pragma unroll
        for (int j = 0; j < W; ++j) { v[j] = (float)((word >> j) & 1u); }
    }
    else { column_load<W>(static_cast<float const *>(x) + (size_t)r * stride + f0, v); }
}

// t = m 4^half with m in [0.5, 2), so that a root is taken in 32 bits whatever the size of t (0, infinities and what is not a number: half 0)
__device__ __forceinline__ float mantissa_of(double t, int &half)
{
    int const e = __builtin_amdgcn_frexp_exp(t) & ~1;
    half = e / 2;
    return (float)__builtin_amdgcn_ldexp(t, -e);
}
__device__ __forceinline__ float root_of(double t)         { int half; float const m = mantissa_of(t, half); return __builtin_amdgcn_ldexpf(sqrtf(m), half); }
__device__ __forceinline__ float inverse_root_of(double t) { int half; float const m = mantissa_of(t, half); return __builtin_amdgcn_ldexpf(1.0f / sqrtf(m), -half); }

// A variance (with eps) of this range comes from 32 bits: what underflows in its sum (2^-149 a square) is nothing to it, and nothing has overflowed.
constexpr float kVarianceLeast = 0x1p-90f, kVarianceMost = 0x1p120f;
__device__ __forceinline__ bool variance_in_range(float t) { return !(t < kVarianceLeast || t > kVarianceMost); }      // (what is not a number stays it)
// A slab's sum of squares beyond this is formed again.  It does not get there while no thread's own sum and mean, of 256 or 1024 threads and at most 2^24 rows, are beyond these.
constexpr float kSquaresMost = 0x1p110f, kThreadSquares = 0x1p98f, kThreadMean = 0x1p40f;

// count, mean and squared deviation of W columns
template <int W>
struct Moments {
    float n = 0.0f, mean[W] = {}, m2[W] = {};
    // (the other's share of the count is 0 where both are empty)
    __device__ __forceinline__ void merge(float on, float const (&omean)[W], float const (&om2)[W])
    {
        float const total = n + on, share = total > 0.0f ? on / total : 0.0f, weight = n * share;
#pragma unroll
        for (int j = 0; j < W; ++j) {
            float const d = omean[j] - mean[j];
            mean[j] = __builtin_fmaf(d, share, mean[j]);
            m2[j]   = __builtin_fmaf(d * weight, d, m2[j] + om2[j]);         // (weight 0: nothing, whatever d * d would be)
        }
        n = total;
    }
};

constexpr int kColShareMax = kColWaves * kWave * 4;     // floats: one value per wavefront and column of the widest tile

// over the lanes and wavefronts of a workgroup that hold the same unit; the result is wavefront 0's.  share: 2 * kColShareMax + kColWaves * kWave floats
template <int W>
__device__ __forceinline__ void merge_workgroup(Moments<W> &m, int log_tx, float *share)
{
    int const lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, tx = lane & ((1 << log_tx) - 1);
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        if (o >= 1 << log_tx) {                                                 // workgroup-uniform
            float om[W], o2[W];
            float const on = lane_xor(m.n, o);
#pragma unroll
            for (int j = 0; j < W; ++j) { om[j] = lane_xor(m.mean[j], o); o2[j] = lane_xor(m.m2[j], o); }
            m.merge(on, om, o2);
        }
    }
    float *const s_mean = share, *const s_m2 = share + kColShareMax, *const s_n = share + 2 * kColShareMax;
    if (lane < (1 << log_tx)) {
        s_n[wave * kWave + tx] = m.n;
#pragma unroll
        for (int j = 0; j < W; ++j) { s_mean[(wave * kWave + tx) * W + j] = m.mean[j]; s_m2[(wave * kWave + tx) * W + j] = m.m2[j]; }
    }
    __syncthreads();
    if (wave == 0) {
        for (int w = 1; w < kColWaves; ++w) {
            float om[W], o2[W];
#pragma unroll
            for (int j = 0; j < W; ++j) { om[j] = s_mean[(w * kWave + tx) * W + j]; o2[j] = s_m2[(w * kWave + tx) * W + j]; }
            m.merge(s_n[w * kWave + tx], om, o2);
        }
    }
}

// the same for two plain sums
template <int W>
__device__ __forceinline__ void add_workgroup(float (&a)[W], float (&b)[W], int log_tx, float *share)
{
    int const lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, tx = lane & ((1 << log_tx) - 1);
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        if (o >= 1 << log_tx) {                                                 // workgroup-uniform
#pragma unroll
            for (int j = 0; j < W; ++j) { a[j] += lane_xor(a[j], o); b[j] += lane_xor(b[j], o); }
        }
    }
    float *const s_a = share, *const s_b = share + kColShareMax;
    if (lane < (1 << log_tx)) {
#pragma unroll
        for (int j = 0; j < W; ++j) { s_a[(wave * kWave + tx) * W + j] = a[j]; s_b[(wave * kWave + tx) * W + j] = b[j]; }
    }
    __syncthreads();
    if (wave == 0) {
        for (int w = 1; w < kColWaves; ++w) {
#pragma unroll
            for (int j = 0; j < W; ++j) { a[j] += s_a[(w * kWave + tx) * W + j]; b[j] += s_b[(w * kWave + tx) * W + j]; }
        }
    }
}

constexpr int kLayerNormBatch = 8;      // rows that a thread has in flight

// The end of a slab that may have columns whose squares leave the range of 32 bits: theirs are summed in 64 about the slab's mean (wavefront 0's m), the rows are read again.
// A column's result goes by its own values alone: those in range keep the bits that they have elsewhere.
template <int W>
__device__ __forceinline__ void layer_norm_stats_far(LayerNormArgs const &a, ColumnThread<W> const &t, ColumnUnit<W> const &u, Moments<W> const &m, float *share)
{
    int const lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, columns = W << a.c.log_tx;       // (no more than threads)
    __syncthreads();                                                            // (the sums in `share` have been read)
    if (threadIdx.x < (1u << a.c.log_tx)) {
#pragma unroll
        for (int j = 0; j < W; ++j) { share[t.tx * W + j] = m.mean[j]; share[kColShareMax + t.tx * W + j] = m.m2[j]; }
    }
    __syncthreads();
    float mean[W];
    double s[W] = {};
#pragma unroll
    for (int j = 0; j < W; ++j) { mean[j] = share[t.tx * W + j]; }
    float const of_column = share[threadIdx.x], m2 = share[kColShareMax + threadIdx.x];                // (of column threadIdx.x, if there is one)
    float const *const x = static_cast<float const *>(a.x) + u.f0;
#pragma unroll 1
    for (int row = t.begin + t.lead; row < t.end; row += t.step) {
        float v[W];
        column_load<W>(x + (size_t)row * a.x_stride, v);
#pragma unroll
        for (int j = 0; j < W; ++j) { double const d = (double)(v[j] - mean[j]); s[j] = __builtin_fma(d, d, s[j]); }
    }
    __syncthreads();                                                            // (all have their means)
    double *const sums = reinterpret_cast<double *>(share);                     // [kColWaves][columns]
#pragma unroll
    for (int j = 0; j < W; ++j) {
        for (int o = 1 << a.c.log_tx; o < kWave; o <<= 1) { s[j] += __shfl_xor(s[j], o); }
        if (lane < (1 << a.c.log_tx)) { sums[wave * columns + t.tx * W + j] = s[j]; }
    }
    __syncthreads();
    if ((int)threadIdx.x < columns && (t.tile << a.c.log_tx) + (int)threadIdx.x / W < a.c.units) {
        double all = 0.0;
        for (int w = 0; w < kColWaves; ++w) { all += sums[w * columns + threadIdx.x]; }
        float const n = (float)(t.end - t.begin);
        bool const out = m2 > kSquaresMost || (a.eps < kVarianceLeast && m2 < kVarianceLeast * n);
        a.partial[(size_t)t.slab * (a.c.units * W) + ((size_t)t.tile << a.c.log_tx) * W + threadIdx.x] = make_float2(of_column, out ? -root_of(all / (double)n) : m2);
    }
}

// mean and squared deviation (packed bits: the ones) of every column over a slab
template <int W, bool BIT>
__global__ __launch_bounds__(kColBlock) void layer_norm_stats_kernel(LayerNormArgs a)
{
    __shared__ __align__(16) float share[2 * kColShareMax + kColWaves * kWave];
    __shared__ int far[kColWaves];
    ColumnThread<W> const t(a.c, a.tiles, blockIdx.x, gridDim.x);
    ColumnUnit<W> const u(a.c, (t.tile << a.c.log_tx) + t.tx);
    constexpr int B = kLayerNormBatch;
    float2 *const partial = a.partial + (size_t)t.slab * (a.c.units * W) + u.column;
    bool const writes = threadIdx.x < (1u << a.c.log_tx) && u.live > 0;

    if constexpr (BIT) {
        float ones[W] = {}, none[W] = {};
        t.template each<B>([&](int base, auto whole) {
            float v[B][W];
#pragma unroll
            for (int i = 0; i < B; ++i) {
                int const row = base + t.lead + i * t.step;
                layer_norm_load<W, true>(a.x, a.x_stride, whole || row < t.end ? row : t.begin, u.f0, v[i]);
            }
#pragma unroll
            for (int i = 0; i < B; ++i) {
                bool const in = whole || base + t.lead + i * t.step < t.end;
#pragma unroll
                for (int j = 0; j < W; ++j) { ones[j] += in ? v[i][j] : 0.0f; }
            }
        });
        add_workgroup<W>(ones, none, a.c.log_tx, share);
        if (writes) {
#pragma unroll
            for (int j = 0; j < W; ++j) { partial[j] = make_float2(ones[j], 0.0f); }
        }
    }
    else {
        Moments<W> m;
        t.template each<B>([&](int base, auto whole) {
            float v[B][W], n = 0.0f;
#pragma unroll
            for (int i = 0; i < B; ++i) {
                int const row = base + t.lead + i * t.step;
                bool const in = whole || row < t.end;
                layer_norm_load<W, false>(a.x, a.x_stride, in ? row : t.begin, u.f0, v[i]);      // (an absent row: another, which counts for nothing)
                n += in ? 1.0f : 0.0f;
            }
            float const rn = whole ? 1.0f / B : n > 0.0f ? 1.0f / n : 0.0f;
            float mean[W], m2[W];
#pragma unroll
            for (int j = 0; j < W; ++j) {
                float s = 0.0f, q = 0.0f;
#pragma unroll
                for (int i = 0; i < B; ++i) { s += whole || base + t.lead + i * t.step < t.end ? v[i][j] : 0.0f; }
                mean[j] = s * rn;
#pragma unroll
                for (int i = 0; i < B; ++i) {
                    float const d = whole || base + t.lead + i * t.step < t.end ? v[i][j] - mean[j] : 0.0f;
                    q = __builtin_fmaf(d, d, q);
                }
                m2[j] = q;
            }
            m.merge(n, mean, m2);
        });
        bool beyond = false;
#pragma unroll
        for (int j = 0; j < W; ++j) { beyond = beyond || (j < u.live && (m.m2[j] > kThreadSquares || fabsf(m.mean[j]) > kThreadMean)); }
        beyond = __any(beyond);
        if (threadIdx.x % kWave == 0) { far[threadIdx.x / kWave] = beyond ? 1 : 0; }
        merge_workgroup<W>(m, a.c.log_tx, share);
        if (a.eps < kVarianceLeast) {                                           // (small sums count, too: those of the whole slab are wavefront 0's)
            bool low = false;
#pragma unroll
            for (int j = 0; j < W; ++j) { low = low || (writes && j < u.live && m.m2[j] < kVarianceLeast * (float)(t.end - t.begin)); }
            if (low) { far[0] = 1; }
            __syncthreads();
        }
        int some = 0;
#pragma unroll
        for (int w = 0; w < kColWaves; ++w) { some |= far[w]; }
        if (some != 0) {                                                        // workgroup-uniform
            layer_norm_stats_far<W>(a, t, u, m, share);
            return;
        }
        if (writes) {
#pragma unroll
            for (int j = 0; j < W; ++j) { partial[j] = make_float2(m.mean[j], m.m2[j]); }
        }
    }
}

// rstd of a column whose variance is beyond the range of 32 bits: its slabs joined in 64.  partial: its entry of the first slab
__device__ __forceinline__ float layer_norm_join_far(LayerNormArgs const &a, float2 const *partial, size_t pitch)
{
    double n = 0.0, mean = 0.0, m2 = 0.0;
#pragma unroll 1
    for (int s = 0; s < a.c.slabs; ++s) {
        float2 const p = partial[s * pitch];
        int const left = a.c.rows - s * a.c.slab_rows;
        double const on = (double)(left < a.c.slab_rows ? left : a.c.slab_rows), d = (double)p.x - mean, share = on / (n + on);
        m2 += (p.y < 0.0f ? (double)p.y * (double)p.y * on : (double)p.y) + d * d * (n * share);
        mean += d * share;
        n += on;
    }
    return inverse_root_of(__builtin_fma(m2, a.inverse_rows, (double)a.eps));
}

// y, from the slabs' sums; the workgroups of the first slab write mean and rstd
template <int W, bool BIT>
__global__ __launch_bounds__(kColBlock) void layer_norm_apply_kernel(LayerNormArgs a)
{
    __shared__ float share[2 * kColShareMax + kColWaves * kWave];
    ColumnThread<W> const t(a.c, a.tiles, backwards(blockIdx.x, gridDim.x), gridDim.x);
    ColumnUnit<W> const u(a.c, (t.tile << a.c.log_tx) + t.tx);
    constexpr int B = 4;
    struct Held { float v[B][W], g[B], b[B]; } held;
    auto const start = [&](int base, Held &h) {
#pragma unroll
        for (int i = 0; i < B; ++i) {
            int const row = base + t.lead + i * t.step;
            if (row < t.end) {
                layer_norm_load<W, BIT>(a.x, a.x_stride, row, u.f0, h.v[i]);
                h.g[i] = a.gamma != nullptr ? a.gamma[row] : 1.0f;
                h.b[i] = a.beta != nullptr ? a.beta[row] : 0.0f;
            }
        }
    };
    start(t.begin, held);
    int const part = (int)threadIdx.x >> a.c.log_tx, parts = kColBlock >> a.c.log_tx;
    Moments<W> m;
    float ones[W] = {}, none[W] = {};
    for (int s = part; s < a.c.slabs; s += parts) {
        float2 const *const p = a.partial + (size_t)s * (a.c.units * W) + u.column;
        int const left = a.c.rows - s * a.c.slab_rows;
        float mean[W], m2[W];
#pragma unroll
        for (int j = 0; j < W; ++j) { float2 const v = p[j]; mean[j] = v.x; m2[j] = v.y; }
        if constexpr (BIT) {
#pragma unroll
            for (int j = 0; j < W; ++j) { ones[j] += mean[j]; }
        }
        else {
#pragma unroll
            for (int j = 0; j < W; ++j) { m2[j] = m2[j] < 0.0f ? __builtin_inff() : m2[j]; }            // (formed in 64 bits: below)
            m.merge((float)(left < a.c.slab_rows ? left : a.c.slab_rows), mean, m2);
        }
    }
    if constexpr (BIT) { add_workgroup<W>(ones, none, a.c.log_tx, share); }
    else               { merge_workgroup<W>(m, a.c.log_tx, share); }
    __syncthreads();                                                            // (the partial sums in `share` have been read)
    if (threadIdx.x < (1u << a.c.log_tx)) {
        float var[W], of[W];
        bool beyond = false;
#pragma unroll
        for (int j = 0; j < W; ++j) {
            float mean;
            if constexpr (BIT) {
                float const rows = (float)a.c.rows;
                mean = ones[j] / rows;
                var[j] = mean * ((rows - ones[j]) / rows);
            }
            else { mean = m.mean[j]; var[j] = m.m2[j] / (float)a.c.rows; beyond = beyond || !variance_in_range(var[j] + a.eps); }
            share[t.tx * W + j] = mean;
            of[j] = 1.0f / sqrtf(var[j] + a.eps);
        }
        if (beyond) {
#pragma unroll
            for (int j = 0; j < W; ++j) {
                if (!variance_in_range(var[j] + a.eps)) { of[j] = layer_norm_join_far(a, a.partial + u.column + j, (size_t)a.c.units * W); }
            }
        }
#pragma unroll
        for (int j = 0; j < W; ++j) { share[kColShareMax + t.tx * W + j] = of[j]; }
    }
    __syncthreads();
    float mean[W], rstd[W];
#pragma unroll
    for (int j = 0; j < W; ++j) { mean[j] = share[t.tx * W + j]; rstd[j] = share[kColShareMax + t.tx * W + j]; }
    if (t.slab == 0 && threadIdx.x < (1u << a.c.log_tx)) {
        if (a.mean != nullptr) { column_store<W>(a.mean + u.f0, u.live, mean); }
        if (a.rstd != nullptr) { column_store<W>(a.rstd + u.f0, u.live, rstd); }
    }
    t.template follow<B>(held, start, [&](int base, Held &h) {
#pragma unroll
        for (int i = 0; i < B; ++i) {
            int const row = base + t.lead + i * t.step;
            if (row < t.end) {
#pragma unroll
                for (int j = 0; j < W; ++j) { h.v[i][j] = __builtin_fmaf((h.v[i][j] - mean[j]) * rstd[j], h.g[i], h.b[i]); }
                column_store<W>(a.out + (size_t)row * a.out_stride + u.f0, u.live, h.v[i]);
            }
        }
    });
}

// Forward pass in one launch, for columns that a workgroup of 1024 threads can hold, R = 4 or 16 rows of a unit per thread: x is read once and the mean is known before
// the deviations are squared.  Packed bits are held as their words.  The squares are summed in 32 bits; where a thread's sum shows that a total might leave
// their range, or a variance is so small that squares below it count, the workgroup sums them again in 64.
constexpr int kWholeBlock = 1024, kWholeWaves = kWholeBlock / kWave;

// the sum over the threads that hold the same unit, in every thread.  share: kWholeWaves * kWave * W floats
template <int W>
__device__ __forceinline__ void whole_sum(float (&v)[W], int log_tx, float *share)
{
    int const lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, tx = lane & ((1 << log_tx) - 1);
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        if (o >= 1 << log_tx) {                                                 // workgroup-uniform
#pragma unroll
            for (int j = 0; j < W; ++j) { v[j] += lane_xor(v[j], o); }
        }
    }
    if (lane < (1 << log_tx)) {
#pragma unroll
        for (int j = 0; j < W; ++j) { share[((wave << log_tx) + tx) * W + j] = v[j]; }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < W; ++j) { v[j] = 0.0f; }
#pragma unroll
    for (int w = 0; w < kWholeWaves; ++w) {
        float o[W];
        column_load<W>(share + ((w << log_tx) + tx) * W, o);
#pragma unroll
        for (int j = 0; j < W; ++j) { v[j] += o[j]; }
    }
}

// The same of one frame of a unit in 64 bits, for the rare call: few registers, so that the common one keeps its own.  share: kWholeWaves * kWave doubles, in use before
__device__ __forceinline__ double whole_sum_double(double v, int log_tx, double *share)
{
    int const lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, tx = lane & ((1 << log_tx) - 1);
    for (int o = 1 << log_tx; o < kWave; o <<= 1) { v += __shfl_xor(v, o); }
    __syncthreads();
    if (lane < (1 << log_tx)) { share[(wave << log_tx) + tx] = v; }
    __syncthreads();
    v = 0.0;
#pragma unroll 1
    for (int w = 0; w < kWholeWaves; ++w) { v += share[(w << log_tx) + tx]; }
    return v;
}

// The rest of the pass for a workgroup with frames whose squares leave the range of 32 bits: theirs are summed in 64, x is read again.  A frame's result goes by its own
// values alone: those in range have the bits that they have elsewhere.  (Behind a return, so that the common call keeps its registers.)
template <int W>
__device__ __forceinline__ void layer_norm_whole_far(LayerNormArgs const &a, ColumnUnit<W> const &u, int ty, int step, float (&mean)[W], float (&var)[W], float (&rstd)[W],
                                                     double *share)
{
    float const *const x = static_cast<float const *>(a.x) + u.f0;
    double s[W] = {};
#pragma unroll 1
    for (int row = ty; row < a.c.rows; row += step) {
        float v[W];
        column_load<W>(x + (size_t)row * a.x_stride, v);
#pragma unroll
        for (int j = 0; j < W; ++j) { double const d = (double)(v[j] - mean[j]); s[j] = __builtin_fma(d, d, s[j]); }
    }
#pragma unroll
    for (int j = 0; j < W; ++j) {
        double const all = whole_sum_double(s[j], a.c.log_tx, share);
        if (!variance_in_range(var[j] + a.eps)) { rstd[j] = inverse_root_of(__builtin_fma(all, a.inverse_rows, (double)a.eps)); }
    }
    if (ty == 0) {
        if (a.mean != nullptr) { column_store<W>(a.mean + u.f0, u.live, mean); }
        if (a.rstd != nullptr) { column_store<W>(a.rstd + u.f0, u.live, rstd); }
    }
#pragma unroll 1
    for (int row = ty; row < a.c.rows; row += step) {
        float const g = a.gamma != nullptr ? a.gamma[row] : 1.0f, b = a.beta != nullptr ? a.beta[row] : 0.0f;
        float v[W];
        column_load<W>(x + (size_t)row * a.x_stride, v);
#pragma unroll
        for (int j = 0; j < W; ++j) { v[j] = __builtin_fmaf((v[j] - mean[j]) * rstd[j], g, b); }
        column_store<W>(a.out + (size_t)row * a.out_stride + u.f0, u.live, v);
    }
}

template <int W, int R, bool BIT>
__global__ __launch_bounds__(kWholeBlock) void layer_norm_whole_kernel(LayerNormArgs a)
{
    __shared__ __align__(16) float share[2][kWholeBlock * W];
    __shared__ int far;
    int const tx = threadIdx.x & ((1 << a.c.log_tx) - 1), ty = (int)threadIdx.x >> a.c.log_tx, step = kWholeBlock >> a.c.log_tx;
    ColumnUnit<W> const u(a.c, (xcd_remap(blockIdx.x, gridDim.x) << a.c.log_tx) + tx);
    float const rows = (float)a.c.rows;
    float v[BIT ? 1 : R][W], mean[W] = {}, q[W] = {};
    uint32_t bits[BIT ? R : 1];
    float const *const mine = static_cast<float const *>(a.x) + (size_t)ty * a.x_stride + u.f0;        // (what is common to a load is added to it in scalar registers)
#pragma unroll
    for (int i = 0; i < R; ++i) {
        int const row = ty + i * step;
        if constexpr (BIT) { bits[i] = row < a.c.rows ? static_cast<uint32_t const *>(a.x)[(size_t)row * a.x_stride + (u.f0 >> 5)] : 0u; }
        else {
            if (row < a.c.rows) { column_load<W>(mine + (size_t)(i * step) * a.x_stride, v[i]); }
            else {
#pragma unroll
                for (int j = 0; j < W; ++j) { v[i][j] = 0.0f; }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
#pragma unroll
        for (int j = 0; j < W; ++j) {
            if constexpr (BIT) { mean[j] += (float)((bits[i] >> ((u.f0 & 31) + j)) & 1u); }
            else               { mean[j] += v[i][j]; }
        }
    }
    if (threadIdx.x == 0) { far = 0; }                                          // (set behind the barrier in the first sum)
    whole_sum<W>(mean, a.c.log_tx, share[0]);
#pragma unroll
    for (int j = 0; j < W; ++j) { mean[j] /= rows; }
    if constexpr (BIT) {
#pragma unroll
        for (int j = 0; j < W; ++j) { q[j] = mean[j] * (1.0f - mean[j]); }
    }
    else {
#pragma unroll
        for (int i = 0; i < R; ++i) {
#pragma unroll
            for (int j = 0; j < W; ++j) {
                float const d = ty + i * step < a.c.rows ? v[i][j] - mean[j] : 0.0f;
                q[j] = __builtin_fmaf(d, d, q[j]);
            }
        }
        bool beyond = false;
#pragma unroll
        for (int j = 0; j < W; ++j) { beyond = beyond || (j < u.live && q[j] > kThreadSquares); }
        if (beyond) { far = 1; }
        whole_sum<W>(q, a.c.log_tx, share[1]);
#pragma unroll
        for (int j = 0; j < W; ++j) { q[j] /= rows; }
    }
    float rstd[W];
#pragma unroll
    for (int j = 0; j < W; ++j) { rstd[j] = 1.0f / sqrtf(q[j] + a.eps); }
    if constexpr (!BIT) {
        if (a.eps < kVarianceLeast) {                                           // (small variances count, too)
            bool low = false;
#pragma unroll
            for (int j = 0; j < W; ++j) { low = low || (j < u.live && q[j] + a.eps < kVarianceLeast); }
            if (low) { far = 1; }
            __syncthreads();
        }
        if (far != 0) {                                                         // workgroup-uniform
            layer_norm_whole_far<W>(a, u, ty, step, mean, q, rstd, reinterpret_cast<double *>(&share[0][0]));
            return;
        }
    }
    if (ty == 0) {
        if (a.mean != nullptr) { column_store<W>(a.mean + u.f0, u.live, mean); }
        if (a.rstd != nullptr) { column_store<W>(a.rstd + u.f0, u.live, rstd); }
    }
    int ry = ty;
    asm volatile("" : "+v"(ry));                                                // (the rows' numbers are formed again: kept over the sums they cost registers that do not suffice: 4096 x 8192 54.5 us and 50.5)
    float *const out = a.out + (size_t)ry * a.out_stride + u.f0;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        int const row = ry + i * step;
        if (row < a.c.rows) {
            float const g = a.gamma != nullptr ? a.gamma[row] : 1.0f, b = a.beta != nullptr ? a.beta[row] : 0.0f;
            float y[W];
#pragma unroll
            for (int j = 0; j < W; ++j) {
                float const x = BIT ? (float)((bits[BIT ? i : 0] >> ((u.f0 & 31) + j)) & 1u) : v[BIT ? 0 : i][j];
                y[j] = __builtin_fmaf((x - mean[j]) * rstd[j], g, b);
            }
            column_store<W, R <= 4>(out + (size_t)(i * step) * a.out_stride, u.live, y);
        }
    }
}

// backward, first launch: per column of the slab sum g and sum g xh, per row of the tile sum dy xh and sum dy
template <int W, bool BIT>
__global__ __launch_bounds__(kColBlock) void layer_norm_backward_sums_kernel(LayerNormArgs a)
{
    __shared__ float share[2 * kColShareMax];
    ColumnThread<W> const t(a.c, a.tiles, blockIdx.x, gridDim.x);
    ColumnUnit<W> const u(a.c, (t.tile << a.c.log_tx) + t.tx);
    constexpr int B = 4;
    float mean[W], rstd[W], c1[W] = {}, c2[W] = {};
    line_load<W>(a.mean + u.f0, u.live, mean);
    line_load<W>(a.rstd + u.f0, u.live, rstd);
    t.template each<B>([&](int base, auto whole) {
        float x[B][W], d[B][W], g[B], s1[B], s2[B];
#pragma unroll
        for (int i = 0; i < B; ++i) {
            int const there = base + t.lead + i * t.step, row = whole || there < t.end ? there : t.begin;
            layer_norm_load<W, BIT>(a.x, a.x_stride, row, u.f0, x[i]);
            column_load<W>(a.dy + (size_t)row * a.out_stride + u.f0, d[i]);
            g[i] = a.gamma != nullptr ? a.gamma[row] : 1.0f;
        }
#pragma unroll
        for (int i = 0; i < B; ++i) {
            bool const in = whole || base + t.lead + i * t.step < t.end;                // (what is not there adds nothing)
            s1[i] = 0.0f; s2[i] = 0.0f;
#pragma unroll
            for (int j = 0; j < W; ++j) {
                float const dj = in && j < u.live ? d[i][j] : 0.0f, xh = in && j < u.live ? (x[i][j] - mean[j]) * rstd[j] : 0.0f, gd = dj * g[i];
                c1[j] += gd;
                c2[j] = __builtin_fmaf(gd, xh, c2[j]);
                s1[i] = __builtin_fmaf(dj, xh, s1[i]);
                s2[i] += dj;
            }
        }
        if (a.row_partial != nullptr) {
#pragma unroll
            for (int o = 1; o < kWave; o <<= 1) {
                if (o < 1 << a.c.log_tx) {                                      // workgroup-uniform
#pragma unroll
                    for (int i = 0; i < B; ++i) { s1[i] += lane_xor(s1[i], o); s2[i] += lane_xor(s2[i], o); }
                }
            }
            if (t.tx == 0) {
#pragma unroll
                for (int i = 0; i < B; ++i) {
                    int const row = base + t.lead + i * t.step;
                    if (whole || row < t.end) { a.row_partial[(size_t)t.tile * a.c.rows + row] = make_float2(s1[i], s2[i]); }
                }
            }
        }
    });
    add_workgroup<W>(c1, c2, a.c.log_tx, share);
    if (threadIdx.x < (1u << a.c.log_tx) && u.live > 0) {
        float2 *const partial = a.partial + (size_t)t.slab * (a.c.units * W) + u.column;
#pragma unroll
        for (int j = 0; j < W; ++j) { partial[j] = make_float2(c1[j], c2[j]); }
    }
}

// backward, second launch: dx; the workgroups behind main_blocks add up the tiles' sums of 64 rows each
template <int W, bool BIT>
__global__ __launch_bounds__(kColBlock) void layer_norm_backward_apply_kernel(LayerNormArgs a)
{
    __shared__ float share[2 * kColShareMax];
    int const lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    if ((int)blockIdx.x >= a.main_blocks) {                                      // workgroup-uniform
        int const row = ((int)blockIdx.x - a.main_blocks) * kWave + lane, from = row < a.c.rows ? row : a.c.rows - 1;
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll 8
        for (int tile = wave; tile < a.c.tiles; tile += kColWaves) {
            float2 const p = a.row_partial[(size_t)tile * a.c.rows + from];
            s1 += p.x; s2 += p.y;
        }
        share[wave * kWave + lane] = s1;
        share[kColShareMax + wave * kWave + lane] = s2;
        __syncthreads();
        if (wave == 0 && row < a.c.rows) {
            for (int w = 1; w < kColWaves; ++w) { s1 += share[w * kWave + lane]; s2 += share[kColShareMax + w * kWave + lane]; }
            if (a.dgamma != nullptr) { a.dgamma[row] = a.accumulate ? a.dgamma[row] + s1 : s1; }
            if (a.dbeta != nullptr)  { a.dbeta[row]  = a.accumulate ? a.dbeta[row] + s2 : s2; }
        }
        return;
    }
    ColumnThread<W> const t(a.c, a.tiles, backwards(blockIdx.x, a.main_blocks), a.main_blocks);
    ColumnUnit<W> const u(a.c, (t.tile << a.c.log_tx) + t.tx);
    constexpr int B = 4;
    struct Held { float x[B][W], d[B][W], g[B]; } held;
    auto const start = [&](int base, Held &h) {
#pragma unroll
        for (int i = 0; i < B; ++i) {
            int const row = base + t.lead + i * t.step;
            if (row < t.end) {
                layer_norm_load<W, BIT>(a.x, a.x_stride, row, u.f0, h.x[i]);
                column_load<W>(a.dy + (size_t)row * a.out_stride + u.f0, h.d[i]);
                h.g[i] = a.gamma != nullptr ? a.gamma[row] : 1.0f;
            }
        }
    };
    start(t.begin, held);
    int const part = (int)threadIdx.x >> a.c.log_tx, parts = kColBlock >> a.c.log_tx;
    float mean[W], rstd[W], c1[W] = {}, c2[W] = {};
    line_load<W>(a.mean + u.f0, u.live, mean);
    line_load<W>(a.rstd + u.f0, u.live, rstd);
    for (int s = part; s < a.c.slabs; s += parts) {
        float2 const *const p = a.partial + (size_t)s * (a.c.units * W) + u.column;
#pragma unroll
        for (int j = 0; j < W; ++j) { float2 const v = p[j]; c1[j] += v.x; c2[j] += v.y; }
    }
    add_workgroup<W>(c1, c2, a.c.log_tx, share);
    __syncthreads();
    if (threadIdx.x < (1u << a.c.log_tx)) {
#pragma unroll
        for (int j = 0; j < W; ++j) { share[t.tx * W + j] = c1[j] * a.reciprocal_rows; share[kColShareMax + t.tx * W + j] = c2[j] * a.reciprocal_rows; }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < W; ++j) { c1[j] = share[t.tx * W + j]; c2[j] = share[kColShareMax + t.tx * W + j]; }
    t.template follow<B>(held, start, [&](int base, Held &h) {
#pragma unroll
        for (int i = 0; i < B; ++i) {
            int const row = base + t.lead + i * t.step;
            if (row < t.end) {
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    float const xh = (h.x[i][j] - mean[j]) * rstd[j];
                    h.d[i][j] = rstd[j] * (__builtin_fmaf(h.d[i][j], h.g[i], -c1[j]) - xh * c2[j]);
                }
                column_store<W>(a.out + (size_t)row * a.out_stride + u.f0, u.live, h.d[i]);
            }
        }
    });
}

}  // namespace bbhip
