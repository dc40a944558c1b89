// Distillation from the logits that a teacher kept.  For every (pixel, frame) with the kept logits z_j of the channels i_j (entries whose channel is
// not one of the layer's are no entries), the student's logits y, the temperature T and the weight w of the place:
//   q_j = exp(z_j / T) / sum_j exp(z_j / T),   p_c = exp(y_c / T) / sum_c exp(y_c / T),
//   loss = w T^2 sum_j q_j (log q_j - log p_{i_j}),   dy_c = w T (p_c - sum_{j : i_j = c} q_j) / weight_sum.
// An entry of minus infinity has no share and is passed over wherever entries are counted: by the table of channels named twice, and by the launch that
// takes the shares off dy, where it would be a second writer of a channel that an entry with a share names.  A place without entries (or whose kept logits are all minus infinity) and one with w = 0 has loss 0 and gradient 0 whatever its logits are.
//
// Two launches.  The first takes, per column and slab of channels, the running maximum m and the sum of exp((y - m) / T) in one pass; workgroups behind
// those read the lists and leave per column the largest z, the reciprocal of their sum E, the largest listed logit y_r of the student, and
//   sum_j q_j ((z_j - z_max) - (y_{i_j} - y_r)) / T - log E,
// to which the second launch adds  log sum_c exp((y_c - y_r) / T)  to have the loss: differences of nearby logits throughout.  A hash table in LDS tells
// whether a list names a channel twice.  The second launch joins the slabs and writes dy: first p for every channel of its slab, then, behind a
// barrier, the few channels of the lists.  Exponents are taken of differences to the maximum, (y - m) * (log2 e / T): the rounding of the product
// grows with the distance from the maximum and weighs as little as the term itself.
// 32768 channels x 2048 frames, lists of 64: sums 44 us = 6.1 TB/s, gradient 112 us = 4.8 TB/s (a copy 5.1): the logits pass the fabric twice.  Up to 32 channels a lane
// holds a whole column and one launch does all (21 channels x 66560 places 41.6 -> 9.3 us).
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
    float4      *lists;             // [units * W]: (z_max, 1 / E (0: no entries, sign bit set: a channel is named twice), the lists' part of the loss, y_r)
    float scale;                    // log2(e) / T
    float reciprocal_t, t_square, coefficient;      // 1 / T, T^2, T / weight_sum
    int   top_size, pix_size, frame_stride, list_stride;
    int   main_blocks, unit_width;
};

constexpr int kListColumns = 4;                                 // columns of a workgroup that reads lists; 64 threads share the entries of each
constexpr int kListParts   = kColBlock / kListColumns;
constexpr int kListHeld    = 256 / kListParts;                  // entries of a thread (lists of up to 256)
constexpr int kListSlots   = 512;                               // hash table of a column: twice the longest list
constexpr int kFoundMost   = 16 * kColBlock;                     // entries that a workgroup looks at at a time
constexpr int kDistillShare = 4 * kColBlock + kListSlots * kListColumns;        // floats: the sums of a tile, or the lists' values and tables
static_assert(kDistillShare >= 2 * kColShareMax, "both uses fit");

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
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        if (o >= 1 << log_tx) {                                                 // workgroup-uniform
            float om[W], os[W];
#pragma unroll
            for (int j = 0; j < W; ++j) { om[j] = lane_xor(m[j], o); os[j] = lane_xor(s[j], o); }
            join_sums<W>(m, s, om, os, scale);
        }
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

// the lists of a few columns.  slots: kListSlots * kListColumns
__device__ __forceinline__ void distillation_lists(DistillArgs const &a, int block, float *share, int *slots)
{
    int const col = threadIdx.x % kListColumns, part = threadIdx.x / kListColumns;
    int const column = block * kListColumns + col, columns = a.pix_size * a.c.frame_size;
    bool const in = column < columns;
    int pix, f;
    split_tile(in ? column : 0, a.frames, pix, f);
    size_t const at = (size_t)pix * a.list_stride + f, entry = (size_t)a.pix_size * a.list_stride;
    size_t const y_at = (size_t)pix * a.frame_stride + f, channel = (size_t)a.pix_size * a.frame_stride;
    for (int s = threadIdx.x; s < kListSlots * kListColumns; s += kColBlock) { slots[s] = -1; }
    float z[kListHeld], y[kListHeld];
    int c[kListHeld];
#pragma unroll
    for (int i = 0; i < kListHeld; ++i) {
        int const j = i * kListParts + part;
        c[i] = -1; z[i] = 0.0f;
        if (i * kListParts < a.top_size && j < a.top_size) { c[i] = a.index[at + j * entry]; z[i] = a.logit[at + j * entry]; }
    }
    float top = -__builtin_inff(), near = -__builtin_inff(), any = 0.0f;
#pragma unroll
    for (int i = 0; i < kListHeld; ++i) {
        y[i] = 0.0f;
        if (i * kListParts < a.top_size) {                                      // workgroup-uniform
            bool const valid = (unsigned)c[i] < (unsigned)a.c.rows && !(z[i] == -__builtin_inff());
            c[i] = valid ? c[i] : -1;
            if (valid) { y[i] = a.y[y_at + c[i] * channel]; any = 1.0f; }
        }
    }
#pragma unroll
    for (int i = 0; i < kListHeld; ++i) {
        top  = c[i] >= 0 ? fmaxf(top, z[i]) : top;
        near = c[i] >= 0 ? fmaxf(near, y[i]) : near;
    }
    __syncthreads();                                                            // (the table is empty)
    float twice = 0.0f;
#pragma unroll
    for (int i = 0; i < kListHeld; ++i) {
        if (c[i] >= 0) {
            unsigned slot = ((unsigned)c[i] * 2654435761u) >> 23;               // (of 512; at most 256 of them are ever taken, so the search ends)
            for (;;) {
                int const there = atomicCAS(&slots[slot * kListColumns + col], -1, c[i]);
                if (there == -1) { break; }
                if (there == c[i]) { twice = 1.0f; break; }
                slot = (slot + 1) % kListSlots;
            }
        }
    }
    // over the threads of a column: its lanes of a wavefront, then the wavefronts
    int const wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
#pragma unroll
    for (int o = kListColumns; o < kWave; o <<= 1) {
        top = fmaxf(top, lane_xor(top, o)); near = fmaxf(near, lane_xor(near, o));
        any = fmaxf(any, lane_xor(any, o)); twice = fmaxf(twice, lane_xor(twice, o));
    }
    float4 *const of_wave = reinterpret_cast<float4 *>(share);                  // [kColWaves][kListColumns]
    if (lane < kListColumns) { of_wave[wave * kListColumns + lane] = make_float4(top, near, any, twice); }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kColWaves; ++w) {
        float4 const o = of_wave[w * kListColumns + col];
        top = fmaxf(top, o.x); near = fmaxf(near, o.y); any = fmaxf(any, o.z); twice = fmaxf(twice, o.w);
    }
    float const r = reference_of(top), yr = reference_of(near);
    float sum = 0.0f, loss = 0.0f;
#pragma unroll
    for (int i = 0; i < kListHeld; ++i) {
        float const d = z[i] == top ? 0.0f : z[i] - r, e = c[i] >= 0 ? exp_scaled(d, a.scale) : 0.0f;
        if (!(e == 0.0f)) {                                                     // (not a number: counts)
            sum += e;
            loss = __builtin_fmaf(e, d - (y[i] - yr), loss);
        }
    }
#pragma unroll
    for (int o = kListColumns; o < kWave; o <<= 1) { sum += lane_xor(sum, o); loss += lane_xor(loss, o); }
    __syncthreads();
    if (lane < kListColumns) { of_wave[wave * kListColumns + lane] = make_float4(sum, loss, 0.0f, 0.0f); }
    __syncthreads();
    if (part == 0 && in) {
        sum = 0.0f; loss = 0.0f;
        for (int w = 0; w < kColWaves; ++w) { sum += of_wave[w * kListColumns + col].x; loss += of_wave[w * kListColumns + col].y; }
        float const q = any > 0.0f ? 1.0f / sum : 0.0f;
        a.lists[(size_t)pix * a.c.units_per_row.count * a.unit_width + f] = make_float4(top, __builtin_copysignf(q, twice > 0.0f ? -1.0f : 1.0f), loss * a.reciprocal_t / sum - logf(sum), yr);
    }
}

template <int W>
__global__ __launch_bounds__(kColBlock) void distillation_sums_kernel(DistillArgs a)
{
    __shared__ __align__(16) float share[kDistillShare];
    if ((int)blockIdx.x >= a.main_blocks) {                                     // workgroup-uniform
        distillation_lists(a, (int)blockIdx.x - a.main_blocks, share, reinterpret_cast<int *>(share + 4 * kColBlock));
        return;
    }
    ColumnThread<W> const t(a.c, a.tiles, blockIdx.x, a.main_blocks);
    ColumnUnit<W> const u(a.c, (t.tile << a.c.log_tx) + t.tx);
    constexpr int B = 8;
    size_t const channel = (size_t)a.pix_size * a.frame_stride;
    float const *const y = a.y + (size_t)u.pix * a.frame_stride + u.f0 + (size_t)t.lead * channel;
    float m[W], s[W] = {};
#pragma unroll
    for (int j = 0; j < W; ++j) { m[j] = -__builtin_inff(); }
    t.template each<B>([&](int base, auto whole) {
        float v[B][W];
#pragma unroll
        for (int i = 0; i < B; ++i) {
            if (whole || base + t.lead + i * t.step < t.end) { column_load<W>(y + (size_t)(base + i * t.step) * channel, v[i]); }
            else {
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
    });
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
    __shared__ int found;
    __shared__ uint16_t found_entry[kFoundMost];                                // listed channels of the slab (a tile has at most 2^16 entries)
    __shared__ float of_m[kWave * W], of_s[kWave * W], of_k[kWave * W];         // per column: reference, 1 / sum, w T / weight_sum (0: nothing to learn)
    ColumnThread<W> const t(a.c, a.tiles, backwards(blockIdx.x, gridDim.x), gridDim.x);
    ColumnUnit<W> const u(a.c, (t.tile << a.c.log_tx) + t.tx);
    int const part = (int)threadIdx.x >> a.c.log_tx, parts = kColBlock >> a.c.log_tx;
    size_t const channel = (size_t)a.pix_size * a.frame_stride, place = (size_t)u.pix * a.frame_stride + u.f0;
    float const *const y = a.y + place + (size_t)t.lead * channel;
    constexpr int B = 4;
    struct Held { float v[B][W]; } held;
    auto const start = [&](int base, Held &h) {
#pragma unroll
        for (int i = 0; i < B; ++i) {
            if (base + t.lead + i * t.step < t.end) { column_load<W>(y + (size_t)(base + i * t.step) * channel, h.v[i]); }
        }
    };
    start(t.begin, held);
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
            bool const none = l.y == 0.0f || w == 0.0f;
            loss[j] = none ? 0.0f : w * a.t_square * (l.z + ((m[j] - l.w) * a.reciprocal_t + logf(s[j])));
            of_m[t.tx * W + j] = reference_of(m[j]);
            of_s[t.tx * W + j] = 1.0f / s[j];
            of_k[t.tx * W + j] = none ? 0.0f : w * a.coefficient;
        }
        if (t.slab == 0) { column_store<W>(a.loss + place, u.live, loss); }
    }
    __syncthreads();
    float *const dy = a.dy + place + (size_t)t.lead * channel;
    float ref[W], gain[W];
    bool learns[W];
#pragma unroll
    for (int j = 0; j < W; ++j) {
        float const k = of_k[t.tx * W + j];
        ref[j] = of_m[t.tx * W + j]; gain[j] = k * of_s[t.tx * W + j]; learns[j] = !(k == 0.0f);
    }
    t.template follow<B>(held, start, [&](int base, Held &h) {
#pragma unroll
        for (int i = 0; i < B; ++i) {
            if (base + t.lead + i * t.step < t.end) {
#pragma unroll
                for (int j = 0; j < W; ++j) { h.v[i][j] = learns[j] ? exp_scaled(h.v[i][j] - ref[j], a.scale) * gain[j] : 0.0f; }
                column_store<W>(dy + (size_t)(base + i * t.step) * channel, u.live, h.v[i]);
            }
        }
    });
    int const log_columns = a.c.log_tx + (W == 4 ? 2 : 0), columns = 1 << log_columns, begin = t.slab * a.c.slab_rows;
    size_t const entry = (size_t)a.pix_size * a.list_stride;
    // A slab holds few of a list's channels: those are gathered first, so that each of the loads that they need is waited for once and not once per entry looked at
    // (32768 channels x 2048 frames, lists of 64: 130 us entry by entry).
    for (int e0 = 0; e0 < columns * a.top_size; e0 += kFoundMost) {             // workgroup-uniform
        if (threadIdx.x == 0) { found = 0; }
        __syncthreads();
        int c[kFoundMost / kColBlock];
#pragma unroll
        for (int i = 0; i < kFoundMost / kColBlock; ++i) {
            int const e = e0 + i * kColBlock + threadIdx.x, col = e & (columns - 1), j = e >> log_columns;
            ColumnUnit<W> const at(a.c, (t.tile << a.c.log_tx) + col / W);
            c[i] = -1;
            if (e < columns * a.top_size && col % W < at.live) { c[i] = a.index[(size_t)at.pix * a.list_stride + at.f0 + col % W + j * entry]; }
        }
#pragma unroll
        for (int i = 0; i < kFoundMost / kColBlock; ++i) {
            if (c[i] >= begin && c[i] < t.end) { found_entry[atomicAdd(&found, 1)] = (uint16_t)(e0 + i * kColBlock + threadIdx.x); }
        }
        // (the store below comes after the one of p above, of another wavefront perhaps: behind a wait for it and a barrier)
        __builtin_amdgcn_s_waitcnt(0x0f70);                                     // vmcnt(0)
        __syncthreads();
        for (int h = threadIdx.x; h < found; h += kColBlock) {
            int const e = found_entry[h], col = e & (columns - 1), j = e >> log_columns;
            float const k = of_k[col];
            if (k == 0.0f) { continue; }
            ColumnUnit<W> const at(a.c, (t.tile << a.c.log_tx) + col / W);
            int const c = a.index[(size_t)at.pix * a.list_stride + at.f0 + col % W + j * entry];
            float const *const logit = a.logit + (size_t)at.pix * a.list_stride + at.f0 + col % W;
            size_t const here = (size_t)at.pix * a.frame_stride + at.f0 + col % W + (size_t)c * channel;
            float4 const l = a.lists[at.column + col % W];
            float const z = logit[j * entry], yc = a.y[here];
            bool const shares = !(z == -__builtin_inff());                      // (else: what stands there is right, or another entry's thread writes it)
            auto weight = [&](float v) { return exp_scaled(v == l.x ? 0.0f : v - reference_of(l.x), a.scale); };
            float q = weight(z);
            if (shares && __builtin_signbitf(l.y)) {                            // a channel may be named twice: its shares are added in the list's order, by its first entry's thread
                int const *const index = a.index + (size_t)at.pix * a.list_stride + at.f0 + col % W;
                int first = a.top_size;
                q = 0.0f;
                for (int o = 0; o < a.top_size; ++o) {
                    float const zo = logit[o * entry];
                    if (index[o * entry] == c && !(zo == -__builtin_inff())) {
                        first = first < o ? first : o;
                        q += weight(zo);
                    }
                }
                if (first != j) { continue; }
            }
            if (shares) { a.dy[here] = k * (exp_scaled(yc - of_m[col], a.scale) * of_s[col] - q * fabsf(l.y)); }
        }
        __syncthreads();
    }
}

// Few channels (at most MOST): a lane takes a column, its logits and the shares of the list in registers.
constexpr int kDistillFew = 32;
template <int MOST>
__global__ __launch_bounds__(kWave) void distillation_few_kernel(DistillArgs a)
{
    ColumnUnit<1> const u(a.c, blockIdx.x * kWave + threadIdx.x);               // (a lane without a column: the first one's, and nothing is stored)
    size_t const channel = (size_t)a.pix_size * a.frame_stride, place = (size_t)u.pix * a.frame_stride + u.f0;
    size_t const entry = (size_t)a.pix_size * a.list_stride, at = (size_t)u.pix * a.list_stride + u.f0;
    float y[MOST], q[MOST];
#pragma unroll
    for (int i = 0; i < MOST; ++i) { y[i] = a.y[place + (i < a.c.rows ? i : 0) * channel]; q[i] = 0.0f; }
    float const w = a.weight != nullptr ? a.weight[place] : 1.0f;
    float top = -__builtin_inff();
    bool any = false;
#pragma unroll 4
    for (int j = 0; j < a.top_size; ++j) {
        bool const valid = (unsigned)a.index[at + j * entry] < (unsigned)a.c.rows;
        float const z = a.logit[at + j * entry];
        any = any || (valid && !(z == -__builtin_inff()));
        top = valid ? fmaxf(top, z) : top;
    }
    float const r = reference_of(top);
    float sum = 0.0f, entropy = 0.0f;
#pragma unroll 4
    for (int j = 0; j < a.top_size; ++j) {
        int const c = a.index[at + j * entry];
        float const z = a.logit[at + j * entry], d = z == top ? 0.0f : z - r;
        float const e = (unsigned)c < (unsigned)a.c.rows ? exp_scaled(d, a.scale) : 0.0f;
        sum += e;
        entropy = e == 0.0f ? entropy : __builtin_fmaf(e, d, entropy);
#pragma unroll
        for (int i = 0; i < MOST; ++i) { q[i] += c == i ? e : 0.0f; }
    }
    float m = -__builtin_inff(), s = 0.0f;
#pragma unroll
    for (int i = 0; i < MOST; ++i) { m = i < a.c.rows ? fmaxf(m, y[i]) : m; }
    float const ref = reference_of(m);
    float loss = entropy;
#pragma unroll
    for (int i = 0; i < MOST; ++i) {
        float const d = y[i] - ref;
        loss = q[i] == 0.0f ? loss : __builtin_fmaf(q[i], -d, loss);
        y[i] = exp_scaled(d, a.scale);
        s += i < a.c.rows ? y[i] : 0.0f;
    }
    bool const none = !any || w == 0.0f;
    float const gain = w * a.coefficient, to_p = 1.0f / s, to_q = 1.0f / sum;
    if (u.live > 0) {
        a.loss[place] = none ? 0.0f : w * a.t_square * (loss * a.reciprocal_t * to_q - logf(sum) + logf(s));
#pragma unroll
        for (int i = 0; i < MOST; ++i) {
            if (i < a.c.rows) { a.dy[place + i * channel] = none ? 0.0f : gain * (y[i] * to_p - q[i] * to_q); }
        }
    }
}

}  // namespace bbhip
