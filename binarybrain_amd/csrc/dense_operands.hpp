// What the products of dense layers read and write, element by element: operands as they lie in frame buffers, gradients formed while they are read, and what
// is done with a finished element of the product.
//
// Every product here is  D[m][n] = sum over k of A(m, k) * B(n, k):
//   forward        z[o][f]  = sum over i of W[o][i] * x[i][f]          m = output, n = frame, k = input
//   input gradient dx[i][f] = sum over o of W[o][i] * dz[o][f]         m = input,  n = frame, k = output
//   weights        dW[o][i] = sum over f of dz[o][f] * x[i][f]         m = output, n = input, k = frame
// An operand's values at consecutive k are neighbours in memory (rows) or a row pitch apart (columns), fp32 or packed bits, and dz is formed from dy and y, or
// from logits, where it is read.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace bbhip {

// activation(z) and its derivative from its value: relu z > 0, sigmoid y * (1 - y), hard tanh inside (-1, 1) as HardTanh has it
enum DenseActivation : int { kActNone = 0, kActRelu = 1, kActSigmoid = 2, kActHardTanh = 3, kActCount = 4, kGradSoftmax = 4 };

enum OperandKind : int {
    kRows        = 0,       // p[row * stride + k]
    kColumns     = 1,       // p[k * stride + row]
    kBitRows     = 2,       // bit k & 31 of word p[row * stride + (k >> 5)]
    kBitColumns  = 3,       // bit row & 31 of word p[k * stride + (row >> 5)]
    kGradRows    = 4,       // dz of (channel row, frame k)
    kGradColumns = 5,       // dz of (channel k, frame row)
};

struct Operand {
    void const  *p;                 // values or words; gradients: dy, or logits
    float const *y;                 // gradients: the activation's values, rows like p's
    long long stride;               // elements from row to row of the buffer
    int   rows, depth;              // how many there are of row and k
    int   mode;                     // gradients: an activation, or kGradSoftmax
    int   vec;                      // rows: 16-byte loads are aligned
    int   ones;                     // a row behind the last one whose values are all 1 (-1: none)
    // of frames (kGradSoftmax): the largest logit, the coefficient over the sum of exponents, the coefficient (0: the frame does not count), the label.
    // kRows with coef: k is a frame, and one that does not count reads as 0 whatever it holds.
    float const *top, *share, *coef;
    int const   *label;
    int   first;                    // channel of the first row (a piece of the channels)
};

// exp(d) for d <= 0 to about an ulp: the product with log2(e) in two parts (one part alone is off by |d| half steps).  Below -150 it is 0 in fp32; so
// is minus infinity, whose two parts would cancel to NaN.
__device__ __forceinline__ float exp_of_nonpositive(float d)
{
    d = d < -150.0f ? -150.0f : d;
    float const t = d * 1.44269502f;
    float const r = fmaf(d, 1.44269502f, -t) + d * 1.92596303e-8f;
    float const e = __builtin_amdgcn_exp2f(t);
    return fmaf(e, r * 0.693147182f, e);
}

__device__ __forceinline__ float activated(float z, int activation)
{
    if (activation == kActRelu)     { return z <= 0.0f ? 0.0f : z; }
    if (activation == kActSigmoid)  { float const e = exp_of_nonpositive(-fabsf(z)); return (z < 0.0f ? e : 1.0f) / (1.0f + e); }
    if (activation == kActHardTanh) { return z <= -1.0f ? -1.0f : z >= 1.0f ? 1.0f : z; }
    return z;
}

// behind a closed activation dy counts as 0 whatever it is
__device__ __forceinline__ float gradient_through(float dy, float y, int activation)
{
    if (activation == kActRelu)     { return y <= 0.0f ? 0.0f : dy; }
    if (activation == kActSigmoid)  { return dy * (y * (1.0f - y)); }
    if (activation == kActHardTanh) { return (y <= -1.0f || y >= 1.0f) ? 0.0f : dy; }
    return dy;
}

// coef * (softmax(z)[channel] - [channel is the label]); share = coef / sum of exponents.  The exponent is of the difference to the largest logit: with log(sum) in one
// number the difference would be off by the rounding of a number as large as the logits.
__device__ __forceinline__ float softmax_gradient(float z, float top, float share, float coef, int label, int channel)
{
    if (coef == 0.0f) { return 0.0f; }
    float const p = exp_of_nonpositive(z - top) * share;
    return channel == label ? p - coef : p;
}

template <int KIND>
__device__ __forceinline__ float operand_at(Operand const &o, int row, int k)
{
    if constexpr (KIND == kRows) {
        if (row == o.ones) { return 1.0f; }
        if (o.coef && o.coef[k] == 0.0f) { return 0.0f; }
        return static_cast<float const *>(o.p)[row * o.stride + k];
    }
    if constexpr (KIND == kColumns) { return static_cast<float const *>(o.p)[k * o.stride + row]; }
    if constexpr (KIND == kBitRows) {
        if (row == o.ones) { return 1.0f; }
        return (float)((static_cast<uint32_t const *>(o.p)[row * o.stride + (k >> 5)] >> (k & 31)) & 1u);
    }
    if constexpr (KIND == kBitColumns) { return (float)((static_cast<uint32_t const *>(o.p)[k * o.stride + (row >> 5)] >> (row & 31)) & 1u); }
    if constexpr (KIND == kGradRows || KIND == kGradColumns) {
        int const channel = KIND == kGradRows ? row : k, frame = KIND == kGradRows ? k : row;
        long long const at = channel * o.stride + frame;
        float const v = static_cast<float const *>(o.p)[at];
        if (o.mode == kGradSoftmax) { return softmax_gradient(v, o.top[frame], o.share[frame], o.coef[frame], o.label[frame], channel + o.first); }
        return o.mode == kActNone ? v : gradient_through(v, o.y[at], o.mode);
    }
}

template <int N>
__device__ __forceinline__ void load_floats(float const *p, bool vec, float (&v)[N])
{
    if (vec) {
#pragma unroll
        for (int j = 0; j < N; j += 4) {
            float4 const q = *reinterpret_cast<float4 const *>(p + j);
            v[j] = q.x; v[j + 1] = q.y; v[j + 2] = q.z; v[j + 3] = q.w;
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < N; ++j) { v[j] = p[j]; }
}

// Values at k, k + 1, ... of a row; behind the last one the last one again, whose use the caller undoes.  `vec`: all exist, and 16-byte loads are aligned.
template <class T, int N>
__device__ __forceinline__ void load_run(T const *p, int k, int depth, bool vec, T (&v)[N])
{
    if (vec) {
#pragma unroll
        for (int j = 0; j < N; j += 4) {
            uint4 const q = *reinterpret_cast<uint4 const *>(p + k + j);
            v[j] = __builtin_bit_cast(T, q.x); v[j + 1] = __builtin_bit_cast(T, q.y); v[j + 2] = __builtin_bit_cast(T, q.z); v[j + 3] = __builtin_bit_cast(T, q.w);
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < N; ++j) { v[j] = p[min(k + j, depth - 1)]; }
}

// the same where consecutive k are a row pitch apart
template <class T, int N>
__device__ __forceinline__ void load_column(T const *p, long long stride, int left, T (&v)[N])
{
    if (left >= N) {
#pragma unroll
        for (int j = 0; j < N; ++j) { v[j] = p[j * stride]; }
        return;
    }
#pragma unroll
    for (int j = 0; j < N; ++j) { v[j] = *p; p += j + 1 < left ? stride : 0; }
}

// gradient_through without a branch (the activation is the same for all)
__device__ __forceinline__ float gradient_of(float dy, float y, int activation)
{
    bool const closed = (activation == kActRelu && y <= 0.0f) || (activation == kActHardTanh && (y <= -1.0f || y >= 1.0f));
    float const slope = activation == kActSigmoid ? y * (1.0f - y) : 1.0f;
    return closed ? 0.0f : dy * slope;
}

// N values from k on, k a multiple of N (8); 0 behind the last one.  The row and the first value exist.  Gradients through an activation take one path for whole and cut runs: the callers unroll this, and a launch
// waits for its code first (with a path per value for cut runs and a branch per value for the activation the packing of a backward pass over 1024 x 1001 x 1000 took 15.0 us instead of 12.0, of
// 4096 x 4096 x 8192 369 instead of 355; values that are only read lose more by the bounds, 14.9 us and 13.4 for 784 x 6144 x 1024).
template <int KIND, int N>
__device__ __forceinline__ void load_values(Operand const &o, int row, int k, float (&v)[N])
{
    int const left = o.depth - k;
    bool const whole = left >= N;
    if (!whole && ((KIND != kGradRows && KIND != kGradColumns) || o.mode == kGradSoftmax)) {
#pragma unroll
        for (int j = 0; j < N; ++j) { v[j] = k + j < o.depth ? operand_at<KIND>(o, row, k + j) : 0.0f; }
        return;
    }
    if constexpr (KIND == kRows) {
        load_run(static_cast<float const *>(o.p) + row * o.stride, k, o.depth, o.vec, v);
        if (o.coef) {
            float c[N];
            load_run(o.coef, k, o.depth, true, c);
#pragma unroll
            for (int j = 0; j < N; ++j) { v[j] = c[j] == 0.0f ? 0.0f : v[j]; }
        }
    }
    if constexpr (KIND == kColumns) { load_column(static_cast<float const *>(o.p) + k * o.stride + row, o.stride, N, v); }
    if constexpr (KIND == kBitRows) {
        uint32_t const w = static_cast<uint32_t const *>(o.p)[row * o.stride + (k >> 5)] >> (k & 31);
#pragma unroll
        for (int j = 0; j < N; ++j) { v[j] = (float)((w >> j) & 1u); }
    }
    if constexpr (KIND == kBitColumns) {
        uint32_t w[N];
        load_column(static_cast<uint32_t const *>(o.p) + k * o.stride + (row >> 5), o.stride, N, w);
#pragma unroll
        for (int j = 0; j < N; ++j) { v[j] = (float)((w[j] >> (row & 31)) & 1u); }
    }
    if constexpr (KIND == kGradRows) {
        long long const at = row * o.stride;
        load_run(static_cast<float const *>(o.p) + at, k, o.depth, o.vec && whole, v);
        if (o.mode == kGradSoftmax) {
            float top[N], share[N], coef[N];
            load_run(o.top, k, o.depth, true, top); load_run(o.share, k, o.depth, true, share); load_run(o.coef, k, o.depth, true, coef);
#pragma unroll
            for (int j = 0; j < N; ++j) { v[j] = softmax_gradient(v[j], top[j], share[j], coef[j], o.label[k + j], row + o.first); }
        }
        else if (o.mode != kActNone) {
            float y[N];
            load_run(o.y + at, k, o.depth, o.vec && whole, y);
#pragma unroll
            for (int j = 0; j < N; ++j) { v[j] = gradient_of(v[j], y[j], o.mode); }
        }
    }
    if constexpr (KIND == kGradColumns) {
        long long const at = k * o.stride + row;
        load_column(static_cast<float const *>(o.p) + at, o.stride, left, v);
        if (o.mode == kGradSoftmax) {
            float const top = o.top[row], share = o.share[row], coef = o.coef[row];
            int const label = o.label[row];
#pragma unroll
            for (int j = 0; j < N; ++j) { v[j] = softmax_gradient(v[j], top, share, coef, label, k + j + o.first); }
        }
        else if (o.mode != kActNone) {
            float y[N];
            load_column(o.y + at, o.stride, left, y);
#pragma unroll
            for (int j = 0; j < N; ++j) { v[j] = gradient_of(v[j], y[j], o.mode); }
        }
    }
    if (!whole) {
#pragma unroll
        for (int j = 0; j < N; ++j) { v[j] = j < left ? v[j] : 0.0f; }
    }
}

// Row of element `reg` of lane `lane` in the result of a 32 x 32 matrix instruction; the column is lane & 31.
__device__ __forceinline__ int acc_row(int reg, int lane) { return (reg & 3) + 8 * (reg >> 2) + 4 * (lane >> 5); }

// ---- what becomes of an element of the product -----------------------------------------------------------------------------------------
enum DenseOutputKind : int {
    kOutForward = 0,        // y = activation(D + bias + residual)
    kOutBits    = 1,        // bit = D + bias + residual > 0
    kOutStore   = 2,        // D, written or added; the column behind the last one goes to `line`
    kOutLogits  = 3,        // D + bias, written if asked for; largest and sum of exponents of the tile's rows per column, the label's logit
};

struct DenseOutput {
    int   kind;
    int   rows, columns;            // of D (without the column of `line`)
    void *out;                      // fp32 rows or words (kOutLogits: may be null)
    long long stride;
    float const *bias;              // null: none
    float const *residual;          // null: none; rows of residual_stride
    long long residual_stride;
    int   activation;
    int   accumulate;
    float *line;
    float2 *partial;                // kOutLogits: [tiles of rows][columns]
    int const *label;
    float *label_logit;
    int   first_channel;            // kOutLogits: channel of row 0 (a piece of the channels)
    int   channels;                 // kOutLogits: of all pieces
    float const *weight;            // kOutLogits: of the frames (null: 1)
};

// kOutLogits: whether anything is made of a frame's logits
__device__ __forceinline__ bool frame_counts(DenseOutput const &o, int n)
{
    int const label = o.label[n];
    return label >= 0 && label < o.channels && !(o.weight && o.weight[n] == 0.0f);
}

__device__ __forceinline__ float before_activation(DenseOutput const &o, float d, int m, int n)
{
    if (o.bias)     { d += o.bias[m]; }
    if (o.residual) { d += o.residual[m * o.residual_stride + n]; }
    return d;
}

__device__ __forceinline__ void store_element(DenseOutput const &o, float d, int m, int n)
{
    float *to = n == o.columns ? o.line + m : static_cast<float *>(o.out) + m * o.stride + n;
    *to = o.accumulate ? *to + d : d;
}

// ---- largest and sum of exponents, joined --------------------------------------------------------------------------------------------------
// (largest, sum of exp(z - largest)); nothing yet: (-inf, 0)
__device__ __forceinline__ float2 joined(float2 a, float2 b)
{
    float const top = fmaxf(a.x, b.x);
    // (a side without any sum adds nothing; its largest may be minus infinity, whose difference to itself is no number)
    float const sa = a.y == 0.0f ? 0.0f : a.y * exp_of_nonpositive(a.x - top), sb = b.y == 0.0f ? 0.0f : b.y * exp_of_nonpositive(b.x - top);
    return make_float2(top, sa + sb);
}

}  // namespace bbhip
