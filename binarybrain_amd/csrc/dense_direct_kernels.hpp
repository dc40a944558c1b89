// Products of dense layers straight from the operands as they lie, in fp32: small problems, and few frames.
//
// dense_direct_kernel: a workgroup owns a tile of 32 x 32 elements; its wavefronts share the k axis (chunks of 32, taken in turn) and add their tiles up through LDS in a fixed order.
// v_mfma_f32_32x32x2_f32 takes one value per lane and operand: lane l holds row l & 31 at the k of its half, l >> 5, so a lane loads 16 consecutive k of one row
// (64 bytes where these are neighbours in memory, 16 times 128 bytes of a half wavefront where rows are) and the 16 instructions of a chunk each take one of them:
// which k meets which in an instruction does not matter as long as both operands agree.  Every product and sum is fp32; no operand is written anywhere.
// What a launch costs is the latency of a chunk's loads and 16 x 64 cycles of matrix instructions per chunk and wavefront; other wavefronts cover the latency (with the next chunk
// held in registers sixteen wavefronts do not fit a compute unit without spilling).  Where there are few tiles and a long k axis several workgroups share it (slabs), and dense_join_kernel
// adds their sums in order.  65 frames of 6144 bits x 1024 outputs take 19 us and 4 to join (25 MB of weights: 5 us; 0.8 GFLOP at 0.15 PFLOP/s: 5.4), a square of 512 over 512 inputs 6.6.
//
// dense_few_frames_kernel: up to eight frames, where a tile of 32 would be mostly empty and the weights are all there is to read.  A wavefront owns an output node and
// walks its row of W 1 KiB at a time, the frames lie in LDS.  1024 x 1024: 4.0 us under a graph, latency; 8192 x 8192 59 us for one frame, 4.6 TB/s of weights, 68 for eight.
#pragma once

#include "dense_operands.hpp"

namespace bbhip {

typedef float DenseAcc __attribute__((ext_vector_type(16)));

constexpr int kDirectTile = 32, kDirectChunk = 32, kDirectRun = 16;

struct DirectProduct {
    Operand     a, b;
    DenseOutput out;
    int n_tiles;                    // tiles side by side
    int tiles;
    int slabs, slab_chunks;         // workgroups that share a tile's k axis
    float *sums;                    // slabs > 1: [slab][m][pitch]
    long long sums_pitch, sums_slab;
    __host__ __device__ int workgroups(void) const { return tiles * slabs; }
};

// An operand from a tile's first row on, as a buffer whose end the loads know: what lies behind it reads as 0, so no load needs a bound of its own, and the code of a chunk stays short (a
// launch of few workgroups waits for its instructions as much as for its data: with bounds per value a backward pass of 330 inputs, 101 outputs and 867 frames took 30 us).
struct TileBuffer { __amdgpu_buffer_rsrc_t r; };
__device__ __forceinline__ TileBuffer tile_buffer(void const *first, long long bytes)
{
    return TileBuffer{__builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(first), 0, (int)(uint32_t)min(bytes, 0xfffffffcLL), 0x00027000)};
}
__device__ __forceinline__ uint32_t load_word(TileBuffer const &b, uint32_t at) { return __builtin_amdgcn_raw_buffer_load_b32(b.r, at, 0, 0); }
__device__ __forceinline__ uint4 load_words(TileBuffer const &b, uint32_t at)
{
    typedef uint32_t V __attribute__((ext_vector_type(4)));
    V const v = __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b128(b.r, at, 0, 0));
    return make_uint4(v.x, v.y, v.z, v.w);
}

// A lane's values of an operand for a chunk: 16 consecutive k of one row.  Behind the last k: columns are behind the buffer's end and read as 0, rows are cleared where `tail`; packed bits
// are some of 0 and 1, which meet a 0 of the other operand.
template <int KIND>
struct RawRun {
    static constexpr int kWords = KIND == kBitRows ? 1 : kDirectRun;
    static constexpr bool kAlongK = KIND == kRows || KIND == kBitRows;
    uint32_t w[kWords];
    float    coef[KIND == kRows ? kDirectRun : 1];

    // the operand from (row0, k0) on (16-byte loads end with the sixteen bytes that the last value lies in)
    static __device__ __forceinline__ TileBuffer buffer(Operand const &o, int row0, int k0)
    {
        uint32_t const *p = static_cast<uint32_t const *>(o.p);
        long long const first = KIND == kRows ? row0 * o.stride + k0 : KIND == kBitRows ? row0 * o.stride + (k0 >> 5) : k0 * o.stride + (KIND == kBitColumns ? row0 >> 5 : row0);
        long long const end = KIND == kRows ? (o.rows - 1) * o.stride + (o.vec ? (o.depth + 3) & ~3 : o.depth) : KIND == kBitRows ? (o.rows - 1) * o.stride + ((o.depth + 31) >> 5) :
                              (o.depth - 1) * o.stride + (KIND == kBitColumns ? (o.rows + 31) >> 5 : o.rows);
        return tile_buffer(p + first, max(end - first, 0LL) * 4);
    }
    // r: the row from row0 on, half: which 16 k
    __device__ __forceinline__ void load(Operand const &o, TileBuffer const &b, int r, int half, int k0)
    {
        uint32_t const pitch = (uint32_t)o.stride * 4;
        if constexpr (KIND == kRows) {
            uint32_t const at = r * pitch + half * 64;
            if (o.vec) {
#pragma unroll
                for (int j = 0; j < kDirectRun; j += 4) {
                    uint4 const q = load_words(b, at + j * 4);
                    w[j] = q.x; w[j + 1] = q.y; w[j + 2] = q.z; w[j + 3] = q.w;
                }
            }
            else {
#pragma unroll
                for (int j = 0; j < kDirectRun; ++j) { w[j] = load_word(b, at + j * 4); }
            }
            if (o.coef) {
                TileBuffer const c = tile_buffer(o.coef + k0, (o.depth - k0) * 4LL);
#pragma unroll
                for (int j = 0; j < kDirectRun; ++j) { coef[j] = __builtin_bit_cast(float, load_word(c, half * 64 + j * 4)); }
            }
        }
        if constexpr (KIND == kColumns || KIND == kBitColumns) {
            uint32_t const at = half * 16 * pitch + (KIND == kColumns ? r * 4 : 0);
#pragma unroll
            for (int j = 0; j < kDirectRun; ++j) { w[j] = load_word(b, at + j * pitch); }
        }
        if constexpr (KIND == kBitRows) { w[0] = load_word(b, r * pitch) >> (half * 16); }
        // (in registers before the first product: the loads overlap)
    }
    __device__ __forceinline__ void clear_behind(Operand const &o, int k)
    {
        if constexpr (KIND == kRows) {
#pragma unroll
            for (int j = 0; j < kDirectRun; ++j) { w[j] = k + j < o.depth ? w[j] : 0u; }
        }
    }
    __device__ __forceinline__ float value(Operand const &o, int r, int j, bool ones) const
    {
        float v;
        if constexpr (KIND == kBitRows)         { v = (float)((w[0] >> j) & 1u); }
        else if constexpr (KIND == kBitColumns) { v = (float)((w[j] >> r) & 1u); }
        else                                    { v = __builtin_bit_cast(float, w[j]); }
        if constexpr (KIND == kRows) { if (o.coef) { v = coef[j] == 0.0f ? 0.0f : v; } }
        return kAlongK && ones ? 1.0f : v;
    }
};

template <int KA, int KB, int WAVES>
__device__ __forceinline__ void direct_product(DirectProduct const &t, int id, float *lds)
{
    int const slab = id / t.tiles, tile = id - slab * t.tiles;
    int const m0 = tile / t.n_tiles * kDirectTile, n0 = (tile % t.n_tiles) * kDirectTile;
    int const lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int const r = lane & 31, half = lane >> 5;
    // (rows behind the last one are 0 or some other value of the buffer: their elements are not stored.  The row of ones meets zeros behind the last k.)
    bool const ones = n0 + r == t.b.ones;
    int const first = slab * t.slab_chunks, chunks = min(first + t.slab_chunks, (t.a.depth + kDirectChunk - 1) / kDirectChunk);
    DenseAcc acc = {};
#pragma nounroll
    for (int c = first + wave; c < chunks; c += WAVES) {
        RawRun<KA> a;
        RawRun<KB> b;
        int const k0 = c * kDirectChunk;
        a.load(t.a, RawRun<KA>::buffer(t.a, m0, k0), r, half, k0);
        b.load(t.b, RawRun<KB>::buffer(t.b, n0, k0), r, half, k0);
        if (k0 + kDirectChunk > t.a.depth) { a.clear_behind(t.a, k0 + half * kDirectRun); b.clear_behind(t.b, k0 + half * kDirectRun); }
#pragma unroll
        for (int j = 0; j < kDirectRun; ++j) { acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.value(t.a, r, j, false), b.value(t.b, r, j, ones), acc, 0, 0, 0); }
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) { lds[(wave * 16 + j) * 64 + lane] = acc[j]; }
    __syncthreads();

    DenseOutput const &o = t.out;
    constexpr int kPer = 16 / WAVES;
    float z[kPer];
    int const n = n0 + r;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        int const reg = e * WAVES + wave;
        float d = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) { d += lds[(w * 16 + reg) * 64 + lane]; }
        int const m = m0 + acc_row(reg, lane);
        bool const inside = m < o.rows && n < o.columns;
        if (t.slabs > 1) {
            if (m < o.rows && (n < o.columns || (n == o.columns && o.line))) { t.sums[slab * t.sums_slab + m * t.sums_pitch + n] = d; }
        }
        else if (o.kind == kOutForward) {
            if (inside) { static_cast<float *>(o.out)[m * o.stride + n] = activated(before_activation(o, d, m, n), o.activation); }
        }
        else if (o.kind == kOutBits) {
            uint64_t const bits = __ballot(inside && before_activation(o, d, inside ? m : 0, inside ? n : 0) > 0.0f);
            if (r == 0 && m < o.rows) { static_cast<uint32_t *>(o.out)[m * o.stride + (n0 >> 5)] = (uint32_t)(bits >> (half * 32)); }
        }
        else if (o.kind == kOutStore) {
            if (m < o.rows && (n < o.columns || (n == o.columns && o.line))) { store_element(o, d, m, n); }
        }
        else {
            z[e] = inside ? before_activation(o, d, m, n) : -INFINITY;
            if (inside) {
                if (o.out) { static_cast<float *>(o.out)[m * o.stride + n] = z[e]; }
                if (o.label[n] == m + o.first_channel) { o.label_logit[n] = z[e]; }
            }
        }
    }
    if (o.kind == kOutLogits && t.slabs == 1) {
        // (largest, sum of exponents) of the tile's rows: of this lane's, the other half's, the other wavefronts'
        float2 s = make_float2(-INFINITY, 0.0f);
#pragma unroll
        for (int e = 0; e < kPer; ++e) { s.x = fmaxf(s.x, z[e]); }
#pragma unroll
        for (int e = 0; e < kPer; ++e) { s.y += z[e] == -INFINITY ? 0.0f : exp_of_nonpositive(z[e] - s.x); }
        s = joined(s, make_float2(__shfl_xor(s.x, 32), __shfl_xor(s.y, 32)));
        __syncthreads();
        float2 *const part = reinterpret_cast<float2 *>(lds);
        if (half == 0) { part[wave * 32 + r] = s; }
        __syncthreads();
        if (threadIdx.x < 32 && n < o.columns) {
#pragma unroll
            for (int w = 1; w < WAVES; ++w) { s = joined(s, part[w * 32 + r]); }
            o.partial[(long long)(m0 / kDirectTile) * o.columns + n] = s;
        }
    }
}

template <int KA, int KB, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void dense_direct_kernel(DirectProduct t)
{
    __shared__ float lds[WAVES * 16 * 64];
    direct_product<KA, KB, WAVES>(t, blockIdx.x, lds);
}

// the weights' gradient (x as KX) and behind it the input's, in one launch; dz as it lies
template <int KX, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void dense_direct_backward_kernel(DirectProduct dw, DirectProduct dx)
{
    __shared__ float lds[WAVES * 16 * 64];
    if ((int)blockIdx.x < dw.workgroups()) { direct_product<kRows, KX, WAVES>(dw, blockIdx.x, lds); }
    else                            { direct_product<kColumns, kColumns, WAVES>(dx, blockIdx.x - dw.workgroups(), lds); }
}

// dz of a call, written: 1024 elements of a row per workgroup, units of a row dealt out by a flat list
struct DzArgs { Operand o; float *dz; long long stride; int per_row; };
__global__ __launch_bounds__(256) void dense_dz_kernel(DzArgs a)
{
    int const row = (int)(blockIdx.x / (unsigned)a.per_row), first = (int)(blockIdx.x % (unsigned)a.per_row) * 1024;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        int const frame = first + i * 256 + threadIdx.x;
        if (frame < a.o.depth) { a.dz[row * a.stride + frame] = operand_at<kGradRows>(a.o, row, frame); }
    }
}

// ---- up to eight frames ---------------------------------------------------------------------------------------------------------------------
constexpr int kFewFrames = 8, kFewWaves = 4, kFewPiece = 1024;             // values of k in LDS at a time

// t.b: columns or packed bits.  A wavefront owns ROWS rows of t.a: what it reads of the frames in LDS serves all of them, and so does what the workgroup reads of the frames, whose values lie
// a row pitch apart.  VEC: lane l takes four neighbouring values of every 256, with one load; else four that lie 64 apart.
template <int KB, int FRAMES, int ROWS, bool VEC>
__global__ __launch_bounds__(kFewWaves * 64) void dense_few_frames_kernel(DirectProduct t)
{
    __shared__ __attribute__((aligned(16))) float x[FRAMES][kFewPiece];
    int const lane = threadIdx.x & 63, m0 = (blockIdx.x * kFewWaves + (threadIdx.x >> 6)) * ROWS;
    Operand const &a = t.a, &b = t.b;
    int const frames = min(FRAMES, b.rows);
    float acc[ROWS][FRAMES] = {};
    for (int k0 = 0; k0 < a.depth; k0 += kFewPiece) {
        int const here = min(kFewPiece, a.depth - k0);
        if (k0) { __syncthreads(); }
        for (int i = threadIdx.x; i < kFewPiece; i += kFewWaves * 64) {
            if constexpr (KB == kBitColumns) {
                uint32_t const bits = i < here ? static_cast<uint32_t const *>(b.p)[(k0 + i) * b.stride] : 0u;
#pragma unroll
                for (int f = 0; f < FRAMES; ++f) { x[f][i] = (float)((bits >> f) & 1u); }
            }
            else if (FRAMES > 1 && b.vec) {
                // (rows of a multiple of four values: the four exist)
#pragma unroll
                for (int f = 0; f < FRAMES; f += 4) {
                    float u[4] = {};
                    if (i < here && f < frames) { load_floats(static_cast<float const *>(b.p) + (k0 + i) * b.stride + f, true, u); }
#pragma unroll
                    for (int h = 0; h < 4; ++h) { if (f + h < FRAMES) { x[f + h < FRAMES ? f + h : 0][i] = f + h < frames ? u[h] : 0.0f; } }
                }
            }
            else {
#pragma unroll
                for (int f = 0; f < FRAMES; ++f) { x[f][i] = i < here && f < frames ? static_cast<float const *>(b.p)[(k0 + i) * b.stride + f] : 0.0f; }
            }
        }
        __syncthreads();
        for (int i = 0; i < here; i += 256) {
            float v[ROWS][4];
#pragma unroll
            for (int q = 0; q < ROWS; ++q) {
                float const *w = static_cast<float const *>(a.p) + min(m0 + q, a.rows - 1) * a.stride + k0 + i;
                if (VEC && i + lane * 4 + 4 <= here) { load_floats(w + lane * 4, true, v[q]); }
                else {
#pragma unroll
                    for (int u = 0; u < 4; ++u) { int const at = VEC ? lane * 4 + u : u * 64 + lane; v[q][u] = i + at < here ? w[at] : 0.0f; }
                }
            }
#pragma unroll
            for (int f = 0; f < FRAMES; ++f) {
                float u[4];
                if (VEC) { load_floats(&x[f][i + lane * 4], true, u); }
                else {
#pragma unroll
                    for (int h = 0; h < 4; ++h) { u[h] = x[f][i + h * 64 + lane]; }
                }
#pragma unroll
                for (int q = 0; q < ROWS; ++q) {
#pragma unroll
                    for (int h = 0; h < 4; ++h) { acc[q][f] = fmaf(v[q][h], u[h], acc[q][f]); }
                }
            }
        }
    }
    DenseOutput const &o = t.out;
#pragma unroll
    for (int q = 0; q < ROWS; ++q) {
        int const m = m0 + q;
#pragma unroll
        for (int f = 0; f < FRAMES; ++f) {
#pragma unroll
            for (int step = 32; step > 0; step /= 2) { acc[q][f] += __shfl_xor(acc[q][f], step); }
        }
        // lane f finishes frame f
        float d = acc[q][0];
#pragma unroll
        for (int f = 1; f < FRAMES; ++f) { d = lane == f ? acc[q][f] : d; }
        bool const inside = m < o.rows && lane < o.columns && lane < FRAMES;
        if (o.kind == kOutBits) {
            uint64_t const bits = __ballot(inside && before_activation(o, d, inside ? m : 0, inside ? lane : 0) > 0.0f);
            if (lane == 0 && m < o.rows) { static_cast<uint32_t *>(o.out)[m * o.stride] = (uint32_t)bits; }
        }
        else if (inside) { static_cast<float *>(o.out)[m * o.stride + lane] = activated(before_activation(o, d, m, lane), o.activation); }
    }
}

}  // namespace bbhip
