// Products of dense layers on the fp16 matrix instructions, to the accuracy of fp32: large problems.
//
// A value v of an operand's row is scaled by a power of two that brings the largest of its row to 2^15 and more, as far as halves hold it, and split into two halves, v 2^e = h + l with
// h = fp16(v 2^e), l = fp16(v 2^e - h): 22 bits, so that  a b = (ah bh + ah bl + al bh) 2^-(ea + eb)  up to 3 * 2^-22 of a product at most (the product of the two lower halves is left
// out) and about 2^-24 on the average: what rounding the factors to fp32 would cost.  The matrix instruction multiplies halves exactly and sums in fp32.  Three fp16 products run
// at 2.5 PFLOP/s / 3 where the fp32 matrix instructions have 0.157; a packed-bit operand is one half without any error, so its products are two.
//
// What the scaling costs, and how it is made good: a value below 2^-18 of the largest of its row keeps fewer bits, one below 2^-41 none, where fp32 would keep all.  That matters where the other
// operand is as much larger there (an input that is not normalised, whose weights are small) or 0 where this one is large (gradients over sparse bits).  So the first launch also leaves what each row lost,
// the sum of what its halves leave of such values, and an element of the product whose sum never got 2^20 times as large as its row and its column can have changed it
//     |sum| < 2^20 * (lost of the row * largest of the column + largest of the row * lost of the column)
// is formed again in fp32 straight from the operands, as one that is no number is (an infinity times a lower half of 0).  What fp32 sums of that length round away is as much.  Sums are looked
// at on the way too (a number that has been large has lost as much in fp32, however small it ends): ordinary operands have next to none of these elements.
//
// The gradients of a softmax do have them, with magnitudes spread over more than 2^100: a twentieth of dx over 32768 channels as training begins, most of all elements as it ends (1024 inputs x 1024
// channels x 4096 frames then took 1.7 to 2.2 ms).  So the products of a loss's gradients take their operands as three pieces of bf16, 24 bits in the
// range of fp32: six products instead of three (three instead of two over packed bits), the smallest first, whatever the values are. The thirds lie apart from the first two pieces and are walked
// ahead of these.  A layer's backward pass keeps halves even where its gradient is a softmax's: 1024 x 1024 x 4096 takes 93 us then, 149 with confident logits, and as triples 139 for any gradient.
//
// Two launches.  The first reads each operand as it lies and leaves its halves in the order in which the matrix instructions want them: blocks of 32 rows x 16 k,
// 1 KiB each, lane l's sixteen bytes (row l & 31, k 8 (l >> 5) .. + 8) at 16 l, so that the second launch moves them to LDS and from there to registers with 16-byte accesses
// that meet no bank twice, without a transposition anywhere.  In the second, a workgroup of eight wavefronts owns 256 x 256 elements (256 x 128 or 128 x 128: four) and walks k in stages of
// 16, the loads of the next three stages to LDS in flight behind the products of the present one (the small tile: of the next four, and its halves one stage ahead in registers).
// Where there are too few tiles for the device, several workgroups share a tile's k axis and a third launch adds their sums in a fixed order.
//
// What bounds it: the matrix instructions and the power they take.  4096 x 4096 x 8192 with packed bits is 550 GFLOP of halves in 442 to 481 us, both products of its backward pass on real
// values 1650 in 1320 to 1500: 1.1 to 1.2 PFLOP/s, where a plain product of halves by the library reaches 1.17 to 1.26.  Five or seven stages ahead changed nothing.  Packing is
// bound by memory and by its two phases, loads and then stores: 207 MB in 60 us, 1.35 GB in 366, 3.5 to 3.7 TB/s.  Small problems are bound by two launches of 13 us and more whose workgroups run once.  Summing what rows lose and looking for
// it costs a large product 1 % and a small one 2 to 3 us of 40; with its triples a loss over 777 x 1001 x 1000 takes 94 us (70 with halves that lose), over 1024 x 32768 x 4096 4.74 ms (3.39).
#pragma once

#include <type_traits>

#include "dense_direct_kernels.hpp"
#include "dense_rules.hpp"

namespace bbhip {

typedef _Float16 DenseHalf8 __attribute__((ext_vector_type(8)));
typedef float    DenseAcc16 __attribute__((ext_vector_type(16)));

struct PackJob {
    Operand src;
    int    kind;
    uint4 *halves;              // [row blocks][k steps][1 or 2][64 lanes]
    int   *exponent;            // of each row (null: packed bits, which are not scaled)
    float *lost;                // of each row: the magnitudes, scaled, of what its halves leave of values that they do not hold to 22 bits; minus infinity: it has no value but 0
    int    k_steps;             // of 16
    int    blocks;              // workgroups
    float *line;                // gradients as rows: their sums (null: not wanted), added with accumulate
    int    accumulate;
    float *dz;                  // gradients as rows: themselves (null: not wanted), rows of dz_stride
    long long dz_stride;
    int    triple;              // three pieces of bf16 instead of halves
    uint4 *thirds;              // the last of them: [row blocks][k steps][64 lanes]; the others lie where halves do
};

// Triples: the largest of a row is brought to 2^40, so that a value 2^-140 as large still has all its pieces (2^-100, and 2^-126 is the least of a third).
constexpr int   kTripleTop = 40;
constexpr float kTripleLeast = 7.88860905e-31f;         // 2^-100

constexpr int kPackJobs = 4;
struct PackArgs { PackJob job[kPackJobs]; };

__device__ __forceinline__ uint32_t two_halves(float a, float b)
{
    typedef _Float16 Half2 __attribute__((ext_vector_type(2)));
    Half2 const h = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, h);
}

__device__ __forceinline__ float to_bf16(float v) { return (float)(__bf16)v; }
__device__ __forceinline__ uint32_t two_bf16(float a, float b)
{
    typedef __bf16 Two __attribute__((ext_vector_type(2)));
    Two const t = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, t);
}

// workgroup -> place in the list of tiles: workgroups go round the eight XCDs, each of which gets a run of neighbours
__device__ __forceinline__ int xcd_run(int id, int total)
{
    int const x = id & 7, q = total >> 3, r = total & 7;
    return x * q + min(x, r) + (id >> 3);
}

// finite magnitude
__device__ __forceinline__ float magnitude(float v) { float const a = fabsf(v); return a < INFINITY ? a : 0.0f; }

// Eight rows and all their k per workgroup: what it writes are whole lines of 128 bytes (eight rows' 16), and with 64 groups of eight k side by side a thread holds all values of a row of up to 4096
// between finding the largest and splitting.  Where rows are columns of the buffer it reads 32 bytes at a time; workgroups that share a line run on one XCD (xcd_run).  With 32 rows per
// workgroup a batch of 65 frames of 6144 bits and as many weights took 14 us longer.
template <int KIND, int THREADS>
__device__ __forceinline__ void pack_rows(PackJob const &j, int block, float *share)
{
    constexpr int ROWS = kPackRows, kOctets = THREADS / ROWS;      // side by side
    constexpr bool kBits = KIND == kBitRows || KIND == kBitColumns;
    constexpr int kPieces = kBits ? 1 : 2;
    int const at = threadIdx.x % ROWS, octet0 = threadIdx.x / ROWS, row = block * ROWS + at;
    int const octets = j.k_steps * 2;
    bool const there = row < j.src.rows;
    float held[kPackHeld][8];
    float top = 0.0f, sum = 0.0f, lost = 0.0f;
    int e = 0;
    if (!kBits) {
        int i = 0;
#pragma unroll
        for (int u = 0; u < kPackHeld; ++u) {
            int const o = octet0 + u * kOctets;
#pragma unroll
            for (int q = 0; q < 8; ++q) { held[u][q] = 0.0f; }
            if (there && o * 8 < j.src.depth) { load_values<KIND, 8>(j.src, row, o * 8, held[u]); }
#pragma unroll
            for (int q = 0; q < 8; ++q) { top = fmaxf(top, magnitude(held[u][q])); sum += held[u][q]; }
        }
        for (i = kPackHeld; octet0 + i * kOctets < octets; ++i) {
            float v[8];
            int const o = octet0 + i * kOctets;
            if (!there || o * 8 >= j.src.depth) { break; }
            load_values<KIND, 8>(j.src, row, o * 8, v);
#pragma unroll
            for (int q = 0; q < 8; ++q) { top = fmaxf(top, magnitude(v[q])); sum += v[q]; }
        }
        // over the threads of a row: within the wavefront, then through LDS in a fixed order
#pragma unroll
        for (int step = ROWS; step < 64; step *= 2) { top = fmaxf(top, __shfl_xor(top, step)); sum += __shfl_xor(sum, step); }
        constexpr int kWaves = THREADS / 64;
        int const wave = threadIdx.x / 64;
        if ((threadIdx.x & 63) < ROWS) { share[wave * ROWS + at] = top; share[(kWaves + wave) * ROWS + at] = sum; }
        __syncthreads();
        top = 0.0f; sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) { top = fmaxf(top, share[w * ROWS + at]); sum += share[(kWaves + w) * ROWS + at]; }
        e = top > 0.0f ? (j.triple ? kTripleTop : 15) - ilogbf(top) : 0;
        if (!j.triple && ldexpf(top, e) >= 65520.0f) { --e; }           // (which halves would round to infinity)
        if (threadIdx.x < ROWS) {
            j.exponent[row] = e;
            if constexpr (KIND == kGradRows) { if (j.line && there) { j.line[row] = j.accumulate ? j.line[row] + sum : sum; } }
        }
    }
    auto const write = [&](int o, float const (&v)[8]) {
        uint4 *to = j.halves + (((long long)(row >> 5) * j.k_steps + (o >> 1)) * kPieces) * 64 + (o & 1) * 32 + (row & 31);
        if constexpr (kBits) {
            if (j.triple) { to[0] = make_uint4(two_bf16(v[0], v[1]), two_bf16(v[2], v[3]), two_bf16(v[4], v[5]), two_bf16(v[6], v[7])); }
            else          { to[0] = make_uint4(two_halves(v[0], v[1]), two_halves(v[2], v[3]), two_halves(v[4], v[5]), two_halves(v[6], v[7])); }
        }
        else if (j.triple) {
            float h[8], m[8], l[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                float const a = ldexpf(v[q], e);
                h[q] = to_bf16(a);
                float const rest = fabsf(h[q]) < INFINITY ? a - h[q] : 0.0f;
                m[q] = to_bf16(rest);
                l[q] = rest - m[q];
                // (whose pieces might leave the range of bf16)
                lost += fabsf(a) < kTripleLeast ? fabsf(a) : 0.0f;
            }
            to[0]  = make_uint4(two_bf16(h[0], h[1]), two_bf16(h[2], h[3]), two_bf16(h[4], h[5]), two_bf16(h[6], h[7]));
            to[64] = make_uint4(two_bf16(m[0], m[1]), two_bf16(m[2], m[3]), two_bf16(m[4], m[5]), two_bf16(m[6], m[7]));
            j.thirds[((long long)(row >> 5) * j.k_steps + (o >> 1)) * 64 + (o & 1) * 32 + (row & 31)] =
                make_uint4(two_bf16(l[0], l[1]), two_bf16(l[2], l[3]), two_bf16(l[4], l[5]), two_bf16(l[6], l[7]));
        }
        else {
            float h[8], l[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                h[q] = ldexpf(v[q], e);
                float const upper = (float)(_Float16)h[q];
                // (the difference of an infinity to itself is no number, its lower half 0)
                l[q] = fabsf(upper) < INFINITY ? h[q] - upper : 0.0f;
                // (below 1/8 the lower half's steps, 2^-24, are more than 2^-21 of the value)
                lost += fabsf(h[q]) < 0.125f ? fabsf(l[q] - (float)(_Float16)l[q]) : 0.0f;
            }
            to[0]  = make_uint4(two_halves(h[0], h[1]), two_halves(h[2], h[3]), two_halves(h[4], h[5]), two_halves(h[6], h[7]));
            to[64] = make_uint4(two_halves(l[0], l[1]), two_halves(l[2], l[3]), two_halves(l[4], l[5]), two_halves(l[6], l[7]));
        }
        if constexpr (KIND == kGradRows) {
            if (j.dz && there) {
                float *d = j.dz + row * j.dz_stride + o * 8;
                if (o * 8 + 8 <= j.src.depth && (reinterpret_cast<uintptr_t>(d) & 15) == 0) {
                    reinterpret_cast<float4 *>(d)[0] = make_float4(v[0], v[1], v[2], v[3]);
                    reinterpret_cast<float4 *>(d)[1] = make_float4(v[4], v[5], v[6], v[7]);
                }
                else {
#pragma unroll
                    for (int q = 0; q < 8; ++q) { if (o * 8 + q < j.src.depth) { d[q] = v[q]; } }
                }
            }
        }
    };
    if (!kBits) {
#pragma unroll
        for (int u = 0; u < kPackHeld; ++u) { if (octet0 + u * kOctets < octets) { write(octet0 + u * kOctets, held[u]); } }
    }
    // what is not held (packed bits: four groups asked for at a time, which are few registers)
    constexpr int kAtATime = kBits ? 4 : 1;
    for (int i = kBits ? 0 : kPackHeld; octet0 + i * kOctets < octets; i += kAtATime) {
        float v[kAtATime][8] = {};
#pragma unroll
        for (int u = 0; u < kAtATime; ++u) {
            int const o = octet0 + (i + u) * kOctets;
            if (there && o * 8 < j.src.depth) { load_values<KIND, 8>(j.src, row, o * 8, v[u]); }
        }
#pragma unroll
        for (int u = 0; u < kAtATime; ++u) {
            if (octet0 + (i + u) * kOctets < octets) { write(octet0 + (i + u) * kOctets, v[u]); }
            if constexpr (kBits) {
#pragma unroll
                for (int q = 0; q < 8; ++q) { top = fmaxf(top, v[u][q]); }
            }
        }
    }
    // (of packed bits only whether any is set; of others every thread has the row's largest)
    constexpr int kWaves = THREADS / 64;
    float mine = kBits ? top : lost;
#pragma unroll
    for (int step = ROWS; step < 64; step *= 2) { mine += __shfl_xor(mine, step); }
    float *const part = share + 2 * kWaves * ROWS;
    if ((threadIdx.x & 63) < ROWS) { part[threadIdx.x / 64 * ROWS + at] = mine; }
    __syncthreads();
    if (threadIdx.x < ROWS) {
        mine = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) { mine += part[w * ROWS + at]; }
        j.lost[row] = kBits ? (mine > 0.0f ? 0.0f : -INFINITY) : top > 0.0f ? mine : -INFINITY;
    }
}

template <int THREADS>
__global__ __launch_bounds__(THREADS, 4) void dense_pack_kernel(PackArgs a)
{
    __shared__ float share[3 * THREADS / 64 * kPackRows];
    int block = blockIdx.x, which = 0;
    while (block >= a.job[which].blocks) { block -= a.job[which].blocks; ++which; }
    PackJob const &j = a.job[which];
    block = xcd_run(block, j.blocks);
    switch (j.kind) {
    case kRows:       pack_rows<kRows, THREADS>(j, block, share); break;
    case kColumns:    pack_rows<kColumns, THREADS>(j, block, share); break;
    case kBitRows:    pack_rows<kBitRows, THREADS>(j, block, share); break;
    case kBitColumns: pack_rows<kBitColumns, THREADS>(j, block, share); break;
    case kGradRows:   pack_rows<kGradRows, THREADS>(j, block, share); break;
    default:          pack_rows<kGradColumns, THREADS>(j, block, share); break;
    }
}

// ---- the product ------------------------------------------------------------------------------------------------------------------------
struct PackedProduct {
    uint4 const *a, *b;             // halves
    int   const *ea, *eb;           // exponents of the rows (eb null: 0)
    float const *lost_a, *lost_b;   // what the rows lost
    uint4 const *thirds_a, *thirds_b;           // triples: their last pieces (packed bits: null)
    int   triple;
    int   a_blocks, b_blocks;       // row blocks of 32
    int   k_steps;
    int   b_pieces;
    int   m_tiles, n_tiles;
    int   slabs, slab_stages;       // of the k axis
    int   workgroups;
    float *sums;                    // slabs > 1: [slab][m][n], n padded to pitch
    long long sums_pitch, sums_slab;
    DenseOutput out;
    Operand src_a, src_b;           // where an element is formed again if it is no number
    int   kind_a, kind_b;           // (sums of products straight from the operands: kind_a negative, there is nothing to form again)
};

// What a launch is for: y or its bits, products as they are (or a slab's sums), logits.
enum PackedUse : int { kUseForward = 0, kUseStore = 1, kUseLogits = 2 };

// 32 x 64 elements of a wavefront lie in LDS as rows of kTilePitch floats.
constexpr int kTilePitch = 68;
// What such a tile has in the place of an element that is not to be stored: a NaN of its own (`marks`: there may be some).  The elements that are stored are never this one: NaN are formed
// again, and plain_nan() is what they are then.
constexpr uint32_t kNotStored = 0x7fb0a5a5u;
__device__ __forceinline__ bool stored(float v) { return __builtin_bit_cast(uint32_t, v) != kNotStored; }
__device__ __forceinline__ float plain_nan(float v) { return v == v ? v : __builtin_bit_cast(float, 0x7fc00000u); }

// ---- elements formed again ----------------------------------------------------------------------------------------------------------------
// The halves of an infinity times a lower half of 0 are no number where the value's product is infinite, and halves lose small values beside large ones: such elements are formed again in fp32
// straight from the operands, so that they are what the formula says; their neighbours keep the bits that they have.

// An element stands where its scaled sum got as large as the limits of its row and its column together: what they lost, times the other's largest (below 2^16, of triples 2^41; bits: 1), times 2^20.  (Where
// either has no value but 0 nothing is lost: minus infinity.)
template <int PB, bool TRIPLE>
__device__ __forceinline__ float limit_of(float lost) { return lost * (PB == 1 ? 1048576.0f : TRIPLE ? 2305843009213693952.0f : 68719476736.0f); }

// By a wavefront: its lanes take the k in turn, N at a time, whose loads overlap.
template <int KA, int KB, int N>
__device__ __forceinline__ float element_again(Operand const &a, Operand const &b, int m, int n, int lane)
{
    float d = 0.0f;
#pragma nounroll
    for (int k0 = lane; k0 < a.depth; k0 += N * 64) {
        float u[N], v[N];
#pragma unroll
        for (int q = 0; q < N; ++q) {
            int const k = min(k0 + q * 64, a.depth - 1);
            u[q] = operand_at<KA>(a, m, k);
            v[q] = operand_at<KB>(b, n, k);
        }
#pragma unroll
        for (int q = 0; q < N; ++q) { if (k0 + q * 64 < a.depth) { d = fmaf(u[q], v[q], d); } }
        if (__any(d != d)) { break; }           // (a sum that is no number stays none: operands full of them are done at once)
    }
#pragma unroll
    for (int step = 32; step > 0; step /= 2) { d += __shfl_xor(d, step); }
    return d;
}

// Values of row row0 + r at k0 + 8 half and the seven behind it, 0 behind the last k (row0 a multiple of 32, k0 of 16, perhaps behind the last k itself; rows behind the last one hold anything)
template <int KIND>
__device__ __forceinline__ void load_eight(Operand const &o, int row0, int k0, int r, int half, float (&v)[8])
{
    constexpr bool kGrad = KIND == kGradRows || KIND == kGradColumns;
    constexpr int kAs = KIND == kGradRows ? kRows : KIND == kGradColumns ? kColumns : KIND;
    constexpr bool kAlong = kAs == kRows || kAs == kBitRows;
    TileBuffer const from = RawRun<kAs>::buffer(o, row0, k0);
    uint32_t const pitch = (uint32_t)o.stride * 4, step = kAlong ? 4 : pitch;
    uint32_t const at = kAlong ? r * pitch + half * 32 : half * 8 * pitch + (kAs == kColumns ? r * 4 : 0);
    int const k = k0 + half * 8;
    if constexpr (KIND == kBitRows) {
        uint32_t const w = load_word(from, r * pitch) >> (k & 31);
#pragma unroll
        for (int j = 0; j < 8; ++j) { v[j] = (float)((w >> j) & 1u); }
    }
    else if (kAs == kRows && o.vec) {
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
            uint4 const q = load_words(from, at + j * 4);
            v[j] = __builtin_bit_cast(float, q.x); v[j + 1] = __builtin_bit_cast(float, q.y); v[j + 2] = __builtin_bit_cast(float, q.z); v[j + 3] = __builtin_bit_cast(float, q.w);
        }
    }
    else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            uint32_t const w = load_word(from, at + j * step);
            v[j] = KIND == kBitColumns ? (float)((w >> r) & 1u) : __builtin_bit_cast(float, w);
        }
    }
    // (values of the frames k: zero behind the last)
    auto const of_frames = [&](void const *p, int j) { return load_word(tile_buffer(static_cast<uint32_t const *>(p) + k0, max(o.depth - k0, 0) * 4LL), (half * 8 + j) * 4); };
    if constexpr (KIND == kRows) {
        if (o.coef) {
#pragma unroll
            for (int j = 0; j < 8; ++j) { v[j] = __builtin_bit_cast(float, of_frames(o.coef, j)) == 0.0f ? 0.0f : v[j]; }
        }
    }
    if constexpr (kGrad) {
        if (o.mode == kGradSoftmax) {
            int const frame = min(row0 + r, o.rows - 1);
            float top = KIND == kGradColumns ? o.top[frame] : 0.0f, share = KIND == kGradColumns ? o.share[frame] : 0.0f, coef = KIND == kGradColumns ? o.coef[frame] : 0.0f;
            int label = KIND == kGradColumns ? o.label[frame] : 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if constexpr (KIND == kGradRows) {
                    top = __builtin_bit_cast(float, of_frames(o.top, j)); share = __builtin_bit_cast(float, of_frames(o.share, j));
                    coef = __builtin_bit_cast(float, of_frames(o.coef, j)); label = (int)of_frames(o.label, j);
                }
                v[j] = softmax_gradient(v[j], top, share, coef, label, (KIND == kGradRows ? row0 + r : k + j) + o.first);
            }
        }
        else if (o.mode != kActNone) {
            Operand y = o;
            y.p = o.y;
            TileBuffer const values = RawRun<kAs>::buffer(y, row0, k0);
#pragma unroll
            for (int j = 0; j < 8; ++j) { v[j] = gradient_of(v[j], __builtin_bit_cast(float, load_word(values, at + j * step)), o.mode); }
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) { v[j] = k + j < o.depth ? v[j] : 0.0f; }
}

// 32 x 32 of them by a wavefront, on the fp32 matrix instructions.  (The loads of several steps overlap: 4096 x 4096 x 8192,
// every element formed again, 4.3 ms in all, 0.4 of it for seeing sums that are no number any more; with one step and without that 4.7.)
template <int KA, int KB>
__device__ __forceinline__ DenseAcc16 block_again(Operand const &a, Operand const &b, int m0, int n0, int lane)
{
    constexpr int kSteps = KA == kGradRows ? 2 : 4;         // (a softmax gradient takes four values of its frame along)
    DenseAcc16 acc = {};
#pragma nounroll
    for (int k0 = 0; k0 < a.depth; k0 += 16 * kSteps) {
        float u[kSteps][8], v[kSteps][8];
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            // (behind the last k everything is 0)
            load_eight<KA>(a, m0, k0 + 16 * s, lane & 31, lane >> 5, u[s]);
            load_eight<KB>(b, n0, k0 + 16 * s, lane & 31, lane >> 5, v[s]);
        }
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
#pragma unroll
            for (int q = 0; q < 8; ++q) { acc = __builtin_amdgcn_mfma_f32_32x32x2f32(u[s][q], v[s][q], acc, 0, 0, 0); }
        }
        bool number = false;
#pragma unroll
        for (int r = 0; r < 16; ++r) { number = number | (acc[r] == acc[r]); }
        if (!__any(number)) { break; }
    }
    return acc;
}

// Those of a tile of 32 x 64 in LDS, rows of `pitch`: bit 16 j + r of a lane's word is element r of block j as a matrix instruction leaves it.  Few by the element (4096 k: about 10 us each, which
// a launch that waits for one wavefront pays), more by the block.
constexpr int kFewAgain = 16;
template <int KA, int KB>
__device__ __forceinline__ void tile_again(Operand const &a, Operand const &b, float *tile, int pitch, uint32_t which, int m0, int n0, int lane)
{
    asm volatile("" : "+v"(lane));              // (so that nothing of this is computed ahead, in registers that the accumulators need)
#pragma nounroll
    for (int j = 0; j < 2; ++j) {
        uint32_t mine = (which >> (16 * j)) & 0xffffu;
        int count = __popc(mine);
#pragma unroll
        for (int step = 32; step > 0; step /= 2) { count += __shfl_xor(count, step); }
        if (count > kFewAgain) {
            DenseAcc16 const acc = block_again<KA, KB>(a, b, m0, n0 + j * 32, lane);
#pragma unroll
            for (int r = 0; r < 16; ++r) { if ((mine >> r) & 1u) { tile[acc_row(r, lane) * pitch + j * 32 + (lane & 31)] = plain_nan(acc[r]); } }
            continue;
        }
        for (uint64_t lanes = __ballot(mine != 0u); lanes != 0; lanes = __ballot(mine != 0u)) {
            int const from = __ffsll((unsigned long long)lanes) - 1, r = __ffs(__builtin_amdgcn_readlane((int)mine, from)) - 1;
            int const row = acc_row(r, from), column = j * 32 + (from & 31);
            float const d = element_again<KA, KB, 16>(a, b, m0 + row, n0 + column, lane);
            if (lane == from) { tile[row * pitch + column] = plain_nan(d); mine &= mine - 1; }
        }
    }
}

// The same for the elements (m, n0 + lane) of a row, d, where `again`: few by the element, more by a lane each (1024 x 1024 x 1024, every element formed again, 0.52 ms).
template <int KA, int KB>
__device__ __forceinline__ void row_again(Operand const &a, Operand const &b, float &d, bool again, int m, int n0, int lane)
{
    uint64_t lanes = __ballot(again);
    if (__popcll(lanes) > kFewAgain) {
        if (!again) { return; }
        float sum[4] = {};                      // (shorter chains of roundings than one sum)
#pragma nounroll
        for (int k0 = 0; k0 < a.depth; k0 += 4) {
            float u[4], v[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                int const k = min(k0 + q, a.depth - 1);
                u[q] = operand_at<KA>(a, m, k);
                v[q] = operand_at<KB>(b, n0 + lane, k);
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) { if (k0 + q < a.depth) { sum[q] = fmaf(u[q], v[q], sum[q]); } }
            d = (sum[0] + sum[1]) + (sum[2] + sum[3]);
            if (!__any(d == d)) { break; }
        }
        return;
    }
    for (; lanes != 0; lanes &= lanes - 1) {
        int const from = __ffsll((unsigned long long)lanes) - 1;
        float const e = element_again<KA, KB, 4>(a, b, m, n0 + from, lane);
        if (lane == from) { d = e; }
    }
}

// whichever kinds the operands are of
__device__ __forceinline__ void logit_again(Operand const &a, Operand const &b, int kind_b, float &d, bool again, int m, int n0, int lane)
{
    if (kind_b == kColumns) { row_again<kRows, kColumns>(a, b, d, again, m, n0, lane); }
    else                    { row_again<kRows, kBitColumns>(a, b, d, again, m, n0, lane); }
}
__device__ __forceinline__ void row_again(Operand const &a, int kind_a, Operand const &b, int kind_b, float &d, bool again, int m, int n0, int lane)
{
    if (kind_a == kRows)           { logit_again(a, b, kind_b, d, again, m, n0, lane); }
    else if (kind_a == kGradRows)  { if (kind_b == kRows) { row_again<kGradRows, kRows>(a, b, d, again, m, n0, lane); }    else { row_again<kGradRows, kBitRows>(a, b, d, again, m, n0, lane); } }
    else                           { row_again<kColumns, kGradColumns>(a, b, d, again, m, n0, lane); }
}

// v[step]: four neighbours of row 4 step + lane / 16 of such a tile, and what they become.  `all`: the four may be moved with 16-byte accesses.
template <int USE>
__device__ __forceinline__ void finish_tile(DenseOutput const &o, float const *tile, float const *bias, int m0, int n0, int lane, bool marks)
{
    int const n = n0 + (lane & 15) * 4, row0 = lane >> 4;
    bool const all = n + 4 <= o.columns && o.stride % 4 == 0 && (reinterpret_cast<uintptr_t>(o.out) & 15) == 0 &&
                     (USE != kUseForward || !o.residual || (o.residual_stride % 4 == 0 && (reinterpret_cast<uintptr_t>(o.residual) & 15) == 0));
    if (n >= o.columns) { return; }
    // what is added is asked for at once, ahead of the first use
    float more[8][4] = {};
    float const *from = USE == kUseForward ? o.residual : o.accumulate ? static_cast<float const *>(o.out) : nullptr;
    long long const pitch = USE == kUseForward ? o.residual_stride : o.stride;
    if (from) {
#pragma unroll
        for (int step = 0; step < 8; ++step) {
            int const m = m0 + step * 4 + row0;
            if (m >= o.rows) { continue; }
            if (all) { load_floats(from + m * pitch + n, true, more[step]); }
            else {
#pragma unroll
                for (int q = 0; q < 4; ++q) { if (n + q < o.columns) { more[step][q] = from[m * pitch + n + q]; } }
            }
        }
    }
#pragma unroll
    for (int step = 0; step < 8; ++step) {
        int const row = step * 4 + row0, m = m0 + row;
        if (m >= o.rows) { continue; }
        float d[4];
        load_floats(tile + row * kTilePitch + (lane & 15) * 4, true, d);
        bool whole = all;
        uint32_t keep = 0xfu;
        if (__builtin_expect(marks, 0)) {
            keep = (stored(d[0]) ? 1u : 0u) | (stored(d[1]) ? 2u : 0u) | (stored(d[2]) ? 4u : 0u) | (stored(d[3]) ? 8u : 0u);
            whole = whole && keep == 0xfu;
        }
        if (USE != kUseStore) {
            float const b = bias[row];
#pragma unroll
            for (int q = 0; q < 4; ++q) { d[q] += b; }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) { d[q] += more[step][q]; }
        if (USE == kUseForward && o.activation != kActNone) {
#pragma unroll
            for (int q = 0; q < 4; ++q) { d[q] = activated(d[q], o.activation); }
        }
        float *to = static_cast<float *>(o.out) + m * o.stride + n;
        if (whole) { *reinterpret_cast<float4 *>(to) = make_float4(d[0], d[1], d[2], d[3]); }
        else {
#pragma unroll
            for (int q = 0; q < 4; ++q) { if (n + q < o.columns && ((keep >> q) & 1u)) { to[q] = d[q]; } }
        }
    }
}

// The same to packed bits: a row of 64 columns is two words.  What is not to be stored is 0 in them; `more`: the bits are added to those of a first pass.
__device__ __forceinline__ void finish_tile_bits(DenseOutput const &o, float const *tile, float const *bias, int m0, int n0, int lane, bool more)
{
    int const n = n0 + lane;
    bool const inside = n < o.columns;
    for (int row = 0; row < 32 && m0 + row < o.rows; ++row) {
        float z = tile[row * kTilePitch + lane] + bias[row];
        if (o.residual && inside) { z += o.residual[(m0 + row) * o.residual_stride + n]; }
        uint64_t const bits = __ballot(inside && z > 0.0f);
        if ((lane & 31) == 0 && inside) {
            uint32_t *const to = static_cast<uint32_t *>(o.out) + (m0 + row) * o.stride + (n >> 5);
            *to = (uint32_t)(bits >> (lane & 32)) | (more ? *to : 0u);
        }
    }
}

// What becomes of a tile of 32 x 64; logits: (largest, sum of exponents) of its rows join `column`, this lane's.
template <int USE>
__device__ __forceinline__ void finish(DenseOutput const &o, bool partial_sums, float const *tile, float const *bias, int m0, int n0, int lane, float2 &column, bool marks, bool more)
{
    if (USE == kUseLogits && !partial_sums && n0 + lane < o.columns) {
        int const n = n0 + lane, rows = min(32, o.rows - m0), label = o.label[n] - o.first_channel - m0;
        float z[32];
        float2 s = make_float2(-INFINITY, 0.0f);
#pragma unroll
        for (int row = 0; row < 32; ++row) {
            z[row] = row < rows ? tile[row * kTilePitch + lane] + bias[row] : -INFINITY;
            s.x = fmaxf(s.x, z[row]);
        }
        if (__builtin_expect(marks, 0)) {
            s.x = -INFINITY;
#pragma unroll
            for (int row = 0; row < 32; ++row) {
                z[row] = stored(tile[row * kTilePitch + lane]) ? z[row] : -INFINITY;
                s.x = fmaxf(s.x, z[row]);
            }
        }
#pragma unroll
        for (int row = 0; row < 32; ++row) { s.y += z[row] == -INFINITY ? 0.0f : exp_of_nonpositive(z[row] - s.x); }
        if (label >= 0 && label < rows && stored(tile[label * kTilePitch + lane])) { o.label_logit[n] = tile[label * kTilePitch + lane] + bias[label]; }
        column = joined(column, s);
    }
    if (USE == kUseForward && o.kind == kOutBits)         { finish_tile_bits(o, tile, bias, m0, n0, lane, more); }
    else if (USE == kUseForward && o.kind == kOutForward) { finish_tile<kUseForward>(o, tile, bias, m0, n0, lane, marks); }
    else if (USE == kUseLogits && !partial_sums)          { if (o.out) { finish_tile<kUseLogits>(o, tile, bias, m0, n0, lane, marks); } }
    else                                                  { finish_tile<kUseStore>(o, tile, bias, m0, n0, lane, marks); }
}

// Waits until at most N of this wavefront's loads are on their way (loads arrive in order) and its reads of LDS are done, then for the workgroup.
template <int N>
__device__ __forceinline__ void arrived(void)
{
    __builtin_amdgcn_s_waitcnt(0xc07f);         // (lgkmcnt 0, where the compiler sees it: it need not wait for these reads again)
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" :: "n"(N) : "memory");
}

template <bool TRIPLE>
__device__ __forceinline__ DenseAcc16 product_of(DenseHalf8 a, DenseHalf8 b, DenseAcc16 c)
{
    typedef __bf16 Bf8 __attribute__((ext_vector_type(8)));
    if constexpr (TRIPLE) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(Bf8, a), __builtin_bit_cast(Bf8, b), c, 0, 0, 0); }
    else                  { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
}

template <int USE, int KA, int KB, bool TRIPLE, int TM, int WM, int WN, int PB, int BUFFERS>
__device__ __forceinline__ void packed_tile(PackedProduct const &p, int id, char *lds, int *scales, float *limits, float *bias)
{
    constexpr int TN = 2, kWaves = WM * WN, kBM = TM * WM, kBN = TN * WN;           // blocks of 32 rows
    constexpr int kOwn = kBM / kWaves;              // row blocks of a that a wavefront loads; of b it loads one
    static_assert(kBM == kWaves * kOwn && kBN == kWaves, "the wavefronts share the loads evenly");
    constexpr int kStageA = kBM * 2048, kStage = kStageA + kBN * 1024 * PB, kLoads = 2 * kOwn + PB, kAhead = BUFFERS - 1;
    int const lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int const tiles = p.m_tiles * p.n_tiles;
    int const slab = id / tiles;
    int const t = xcd_run(id % tiles, tiles);
    // runs of eight tiles down, then across: what a run's workgroups read at a time is a few row blocks of either operand
    int const band = t / (8 * p.n_tiles), rest = t - band * 8 * p.n_tiles, high = min(8, p.m_tiles - band * 8);
    int const m_tile = band * 8 + rest % high, n_tile = rest / high;
    int const rb_a = m_tile * kBM, rb_b = n_tile * kBN;
    int const first = slab * p.slab_stages, stages = min(p.slab_stages, p.k_steps - first);

    // a stage is 16 k: of each row block two (packed bits: one) blocks of 1 KiB, which a wavefront moves to LDS as they are
    char const *from_a[kOwn];
#pragma unroll
    for (int i = 0; i < kOwn; ++i) { from_a[i] = reinterpret_cast<char const *>(p.a) + ((long long)min(rb_a + wave * kOwn + i, p.a_blocks - 1) * p.k_steps + first) * 2048; }
    char const *from_b = reinterpret_cast<char const *>(p.b) + ((long long)min(rb_b + wave, p.b_blocks - 1) * p.k_steps + first) * (1024 * PB);
    uint32_t const at_lds = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds);
    auto const fetch = [&](int buffer) {
        // (as assembly: the compiler would wait for all of them ahead of every read of LDS, whichever buffer it reads.  Each lane's sixteen bytes go to M0 + offset + 16 lane.)
        uint32_t const to_a = at_lds + buffer * kStage + wave * kOwn * 2048, to_b = at_lds + buffer * kStage + kStageA + wave * 1024 * PB;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            char const *const a = from_a[i] + lane * 16;
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\tglobal_load_lds_dwordx4 %1, off offset:1024" :: "s"(to_a + i * 2048), "v"(a) : "memory", "m0");
            from_a[i] += 2048;
        }
        char const *const b = from_b + lane * 16;
        if constexpr (PB == 2) {
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\tglobal_load_lds_dwordx4 %1, off offset:1024" :: "s"(to_b), "v"(b) : "memory", "m0");
        }
        else { asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" :: "s"(to_b), "v"(b) : "memory", "m0"); }
        from_b += 1024 * PB;
    };

    // what is needed behind the products: the scales and biases of the tile's rows (the barriers of the stages are between this and its use)
    DenseOutput o = p.out;
    int const *const scale_a = scales, *const scale_b = scales + kBM * 32;
    float const *const limit_a = limits, *const limit_b = limits + kBM * 32;
    for (int i = threadIdx.x; i < kBM * 32; i += kWaves * 64) {
        scales[i] = p.ea[min(rb_a * 32 + i, p.a_blocks * 32 - 1)];
        limits[i] = limit_of<PB, TRIPLE>(p.lost_a[min(rb_a * 32 + i, p.a_blocks * 32 - 1)]);
        if (USE != kUseStore) { bias[i] = o.bias && rb_a * 32 + i < o.rows ? o.bias[rb_a * 32 + i] : 0.0f; }
    }
    for (int i = threadIdx.x; i < kBN * 32; i += kWaves * 64) {
        scales[kBM * 32 + i] = PB == 2 ? p.eb[min(rb_b * 32 + i, p.b_blocks * 32 - 1)] : 0;
        limits[kBM * 32 + i] = limit_of<PB, TRIPLE>(p.lost_b[min(rb_b * 32 + i, p.b_blocks * 32 - 1)]);
    }

    int const wm = wave / WN, wn = wave % WN;
    DenseAcc16 acc[TM][TN] = {};
    if constexpr (TRIPLE) {
        // Thirds of one operand times firsts of the other ahead of everything else, two steps of k at a time.
        auto const thirds = [&](auto of_a) {
            constexpr bool kOfA = decltype(of_a)::value;
            constexpr int kThirdStage = (kBM + kBN) * 2048, kThirdLoads = 2 * kOwn + 2;
            constexpr long long kStepA = kOfA ? 1024 : 2048, kStepB = kOfA ? 1024 * PB : 1024;          // bytes from step to step
            char const *third_a[kOwn];
#pragma unroll
            for (int i = 0; i < kOwn; ++i) {
                third_a[i] = reinterpret_cast<char const *>(kOfA ? p.thirds_a : p.a) + ((long long)min(rb_a + wave * kOwn + i, p.a_blocks - 1) * p.k_steps + first) * kStepA + lane * 16;
            }
            char const *third_b = reinterpret_cast<char const *>(kOfA ? p.b : p.thirds_b) + ((long long)min(rb_b + wave, p.b_blocks - 1) * p.k_steps + first) * kStepB + lane * 16;
            auto const fetch_two = [&](int buffer, int s) {
                bool const both = 2 * s + 1 < stages;           // (else the first step once more, which is not used)
                auto const two = [&](uint32_t to, char const *from, long long step) {
                    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" :: "s"(to), "v"(from) : "memory", "m0");
                    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" :: "s"(to + 1024), "v"(from + (both ? step : 0)) : "memory", "m0");
                };
#pragma unroll
                for (int i = 0; i < kOwn; ++i) { two(at_lds + buffer * kThirdStage + (wave * kOwn + i) * 2048, third_a[i], kStepA); third_a[i] += 2 * kStepA; }
                two(at_lds + buffer * kThirdStage + (kBM + wave) * 2048, third_b, kStepB);
                third_b += 2 * kStepB;
            };
            int const pairs = (stages + 1) / 2;
            for (int s = 0; s < min(kAhead, pairs); ++s) { fetch_two(s, s); }
            int buffer = 0, free = kAhead;
#pragma nounroll
            for (int s = 0; s < pairs; ++s) {
                if (s + kAhead < pairs) { arrived<(kAhead - 1) * kThirdLoads>(); fetch_two(free, s + kAhead); }
                else                    { arrived<0>(); }
                char const *const from = lds + buffer * kThirdStage + lane * 16;
                DenseHalf8 u[TM][2], v[TN][2];
#pragma unroll
                for (int q = 0; q < 2; ++q) {
#pragma unroll
                    for (int j = 0; j < TN; ++j) { v[j][q] = *reinterpret_cast<DenseHalf8 const *>(from + (kBM + wn * TN + j) * 2048 + q * 1024); }
#pragma unroll
                    for (int i = 0; i < TM; ++i) { u[i][q] = *reinterpret_cast<DenseHalf8 const *>(from + (wm * TM + i) * 2048 + q * 1024); }
                }
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    if (q == 1 && 2 * s + 1 >= stages) { break; }
#pragma unroll
                    for (int i = 0; i < TM; ++i) {
#pragma unroll
                        for (int j = 0; j < TN; ++j) { acc[i][j] = product_of<true>(u[i][q], v[j][q], acc[i][j]); }
                    }
                }
                free = buffer;
                buffer = buffer + 1 == BUFFERS ? 0 : buffer + 1;
            }
            __syncthreads();                    // (nobody reads LDS any more, where the next loads go)
        };
        thirds(std::true_type{});
        if constexpr (PB == 2) { thirds(std::false_type{}); }
    }
    struct Halves { DenseHalf8 a[TM][2], b[TN][PB]; };
    auto const read = [&](int buffer, Halves &h) {
        char const *from = lds + buffer * kStage + lane * 16;
#pragma unroll
        for (int j = 0; j < TN; ++j) {
#pragma unroll
            for (int q = 0; q < PB; ++q) { h.b[j][q] = *reinterpret_cast<DenseHalf8 const *>(from + kStageA + ((wn * TN + j) * PB + q) * 1024); }
        }
#pragma unroll
        for (int i = 0; i < TM; ++i) {
#pragma unroll
            for (int q = 0; q < 2; ++q) { h.a[i][q] = *reinterpret_cast<DenseHalf8 const *>(from + ((wm * TM + i) * 2 + q) * 1024); }
            // (all reads are asked for ahead of the first product, in the order in which the products want them: a product waits for no read behind its own)
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto const multiply = [&](Halves const &h) {
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            if constexpr (TRIPLE && PB == 2) {
#pragma unroll
                for (int j = 0; j < TN; ++j) { acc[i][j] = product_of<TRIPLE>(h.a[i][1], h.b[j][1], acc[i][j]); }
            }
#pragma unroll
            for (int j = 0; j < TN; ++j) { acc[i][j] = product_of<TRIPLE>(h.a[i][1], h.b[j][0], acc[i][j]); }
            if constexpr (PB == 2) {
#pragma unroll
                for (int j = 0; j < TN; ++j) { acc[i][j] = product_of<TRIPLE>(h.a[i][0], h.b[j][1], acc[i][j]); }
            }
#pragma unroll
            for (int j = 0; j < TN; ++j) { acc[i][j] = product_of<TRIPLE>(h.a[i][0], h.b[j][0], acc[i][j]); }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // Of each element whether its sum has not been as large as its limit yet, bit 16 j + r; later whether it is formed again.  Looked at up to eight times on the way, every 1024 k or more: with
    // fewer a sum is seldom that small at the end.  Nor where the limits are below 2^12 (sums of scaled values are 2^27 and more): all rows of a wavefront have that in common.
    uint32_t again[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i) { again[i] = 0xffffffffu; }
    int const look_every = max(64, (stages / 8 + 1) & ~1);
    int look = look_every;
    auto const look_at_sums = [&] {
        look += look_every;
        float lb[TN], most = 0.0f;
#pragma unroll
        for (int j = 0; j < TN; ++j) { lb[j] = limit_b[(wn * TN + j) * 32 + (lane & 31)]; most = fmaxf(most, lb[j]); }
#pragma unroll
        for (int i = 0; i < TM; ++i) { most = fmaxf(most, limit_a[(wm * TM + i) * 32 + (lane & 31)]); }
        if (!__any(most >= 4096.0f)) { look = 0x7fffffff; return; }
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            // (the sign of the difference goes in at the bottom, from the last element to the first)
            uint32_t small = 0;
#pragma unroll
            for (int e = 16 * TN - 1; e >= 0; --e) {
                float const left = fabsf(acc[i][e / 16][e % 16]) - (limit_a[(wm * TM + i) * 32 + acc_row(e % 16, lane)] + lb[e / 16]);
                small = __builtin_amdgcn_alignbit(small, __builtin_bit_cast(uint32_t, left), 31);
                if (e % 4 == 0) { __builtin_amdgcn_sched_barrier(0); }
            }
            again[i] &= small;
        }
    };
    __builtin_amdgcn_s_waitcnt(0xc07f);         // (no scalar load on its way: with one the compiler could not count reads of LDS and would wait for all of them at once)
    if constexpr (TM == 2) {
        // A small tile's halves fit the registers twice: the next stage's are read behind the present one's products, which nothing else would cover where a compute unit has one such
        // workgroup.  A stage's buffer is free as soon as its halves are in registers, so the loads are four stages ahead.
        static_assert(BUFFERS == 4, "the stage's buffer is its number modulo four");
        Halves even, odd;
        int const ahead = min(BUFFERS, stages);
        for (int s = 0; s < ahead; ++s) { fetch(s); }
        if (stages >= 4) { arrived<3 * kLoads>(); } else { arrived<0>(); }
        read(0, even);
        auto const step = [&](int s, Halves const &now, Halves &next) {
            if (s + 1 < stages) {
                if (s + 3 < stages) { arrived<2 * kLoads>(); } else { arrived<0>(); }
                if (s + 4 < stages) { fetch(s & 3); }
                read((s + 1) & 3, next);
            }
            multiply(now);
        };
        auto const full_step = [&](int s, Halves const &now, Halves &next) {           // (without a branch between the reads and the products, so that these wait for none of them)
            arrived<2 * kLoads>();
            fetch(s & 3);
            read((s + 1) & 3, next);
            multiply(now);
        };
        int s = 0;
        for (;;) {
            for (int const end = min(stages - 5, look); s < end; s += 2) {
                full_step(s, even, odd);
                full_step(s + 1, odd, even);
            }
            if (s < look) { break; }
            look_at_sums();
        }
#pragma nounroll
        for (; s < stages; s += 2) {
            step(s, even, odd);
            if (s + 1 < stages) { step(s + 1, odd, even); }
        }
    }
    else {
        // A stage's loads are asked for kAhead stages before.  Behind the barrier all wavefronts' loads of the stage have arrived, and nobody reads the buffer of the stage before any
        // more, which the next loads go to.
        Halves h;
        int const ahead = min(kAhead, stages);
        for (int s = 0; s < ahead; ++s) { fetch(s); }
        int buffer = 0, free = kAhead;
        int s = 0;
        for (;;) {
            for (int const end = min(stages - kAhead, look); s < end; ++s) {
                arrived<(kAhead - 1) * kLoads>();
                fetch(free);
                read(buffer, h);
                multiply(h);
                free = buffer;
                buffer = buffer + 1 == BUFFERS ? 0 : buffer + 1;
            }
            if (s < look) { break; }
            look_at_sums();
        }
        for (; s < stages; ++s) {
            arrived<0>();
            read(buffer, h);
            multiply(h);
            buffer = buffer + 1 == BUFFERS ? 0 : buffer + 1;
        }
    }

    // 32 x 64 elements at a time go through LDS, so that a lane has neighbours of a row to store, or the rows of a column to sum
    if (p.slabs > 1) {
        o.kind = kOutStore; o.out = p.sums + slab * p.sums_slab; o.stride = p.sums_pitch; o.accumulate = 0;
    }
    float *const tile = reinterpret_cast<float *>(lds) + wave * 32 * kTilePitch;
    int const n0 = (rb_b + wn * TN) * 32;
    __syncthreads();                            // (the stages are done with LDS)
    float2 column = make_float2(-INFINITY, 0.0f);
#pragma unroll
    for (int i = 0; i < TM; ++i) { if (rb_a + wm * TM + i >= p.a_blocks) { again[i] = 0; } }
#pragma nounroll
    for (int i = 0; i < TM; ++i) {
        int const rb = rb_a + wm * TM + i, m0 = rb * 32;
        if (rb >= p.a_blocks) { break; }
        int eb[TN];
        float lb[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j) { eb[j] = scale_b[(wn * TN + j) * 32 + (lane & 31)]; lb[j] = limit_b[(wn * TN + j) * 32 + (lane & 31)]; }
        // (registers have no index; `which` is i, and the compiler does not know it: it would write the loop out, with all its addresses in registers at once)
        int which = i;
        asm volatile("" : "+s"(which));
        DenseAcc16 now[TN];
        uint32_t small = 0;
#pragma unroll
        for (int u = 0; u < TM; ++u) {
            if (u != which) { continue; }
#pragma unroll
            for (int j = 0; j < TN; ++j) { now[j] = acc[u][j]; }
            small = again[u];
        }
        bool odd = false;                           // some sum is below its limit, or no number
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            int const row = acc_row(r, lane), ea = scale_a[(wm * TM + i) * 32 + row];
            float const la = limit_a[(wm * TM + i) * 32 + row];
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                odd = odd | !(fabsf(now[j][r]) >= la + lb[j]);
                tile[row * kTilePitch + j * 32 + (lane & 31)] = ldexpf(now[j][r], -(ea + eb[j]));           // the scales come off
            }
        }
        bool const marks = p.slabs == 1 && __any(odd);
        uint32_t formed = 0;
        if (__builtin_expect(marks, 0)) {
            int at = lane;
            asm volatile("" : "+v"(at));            // (or the sums of limits from above stay in registers)
            uint32_t below = 0;                     // as look_at_sums has it
#pragma unroll
            for (int e = 16 * TN - 1; e >= 0; --e) {
                float const left = fabsf(now[e / 16][e % 16]) - (limit_a[(wm * TM + i) * 32 + acc_row(e % 16, at)] + limit_b[(wn * TN + e / 16) * 32 + (at & 31)]);
                below = __builtin_amdgcn_alignbit(below, __builtin_bit_cast(uint32_t, left), 31);
                if (e % 4 == 0) { __builtin_amdgcn_sched_barrier(0); }
            }
            below &= small;
#pragma unroll
            for (int e = 0; e < 16 * TN; ++e) {
                float *const d = tile + acc_row(e % 16, at) * kTilePitch + e / 16 * 32 + (at & 31);
                if (*d != *d || ((below >> e) & 1u)) {
                    formed |= 1u << e;
                    *d = __builtin_bit_cast(float, kNotStored);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < TM; ++u) { again[u] = u == which ? formed : again[u]; }
        int at = lane;
        asm volatile("" : "+v"(at));                // (nor are its addresses kept from one round to the next)
        finish<USE>(o, p.slabs > 1, tile, bias + (wm * TM + i) * 32, m0, n0, at, column, marks, false);
    }
    // A second time round for what is formed again (its code needs the registers that the accumulators have had)
    uint32_t any = 0;
#pragma unroll
    for (int u = 0; u < TM; ++u) { any |= again[u]; }
    if (__builtin_expect(p.slabs == 1 && __any(any != 0u), 0)) {
#pragma nounroll
        for (int i = 0; i < TM; ++i) {
            int const m0 = (rb_a + wm * TM + i) * 32;
            uint32_t here = 0;
#pragma unroll
            for (int u = 0; u < TM; ++u) { here = u == i ? again[u] : here; }
            // (not those outside, nor of frames that nothing is made of)
            for (int r = 0; r < 16; ++r) { if (m0 + acc_row(r, lane) >= o.rows) { here &= ~(0x10001u << r); } }
            for (int j = 0; j < TN; ++j) {
                int const n = n0 + j * 32 + (lane & 31);
                if (n >= o.columns || (USE == kUseLogits && !frame_counts(o, n))) { here &= ~(0xffffu << (16 * j)); }
            }
            if (!__any(here != 0u)) { continue; }
            for (int row = 0; row < 32; ++row) { tile[row * kTilePitch + lane] = __builtin_bit_cast(float, kNotStored); }
            tile_again<KA, KB>(p.src_a, p.src_b, tile, kTilePitch, here, m0, n0, lane);
            finish<USE>(o, false, tile, bias + (wm * TM + i) * 32, m0, n0, lane, column, true, true);
        }
    }
    if (USE == kUseLogits && p.slabs == 1 && n0 + lane < o.columns && rb_a + wm * TM < p.a_blocks) {
        o.partial[(long long)((rb_a + wm * TM) / TM) * o.columns + n0 + lane] = column;
    }
}

template <int TM, int WM, int WN, int BUFFERS>
constexpr int packed_lds(void)
{
    constexpr int kStages = BUFFERS * (TM * WM + 2 * WN) * 2048, kTiles = WM * WN * 32 * kTilePitch * 4;
    return kStages > kTiles ? kStages : kTiles;
}

template <int USE, int TM, int WM, int WN, int PB, int BUFFERS>
__global__ __launch_bounds__(WM * WN * 64, 2) void dense_packed_kernel(PackedProduct p)
{
    __shared__ __attribute__((aligned(1024))) char lds[packed_lds<TM, WM, WN, BUFFERS>()];
    __shared__ int scales[(TM * WM + 2 * WN) * 32];
    __shared__ float limits[(TM * WM + 2 * WN) * 32];
    __shared__ float bias[TM * WM * 32];
    packed_tile<USE, kRows, PB == 1 ? kBitColumns : kColumns, false, TM, WM, WN, PB, BUFFERS>(p, blockIdx.x, lds, scales, limits, bias);
}

// the weights' gradient, and behind it the input's (either may have no workgroups)
template <bool TRIPLE, int TM, int WM, int WN, int PB, int BUFFERS>
__global__ __launch_bounds__(WM * WN * 64, 2) void dense_packed_pair_kernel(PackedProduct p, PackedProduct q)
{
    __shared__ __attribute__((aligned(1024))) char lds[packed_lds<TM, WM, WN, BUFFERS>()];
    __shared__ int scales[(TM * WM + 2 * WN) * 32];
    __shared__ float limits[(TM * WM + 2 * WN) * 32];
    if ((int)blockIdx.x < p.workgroups) { packed_tile<kUseStore, kGradRows, PB == 1 ? kBitRows : kRows, TRIPLE, TM, WM, WN, PB, BUFFERS>(p, blockIdx.x, lds, scales, limits, nullptr); }
    else                                { packed_tile<kUseStore, kColumns, kGradColumns, TRIPLE, TM, WM, WN, 2, BUFFERS>(q, blockIdx.x - p.workgroups, lds, scales, limits, nullptr); }
}

// `top`: the largest magnitude of the sums
__device__ __forceinline__ float sum_of_slabs(PackedProduct const &p, int m, int n, float &top)
{
    float const *from = p.sums + m * p.sums_pitch + n;
    float d = 0.0f;
    int s = 0;
    for (; s + 4 <= p.slabs; s += 4) {
        float const a = from[s * p.sums_slab], b = from[(s + 1) * p.sums_slab], c = from[(s + 2) * p.sums_slab], e = from[(s + 3) * p.sums_slab];
        d = (((d + a) + b) + c) + e;
        top = fmaxf(fmaxf(fmaxf(fmaxf(top, fabsf(a)), fabsf(b)), fabsf(c)), fabsf(e));
    }
    for (; s < p.slabs; ++s) { float const a = from[s * p.sums_slab]; d += a; top = fmaxf(top, fabsf(a)); }
    top = fmaxf(top, fabsf(d));
    return d;
}

// as the tiles have it, with the scales off
__device__ __forceinline__ float limit_at(PackedProduct const &p, int m, int n)
{
    float const lost = p.lost_a[m] + p.lost_b[n];
    return p.b_pieces == 2 ? ldexpf(p.triple ? limit_of<2, true>(lost) : limit_of<2, false>(lost), -(p.ea[m] + p.eb[n])) : ldexpf(limit_of<1, false>(lost), -p.ea[m]);
}

// The slabs' sums of a product, in order, and what becomes of them: a wavefront takes 64 neighbours of a row.
__device__ __forceinline__ void join_slabs(PackedProduct const &p, unsigned id)
{
    DenseOutput const &o = p.out;
    unsigned const across = (unsigned)(p.sums_pitch / 64), unit = id * 4 + threadIdx.x / 64;
    int const lane = threadIdx.x & 63, m = (int)(unit / across), n = (int)(unit % across) * 64 + lane;
    if (m >= o.rows) { return; }
    bool const inside = n < o.columns || (n == o.columns && o.line && o.kind == kOutStore);
    float d = 0.0f;
    bool again = false;
    if (inside) {
        float const limit = p.kind_a >= 0 ? limit_at(p, m, n) : -INFINITY;
        float top = 0.0f;
        d = sum_of_slabs(p, m, n, top);
        again = p.kind_a >= 0 && (d != d || top < limit);
    }
    if (__builtin_expect(__any(again), 0)) { row_again(p.src_a, p.kind_a, p.src_b, p.kind_b, d, again, m, n - lane, lane); }
    if (o.kind == kOutForward) { if (inside) { static_cast<float *>(o.out)[m * o.stride + n] = activated(before_activation(o, d, m, n), o.activation); } }
    else if (o.kind == kOutBits) {
        uint64_t const bits = __ballot(inside && before_activation(o, d, m, inside ? n : 0) > 0.0f);
        if ((lane & 31) == 0 && inside) { static_cast<uint32_t *>(o.out)[m * o.stride + (n >> 5)] = (uint32_t)(bits >> (lane & 32)); }
    }
    else if (inside) { store_element(o, d, m, n); }
}

__global__ __launch_bounds__(256) void dense_join_kernel(PackedProduct p, PackedProduct q, unsigned first_blocks)
{
    if (blockIdx.x < first_blocks) { join_slabs(p, blockIdx.x); }
    else                           { join_slabs(q, blockIdx.x - first_blocks); }
}

// The same for logits: a workgroup takes 32 rows of 64 columns, each of its sixteen wavefronts two of the rows, four slabs of both at a time.
constexpr int kJoinLogitWaves = 16;
__global__ __launch_bounds__(kJoinLogitWaves * 64, 8) void dense_join_logits_kernel(PackedProduct p)
{
    __shared__ float2 part[kJoinLogitWaves][64];
    DenseOutput const &o = p.out;
    unsigned const across = (unsigned)(p.sums_pitch / 64);
    int const lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tile = (int)(blockIdx.x / across), n = (int)(blockIdx.x % across) * 64 + lane;
    int const m0 = tile * 32 + wave * 2;
    bool const inside = n < o.columns;
    int const label = inside ? o.label[n] - o.first_channel : -1;
    float z[2] = {}, top[2] = {}, limit[2] = {-INFINITY, -INFINITY};
    if (inside && p.kind_a >= 0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) { limit[i] = limit_at(p, min(m0 + i, o.rows - 1), n); }
    }
    if (inside) {
        // (a row behind the last one reads the last one)
        float const *const a = p.sums + min(m0, o.rows - 1) * p.sums_pitch + n, *const b = p.sums + min(m0 + 1, o.rows - 1) * p.sums_pitch + n;
        for (int s = 0; s < p.slabs; s += 4) {
            float u[4], v[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                long long const at = min(s + q, p.slabs - 1) * p.sums_slab;
                u[q] = a[at]; v[q] = b[at];
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                z[0] += s + q < p.slabs ? u[q] : 0.0f; z[1] += s + q < p.slabs ? v[q] : 0.0f;
                top[0] = fmaxf(top[0], fabsf(u[q])); top[1] = fmaxf(top[1], fabsf(v[q]));
            }
        }
    }
    bool again[2] = {};
    if (inside && p.kind_a >= 0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) { again[i] = z[i] != z[i] || fmaxf(top[i], fabsf(z[i])) < limit[i]; }
    }
    if (__builtin_expect(__any(again[0] || again[1]), 0)) {
#pragma nounroll
        for (int i = 0; i < 2; ++i) {
            float d = i ? z[1] : z[0];
            if (m0 + i < o.rows) { logit_again(p.src_a, p.src_b, p.kind_b, d, (i ? again[1] : again[0]) && frame_counts(o, n), m0 + i, n - lane, lane); }
            if (i) { z[1] = d; } else { z[0] = d; }
        }
    }
    float2 s = make_float2(-INFINITY, 0.0f);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        int const m = m0 + i;
        if (!inside || m >= o.rows) { z[i] = -INFINITY; continue; }
        z[i] += o.bias ? o.bias[m] : 0.0f;
        if (o.out) { static_cast<float *>(o.out)[m * o.stride + n] = z[i]; }
        if (label == m) { o.label_logit[n] = z[i]; }
        s.x = fmaxf(s.x, z[i]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) { s.y += z[i] == -INFINITY ? 0.0f : exp_of_nonpositive(z[i] - s.x); }
    part[wave][lane] = s;
    for (int step = kJoinLogitWaves / 2; step > 0; step /= 2) {
        __syncthreads();
        if (wave < step) { s = joined(s, part[wave + step][lane]); part[wave][lane] = s; }
    }
    if (wave == 0 && inside) { o.partial[(long long)tile * o.columns + n] = s; }
}

}  // namespace bbhip
