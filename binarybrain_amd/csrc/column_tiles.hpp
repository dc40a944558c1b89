// Sums and maxima down the columns of node-major, frame-minor buffers: a column is one (pixel, frame), its elements lie one row pitch (times
// the pixels) apart.  Shared by the operators that work frame by frame over all nodes: layer normalisation and what reads the logits.
//
// A unit is W consecutive frames of one row (W = 4: one 128-bit access where rows start on 16 bytes, else W = 1).  A workgroup owns a tile
// of `tx` consecutive units (a power of two up to the wavefront) and a slab of rows; lane l of a wavefront takes unit l % tx and
// row l / tx of the 64 / tx rows that the wavefront reads at once, so a load covers segments of 16 * tx bytes.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "lut_kernels.hpp"

namespace bbhip {

constexpr int kColBlock = 256;
constexpr int kColWaves = kColBlock / kWave;

struct ColumnSpace {
    TileDivisor units_per_row;      // units of one (pixel) row: ceil(frame_size / W)
    int units;                      // pix_size * units_per_row
    int frame_size;
    int log_tx;                     // tile width, log2
    int tiles;                      // ceil(units / tx)
    int rows, slab_rows, slabs;     // rows = nodes or channels
};

// the unit of a lane: where it lies in its row block and how many of its W frames exist (live 0: no such unit; it loads the first one)
template <int W>
struct ColumnUnit {
    int pix, f0, live, column;      // column: of its first frame, in the compact order of units
    __device__ __forceinline__ ColumnUnit(ColumnSpace const &c, int unit)
    {
        bool const in = unit < c.units;
        int const u = in ? unit : 0;
        int q;
        split_tile(u, c.units_per_row, pix, q);
        f0     = q * W;
        live   = in ? (c.frame_size - f0 < W ? c.frame_size - f0 : W) : 0;
        column = u * W;
    }
};

// W frames at p.  Whole: where the last unit of a row is not, what lies behind the frames is read too (a row's pitch is a multiple of W) and counts for nothing.
template <int W>
__device__ __forceinline__ void column_load(float const *__restrict__ p, float (&v)[W])
{
    if constexpr (W == 4) {
        float4 const t = *reinterpret_cast<float4 const *>(p);
        v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
    }
    else { v[0] = p[0]; }
}

// the same of an array that ends with its last frame: the absent ones 0
template <int W>
__device__ __forceinline__ void line_load(float const *__restrict__ p, int live, float (&v)[W])
{
#pragma unroll
    for (int j = 0; j < W; ++j) { v[j] = j < live ? p[j] : 0.0f; }
}

// STREAM: past the caches (what a second launch reads again would lose its place in them to the output).  Large outputs in segments of less than a cache line go through
// them, which joins the neighbours' halves: 4096 x 8192 frames in tiles of 64 bytes 68 us past the caches, 58 through them (1024 x 8192 14.4 and 16.3).
template <int W, bool STREAM = true>
__device__ __forceinline__ void column_store(float *__restrict__ p, int live, float const (&v)[W])
{
    if constexpr (W == 4) {
        if (live == 4) {
            using V = float __attribute__((ext_vector_type(4)));
            if constexpr (STREAM) { __builtin_nontemporal_store(V{v[0], v[1], v[2], v[3]}, reinterpret_cast<V *>(p)); }
            else                  { *reinterpret_cast<V *>(p) = V{v[0], v[1], v[2], v[3]}; }
            return;
        }
    }
#pragma unroll
    for (int j = 0; j < W; ++j) { if (j < live) { p[j] = v[j]; } }
}

// A second launch over the same data goes through it backwards (`block` of ColumnThread counted from the end): what the first launch read last is still in
// the 256 MiB memory-side cache.
__device__ __forceinline__ int backwards(int block, int blocks) { return blocks - 1 - block; }

// where a thread of a workgroup stands: one unit, rows begin + lead, + step, ... below end of its slab
template <int W>
struct ColumnThread {
    int slab, tile, tx, begin, lead, step, end;
    __device__ __forceinline__ ColumnThread(ColumnSpace const &c, TileDivisor const &tiles, int block, int blocks)
    {
        int const lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
        split_tile(xcd_remap(block, blocks), tiles, slab, tile);
        tx = lane & ((1 << c.log_tx) - 1);
        int const at_once = kWave >> c.log_tx;
        begin = slab * c.slab_rows;
        lead  = wave * at_once + (lane >> c.log_tx);
        step  = kColWaves * at_once;
        end   = begin + c.slab_rows < c.rows ? begin + c.slab_rows : c.rows;
    }
    // body(base, whole) for every B rows of a thread, rows base + lead + i * step; whole (a compile-time truth): all of them exist
    template <int B, class F>
    __device__ __forceinline__ void each(F body) const
    {
        int base = begin;
        for (; base + B * step <= end; base += B * step) { body(base, std::true_type()); }      // workgroup-uniform
        if (base < end) { body(base, std::false_type()); }
    }
    // The same with the loads of the next B rows issued before the present ones are used: start(base, held) before what the use waits for anyway, then
    // follow(held, start, use).  start loads only rows below end, use(base, held) uses only those.
    template <int B, class Held, class S, class U>
    __device__ __forceinline__ void follow(Held &held, S start, U use) const
    {
        for (int base = begin; base < end; base += B * step) {                  // workgroup-uniform
            Held next = held;
            if (base + B * step < end) { start(base + B * step, next); }
            use(base, held);
            held = next;
        }
    }
};

}  // namespace bbhip
