// The largest logits of every (pixel, frame), and a category drawn from them.
//
// Order: descending, equal values by ascending channel, anything that is not a number before all numbers, -0 equal to +0 (and returned as +0).  A value
// becomes a 32-bit key that orders as an unsigned number; with the channel behind it no two entries of a column are equal, so the result is unique.
//
// One pass over the logits.  A workgroup owns the columns of a tile and a slab of channels and reads 256 channels of each column at a time.  What is not above the
// column's bound (the k-th largest so far) is dropped by one comparison; the rest is appended to the column's list in LDS, in any order, and when a
// list could overflow with the next 256 channels, one wavefront per column cuts it to its k largest and raises the bound.  With random logits a column appends
// about k (1 + ln(channels / 256)) entries and is cut a few times.  Few columns are shared by several workgroups, a slab of channels each; a second launch
// selects from their lists.
//
// The k-th largest of a list is found bit by bit from the top: the count of keys that reach a candidate is the number of bits of a few ballots.
#pragma once

#include "column_tiles.hpp"
#include "corner_index.hpp"

namespace bbhip {

constexpr int kTopMost  = 256;                  // largest k
constexpr int kTopChunk = 256;                  // channels that a workgroup reads at a time, of each column
constexpr int kTopList  = kTopMost + kTopChunk; // entries of a column's list: cut to k <= kTopMost before each chunk that might not fit
constexpr int kTopJoin  = 1024;                 // entries that the second launch selects from

struct TopArgs {
    ColumnSpace c;                  // rows = channels
    TileDivisor tiles;
    float const *y;
    int         *index;             // top logits: [top * pix][list_stride]
    float       *logit;
    float const *u;                 // sampling: [pix][frame_stride], and so are
    int         *category;
    float       *share;             // the drawn category's share, or NULL
    uint2       *candidates;        // [slabs][units * W][top]: (key, channel), where several slabs share a column
    float temperature, top_p, min_p;
    int   top_size, pix_size, frame_stride, list_stride;
};

__device__ __forceinline__ uint32_t order_key(float v)
{
    uint32_t const b = v == 0.0f ? 0u : __float_as_uint(v);
    uint32_t const k = b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
    return v != v ? 0xffffffffu : k;
}
__device__ __forceinline__ float value_of_key(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu)); }

__device__ __forceinline__ int bits_below_lane(uint64_t mask)
{
    return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
}

// The k largest of n > k entries, entry i * 64 + lane in register i, to the front of key_out / index_out in any order; returns a lower bound of their keys.
// rows: above every channel.  A whole wavefront calls this.
template <int PER>
__device__ __forceinline__ uint32_t select_largest(uint32_t const (&key)[PER], int const (&index)[PER], int n, int k, int rows, uint32_t *key_out, int *index_out)
{
    int const lane = threadIdx.x % kWave;
    uint32_t bound = 0u;
    int reach = n;
    for (int bit = 31; bit >= 0 && reach != k; --bit) {
        uint32_t const candidate = bound | (1u << bit);
        int count = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) { count += __popcll(__ballot(i * kWave + lane < n && key[i] >= candidate)); }
        if (count >= k) { bound = candidate; reach = count; }
    }
    int last = rows;                                                            // of the entries that equal the bound, those up to here
    if (reach != k) {                                                           // (bound is the k-th largest key, and more than k entries reach it)
        int above = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) { above += __popcll(__ballot(i * kWave + lane < n && key[i] > bound)); }
        int const wanted = k - above;                                           // >= 1
        last = 0;
        for (int bit = 31 - __clz(rows); bit >= 0; --bit) {                     // the wanted-th smallest channel
            int const candidate = last | (1 << bit);
            int count = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i) { count += __popcll(__ballot(i * kWave + lane < n && key[i] == bound && index[i] < candidate)); }
            if (count < wanted) { last = candidate; }
        }
    }
    int base = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        bool const taken = i * kWave + lane < n && (key[i] > bound || (key[i] == bound && index[i] <= last));
        uint64_t const mask = __ballot(taken);
        if (taken) {
            int const at = base + bits_below_lane(mask);
            key_out[at] = key[i]; index_out[at] = index[i];
        }
        base += __popcll(mask);
    }
    return bound;
}

// k entries in LDS into their order, by counting for each those before it.  A whole wavefront calls this.
__device__ __forceinline__ void order_entries(uint32_t *key, int *index, int k)
{
    constexpr int PER = kTopMost / kWave;
    int const lane = threadIdx.x % kWave;
    uint32_t mine[PER];
    int at[PER], rank[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        int const e = i * kWave + lane;
        mine[i] = e < k ? key[e] : 0u;
        at[i]   = e < k ? index[e] : 0;
        rank[i] = 0;
    }
    for (int e = 0; e < k; ++e) {
        uint32_t const other = key[e];
        int const where = index[e];
#pragma unroll
        for (int i = 0; i < PER; ++i) { rank[i] += (other > mine[i] || (other == mine[i] && where < at[i])) ? 1 : 0; }
    }
    wave_fence();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if (i * kWave + lane < k) { key[rank[i]] = mine[i]; index[rank[i]] = at[i]; }
    }
    wave_fence();
}

// One category of k ordered entries: weights exp((z - z_0) / T); kept is the shortest prefix that holds top_p of their sum, of it those of at least min_p times the
// largest; drawn is the first whose sum with those before it exceeds u times the sum of the kept.  All of it in 64 bits: the drawn index is a whole number that the
// rounding of a sum must not move.  z_0 minus infinity or not a number: category -1, share 0.  A whole wavefront calls this.
__device__ __forceinline__ void draw_category(uint32_t const *key, int const *index, int k, float u, float temperature, float top_p, float min_p, int &category, float &share)
{
    constexpr int PER = kTopMost / kWave;
    int const lane = threadIdx.x % kWave;
    float const z0 = value_of_key(key[0]);
    if (!(z0 > -__builtin_inff())) { category = -1; share = 0.0f; return; }     // wave-uniform
    double weight[PER], up_to[PER], before = 0.0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        int const e = i * kWave + lane;
        float const z = e < k ? value_of_key(key[e]) : -__builtin_inff();
        weight[i] = z == z0 ? 1.0 : exp(((double)z - (double)z0) / (double)temperature);
        double sum = weight[i];
        if (i * kWave < k) {                                                    // wave-uniform
            for (int o = 1; o < kWave; o <<= 1) {
                double const left = __shfl_up(sum, o);
                if (lane >= o) { sum += left; }
            }
        }
        up_to[i] = before + sum;
        before += __shfl(sum, kWave - 1);
    }
    int kept = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        int const e = i * kWave + lane;
        bool const in = weight[i] > 0.0 && weight[i] >= (double)min_p && (top_p >= 1.0f || up_to[i] - weight[i] < (double)top_p * before);
        kept += __popcll(__ballot(e < k && (e == 0 || in)));
    }
    double total = 0.0;
#pragma unroll
    for (int i = 0; i < PER; ++i) { if ((kept - 1) / kWave == i) { total = __shfl(up_to[i], (kept - 1) % kWave); } }
    int drawn = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) { drawn += __popcll(__ballot(i * kWave + lane < kept && up_to[i] <= (double)u * total)); }
    drawn = drawn < kept ? drawn : kept - 1;
    category = index[drawn];
    double w = 0.0;
#pragma unroll
    for (int i = 0; i < PER; ++i) { if (drawn / kWave == i) { w = __shfl(weight[i], drawn % kWave); } }
    share = (float)(w / total);
}

// W = 4: a thread reads four frames of a channel, W = 1: one; TX threads side by side.  DRAW: a category instead of the list
template <int W, int TX, bool DRAW>
__global__ __launch_bounds__(kTopChunk * TX) void top_logits_scan_kernel(TopArgs a)
{
    constexpr int COLS = W * TX, AHEAD = 4;
    static_assert(COLS <= kTopChunk * TX / kWave, "a wavefront per column");
    __shared__ uint32_t key[COLS][kTopList];
    __shared__ int index[COLS][kTopList];
    __shared__ int count[COLS];
    __shared__ float bound[COLS];
    __shared__ int full[3];
    int const lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    int slab, tile;
    split_tile(xcd_remap(blockIdx.x, gridDim.x), a.tiles, slab, tile);
    int const tx = threadIdx.x % TX, ty = threadIdx.x / TX;
    ColumnUnit<W> const u(a.c, tile * TX + tx);
    int const begin = slab * a.c.slab_rows, end = begin + a.c.slab_rows < a.c.rows ? begin + a.c.slab_rows : a.c.rows;
    int const chunks = (end - begin + kTopChunk - 1) / kTopChunk, k = a.top_size;
    size_t const channel = (size_t)a.pix_size * a.frame_stride;
    float const *const y = a.y + (size_t)u.pix * a.frame_stride + u.f0;

    if (threadIdx.x < COLS) { count[threadIdx.x] = 0; bound[threadIdx.x] = __builtin_nanf(""); }
    if (threadIdx.x < 3) { full[threadIdx.x] = 0; }
    float v[AHEAD][W], drop[W];
    auto request = [&](int n, float (&to)[W]) {
        int const row = begin + n * kTopChunk + ty;
        column_load<W>(y + (size_t)(row < end ? row : begin) * channel, row < end ? u.live : 0, to);
    };
#pragma unroll
    for (int p = 0; p < AHEAD; ++p) { if (p < chunks) { request(p, v[p]); } }
#pragma unroll
    for (int j = 0; j < W; ++j) { drop[j] = __builtin_nanf(""); }               // (nothing is dropped)
    __syncthreads();
    for (int n0 = 0; n0 < chunks; n0 += AHEAD) {
#pragma unroll
        for (int p = 0; p < AHEAD; ++p) {
            int const n = n0 + p;
            if (n >= chunks) { break; }                                         // workgroup-uniform
            int const row = begin + n * kTopChunk + ty;
#pragma unroll
            for (int j = 0; j < W; ++j) {
                if (row < end && j < u.live && !(v[p][j] <= drop[j])) {
                    int const col = tx * W + j, at = atomicAdd(&count[col], 1);
                    key[col][at] = order_key(v[p][j]);
                    index[col][at] = row;
                    if (at >= kTopMost) { full[n % 3] = 1; }                    // the next chunk might not fit
                }
            }
            if (n + AHEAD < chunks) { request(n + AHEAD, v[p]); }
            __syncthreads();
            // (three flags in turn: the one read now is written again three chunks on, and cleared behind the next barrier, which no one passes before all have read it)
            bool const cut = full[n % 3] != 0;
            if (threadIdx.x == 0) { full[(n + 2) % 3] = 0; }
            if (cut) {                                                          // workgroup-uniform
                if (wave < COLS && count[wave] > kTopMost) {
                    constexpr int PER = kTopList / kWave;
                    int const entries = count[wave];
                    uint32_t ks[PER];
                    int is[PER];
#pragma unroll
                    for (int i = 0; i < PER; ++i) {
                        int const e = i * kWave + lane;
                        ks[i] = e < entries ? key[wave][e] : 0u;
                        is[i] = e < entries ? index[wave][e] : 0;
                    }
                    wave_fence();
                    uint32_t const low = select_largest<PER>(ks, is, entries, k, a.c.rows, key[wave], index[wave]);
                    if (lane == 0) { count[wave] = k; bound[wave] = value_of_key(low); }
                }
                __syncthreads();
#pragma unroll
                for (int j = 0; j < W; ++j) { drop[j] = bound[tx * W + j]; }
            }
        }
    }
    if (wave < COLS) {
        constexpr int PER = kTopList / kWave;
        int entries = count[wave];
        if (entries > k) {
            uint32_t ks[PER];
            int is[PER];
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                int const e = i * kWave + lane;
                ks[i] = e < entries ? key[wave][e] : 0u;
                is[i] = e < entries ? index[wave][e] : 0;
            }
            wave_fence();
            (void)select_largest<PER>(ks, is, entries, k, a.c.rows, key[wave], index[wave]);
            wave_fence();
            entries = k;
        }
        ColumnUnit<W> const mine(a.c, tile * TX + wave / W);
        if (wave % W < mine.live) {
            if (a.c.slabs > 1) {
                uint2 *const to = a.candidates + ((size_t)slab * (a.c.units * W) + mine.column + wave % W) * k;
                for (int e = lane; e < k; e += kWave) { to[e] = e < entries ? make_uint2(key[wave][e], (uint32_t)index[wave][e]) : make_uint2(0u, 0u); }    // (key 0: below every value)
            }
            else {
                order_entries(key[wave], index[wave], k);
                if (DRAW) {
                    size_t const at = (size_t)mine.pix * a.frame_stride + mine.f0 + wave % W;
                    int category;
                    float share;
                    draw_category(key[wave], index[wave], k, a.u[at], a.temperature, a.top_p, a.min_p, category, share);
                    if (lane == 0) {
                        a.category[at] = category;
                        if (a.share != nullptr) { a.share[at] = share; }
                    }
                }
            }
        }
    }
    if (!DRAW && a.c.slabs == 1) {
        __syncthreads();
        for (int e = threadIdx.x; e < k * COLS; e += kTopChunk * TX) {          // neighbouring columns side by side
            int const col = e % COLS, j = e / COLS;
            ColumnUnit<W> const of(a.c, tile * TX + col / W);
            if (col % W < of.live) {
                size_t const at = ((size_t)j * a.pix_size + of.pix) * a.list_stride + of.f0 + col % W;
                a.index[at] = index[col][j];
                a.logit[at] = value_of_key(key[col][j]);
            }
        }
    }
}

// the largest of the slabs' lists: a wavefront per column
template <int W, bool DRAW>
__global__ __launch_bounds__(kColBlock) void top_logits_join_kernel(TopArgs a)
{
    constexpr int PER = kTopJoin / kWave;
    __shared__ uint32_t key[kColWaves][kTopMost];
    __shared__ int index[kColWaves][kTopMost];
    int const lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, k = a.top_size, n = a.c.slabs * k;
    int const column = blockIdx.x * kColWaves + wave;
    ColumnUnit<W> const u(a.c, column / W);
    if (column % W >= u.live) { return; }                                       // (wavefronts of this kernel do not meet)
    uint32_t ks[PER];
    int is[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        int const e = i * kWave + lane;
        uint2 v = make_uint2(0u, 0u);
        if (e < n) {
            int const slab = e / k;
            v = a.candidates[((size_t)slab * (a.c.units * W) + column) * k + (e - slab * k)];
        }
        ks[i] = v.x; is[i] = (int)v.y;
    }
    (void)select_largest<PER>(ks, is, n, k, a.c.rows, key[wave], index[wave]);
    wave_fence();
    order_entries(key[wave], index[wave], k);
    if (DRAW) {
        size_t const at = (size_t)u.pix * a.frame_stride + u.f0 + column % W;
        int category;
        float share;
        draw_category(key[wave], index[wave], k, a.u[at], a.temperature, a.top_p, a.min_p, category, share);
        if (lane == 0) {
            a.category[at] = category;
            if (a.share != nullptr) { a.share[at] = share; }
        }
    }
    else {
        for (int j = lane; j < k; j += kWave) {
            size_t const at = ((size_t)j * a.pix_size + u.pix) * a.list_stride + u.f0 + column % W;
            a.index[at] = index[wave][j];
            a.logit[at] = value_of_key(key[wave][j]);
        }
    }
}

}  // namespace bbhip
