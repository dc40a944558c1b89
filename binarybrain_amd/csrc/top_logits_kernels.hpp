// The largest logits of every (pixel, frame), and a category drawn from them.
//
// Order: descending, equal values by ascending channel, anything that is not a number before all numbers, -0 equal to +0 (and returned as +0).  A value
// becomes a 32-bit key that orders as an unsigned number; with the channel behind it no two entries of a column are equal, so the result is unique.
//
// One pass over the logits.  A workgroup owns the columns of a tile and a slab of channels; its threads hold 12 channels of their columns in registers at a time.  Of the
// first ones the maxima of 256 or 512 groups of channels are taken: the k-th largest of those bounds the k-th largest logit from below, and with random logits
// 72 of 1536 reach the bound of k = 64.  What is below is dropped by one comparison, the rest is appended to the column's list in LDS, in any order, and the next channels are
// requested.  Logits that defeat the bound (ascending ones, ties) make a list overflow: those channels are appended again, a few at a time, with the lists cut to their k
// largest in between.  Few columns are shared by several workgroups, a slab of channels each; a second launch selects from their lists.
// 32768 channels x 1024 frames, k = 64, logits with many ties: 51 us for the scan (33 without bounds and lists: the loads; the bounds take about 5, the appends 3, the
// cuts of the lists 10) and 9 us for the join; 27 vector instructions per logit, a little less than half of the time.
//
// The k-th largest of a list is found bit by bit from the top: the count of keys that reach a candidate is the number of bits of a few ballots.
#pragma once

#include "column_tiles.hpp"
#include "corner_index.hpp"

namespace bbhip {

constexpr int kTopMost = 256;                   // largest k
constexpr int kTopJoin = 1024;                  // entries that the second launch selects from
constexpr int kTopFew  = 32;                    // channels up to which a lane takes a column by itself

// TX threads side by side: a workgroup reads this many channels of each column with one load per thread ...
template <int TX> constexpr int kTopRows = TX == 1 ? 256 : 128;
// ... of which it holds so many at a time (128 registers let two workgroups share a compute unit) ...
constexpr int kTopHeld = 12;
// ... and a column's list holds these besides the kTopMost that it is cut to
template <int TX> constexpr int kTopList = kTopMost + kTopRows<TX>;

// up to this k the bounds come from 256 groups of channels, above from 512 (72 of 1536 random logits reach the bound of k = 64, 316 that of k = 256)
constexpr int kTopFewGroups = 96;

struct TopArgs {
    ColumnSpace c;                  // rows = channels
    TileDivisor tiles, entries;     // entries: top_size
    float const *y;
    int         *index;             // top logits: [top * pix][list_stride]
    float       *logit;
    float const *u;                 // sampling: [pix][frame_stride], and so are
    int         *category;
    float       *share;             // the drawn category's share, or NULL
    uint64_t    *candidates;        // [slabs][units * W][top], where several slabs share a column
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

// an entry of a list: of two, the larger number comes first
__device__ __forceinline__ uint64_t entry_of(uint32_t key, int channel) { return ((uint64_t)key << 32) | (uint32_t)~channel; }
__device__ __forceinline__ uint32_t key_of(uint64_t entry)              { return (uint32_t)(entry >> 32); }
__device__ __forceinline__ int      channel_of(uint64_t entry)          { return (int)~(uint32_t)entry; }

// The k-th largest of n >= k keys, key i * 64 + lane in register i (0 behind them): bit by bit from the top, the keys that reach a candidate counted by ballots; bits
// that all keys agree in are passed over.  `reach`: how many keys reach the returned bound; k where the search could stop early, and then the bound itself need not be a
// key.  A whole wavefront calls this.
template <int PER>
__device__ __forceinline__ uint32_t kth_key(uint32_t const (&key)[PER], int n, int k, int &reach)
{
    int const lane = threadIdx.x % kWave;
    uint32_t const one = (uint32_t)__builtin_amdgcn_readfirstlane((int)key[0]);
    uint32_t differ = 0u;
#pragma unroll
    for (int i = 0; i < PER; ++i) { differ |= i * kWave + lane < n ? key[i] ^ one : 0u; }
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) { differ |= lane_xor(differ, o); }
    uint32_t open = (uint32_t)__builtin_amdgcn_readfirstlane((int)differ), bound = one & ~open;
    reach = n;
    while (open != 0u && reach != k) {
        uint32_t const bit = 0x80000000u >> __clz((int)open), candidate = bound | bit;
        open &= ~bit;
        int count = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) { count += __popcll(__ballot(key[i] >= candidate)); }
        if (count >= k) { bound = candidate; reach = count; }
    }
    return bound;
}

// The k largest of n > k entries, entry i * 64 + lane in register i (key 0 behind them), to the front of `list` in any order; returns a lower bound of their keys.  rows:
// above every channel.  A whole wavefront calls this.
template <int PER>
__device__ __forceinline__ uint32_t select_entries(uint32_t const (&key)[PER], int const (&channel)[PER], int n, int k, int rows, uint64_t *list)
{
    int reach;
    uint32_t const bound = kth_key<PER>(key, n, k, reach);                      // (above 0: so is every key, and what is behind the entries is not taken)
    int last = rows;                                                            // of the entries that equal the bound, those up to here
    if (reach != k) {                                                           // (bound is the k-th largest key, and more than k entries reach it)
        int above = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) { above += __popcll(__ballot(key[i] > bound)); }
        int const wanted = k - above;                                           // >= 1
        last = 0;
        for (int bit = 31 - __clz(rows); bit >= 0; --bit) {                     // the wanted-th smallest channel
            int const candidate = last | (1 << bit);
            int count = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i) { count += __popcll(__ballot(key[i] == bound && channel[i] < candidate)); }
            if (count < wanted) { last = candidate; }
        }
    }
    int base = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        bool const taken = key[i] > bound || (key[i] == bound && channel[i] <= last);
        uint64_t const mask = __ballot(taken);
        if (taken) { list[base + bits_below_lane(mask)] = entry_of(key[i], channel[i]); }
        base += __popcll(mask);
    }
    wave_fence();
    return bound;
}
// the same within a list in LDS
template <int PER>
__device__ __forceinline__ uint32_t cut_list_of(uint64_t *list, int n, int k, int rows)
{
    int const lane = threadIdx.x % kWave;
    uint32_t key[PER];
    int channel[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        int const e = i * kWave + lane;
        uint64_t const v = e < n ? list[e] : 0u;
        key[i] = key_of(v); channel[i] = channel_of(v);
    }
    wave_fence();
    return select_entries<PER>(key, channel, n, k, rows, list);
}
// with as many registers as the list needs
template <int MOST>
__device__ __forceinline__ uint32_t cut_list(uint64_t *list, int n, int k, int rows)
{
    if (n <= 4 * kWave) { return cut_list_of<4>(list, n, k, rows); }
    return cut_list_of<MOST / kWave>(list, n, k, rows);
}

// k entries in LDS into their order, by counting for each those before it.  A whole wavefront calls this.
template <int PER>
__device__ __forceinline__ void order_list_of(uint64_t *list, int k)
{
    int const lane = threadIdx.x % kWave;
    uint64_t mine[PER];
    int rank[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) { mine[i] = i * kWave + lane < k ? list[i * kWave + lane] : 0u; rank[i] = 0; }
#pragma unroll 4
    for (int e = 0; e < k; ++e) {
        uint64_t const other = list[e];
#pragma unroll
        for (int i = 0; i < PER; ++i) { rank[i] += other > mine[i] ? 1 : 0; }
    }
    wave_fence();
#pragma unroll
    for (int i = 0; i < PER; ++i) { if (i * kWave + lane < k) { list[rank[i]] = mine[i]; } }
    wave_fence();
}
__device__ __forceinline__ void order_list(uint64_t *list, int k)
{
    if (k <= kWave) { order_list_of<1>(list, k); }
    else            { order_list_of<kTopMost / kWave>(list, k); }
}

// One category of k ordered entries: weights exp((z - z_0) / T); kept is the shortest prefix that holds top_p of their sum, of it those of at least min_p times the
// largest; drawn is the first whose sum with those before it exceeds u times the sum of the kept.  All of it in 64 bits: the drawn index is a whole number that the
// rounding of a sum must not move.  z_0 minus infinity or not a number: category -1, share 0.  A whole wavefront calls this.
template <int PER>
__device__ __forceinline__ void draw_of(uint64_t const *list, int k, float u, float temperature, float top_p, float min_p, int &category, float &share)
{
    int const lane = threadIdx.x % kWave;
    float const z0 = value_of_key(key_of(list[0]));
    if (!(z0 > -__builtin_inff())) { category = -1; share = 0.0f; return; }     // wave-uniform
    double weight[PER], up_to[PER], before = 0.0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        int const e = i * kWave + lane;
        float const z = e < k ? value_of_key(key_of(list[e])) : -__builtin_inff();
        weight[i] = z == z0 ? 1.0 : exp(((double)z - (double)z0) / (double)temperature);
        double sum = weight[i];
        for (int o = 1; o < kWave; o <<= 1) {
            double const left = __shfl_up(sum, o);
            if (lane >= o) { sum += left; }
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
    category = channel_of(list[drawn]);
    double w = 0.0;
#pragma unroll
    for (int i = 0; i < PER; ++i) { if (drawn / kWave == i) { w = __shfl(weight[i], drawn % kWave); } }
    share = (float)(w / total);
}
// of the column at `at` of the buffers of one row per pixel
__device__ __forceinline__ void draw_category(TopArgs const &a, uint64_t const *list, size_t at)
{
    int category;
    float share;
    if (a.top_size <= kWave) { draw_of<1>(list, a.top_size, a.u[at], a.temperature, a.top_p, a.min_p, category, share); }
    else                     { draw_of<kTopMost / kWave>(list, a.top_size, a.u[at], a.temperature, a.top_p, a.min_p, category, share); }
    if (threadIdx.x % kWave == 0) {
        a.category[at] = category;
        if (a.share != nullptr) { a.share[at] = share; }
    }
}

// W = 4: a thread reads four frames of a channel, W = 1: one; TX threads side by side.  DRAW: a category instead of the list.  GROUPS: of channels, whose maxima give the bounds
template <int W, int TX, bool DRAW, int GROUPS>
__global__ __launch_bounds__(kTopRows<TX> * TX, 4) void top_logits_scan_kernel(TopArgs a)
{
    constexpr int COLS = W * TX, ROWS = kTopRows<TX>, BLOCK = ROWS * TX, WAVES = BLOCK / kWave, HELD = kTopHeld, LIST = kTopList<TX>;
    __shared__ uint64_t list[COLS][LIST];
    __shared__ int count[COLS], before[COLS];
    __shared__ float bound[COLS];
    __shared__ int full[3], over;
    int const lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    int slab, tile;
    split_tile(xcd_remap(blockIdx.x, gridDim.x), a.tiles, slab, tile);
    int const tx = threadIdx.x % TX, ty = threadIdx.x / TX;
    ColumnUnit<W> const u(a.c, tile * TX + tx);
    int const begin = slab * a.c.slab_rows, end = begin + a.c.slab_rows < a.c.rows ? begin + a.c.slab_rows : a.c.rows;
    int const k = a.top_size;
    size_t const channel = (size_t)a.pix_size * a.frame_stride;
    float const *const y = a.y + (size_t)u.pix * a.frame_stride + u.f0;

    float v[HELD][W], drop[W];
    float const *const mine = y + (size_t)ty * channel;                         // (what is common to a load is added to it in scalar registers)
    auto request = [&](int from) {
        if (from + HELD * ROWS <= end) {                                        // workgroup-uniform
#pragma unroll
            for (int i = 0; i < HELD; ++i) { column_load<W>(mine + (size_t)(from + i * ROWS) * channel, v[i]); }
        }
        else {
#pragma unroll
            for (int i = 0; i < HELD; ++i) { if (from + i * ROWS + ty < end) { column_load<W>(mine + (size_t)(from + i * ROWS) * channel, v[i]); } }
        }
    };
    // (not a number drops nothing)
#pragma unroll
    for (int j = 0; j < W; ++j) { drop[j] = __builtin_nanf(""); }
    if (threadIdx.x < COLS) { count[threadIdx.x] = 0; }
    if (threadIdx.x == 0) { over = 0; }
    if (threadIdx.x < 3) { full[threadIdx.x] = 0; }

    request(begin);
    for (int from = begin; from < end; from += HELD * ROWS) {
        if (from == begin && end - begin >= 2 * kTopMost) {
            // The k-th largest of the maxima of the groups: as many entries are no smaller, so it bounds the k-th largest entry from below, and hardly more than k entries
            // reach it where the groups are many against k.
            constexpr int PARTS = GROUPS / ROWS, PER = GROUPS / kWave;
            uint32_t *const maxima = reinterpret_cast<uint32_t *>(&list[0][0]);                          // [COLS][GROUPS]
            static_assert(GROUPS * sizeof(uint32_t) <= LIST * sizeof(uint64_t) && HELD % PARTS == 0, "they fit where the lists will be");
#pragma unroll
            for (int g = 0; g < PARTS; ++g) {
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    float top = -__builtin_inff();
#pragma unroll
                    for (int i = g * HELD / PARTS; i < (g + 1) * HELD / PARTS; ++i) { top = fmaxf(top, from + i * ROWS + ty < end ? v[i][j] : top); }
                    maxima[(tx * W + j) * GROUPS + g * ROWS + ty] = from + g * HELD / PARTS * ROWS + ty < end ? order_key(top) : 0u;      // (0: a group without channels)
                }
            }
            __syncthreads();
            for (int col = wave; col < COLS; col += WAVES) {
                uint32_t key[PER];
                int reach;
#pragma unroll
                for (int i = 0; i < PER; ++i) { key[i] = maxima[col * GROUPS + i * kWave + lane]; }
                uint32_t low = kth_key<PER>(key, GROUPS, k, reach);
                // entries equal to the bound count: dropped is what is not above the key before it (that of -0 is no value's: the one before that)
                low = low == 0u ? 0u : low == 0x80000000u ? low - 2u : low - 1u;
                if (lane == 0) { bound[col] = value_of_key(low); }
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < W; ++j) { drop[j] = bound[tx * W + j]; }
        }
        // What is left goes to the lists, in any order.  All held channels at once; where a list would overflow they are taken back and appended with one load of channels
        // at a time, each time cutting the lists that might not hold the next.
        if (threadIdx.x < COLS) { before[threadIdx.x] = count[threadIdx.x]; }
        __syncthreads();
        // (one request for a place per thread and column, for all that it has)
        int at[W];
        bool any = false;
#pragma unroll
        for (int j = 0; j < W; ++j) {
            int mine_of = 0;
#pragma unroll
            for (int i = 0; i < HELD; ++i) { mine_of += from + i * ROWS + ty < end && !(v[i][j] <= drop[j]) ? 1 : 0; }
            mine_of = j < u.live ? mine_of : 0;
            at[j] = LIST;
            if (mine_of > 0) {
                any = true;
                at[j] = atomicAdd(&count[tx * W + j], mine_of);
                if (at[j] + mine_of > LIST) { over = 1; }
            }
        }
        if (any) {
#pragma unroll
            for (int i = 0; i < HELD; ++i) {
                int const row = from + i * ROWS + ty;
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    if (row < end && !(v[i][j] <= drop[j])) {
                        if (at[j] < LIST) { list[tx * W + j][at[j]] = entry_of(order_key(v[i][j]), row); }
                        at[j] += 1;
                    }
                }
            }
        }
        __syncthreads();
        if (over != 0) {                                                        // workgroup-uniform
            __syncthreads();
            if (threadIdx.x < COLS) { count[threadIdx.x] = before[threadIdx.x]; }
            if (threadIdx.x == 0) { over = 0; }
            // (the lists hold at most kTopMost entries here: those of the channels before were cut)
            __syncthreads();
            for (int i = 0; i < HELD; ++i) {                                    // (read again: a loop cannot index registers, and unrolled it would not fit the instruction cache)
                int const row = from + i * ROWS + ty;
                float r[W];
                if (row < end) { column_load<W>(mine + (size_t)(from + i * ROWS) * channel, r); }
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    if (row < end && j < u.live && !(r[j] <= drop[j])) {
                        int const col = tx * W + j, at = atomicAdd(&count[col], 1);
                        list[col][at] = entry_of(order_key(r[j]), row);
                        if (at >= kTopMost) { full[i % 3] = 1; }                // the next channels might not fit
                    }
                }
                __syncthreads();
                // (three flags in turn: the one read now is written again three loads on, and cleared behind the next barrier, which no one passes before all have read it)
                bool const some = full[i % 3] != 0;
                if (threadIdx.x == 0) { full[(i + 2) % 3] = 0; }
                if (some) {                                                     // workgroup-uniform
                    for (int col = wave; col < COLS; col += WAVES) {
                        int const entries = count[col];
                        if (entries > kTopMost) {
                            uint32_t const low = cut_list<LIST>(list[col], entries, k, a.c.rows);
                            if (lane == 0) { count[col] = k; bound[col] = value_of_key(low); }
                        }
                        else if (lane == 0) { bound[col] = __builtin_nanf(""); }
                    }
                    __syncthreads();
#pragma unroll
                    for (int j = 0; j < W; ++j) {
                        float const b = bound[tx * W + j];
                        if (b == b) { drop[j] = b; }
                    }
                }
            }
            __syncthreads();
            if (threadIdx.x < 3) { full[threadIdx.x] = 0; }
        }
        if (from + HELD * ROWS < end) {
            // (more to come: lists that hold more than kTopMost entries are cut, which also raises their bounds.  The next channels are on their way meanwhile)
            request(from + HELD * ROWS);
            for (int col = wave; col < COLS; col += WAVES) {
                int const entries = count[col];
                float low = __builtin_nanf("");
                if (entries > kTopMost) {
                    low = value_of_key(cut_list<LIST>(list[col], entries, k, a.c.rows));
                    if (lane == 0) { count[col] = k; }
                }
                if (lane == 0) { bound[col] = low; }
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < W; ++j) {
                float const b = bound[tx * W + j];
                if (b == b) { drop[j] = b; }                                    // (a bound that is not a number, or none: the one before stays)
            }
        }
    }
    for (int col = wave; col < COLS; col += WAVES) {
        int entries = count[col];
        ColumnUnit<W> const of(a.c, tile * TX + col / W);
        if (col % W >= of.live) { continue; }                                 // wave-uniform
        if (entries > k) {
            (void)cut_list<LIST>(list[col], entries, k, a.c.rows);
            entries = k;
        }
        if (a.c.slabs > 1) {
            uint64_t *const to = a.candidates + ((size_t)slab * (a.c.units * W) + of.column + col % W) * k;
            for (int e = lane; e < k; e += kWave) { to[e] = e < entries ? list[col][e] : 0u; }          // (0: below every entry)
        }
        else {
            order_list(list[col], k);
            if (DRAW) { draw_category(a, list[col], (size_t)of.pix * a.frame_stride + of.f0 + col % W); }
        }
    }
    if (!DRAW && a.c.slabs == 1) {
        __syncthreads();
        for (int e = threadIdx.x; e < k * COLS; e += BLOCK) {                   // neighbouring columns side by side
            int const col = e % COLS, j = e / COLS;
            ColumnUnit<W> const of(a.c, tile * TX + col / W);
            if (col % W < of.live) {
                size_t const at = ((size_t)j * a.pix_size + of.pix) * a.list_stride + of.f0 + col % W;
                a.index[at] = channel_of(list[col][j]);
                a.logit[at] = value_of_key(key_of(list[col][j]));
            }
        }
    }
}

// the largest of the slabs' lists: a wavefront per column, PER entries per lane
template <int W, bool DRAW, int PER>
__global__ __launch_bounds__(kColBlock) void top_logits_join_kernel(TopArgs a)
{
    __shared__ uint64_t lists[kColWaves][kTopMost];
    int const lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, k = a.top_size, n = a.c.slabs * k;
    int const column = blockIdx.x * kColWaves + wave;
    ColumnUnit<W> const u(a.c, column / W);
    if (column % W >= u.live) { return; }                                       // (wavefronts of this kernel do not meet)
    uint64_t *const list = lists[wave];
    uint64_t v[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {                                             // (all requested before the first is waited for)
        int slab, j;
        split_tile(i * kWave + lane < n ? i * kWave + lane : 0, a.entries, slab, j);
        v[i] = a.candidates[((size_t)slab * (a.c.units * W) + column) * k + j];
    }
    uint32_t key[PER];
    int channel[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) { key[i] = i * kWave + lane < n ? key_of(v[i]) : 0u; channel[i] = channel_of(v[i]); }
    (void)select_entries<PER>(key, channel, n, k, a.c.rows, list);
    order_list(list, k);
    if (DRAW) { draw_category(a, list, (size_t)u.pix * a.frame_stride + u.f0 + column % W); }
    else {
        for (int j = lane; j < k; j += kWave) {
            size_t const at = ((size_t)j * a.pix_size + u.pix) * a.list_stride + u.f0 + column % W;
            a.index[at] = channel_of(list[j]);
            a.logit[at] = value_of_key(key_of(list[j]));
        }
    }
}

// Few channels (at most MOST): a lane takes a column, its keys in registers, and finds one entry after the other.
template <int MOST, bool DRAW>
__global__ __launch_bounds__(kWave) void top_logits_few_kernel(TopArgs a)
{
    __shared__ double weight[DRAW ? MOST : 1][kWave];
    __shared__ int which[DRAW ? MOST : 1][kWave];
    int const lane = threadIdx.x, column = blockIdx.x * kWave + lane, k = a.top_size;
    ColumnUnit<1> const u(a.c, column);
    size_t const channel = (size_t)a.pix_size * a.frame_stride, at = (size_t)u.pix * a.frame_stride + u.f0;
    float v[MOST];
    uint32_t key[MOST];
#pragma unroll
    for (int i = 0; i < MOST; ++i) { v[i] = a.y[at + (i < a.c.rows ? i : 0) * channel]; }                       // (a lane without a column: the first one's)
#pragma unroll
    for (int i = 0; i < MOST; ++i) { key[i] = i < a.c.rows ? order_key(v[i]) : 0u; }
    float z0 = 0.0f;
    double all = 0.0;
    for (int j = 0; j < k; ++j) {
        uint32_t top = 0u;
        int found = 0;
#pragma unroll
        for (int i = 0; i < MOST; ++i) {
            if (key[i] > top) { top = key[i]; found = i; }
        }
#pragma unroll
        for (int i = 0; i < MOST; ++i) { key[i] = i == found ? 0u : key[i]; }
        if (DRAW) {
            float const z = value_of_key(top);
            if (j == 0) { z0 = z; }
            double const w = z == z0 ? 1.0 : exp(((double)z - (double)z0) / (double)a.temperature);
            weight[j][lane] = w; which[j][lane] = found;
            all += w;
        }
        else if (u.live > 0) {
            size_t const to = ((size_t)j * a.pix_size + u.pix) * a.list_stride + u.f0;
            a.index[to] = found;
            a.logit[to] = value_of_key(top);
        }
    }
    if (DRAW) {
        int category = -1;
        float share = 0.0f;
        if (z0 > -__builtin_inff()) {
            double total = 0.0, sum = 0.0, w = 1.0;
            int kept = 0;
            for (; kept < k; ++kept) {
                w = weight[kept][lane];
                if (kept > 0 && !(w > 0.0 && w >= (double)a.min_p && (a.top_p >= 1.0f || total < (double)a.top_p * all))) { break; }
                total += w;
            }
            double const reach = (double)a.u[at] * total;
            int drawn = 0;
            for (; ; ++drawn) {
                w = weight[drawn][lane];
                sum += w;
                if (drawn == kept - 1 || !(sum <= reach)) { break; }
            }
            category = which[drawn][lane];
            share = (float)(w / total);
        }
        if (u.live > 0) {
            a.category[at] = category;
            if (a.share != nullptr) { a.share[at] = share; }
        }
    }
}

}  // namespace bbhip
