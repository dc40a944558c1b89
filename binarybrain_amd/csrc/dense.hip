// Host side of the entries of dense layers, of the loss on top of one and of the clipping of gradients (include/bbhip.h): argument checks, how a call is divided,
// launches.  The kernels are in dense_*.hpp and gradient_norm_kernels.hpp.

#include <hip/hip_runtime.h>

#include <new>

#include "../../include/bbhip.h"
#include "host_calls.hpp"
#include "launch_rules.hpp"
#include "dense_rules.hpp"
#include "dense_direct_kernels.hpp"
#include "dense_loss_kernels.hpp"
#include "dense_packed_kernels.hpp"
#include "gradient_norm_kernels.hpp"

using namespace bbhip;

namespace {

// a product as the entries describe it, before it is known how it is computed
struct Product {
    Operand     a, b;
    int         kind_a, kind_b;
    DenseOutput out;
    bool wanted = true;
};

Operand rows_of(float const *p, long long stride, int rows, int depth)
{
    Operand o{};
    o.p = p; o.stride = stride; o.rows = rows; o.depth = depth; o.ones = -1;
    o.vec = starts_on_16_bytes(p) && stride % 4 == 0;
    return o;
}

int check_tiles(long long tiles, int threads, char const *name)
{
    if (tiles > 0 && !launch_holds(tiles, threads)) { return fail("%s: a launch of %lld workgroups of %d threads: 2^32 threads or more", name, tiles, threads); }
    return 0;
}

// Takes pieces of a workspace, or counts them (base null)
struct Carver {
    char *base;
    size_t at = 0;
    template <class E> E *take(size_t count)
    {
        E *const p = base ? reinterpret_cast<E *>(base + at) : nullptr;
        at += align256(count * sizeof(E));
        return p;
    }
};

// the sums of workgroups that share a product's k axis (columns and perhaps one more)
long long sums_pitch(int columns) { return ceil_div(columns, 64) * 64LL; }
float *sums_of(Carver &c, int slabs, int rows, int columns) { return slabs > 1 ? c.take<float>((size_t)slabs * rows * sums_pitch(columns)) : nullptr; }

// added up, and what becomes of them; q may have none
int join(PackedProduct const &p, PackedProduct const &q, hipStream_t st, char const *name)
{
    if (p.slabs > 1 && p.out.kind == kOutLogits) {
        long long const blocks = ceil_div(p.out.rows, 32) * (p.sums_pitch / 64);
        if (check_tiles(blocks, kJoinLogitWaves * 64, name)) { return 1; }
        launch(dense_join_logits_kernel, dim3((unsigned)blocks), dim3(kJoinLogitWaves * 64), 0, st, p);
        BBHIP_LAUNCH_CHECK();
        return 0;
    }
    auto const blocks = [](PackedProduct const &d) { return d.slabs > 1 ? ((long long)d.out.rows * d.sums_pitch + 255) / 256 : 0; };
    long long const first = blocks(p), second = blocks(q);
    if (first + second == 0) { return 0; }
    if (check_tiles(first + second, 256, name)) { return 1; }
    launch(dense_join_kernel, dim3((unsigned)(first + second)), dim3(256), 0, st, p, q, (unsigned)first);
    BBHIP_LAUNCH_CHECK();
    return 0;
}

// ---- products straight from the operands ----
int direct(DirectProduct &d, Product const &p, DirectShape const &s, float *sums, int columns, char const *name)
{
    d = DirectProduct{};
    d.slabs = 1;
    if (!p.wanted) { return 0; }
    d.a = p.a; d.b = p.b; d.out = p.out;
    d.n_tiles = s.n_tiles; d.slabs = s.slabs; d.slab_chunks = s.slab_chunks;
    d.sums = sums; d.sums_pitch = sums_pitch(columns); d.sums_slab = d.sums_pitch * p.out.rows;
    if (check_tiles(s.tiles * s.slabs, s.waves * 64, name)) { return 1; }
    d.tiles = (int)s.tiles;
    return 0;
}

PackedProduct sums_to_join(DirectProduct const &d)
{
    PackedProduct p{};
    p.slabs = d.tiles ? d.slabs : 1; p.sums = d.sums; p.sums_pitch = d.sums_pitch; p.sums_slab = d.sums_slab; p.out = d.out; p.kind_a = -1;
    return p;
}

bool few_frames(Product const &p) { return p.out.columns <= kFewFrames && p.out.kind != kOutLogits; }

int few_frames_forward(Product const &p, bool bit, hipStream_t st, char const *name)
{
    DirectProduct d{};
    d.a = p.a; d.b = p.b; d.out = p.out;
    // Four rows for a wavefront, which read a frame's value once, where wavefronts of one row would not run all at once (32 KB of LDS per workgroup: five on a compute unit).  1024 inputs, one frame:
    // 4096 outputs 5.3 us with one row and 7.1 with four, 8192 10.2 and 8.4; eight frames: 9.6 and 10.8, 20.2 and 13.4; 8192 x 8192 x 8 frames 131 and 68.
    bool const four = p.out.rows > 5 * 256 * kFewWaves;
    long long const blocks = ceil_div(p.out.rows, kFewWaves * (four ? 4 : 1));
    if (check_tiles(blocks, kFewWaves * 64, name)) { return 1; }
    dim3 const grid((unsigned)blocks), block(kFewWaves * 64);
#define BBHIP_FEW(KIND, FRAMES)                                                                                         \
    do {                                                                                                                \
        if (four) { if (p.a.vec) { launch((dense_few_frames_kernel<KIND, FRAMES, 4, true>), grid, block, 0, st, d); }   \
                    else         { launch((dense_few_frames_kernel<KIND, FRAMES, 4, false>), grid, block, 0, st, d); } } \
        else      { if (p.a.vec) { launch((dense_few_frames_kernel<KIND, FRAMES, 1, true>), grid, block, 0, st, d); }   \
                    else         { launch((dense_few_frames_kernel<KIND, FRAMES, 1, false>), grid, block, 0, st, d); } } \
    } while (0)
    if (p.out.columns == 1) { if (bit) { BBHIP_FEW(kBitColumns, 1); } else { BBHIP_FEW(kColumns, 1); } }
    else                    { if (bit) { BBHIP_FEW(kBitColumns, kFewFrames); } else { BBHIP_FEW(kColumns, kFewFrames); } }
#undef BBHIP_FEW
    BBHIP_LAUNCH_CHECK();
    return 0;
}

int direct_forward(Product const &p, bool bit, float *sums, hipStream_t st, char const *name)
{
    DirectShape const s = p.out.kind == kOutLogits ? logits_shape(p.out.rows, p.out.columns, p.a.depth) : direct_shape(p.out.rows, p.out.columns, p.a.depth);
    DirectProduct d;
    if (direct(d, p, s, sums, p.out.columns, name)) { return 1; }
    dim3 const grid((unsigned)d.workgroups()), block((unsigned)s.waves * 64);
#define BBHIP_DIRECT(WAVES)                                                                             \
    do {                                                                                                \
        if (bit) { launch((dense_direct_kernel<kRows, kBitColumns, WAVES>), grid, block, 0, st, d); }   \
        else     { launch((dense_direct_kernel<kRows, kColumns, WAVES>), grid, block, 0, st, d); }      \
    } while (0)
    if (s.waves == 8)      { BBHIP_DIRECT(8); }
    else if (s.waves == 4) { BBHIP_DIRECT(4); }
    else if (s.waves == 1) { BBHIP_DIRECT(1); }
    else                   { return fail("%s: no kernel of %d wavefronts", name, s.waves); }
#undef BBHIP_DIRECT
    BBHIP_LAUNCH_CHECK();
    return join(sums_to_join(d), PackedProduct{}, st, name);
}

// of a small backward pass: how it is divided, and its places in a workspace
struct DirectBackwardSpace {
    DirectShape w, x;
    float *dz, *w_sums, *x_sums;
    DirectBackwardSpace(Carver &c, int inputs, int outputs, int frames, bool with_dz)
    {
        direct_shapes(outputs, inputs + 1, frames, inputs, frames, outputs, w, x);
        dz = with_dz ? c.take<float>((size_t)outputs * (ceil_div(frames, 64) * 64)) : nullptr;
        w_sums = sums_of(c, w.slabs, outputs, inputs + 1);
        x_sums = sums_of(c, x.slabs, inputs, frames);
    }
};

// dw.a and dx.b are gradients; where these are more than dy itself, or wanted, they are formed first and lie in `dz`
int direct_backward(Product const &dw, Product const &dx, DirectBackwardSpace const &s, float *dz, long long dz_stride, bool bit, hipStream_t st, char const *name)
{
    DirectProduct w, x;
    Product with_line = dw, from_dz = dx;
    if (dz) {
        DzArgs z{dw.a, dz, dz_stride, ceil_div(dw.a.depth, 1024)};
        long long const blocks = (long long)z.per_row * dw.a.rows;
        if (check_tiles(blocks, 256, name)) { return 1; }
        launch(dense_dz_kernel, dim3((unsigned)blocks), dim3(256), 0, st, z);
        BBHIP_LAUNCH_CHECK();
        with_line.a = rows_of(dz, dz_stride, dw.a.rows, dw.a.depth);
        from_dz.b = rows_of(dz, dz_stride, dx.b.rows, dx.b.depth);
    }
    with_line.b.ones = dw.out.line ? dw.b.rows : -1;
    if (direct(w, with_line, s.w, s.w_sums, dw.out.columns + 1, name) || direct(x, from_dz, s.x, s.x_sums, dx.out.columns, name)) { return 1; }
    // in one launch where both take as many wavefronts
    bool const together = s.w.waves == s.x.waves && launch_holds((long long)w.workgroups() + x.workgroups() + 1, s.w.waves * 64);
    DirectProduct none{};
    none.slabs = 1;
    for (int part = together ? 1 : 0; part < 2; ++part) {
        DirectProduct const &a = together || part == 0 ? w : none, &b = together || part == 1 ? x : none;
        int const waves = part == 0 ? s.w.waves : s.x.waves;
        if (a.workgroups() + b.workgroups() == 0) { continue; }
        dim3 const grid((unsigned)(a.workgroups() + b.workgroups())), block((unsigned)waves * 64);
#define BBHIP_DIRECT(WAVES)                                                                             \
        do {                                                                                            \
            if (bit) { launch((dense_direct_backward_kernel<kBitRows, WAVES>), grid, block, 0, st, a, b); } \
            else     { launch((dense_direct_backward_kernel<kRows, WAVES>), grid, block, 0, st, a, b); }    \
        } while (0)
        if (waves == 8)      { BBHIP_DIRECT(8); }
        else if (waves == 4) { BBHIP_DIRECT(4); }
        else if (waves == 1) { BBHIP_DIRECT(1); }
        else                 { return fail("%s: no kernel of %d wavefronts", name, waves); }
#undef BBHIP_DIRECT
        BBHIP_LAUNCH_CHECK();
    }
    return join(sums_to_join(w), sums_to_join(x), st, name);
}

// ---- products by way of packed halves ----
// an operand's halves and scales in a workspace, and the job that writes them
struct Packed {
    uint4 *halves;
    int   *exponent;
    float *lost;
    uint4 *thirds = nullptr;
    int    blocks, steps, pieces, triple;
    Packed() = default;
    Packed(Carver &c, int rows, int depth, bool bits, bool as_triple = false) : blocks(ceil_div(rows, 32)), steps(pack_steps(depth)), pieces(bits ? 1 : 2), triple(as_triple)
    {
        halves = c.take<uint4>((size_t)blocks * steps * pieces * 64);
        exponent = bits ? nullptr : c.take<int>((size_t)blocks * 32);
        lost = c.take<float>((size_t)blocks * 32);
        if (as_triple && !bits) { thirds = c.take<uint4>((size_t)blocks * steps * 64); }
    }
    PackJob job(Operand const &o, int kind) const
    {
        PackJob j{};
        j.src = o; j.kind = kind; j.halves = halves; j.exponent = exponent; j.lost = lost; j.triple = triple; j.thirds = thirds; j.k_steps = steps;
        j.blocks = blocks * (32 / kPackRows);
        return j;
    }
};

struct Jobs {
    PackArgs a{};
    int count = 0, deepest = 0;
    void add(PackJob const &j)
    {
        a.job[count++] = j;
        if (j.exponent && j.src.depth > deepest) { deepest = j.src.depth; }
    }
    int run(hipStream_t st, char const *name) const
    {
        long long total = 0;
        for (int i = 0; i < count; ++i) { total += a.job[i].blocks; }
        bool const wide = pack_is_wide(deepest);
        if (check_tiles(total, wide ? 1024 : 512, name)) { return 1; }
        if (wide) { launch(dense_pack_kernel<1024>, dim3((unsigned)total), dim3(1024), 0, st, a); }
        else      { launch(dense_pack_kernel<512>, dim3((unsigned)total), dim3(512), 0, st, a); }
        BBHIP_LAUNCH_CHECK();
        return 0;
    }
};

int packed_product(PackedProduct &d, Product const &p, PackedShape const &s, Packed const &a, Packed const &b, float *sums, char const *name)
{
    d = PackedProduct{};
    if (!p.wanted) { d.b_pieces = 2; return 0; }
    d.a = a.halves; d.ea = a.exponent; d.lost_a = a.lost; d.a_blocks = a.blocks;
    d.b = b.halves; d.eb = b.exponent; d.lost_b = b.lost; d.thirds_a = a.thirds; d.thirds_b = b.thirds; d.triple = a.triple; d.b_blocks = b.blocks; d.b_pieces = b.pieces;
    d.k_steps = s.k_steps; d.m_tiles = s.m_tiles; d.n_tiles = s.n_tiles; d.slabs = s.slabs; d.slab_stages = s.slab_stages;
    if (check_tiles(s.workgroups(), kTileThreads[s.size], name)) { return 1; }
    d.workgroups = (int)s.workgroups();
    d.sums = sums; d.sums_pitch = sums_pitch(p.out.columns); d.sums_slab = d.sums_pitch * p.out.rows;
    d.out = p.out;
    d.out.line = nullptr;               // (summed where the halves are written)
    d.src_a = p.a; d.src_b = p.b; d.kind_a = p.kind_a; d.kind_b = p.kind_b;
    return 0;
}

int packed_run(PackedProduct const &p, int size, hipStream_t st, char const *name)
{
    dim3 const grid((unsigned)p.workgroups), block((unsigned)kTileThreads[size]);
#define BBHIP_PACKED(USE, ...)                                                                          \
    do {                                                                                                \
        if (p.b_pieces == 1) { launch((dense_packed_kernel<USE, __VA_ARGS__, 1, kTileBuffers[size_]>), grid, block, 0, st, p); } \
        else                 { launch((dense_packed_kernel<USE, __VA_ARGS__, 2, kTileBuffers[size_]>), grid, block, 0, st, p); } \
    } while (0)
#define BBHIP_PACKED_SIZES(USE)                                                                         \
    do {                                                                                                \
        if (size == kTileLarge)       { constexpr int size_ = kTileLarge;  BBHIP_PACKED(USE, 4, 2, 4); } \
        else if (size == kTileMiddle) { constexpr int size_ = kTileMiddle; BBHIP_PACKED(USE, 4, 2, 2); } \
        else                          { constexpr int size_ = kTileSmall;  BBHIP_PACKED(USE, 2, 2, 2); } \
    } while (0)
    if (p.out.kind == kOutLogits) { BBHIP_PACKED_SIZES(kUseLogits); }
    else                          { BBHIP_PACKED_SIZES(kUseForward); }
#undef BBHIP_PACKED_SIZES
#undef BBHIP_PACKED
    BBHIP_LAUNCH_CHECK();
    return join(p, PackedProduct{}, st, name);
}

// p and behind it q, whose operands are not packed bits
int packed_run(PackedProduct const &p, PackedProduct const &q, int size, hipStream_t st, char const *name)
{
    if (check_tiles((long long)p.workgroups + q.workgroups, kTileThreads[size], name)) { return 1; }
    if (p.workgroups + q.workgroups == 0) { return 0; }
    dim3 const grid((unsigned)(p.workgroups + q.workgroups)), block((unsigned)kTileThreads[size]);
    bool const triple = p.triple || q.triple;
#define BBHIP_PACKED(...)                                                                               \
    do {                                                                                                \
        if (triple) {                                                                                   \
            if (p.b_pieces == 1) { launch((dense_packed_pair_kernel<true, __VA_ARGS__, 1, kTileBuffers[size_]>), grid, block, 0, st, p, q); } \
            else                 { launch((dense_packed_pair_kernel<true, __VA_ARGS__, 2, kTileBuffers[size_]>), grid, block, 0, st, p, q); } \
        }                                                                                               \
        else {                                                                                          \
            if (p.b_pieces == 1) { launch((dense_packed_pair_kernel<false, __VA_ARGS__, 1, kTileBuffers[size_]>), grid, block, 0, st, p, q); } \
            else                 { launch((dense_packed_pair_kernel<false, __VA_ARGS__, 2, kTileBuffers[size_]>), grid, block, 0, st, p, q); } \
        }                                                                                               \
    } while (0)
    if (size == kTileLarge)       { constexpr int size_ = kTileLarge;  BBHIP_PACKED(4, 2, 4); }
    else if (size == kTileMiddle) { constexpr int size_ = kTileMiddle; BBHIP_PACKED(4, 2, 2); }
    else                          { constexpr int size_ = kTileSmall;  BBHIP_PACKED(2, 2, 2); }
#undef BBHIP_PACKED
    BBHIP_LAUNCH_CHECK();
    return join(p, q, st, name);
}

// of a layer's forward pass
struct ForwardSpace {
    PackedShape shape;
    Packed W, x;
    float *sums;
    ForwardSpace(Carver &c, int inputs, int outputs, int frames, bool bit)
        : shape(best_shape(outputs, frames, inputs)), W(c, outputs, inputs, false), x(c, frames, inputs, bit), sums(sums_of(c, shape.slabs, outputs, frames)) {}
};

// of its backward pass
struct BackwardSpace {
    PackedShape dw, dx;
    Packed dz_rows, x, W, dz_columns;
    float *dw_sums, *dx_sums;
    BackwardSpace(Carver &c, int inputs, int outputs, int frames, bool bit, bool triple)
    {
        best_shapes(outputs, inputs, frames, inputs, frames, outputs, dw, dx);
        dz_rows = Packed(c, outputs, frames, false, triple);
        x = Packed(c, inputs, frames, bit, triple);
        W = Packed(c, inputs, outputs, false, triple);
        dz_columns = Packed(c, frames, outputs, false, triple);
        dw_sums = sums_of(c, dw.slabs, outputs, inputs);
        dx_sums = sums_of(c, dx.slabs, inputs, frames);
    }
    // the last piece of a loss, of fewer channels: the same places, the same divisions of the k axis or fewer
    void cut(int inputs, int outputs, int frames)
    {
        dw = packed_shape(dw.size, dw.slabs, outputs, inputs, frames);
        dx = packed_shape(dx.size, dx.slabs, inputs, frames, outputs);
        dz_rows.blocks = ceil_div(outputs, 32);
        W.steps = dz_columns.steps = pack_steps(outputs);
    }
    // jobs of both products (x apart: the pieces of a loss share it); the rows' job may leave db and dz on its way
    void add_jobs(Jobs &jobs, Product const &w, Product const &i, bool with_x, float *db, int accumulate, float *dz, long long dz_stride) const
    {
        if (w.wanted || dz) {
            PackJob j = dz_rows.job(w.a, kGradRows);
            j.line = db; j.accumulate = accumulate; j.dz = dz; j.dz_stride = dz_stride;
            jobs.add(j);
        }
        if (w.wanted && with_x) { jobs.add(x.job(w.b, w.kind_b)); }
        if (i.wanted) { jobs.add(W.job(i.a, i.kind_a)); jobs.add(dz_columns.job(i.b, i.kind_b)); }
    }
    int run(Product const &w, Product const &i, hipStream_t st, char const *name) const
    {
        PackedProduct p, q;
        if (packed_product(p, w, dw, dz_rows, x, dw_sums, name) || packed_product(q, i, dx, W, dz_columns, dx_sums, name)) { return 1; }
        return packed_run(p, q, dw.size, st, name);
    }
};

// ---- what an entry checks ----
int check_sizes(int inputs, int outputs, int frames, char const *name)
{
    if (!(inputs > 0 && outputs > 0 && frames > 0)) { return fail("%s: sizes must be positive", name); }
    if (inputs > kDenseNodesMost || outputs > kDenseNodesMost || frames > kDenseFramesMost) {
        return fail("%s: more than 2^24 nodes or 2^25 frames", name);
    }
    return 0;
}

int check_stride(bool bit, int stride, int frames, char const *name)
{
    if ((bit ? (long long)stride * 32 : stride) < frames) { return fail("%s: frame stride shorter than the frames", name); }
    if (stride > kDenseStrideMost) { return fail("%s: a frame stride of %d: at most %d", name, stride, kDenseStrideMost); }
    return 0;
}

Operand frames_as_columns(void const *x, int stride, int inputs, int frames)
{
    Operand o{};
    o.p = x; o.stride = stride; o.rows = frames; o.depth = inputs; o.ones = -1;
    o.vec = starts_on_16_bytes(x) && stride % 4 == 0;
    return o;
}

Operand frames_as_depth(void const *x, bool bit, int stride, int inputs, int frames)
{
    Operand o = rows_of(static_cast<float const *>(x), stride, inputs, frames);
    if (bit) { o.vec = 0; }
    return o;
}

int dense_forward(void const *x, bool bit, void *y, bool bit_out, float const *W, float const *b, float const *residual, int activation, int inputs, int outputs,
                  int frames, int x_stride, int y_stride, int residual_stride, void *workspace, size_t workspace_size, void *stream, char const *name)
{
    clear_hints();
    if (!(x && y && W)) { return fail("%s: null buffer", name); }
    if (check_sizes(inputs, outputs, frames, name)) { return 1; }
    if (check_stride(bit, x_stride, frames, name) || check_stride(bit_out, y_stride, frames, name) || (residual && check_stride(false, residual_stride, frames, name))) { return 1; }
    if (activation < 0 || activation >= kActCount) { return fail("%s: activation=%d is none of 0 .. %d", name, activation, kActCount - 1); }
    Product p;
    p.a = rows_of(W, inputs, outputs, inputs);
    p.b = frames_as_columns(x, x_stride, inputs, frames);
    p.kind_a = kRows; p.kind_b = bit ? kBitColumns : kColumns;
    p.out = DenseOutput{};
    p.out.kind = bit_out ? kOutBits : kOutForward;
    p.out.rows = outputs; p.out.columns = frames; p.out.out = y; p.out.stride = y_stride;
    p.out.bias = b; p.out.residual = residual; p.out.residual_stride = residual_stride; p.out.activation = activation;
    hipStream_t const st = static_cast<hipStream_t>(stream);
    Carver c{static_cast<char *>(workspace)};
    if (few_frames(p)) {
        ScopedTimer tm(kTimeOther, st);
        return few_frames_forward(p, bit, st, name);
    }
    if (!forward_packed(inputs, outputs, frames)) {
        float *const sums = sums_of(c, direct_shape(outputs, frames, inputs).slabs, outputs, frames);
        if (check_workspace(workspace, workspace_size, c.at, name)) { return 1; }
        ScopedTimer tm(kTimeOther, st);
        return direct_forward(p, bit, sums, st, name);
    }
    ForwardSpace const s(c, inputs, outputs, frames, bit);
    if (check_workspace(workspace, workspace_size, c.at, name)) { return 1; }
    ScopedTimer tm(kTimeOther, st);
    Jobs jobs;
    jobs.add(s.W.job(p.a, p.kind_a));
    jobs.add(s.x.job(p.b, p.kind_b));
    PackedProduct d;
    return jobs.run(st, name) || packed_product(d, p, s.shape, s.W, s.x, s.sums, name) || packed_run(d, s.shape.size, st, name);
}

int dense_backward(void const *x, bool bit, float const *dy, float const *y, float const *W, float *dx, float *dW, float *db, float *dr, int activation,
                   int accumulate, int inputs, int outputs, int frames, int x_stride, int dx_stride, int stride, void *workspace, size_t workspace_size, void *stream,
                   char const *name)
{
    clear_hints();
    if (!dy || (!dx && !dW && !dr) || (dx && !W) || (dW && !x)) { return fail("%s: null buffer", name); }
    if (db && !dW) { return fail("%s: db is formed with dW", name); }
    if (activation < 0 || activation >= kActCount) { return fail("%s: activation=%d is none of 0 .. %d", name, activation, kActCount - 1); }
    if (activation != kActNone && !y) { return fail("%s: the activation's gradient needs the forward pass's output", name); }
    if (check_sizes(inputs, outputs, frames, name)) { return 1; }
    if ((dW && check_stride(bit, x_stride, frames, name)) || check_stride(false, stride, frames, name) || (dx && check_stride(false, dx_stride, frames, name))) { return 1; }
    Operand g{};
    g.p = dy; g.y = y; g.stride = stride; g.mode = activation; g.ones = -1;
    g.vec = starts_on_16_bytes(dy) && starts_on_16_bytes(y) && stride % 4 == 0;
    Product w, i;
    w.wanted = dW != nullptr;
    w.a = g; w.a.rows = outputs; w.a.depth = frames;
    w.b = frames_as_depth(x, bit, x_stride, inputs, frames);
    w.kind_a = kGradRows; w.kind_b = bit ? kBitRows : kRows;
    w.out = DenseOutput{};
    w.out.kind = kOutStore; w.out.rows = outputs; w.out.columns = inputs; w.out.out = dW; w.out.stride = inputs; w.out.accumulate = accumulate; w.out.line = db;
    i.wanted = dx != nullptr;
    i.a = rows_of(W, inputs, inputs, outputs);
    i.b = g; i.b.rows = frames; i.b.depth = outputs;
    i.kind_a = kColumns; i.kind_b = kGradColumns;
    i.out = DenseOutput{};
    i.out.kind = kOutStore; i.out.rows = inputs; i.out.columns = frames; i.out.out = dx; i.out.stride = dx_stride;
    hipStream_t const st = static_cast<hipStream_t>(stream);
    if (backward_packed(inputs, outputs, frames)) {
        Carver c{static_cast<char *>(workspace)};
        BackwardSpace const s(c, inputs, outputs, frames, bit, false);
        if (check_workspace(workspace, workspace_size, c.at, name)) { return 1; }
        ScopedTimer tm(kTimeOther, st);
        Jobs jobs;
        s.add_jobs(jobs, w, i, true, db, accumulate, dr, stride);
        return jobs.run(st, name) || s.run(w, i, st, name);
    }
    Carver c{static_cast<char *>(workspace)};
    bool const own = !dr && activation != kActNone;
    DirectBackwardSpace const d(c, inputs, outputs, frames, own);
    if (check_workspace(workspace, workspace_size, c.at, name)) { return 1; }
    ScopedTimer tm(kTimeOther, st);
    return direct_backward(w, i, d, own ? d.dz : dr, own ? ceil_div(frames, 64) * 64 : stride, bit, st, name);
}

// ---- the loss on top of a dense layer ----
struct LossSpace {
    LossPlan plan;
    float2 *partial;
    float *label_logit, *top = nullptr, *share = nullptr, *coef = nullptr, *logits = nullptr, *logit_sums = nullptr;
    char *direct_space = nullptr;       // not packed: of a piece's gradients
    Packed W, x;                        // packed: of a piece's logits
    alignas(BackwardSpace) char backward_space[sizeof(BackwardSpace)];
    size_t total;
    BackwardSpace const &backward(void) const { return *reinterpret_cast<BackwardSpace const *>(backward_space); }
    LossSpace(char *base, int inputs, int channels, int frames, bool bit, bool gradients) : plan(loss_plan(inputs, channels, frames))
    {
        Carver c{base};
        partial     = c.take<float2>((size_t)plan.tiles * frames);
        label_logit = c.take<float>((size_t)frames);
        if (gradients) {
            top    = c.take<float>((size_t)frames);
            share  = c.take<float>((size_t)frames);
            coef   = c.take<float>((size_t)frames);
            logits = c.take<float>((size_t)plan.piece * plan.stride);
        }
        if (plan.packed) {
            W = Packed(c, plan.piece, inputs, false);
            x = Packed(c, frames, inputs, bit);
            logit_sums = sums_of(c, plan.logits.slabs, plan.piece, frames);
            if (gradients) { new (backward_space) BackwardSpace(c, inputs, plan.piece, frames, bit, true); }
        }
        else {
            // (the last piece, of fewer channels, may be divided otherwise)
            int const last = channels - (channels - 1) / plan.piece * plan.piece;
            size_t most = 0, most_sums = 0;
            for (int count : {plan.piece, last}) {
                Carver d{nullptr}, e{nullptr};
                DirectBackwardSpace const space(d, inputs, count, frames, false);
                sums_of(e, logits_shape(count, frames, inputs).slabs, count, frames);
                most = d.at > most ? d.at : most;
                most_sums = e.at > most_sums ? e.at : most_sums;
            }
            logit_sums = c.take<float>(most_sums / sizeof(float));
            if (gradients) { direct_space = c.take<char>(most); }
        }
        total = c.at;
    }
};

int dense_loss(void const *x, bool bit, float const *W, float const *b, int const *label, float const *weight, float *dx, float *dW, float *db, float *loss,
               float weight_sum, int accumulate, int inputs, int channels, int frames, int x_stride, int dx_stride, void *workspace, size_t workspace_size, void *stream,
               char const *name)
{
    clear_hints();
    if (!(x && W && label && loss)) { return fail("%s: null buffer", name); }
    if (db && !dW) { return fail("%s: db is formed with dW", name); }
    if (check_sizes(inputs, channels, frames, name)) { return 1; }
    if (check_stride(bit, x_stride, frames, name) || (dx && check_stride(false, dx_stride, frames, name))) { return 1; }
    bool const gradients = dx || dW;
    LossSpace const s(static_cast<char *>(workspace), inputs, channels, frames, bit, gradients);
    if (check_workspace(workspace, workspace_size, s.total, name)) { return 1; }
    float *const logits = s.logits, *const coef = s.coef;
    hipStream_t const st = static_cast<hipStream_t>(stream);
    ScopedTimer tm(kTimeOther, st);
    int const pieces = ceil_div(channels, s.plan.piece);
    bool x_packed = false, x_rows_packed = false;
    auto const logit_piece = [&](int piece, bool store) {
        int const first = piece * s.plan.piece, count = channels - first < s.plan.piece ? channels - first : s.plan.piece;
        Product p;
        p.a = rows_of(W + (size_t)first * inputs, inputs, count, inputs);
        p.b = frames_as_columns(x, x_stride, inputs, frames);
        p.kind_a = kRows; p.kind_b = bit ? kBitColumns : kColumns;
        p.out = DenseOutput{};
        p.out.kind = kOutLogits; p.out.rows = count; p.out.columns = frames; p.out.out = store ? logits : nullptr; p.out.stride = s.plan.stride;
        p.out.bias = b ? b + first : nullptr;
        p.out.partial = s.partial + (size_t)(first / s.plan.tile) * frames;
        p.out.label = label; p.out.label_logit = s.label_logit; p.out.first_channel = first;
        p.out.channels = channels; p.out.weight = weight;
        if (!s.plan.packed) { return direct_forward(p, bit, s.logit_sums, st, name); }
        Jobs jobs;
        jobs.add(s.W.job(p.a, p.kind_a));
        if (!x_packed) { jobs.add(s.x.job(p.b, p.kind_b)); x_packed = true; }
        PackedShape const shape = packed_shape(s.plan.logits.size, s.plan.logits.slabs, count, frames, inputs);
        PackedProduct d;
        Packed W_piece = s.W;
        W_piece.blocks = ceil_div(count, 32);
        return (int)(jobs.run(st, name) || packed_product(d, p, shape, W_piece, s.x, s.logit_sums, name) || packed_run(d, shape.size, st, name));
    };
    // the pieces' largest logits and sums; the last piece's logits stay for its gradient
    for (int piece = 0; piece < pieces; ++piece) { if (logit_piece(piece, gradients && piece == pieces - 1)) { return 1; } }
    LossFinishArgs f{};
    f.partial = s.partial; f.label_logit = s.label_logit;
    f.label = label; f.weight = weight; f.loss = loss;
    f.top = s.top; f.share = s.share; f.coef = coef;
    f.reciprocal_weight_sum = (float)(1.0 / (double)weight_sum);
    f.tiles = s.plan.tiles; f.frames = frames; f.channels = channels;
    launch(dense_loss_finish_kernel, dim3((unsigned)ceil_div(frames, kFinishFrames)), dim3(kFinishFrames * kFinishGroups), 0, st, f);
    BBHIP_LAUNCH_CHECK();
    if (!gradients) { return 0; }
    for (int piece = pieces - 1; piece >= 0; --piece) {
        int const first = piece * s.plan.piece, count = channels - first < s.plan.piece ? channels - first : s.plan.piece;
        if (piece != pieces - 1 && logit_piece(piece, true)) { return 1; }
        Operand g{};
        g.p = logits; g.stride = s.plan.stride; g.mode = kGradSoftmax; g.ones = -1; g.vec = 1; g.first = first;
        g.top = f.top; g.share = f.share; g.coef = f.coef; g.label = label;
        Product w, i;
        w.wanted = dW != nullptr;
        w.a = g; w.a.rows = count; w.a.depth = frames;
        w.b = frames_as_depth(x, bit, x_stride, inputs, frames);
        if (!bit) { w.b.coef = coef; }
        w.kind_a = kGradRows; w.kind_b = bit ? kBitRows : kRows;
        w.out = DenseOutput{};
        w.out.kind = kOutStore; w.out.rows = count; w.out.columns = inputs; w.out.out = dW + (size_t)first * inputs; w.out.stride = inputs;
        w.out.accumulate = accumulate; w.out.line = db ? db + first : nullptr;
        i.wanted = dx != nullptr;
        i.a = rows_of(W + (size_t)first * inputs, inputs, inputs, count);
        i.b = g; i.b.rows = frames; i.b.depth = count;
        i.kind_a = kColumns; i.kind_b = kGradColumns;
        i.out = DenseOutput{};
        i.out.kind = kOutStore; i.out.rows = inputs; i.out.columns = frames; i.out.out = dx; i.out.stride = dx_stride; i.out.accumulate = piece != pieces - 1;
        if (!s.plan.packed) {
            // (in the place of the logits)
            Carver c{s.direct_space};
            DirectBackwardSpace const d(c, inputs, count, frames, false);
            if (direct_backward(w, i, d, logits, s.plan.stride, bit, st, name)) { return 1; }
            continue;
        }
        Jobs jobs;
        BackwardSpace b = s.backward();
        if (count != s.plan.piece) { b.cut(inputs, count, frames); }
        b.add_jobs(jobs, w, i, !x_rows_packed, w.out.line, accumulate, nullptr, 0);
        x_rows_packed = true;
        if (jobs.run(st, name) || b.run(w, i, st, name)) { return 1; }
    }
    return 0;
}

int check_list(int size, void const *a, void const *b, float max_norm, float const *norm, char const *name)
{
    if (size < 0) { return fail("%s: size=%d", name, size); }
    if (!norm || (size > 0 && !(a && b))) { return fail("%s: null buffer", name); }
    if (!(max_norm >= 0.0f)) { return fail("%s: max_norm must not be negative", name); }
    return 0;
}

int squares(int size, int const *sizes, float *const *grads, void *workspace, size_t workspace_size, hipStream_t st, char const *name)
{
    if (check_workspace(workspace, workspace_size, bbhip_GradientNorm_WorkspaceBytes(), name)) { return 1; }
    launch(gradient_squares_kernel, dim3(kNormGrid), dim3(kNormBlock), 0, st, size, sizes, reinterpret_cast<float const *const *>(grads), static_cast<double *>(workspace));
    BBHIP_LAUNCH_CHECK();
    return 0;
}

}  // namespace

size_t bbhip_DenseAffine_Forward_WorkspaceBytes(int input_node_size, int output_node_size, int frame_size, int bit_input)
{
    if (check_sizes(input_node_size, output_node_size, frame_size, __func__)) { return 0; }
    Carver forward{nullptr};
    if (frame_size <= kFewFrames) { return 0; }
    if (forward_packed(input_node_size, output_node_size, frame_size)) { ForwardSpace const f(forward, input_node_size, output_node_size, frame_size, bit_input != 0); }
    else { sums_of(forward, direct_shape(output_node_size, frame_size, input_node_size).slabs, output_node_size, frame_size); }
    return forward.at;
}

size_t bbhip_DenseAffine_WorkspaceBytes(int input_node_size, int output_node_size, int frame_size)
{
    if (check_sizes(input_node_size, output_node_size, frame_size, __func__)) { return 0; }
    size_t const forward = bbhip_DenseAffine_Forward_WorkspaceBytes(input_node_size, output_node_size, frame_size, 0);
    Carver backward{nullptr};
    if (backward_packed(input_node_size, output_node_size, frame_size)) { BackwardSpace const b(backward, input_node_size, output_node_size, frame_size, false, false); }
    else { DirectBackwardSpace const d(backward, input_node_size, output_node_size, frame_size, true); }
    return forward > backward.at ? forward : backward.at;
}

int bbhip_fp32_DenseAffine_Forward(float const *dev_x_buf, float *dev_y_buf, float const *dev_W, float const *dev_b, float const *dev_residual_buf, int activation,
                                   int input_node_size, int output_node_size, int frame_size, int x_frame_stride, int y_frame_stride, int residual_frame_stride,
                                   void *dev_workspace, size_t workspace_size, void *stream)
{
    return dense_forward(dev_x_buf, false, dev_y_buf, false, dev_W, dev_b, dev_residual_buf, activation, input_node_size, output_node_size, frame_size, x_frame_stride,
                         y_frame_stride, residual_frame_stride, dev_workspace, workspace_size, stream, __func__);
}

int bbhip_bit_fp32_DenseAffine_Forward(int const *dev_x_buf, float *dev_y_buf, float const *dev_W, float const *dev_b, float const *dev_residual_buf, int activation,
                                       int input_node_size, int output_node_size, int frame_size, int x_frame_stride, int y_frame_stride, int residual_frame_stride,
                                       void *dev_workspace, size_t workspace_size, void *stream)
{
    return dense_forward(dev_x_buf, true, dev_y_buf, false, dev_W, dev_b, dev_residual_buf, activation, input_node_size, output_node_size, frame_size, x_frame_stride,
                         y_frame_stride, residual_frame_stride, dev_workspace, workspace_size, stream, __func__);
}

int bbhip_fp32_bit_DenseAffine_Forward(float const *dev_x_buf, int *dev_y_buf, float const *dev_W, float const *dev_b, float const *dev_residual_buf, int input_node_size,
                                       int output_node_size, int frame_size, int x_frame_stride, int y_frame_stride, int residual_frame_stride, void *dev_workspace,
                                       size_t workspace_size, void *stream)
{
    return dense_forward(dev_x_buf, false, dev_y_buf, true, dev_W, dev_b, dev_residual_buf, kActNone, input_node_size, output_node_size, frame_size, x_frame_stride,
                         y_frame_stride, residual_frame_stride, dev_workspace, workspace_size, stream, __func__);
}

int bbhip_bit_bit_DenseAffine_Forward(int const *dev_x_buf, int *dev_y_buf, float const *dev_W, float const *dev_b, float const *dev_residual_buf, int input_node_size,
                                      int output_node_size, int frame_size, int x_frame_stride, int y_frame_stride, int residual_frame_stride, void *dev_workspace,
                                      size_t workspace_size, void *stream)
{
    return dense_forward(dev_x_buf, true, dev_y_buf, true, dev_W, dev_b, dev_residual_buf, kActNone, input_node_size, output_node_size, frame_size, x_frame_stride,
                         y_frame_stride, residual_frame_stride, dev_workspace, workspace_size, stream, __func__);
}

int bbhip_fp32_DenseAffine_Backward(float const *dev_x_buf, float const *dev_dy_buf, float const *dev_y_buf, float const *dev_W, float *dev_dx_buf, float *dev_dW,
                                    float *dev_db, float *dev_dr_buf, int activation, int accumulate, int input_node_size, int output_node_size, int frame_size,
                                    int x_frame_stride, int dx_frame_stride, int frame_stride, void *dev_workspace, size_t workspace_size, void *stream)
{
    return dense_backward(dev_x_buf, false, dev_dy_buf, dev_y_buf, dev_W, dev_dx_buf, dev_dW, dev_db, dev_dr_buf, activation, accumulate, input_node_size, output_node_size,
                          frame_size, x_frame_stride, dx_frame_stride, frame_stride, dev_workspace, workspace_size, stream, __func__);
}

int bbhip_bit_fp32_DenseAffine_Backward(int const *dev_x_buf, float const *dev_dy_buf, float const *dev_y_buf, float const *dev_W, float *dev_dx_buf, float *dev_dW,
                                        float *dev_db, float *dev_dr_buf, int activation, int accumulate, int input_node_size, int output_node_size, int frame_size,
                                        int x_frame_stride, int dx_frame_stride, int frame_stride, void *dev_workspace, size_t workspace_size, void *stream)
{
    return dense_backward(dev_x_buf, true, dev_dy_buf, dev_y_buf, dev_W, dev_dx_buf, dev_dW, dev_db, dev_dr_buf, activation, accumulate, input_node_size, output_node_size,
                          frame_size, x_frame_stride, dx_frame_stride, frame_stride, dev_workspace, workspace_size, stream, __func__);
}

size_t bbhip_LossDenseSoftmaxCrossEntropy_WorkspaceBytes(int input_node_size, int ch_size, int frame_size, int gradients)
{
    if (check_sizes(input_node_size, ch_size, frame_size, __func__)) { return 0; }
    size_t const bits = LossSpace(nullptr, input_node_size, ch_size, frame_size, true, gradients != 0).total;
    size_t const values = LossSpace(nullptr, input_node_size, ch_size, frame_size, false, gradients != 0).total;
    return bits > values ? bits : values;
}

int bbhip_fp32_LossDenseSoftmaxCrossEntropy(float const *dev_x_buf, float const *dev_W, float const *dev_b, int const *dev_label_buf, float const *dev_weight_buf,
                                            float *dev_dx_buf, float *dev_dW, float *dev_db, float *dev_loss_buf, float weight_sum, int accumulate, int input_node_size,
                                            int ch_size, int frame_size, int x_frame_stride, int dx_frame_stride, void *dev_workspace, size_t workspace_size, void *stream)
{
    return dense_loss(dev_x_buf, false, dev_W, dev_b, dev_label_buf, dev_weight_buf, dev_dx_buf, dev_dW, dev_db, dev_loss_buf, weight_sum, accumulate, input_node_size,
                      ch_size, frame_size, x_frame_stride, dx_frame_stride, dev_workspace, workspace_size, stream, __func__);
}

int bbhip_bit_fp32_LossDenseSoftmaxCrossEntropy(int const *dev_x_buf, float const *dev_W, float const *dev_b, int const *dev_label_buf, float const *dev_weight_buf,
                                                float *dev_dx_buf, float *dev_dW, float *dev_db, float *dev_loss_buf, float weight_sum, int accumulate,
                                                int input_node_size, int ch_size, int frame_size, int x_frame_stride, int dx_frame_stride, void *dev_workspace,
                                                size_t workspace_size, void *stream)
{
    return dense_loss(dev_x_buf, true, dev_W, dev_b, dev_label_buf, dev_weight_buf, dev_dx_buf, dev_dW, dev_db, dev_loss_buf, weight_sum, accumulate, input_node_size,
                      ch_size, frame_size, x_frame_stride, dx_frame_stride, dev_workspace, workspace_size, stream, __func__);
}

// ---- the norm of a list of gradients ----
size_t bbhip_GradientNorm_WorkspaceBytes(void) { return align256(kNormGrid * sizeof(double)); }

int bbhip_fp32_GradientNorm(int size, int const *dev_size_table, float *const *dev_grads_buf_table, float max_norm, float *dev_norm, void *dev_workspace,
                            size_t workspace_size, void *stream)
{
    clear_hints();
    if (check_list(size, dev_size_table, dev_grads_buf_table, max_norm, dev_norm, __func__)) { return 1; }
    hipStream_t const st = static_cast<hipStream_t>(stream);
    ScopedTimer tm(kTimeOther, st);
    if (squares(size, dev_size_table, dev_grads_buf_table, dev_workspace, workspace_size, st, __func__)) { return 1; }
    launch(gradient_norm_kernel, dim3(1), dim3(kNormBlock), 0, st, static_cast<double const *>(dev_workspace), max_norm, dev_norm);
    BBHIP_LAUNCH_CHECK();
    return 0;
}

int bbhip_fp32_GradientClip(int size, int const *dev_size_table, float *const *dev_grads_buf_table, float max_norm, float *dev_norm, void *dev_workspace,
                            size_t workspace_size, void *stream)
{
    clear_hints();
    if (check_list(size, dev_size_table, dev_grads_buf_table, max_norm, dev_norm, __func__)) { return 1; }
    hipStream_t const st = static_cast<hipStream_t>(stream);
    ScopedTimer tm(kTimeOther, st);
    if (squares(size, dev_size_table, dev_grads_buf_table, dev_workspace, workspace_size, st, __func__)) { return 1; }
    launch(gradient_clip_kernel, dim3(kNormGrid), dim3(kNormBlock), 0, st, size, dev_size_table, dev_grads_buf_table, static_cast<double const *>(dev_workspace), max_norm, dev_norm);
    BBHIP_LAUNCH_CHECK();
    return 0;
}

int bbhip_fp32_OptimizerAdam_Clipped(int size, int const *dev_size_table, float *const *dev_params_buf_table, float *const *dev_grads_buf_table,
                                     float *const *dev_m_buf_table, float *const *dev_v_buf_table, float lr_t, double beta1, double beta2, float max_norm, float *dev_norm,
                                     int zero_grads, void *dev_workspace, size_t workspace_size, void *stream)
{
    clear_hints();
    if (check_list(size, dev_size_table, dev_grads_buf_table, max_norm, dev_norm, __func__)) { return 1; }
    if (size > 0 && !(dev_params_buf_table && dev_m_buf_table && dev_v_buf_table)) { return fail("%s: null buffer", __func__); }
    hipStream_t const st = static_cast<hipStream_t>(stream);
    ScopedTimer tm(kTimeOther, st);
    if (squares(size, dev_size_table, dev_grads_buf_table, dev_workspace, workspace_size, st, __func__)) { return 1; }
    auto const step = zero_grads ? adam_clipped_kernel<true> : adam_clipped_kernel<false>;
    launch(step, dim3(kNormGrid), dim3(kNormBlock), 0, st, size, dev_size_table, dev_params_buf_table, dev_grads_buf_table, dev_m_buf_table, dev_v_buf_table, lr_t,
           (float)(1.0 - beta1), (float)(1.0 - beta2), static_cast<double const *>(dev_workspace), max_norm, dev_norm);
    BBHIP_LAUNCH_CHECK();
    return 0;
}
