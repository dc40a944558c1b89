// Host side of the entries of dense layers, of the loss on top of one and of the clipping of gradients (include/bbhip.h): argument checks, how a call is divided,
// launches.  The kernels are in dense_*.hpp and gradient_norm_kernels.hpp.

#include <hip/hip_runtime.h>

#include "../../include/bbhip.h"
#include "host_calls.hpp"
#include "launch_rules.hpp"
#include "dense_rules.hpp"
#include "dense_direct_kernels.hpp"
#include "dense_loss_kernels.hpp"
#include "gradient_norm_kernels.hpp"

using namespace bbhip;

namespace {

// a product as the entries describe it, before it is known how it is computed
struct Product {
    Operand     a, b;
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

// ---- products straight from the operands ----
int direct(DirectProduct &d, Product const &p, int columns, char const *name, int waves)
{
    d.a = p.a; d.b = p.b; d.out = p.out;
    d.n_tiles = ceil_div(columns, kDirectTile);
    long long const tiles = p.wanted ? (long long)ceil_div(p.out.rows, kDirectTile) * d.n_tiles : 0;
    if (check_tiles(tiles, waves * 64, name)) { return 1; }
    d.tiles = (int)tiles;
    return 0;
}

int direct_forward(Product const &p, bool bit, hipStream_t st, char const *name)
{
    int const waves = direct_waves(p.a.depth);
    DirectProduct d;
    if (direct(d, p, p.out.columns, name, waves)) { return 1; }
    dim3 const grid((unsigned)d.tiles), block((unsigned)waves * 64);
    if (waves == 16) {
        if (bit) { launch((dense_direct_kernel<kRows, kBitColumns, 16>), grid, block, 0, st, d); }
        else     { launch((dense_direct_kernel<kRows, kColumns, 16>), grid, block, 0, st, d); }
    }
    else {
        if (bit) { launch((dense_direct_kernel<kRows, kBitColumns, 4>), grid, block, 0, st, d); }
        else     { launch((dense_direct_kernel<kRows, kColumns, 4>), grid, block, 0, st, d); }
    }
    BBHIP_LAUNCH_CHECK();
    return 0;
}

int direct_backward(Product const &dw, Product const &dx, bool bit, hipStream_t st, char const *name)
{
    int const waves = direct_waves(dw.wanted && dw.a.depth > dx.a.depth ? dw.a.depth : dx.a.depth);
    DirectProduct w, x;
    Product with_line = dw;
    if (dw.out.line) { with_line.b.ones = dw.b.rows; }
    if (direct(w, with_line, dw.out.columns + (dw.out.line ? 1 : 0), name, waves) || direct(x, dx, dx.out.columns, name, waves) ||
        check_tiles((long long)w.tiles + x.tiles, waves * 64, name)) { return 1; }
    if (w.tiles + x.tiles == 0) { return 0; }
    dim3 const grid((unsigned)(w.tiles + x.tiles)), block((unsigned)waves * 64);
    if (waves == 16) {
        if (bit) { launch((dense_direct_backward_kernel<kBitRows, 16>), grid, block, 0, st, w, x); }
        else     { launch((dense_direct_backward_kernel<kRows, 16>), grid, block, 0, st, w, x); }
    }
    else {
        if (bit) { launch((dense_direct_backward_kernel<kBitRows, 4>), grid, block, 0, st, w, x); }
        else     { launch((dense_direct_backward_kernel<kRows, 4>), grid, block, 0, st, w, x); }
    }
    BBHIP_LAUNCH_CHECK();
    return 0;
}

// ---- what an entry checks ----
int check_sizes(int inputs, int outputs, int frames, char const *name)
{
    if (!(inputs > 0 && outputs > 0 && frames > 0)) { return fail("%s: sizes must be positive", name); }
    if (inputs > kDenseNodesMost || outputs > kDenseNodesMost || frames > kDenseFramesMost) {
        return fail("%s: more than 2^%d nodes or 2^%d frames", name, 24, 26);
    }
    return 0;
}

int check_stride(bool bit, int stride, int frames, char const *name)
{
    if ((bit ? (long long)stride * 32 : stride) < frames) { return fail("%s: frame stride shorter than the frames", name); }
    return 0;
}

Operand frames_as_columns(void const *x, int stride, int inputs, int frames)
{
    Operand o{};
    o.p = x; o.stride = stride; o.rows = frames; o.depth = inputs; o.ones = -1;
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
    p.out = DenseOutput{};
    p.out.kind = bit_out ? kOutBits : kOutForward;
    p.out.rows = outputs; p.out.columns = frames; p.out.out = y; p.out.stride = y_stride;
    p.out.bias = b; p.out.residual = residual; p.out.residual_stride = residual_stride; p.out.activation = activation;
    hipStream_t const st = static_cast<hipStream_t>(stream);
    if (check_workspace(workspace, workspace_size, 0, name)) { return 1; }
    ScopedTimer tm(kTimeOther, st);
    return direct_forward(p, bit, st, name);
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
    w.out = DenseOutput{};
    w.out.kind = kOutStore; w.out.rows = outputs; w.out.columns = inputs; w.out.out = dW; w.out.stride = inputs; w.out.accumulate = accumulate; w.out.line = db;
    i.wanted = dx != nullptr;
    i.a = rows_of(W, inputs, inputs, outputs);
    i.b = g; i.b.rows = frames; i.b.depth = outputs;
    i.out = DenseOutput{};
    i.out.kind = kOutStore; i.out.rows = inputs; i.out.columns = frames; i.out.out = dx; i.out.stride = dx_stride;
    hipStream_t const st = static_cast<hipStream_t>(stream);
    if (check_workspace(workspace, workspace_size, 0, name)) { return 1; }
    ScopedTimer tm(kTimeOther, st);
    if (direct_backward(w, i, bit, st, name)) { return 1; }
    if (dr) {
        Operand o = g;
        o.rows = outputs; o.depth = frames;
        launch(dense_dz_kernel, dim3((unsigned)ceil_div(frames, 256), (unsigned)(outputs < 65535 ? outputs : 65535), (unsigned)ceil_div(outputs, 65535)), dim3(256), 0, st, o, dr, (long long)stride);
        BBHIP_LAUNCH_CHECK();
    }
    return 0;
}

// ---- the loss on top of a dense layer ----
struct LossSpace {
    LossPlan plan;
    size_t partial, label_logit, top, share, coef, logits, total;          // offsets
    LossSpace(int inputs, int channels, int frames, bool gradients) : plan(loss_plan(inputs, channels, frames))
    {
        size_t at = 0;
        auto const take = [&](size_t bytes) { size_t const was = at; at += align256(bytes); return was; };
        partial     = take((size_t)plan.tiles * frames * sizeof(float2));
        label_logit = take((size_t)frames * 4);
        top         = take(gradients ? (size_t)frames * 4 : 0);
        share       = take(gradients ? (size_t)frames * 4 : 0);
        coef        = take(gradients ? (size_t)frames * 4 : 0);
        logits      = take(gradients ? (size_t)plan.piece * plan.stride * 4 : 0);
        total       = at;
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
    LossSpace const s(inputs, channels, frames, gradients);
    if (check_workspace(workspace, workspace_size, s.total, name)) { return 1; }
    char *const base = static_cast<char *>(workspace);
    float *const logits = reinterpret_cast<float *>(base + s.logits), *const coef = reinterpret_cast<float *>(base + s.coef);
    hipStream_t const st = static_cast<hipStream_t>(stream);
    ScopedTimer tm(kTimeOther, st);
    int const pieces = ceil_div(channels, s.plan.piece);
    auto const logit_piece = [&](int piece, bool store) {
        int const first = piece * s.plan.piece, count = channels - first < s.plan.piece ? channels - first : s.plan.piece;
        Product p;
        p.a = rows_of(W + (size_t)first * inputs, inputs, count, inputs);
        p.b = frames_as_columns(x, x_stride, inputs, frames);
        p.out = DenseOutput{};
        p.out.kind = kOutLogits; p.out.rows = count; p.out.columns = frames; p.out.out = store ? logits : nullptr; p.out.stride = s.plan.stride;
        p.out.bias = b ? b + first : nullptr;
        p.out.partial = reinterpret_cast<float2 *>(base + s.partial) + (size_t)(first / kLossTile) * frames;
        p.out.label = label; p.out.label_logit = reinterpret_cast<float *>(base + s.label_logit); p.out.first_channel = first;
        return direct_forward(p, bit, st, name);
    };
    // the pieces' largest logits and sums; the last piece's logits stay for its gradient
    for (int piece = 0; piece < pieces; ++piece) { if (logit_piece(piece, gradients && piece == pieces - 1)) { return 1; } }
    LossFinishArgs f{};
    f.partial = reinterpret_cast<float2 const *>(base + s.partial); f.label_logit = reinterpret_cast<float const *>(base + s.label_logit);
    f.label = label; f.weight = weight; f.loss = loss;
    f.top = gradients ? reinterpret_cast<float *>(base + s.top) : nullptr;
    f.share = gradients ? reinterpret_cast<float *>(base + s.share) : nullptr;
    f.coef = gradients ? coef : nullptr;
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
        w.out = DenseOutput{};
        w.out.kind = kOutStore; w.out.rows = count; w.out.columns = inputs; w.out.out = dW + (size_t)first * inputs; w.out.stride = inputs;
        w.out.accumulate = accumulate; w.out.line = db ? db + first : nullptr;
        i.wanted = dx != nullptr;
        i.a = rows_of(W + (size_t)first * inputs, inputs, inputs, count);
        i.b = g; i.b.rows = frames; i.b.depth = count;
        i.out = DenseOutput{};
        i.out.kind = kOutStore; i.out.rows = inputs; i.out.columns = frames; i.out.out = dx; i.out.stride = dx_stride; i.out.accumulate = piece != pieces - 1;
        if (direct_backward(w, i, bit, st, name)) { return 1; }
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

size_t bbhip_DenseAffine_WorkspaceBytes(int input_node_size, int output_node_size, int frame_size)
{
    (void)input_node_size; (void)output_node_size; (void)frame_size;
    return 0;
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
    return LossSpace(input_node_size, ch_size, frame_size, gradients != 0).total;
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
