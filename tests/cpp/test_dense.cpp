// The host classes of dense layers: bb::DenseAffine, LossDenseSoftmaxCrossEntropy, GradientNorm, and OptimizerAdam with clipped gradients.
//   test_dense          on the device: values against 64-bit loops, accumulation, stacked passes, a convolution of a dense layer, a training step of all of them
//   test_dense --rules  on the CPU: how the products are divided, over many sizes; objects that need no device
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <random>
#include <sstream>
#include <vector>

#include "../../binarybrain_amd/csrc/dense_rules.hpp"
#include "bb/Convolution2d.h"
#include "bb/DenseAffine.h"
#include "bb/GradientNorm.h"
#include "bb/LossDenseSoftmaxCrossEntropy.h"
#include "bb/ObjectLoader.h"
#include "bb/OptimizerAdam.h"
#include "bb/Sequential.h"

static int g_failures = 0;
static void check(bool ok, char const *what, double a = 0, double b = 0)
{
    if (!ok) { ++g_failures; std::printf("FAILED %s (%g, %g)\n", what, a, b); }
}

// every tile and every step of the k axis belongs to one workgroup, none is empty
static void test_rules(void)
{
    std::mt19937 mt(1);
    auto pick = [&](int most) { return 1 + (int)(mt() % (unsigned)(mt() % 3 == 0 ? 100 : most)); };
    for (int i = 0; i < 100000; ++i) {
        int const m = pick(i % 5 ? 9000 : bbhip::kDenseNodesMost), n = pick(i % 7 ? 9000 : bbhip::kDenseFramesMost), k = pick(i % 2 ? 9000 : 2000000), m1 = pick(9000), k1 = pick(9000);
        bbhip::DirectShape const d = bbhip::direct_shape(m, n, k);
        int const chunks = (k + 31) / 32;
        check(d.slabs >= 1 && (long long)d.slabs * d.slab_chunks >= chunks && (long long)(d.slabs - 1) * d.slab_chunks < chunks, "direct slabs", m, k);
        check(d.slabs == 1 || d.tiles * d.slabs <= 1024, "direct workgroups", m, n);
        check((d.waves == 1 || d.waves == 4 || d.waves == 8 || d.waves == 16) && d.tiles == (long long)((m + 31) / 32) * ((n + 31) / 32), "direct tiles", m, n);
        bbhip::PackedShape s{}, t{}, one = bbhip::best_shape(m, n, k);
        bbhip::best_shapes(m, n, k, m1, n, k1, s, t);
        for (auto const &p : {s, t, one}) {
            check(p.slabs >= 1 && p.slab_stages >= 1 && (long long)p.slabs * p.slab_stages >= p.k_steps && (long long)(p.slabs - 1) * p.slab_stages < p.k_steps, "packed slabs", m, k);
        }
        check(s.size == t.size, "one size of tiles for a launch", s.size, t.size);
        check((long long)one.m_tiles * bbhip::kTileRows[one.size] >= m && (long long)(one.m_tiles - 1) * bbhip::kTileRows[one.size] < m, "packed rows", m);
        check((long long)one.n_tiles * bbhip::kTileColumns[one.size] >= n && (long long)(one.n_tiles - 1) * bbhip::kTileColumns[one.size] < n, "packed columns", n);
        bbhip::LossPlan const l = bbhip::loss_plan(k1, m, n);
        check(l.piece >= 1 && l.piece <= m && (l.piece == m || l.piece % 256 == 0) && l.stride % 64 == 0 && l.stride >= n, "pieces of a loss", m, n);
        check((long long)l.tiles * l.tile >= m && (long long)(l.tiles - 1) * l.tile < m && (l.piece == m || l.piece % l.tile == 0), "tiles of a loss", m, n);
        // (what is held of the logits does not grow with the channels, but for the smallest piece)
        check((long long)l.piece * l.stride <= (64LL << 20) || l.piece <= 256, "size of a piece", l.piece, l.stride);
    }
    int const stride = bbhip::kDenseStrideMost;
    check(31LL * stride * 4 + 4096 < (1LL << 32) && stride >= bbhip::kDenseFramesMost + 128, "offsets of 32 bits", stride);
}

static void test_objects(void)
{
    auto layer = bb::DenseAffine<float, float>::Create(bb::indices_t({2, 3}), "hard_tanh", 7);
    layer->SetName("dense");
    check(layer->SetInputShape({4, 5}) == bb::indices_t({2, 3}) && layer->GetParameters().GetSize() == 2 && layer->GetGradients().GetSize() == 2, "shape and parameters");
    double square = 0;
    { auto W = layer->lock_W_const(); auto b = layer->lock_b_const(); for (int i = 0; i < 120; ++i) { square += (double)W[i] * W[i]; check(i >= 6 || b[i] == 0.0f, "b starts at 0"); } }
    check(square > 2 && square < 12, "W starts with a deviation of 1 / sqrt(20)", square);
    std::stringstream ss;
    layer->DumpObject(ss);
    auto again = std::dynamic_pointer_cast<bb::DenseAffine<float, float>>(bb::Object_Load(ss));
    check((bool)again, "loaded by its name");
    if (again) {
        check(again->GetName() == "dense" && again->GetInputShape() == bb::indices_t({4, 5}) && again->GetOutputShape() == bb::indices_t({2, 3}) && again->GetActivation() == 3, "loaded fields");
        auto W = layer->lock_W_const(), V = again->lock_W_const(); auto d = again->lock_dW_const();
        for (int i = 0; i < 120; ++i) { check(W[i] == V[i] && d[i] == 0.0f, "loaded weights"); }
    }
    std::vector<double> x(20, 0.0);
    x[3] = 100.0;
    { auto W = layer->lock_W_const(); check(layer->ForwardNode(1, x)[0] == (W[23] > 0.01f ? 1.0 : W[23] < -0.01f ? -1.0 : 100.0 * (double)W[23]), "ForwardNode"); }
    layer->SendCommand("parameter_lock true");
    check(layer->GetParameters().GetSize() == 0 && layer->GetGradients().GetSize() == 0, "parameter_lock");
    int threw = 0;
    try { (void)bb::DenseAffine<float, float>::Create((bb::index_t)3, "gelu"); } catch (bb::Exception const &) { ++threw; }
    try { (void)bb::LossDenseSoftmaxCrossEntropy<float>::Create(layer); } catch (bb::Exception const &) { ++threw; }
    check(threw == 2, "refusals", threw);
    auto bits = bb::DenseAffine<bb::Bit, float>::Create((bb::index_t)3);
    std::stringstream sb;
    bits->DumpObject(sb);
    check((bool)std::dynamic_pointer_cast<bb::DenseAffine<bb::Bit, float>>(bb::Object_Load(sb)), "bits loaded by its name");
    check(bb::LossDenseSoftmaxCrossEntropy<bb::Bit>::Create(bits)->GetLoss() == 0, "a loss of nothing");
}

static bb::FrameBuffer random_frames(std::mt19937 &mt, int frames, bb::indices_t shape)
{
    std::normal_distribution<float> dist(0.25f, 1.0f);
    bb::FrameBuffer buf(frames, shape, BB_TYPE_FP32);
    auto p = buf.Lock<float>();
    for (int n = 0; n < buf.GetNodeSize(); ++n) { for (int f = 0; f < frames; ++f) { p.Set(f, n, dist(mt)); } }
    return buf;
}

static bb::FrameBuffer random_bits(std::mt19937 &mt, int frames, bb::indices_t shape)
{
    bb::FrameBuffer buf(frames, shape, BB_TYPE_BIT);
    auto p = buf.Lock<bb::Bit>();
    for (int n = 0; n < buf.GetNodeSize(); ++n) { for (int f = 0; f < frames; ++f) { p.Set(f, n, bb::Bit((mt() >> 7) % 3 == 0)); } }
    return buf;
}

// two stacked passes with a residual: each finds its own input, the weights' gradients add up
template <typename BinType>
static void test_layer(int inputs, int outputs, int frames, char const *activation)
{
    std::mt19937 mt(inputs + frames);
    bool const bit = std::is_same<BinType, bb::Bit>::value;
    auto layer = bb::DenseAffine<BinType, float>::Create((bb::index_t)outputs, activation);
    layer->SetInputShape({inputs});
    { auto b = layer->lock_b(); for (int o = 0; o < outputs; ++o) { b[o] = 0.01f * (float)(o % 50); } }
    bb::FrameBuffer x[2], r[2], dy[2], y[2], dx[2], dr[2];
    for (int k = 0; k < 2; ++k) {
        x[k] = bit ? random_bits(mt, frames, {inputs}) : random_frames(mt, frames, {inputs});
        r[k] = random_frames(mt, frames, {outputs}); dy[k] = random_frames(mt, frames, {outputs});
    }
    for (int k = 0; k < 2; ++k) { y[k] = layer->Forward(x[k], r[k], true); }
    for (int k = 1; k >= 0; --k) { dx[k] = layer->Backward(dy[k], &dr[k]); }
    int const kind = layer->GetActivation();
    std::vector<double> dW((std::size_t)inputs * outputs, 0.0), db(outputs, 0.0);
    auto W = layer->lock_W_const(); auto b = layer->lock_b_const();
    double worst_y = 0, worst_dx = 0, worst_dr = 0;
    for (int k = 0; k < 2; ++k) {
        auto py = y[k].template LockConst<float>(); auto pr = r[k].template LockConst<float>(); auto pd = dy[k].template LockConst<float>();
        auto pdx = dx[k].template LockConst<float>(); auto pdr = dr[k].template LockConst<float>();
        for (int f = 0; f < frames; ++f) {
            std::vector<double> v(inputs), back(inputs, 0.0);
            for (int i = 0; i < inputs; ++i) { v[i] = bit ? (double)(bool)x[k].template LockConst<bb::Bit>().Get(f, i) : (double)x[k].template LockConst<float>().Get(f, i); }
            for (int o = 0; o < outputs; ++o) {
                double z = (double)b[o] + pr.Get(f, o);
                for (int i = 0; i < inputs; ++i) { z += (double)W[(bb::index_t)o * inputs + i] * v[i]; }
                double const a = kind == 1 ? std::max(z, 0.0) : kind == 2 ? 1 / (1 + std::exp(-z)) : kind == 3 ? std::min(std::max(z, -1.0), 1.0) : z;
                worst_y = std::max(worst_y, std::fabs(py.Get(f, o) - a));
                // (the derivative is of the value that the forward pass gave)
                double const s = py.Get(f, o), slope = kind == 1 ? s > 0 : kind == 2 ? s * (1 - s) : kind == 3 ? s > -1 && s < 1 : 1.0, d = pd.Get(f, o) * slope;
                worst_dr = std::max(worst_dr, std::fabs(pdr.Get(f, o) - d));
                db[o] += d;
                for (int i = 0; i < inputs; ++i) { back[i] += (double)W[(bb::index_t)o * inputs + i] * d; dW[(std::size_t)o * inputs + i] += d * v[i]; }
            }
            for (int i = 0; i < inputs; ++i) { worst_dx = std::max(worst_dx, std::fabs(pdx.Get(f, i) - back[i])); }
        }
    }
    // sums of up to 2000 products whose magnitudes add up to 100 at most, each rounded to 2^-24
    check(worst_y < 1e-4 && worst_dx < 1e-4 && worst_dr < 1e-5, "dense y, dx, dr", worst_y, worst_dx);
    double worst = 0;
    { auto p = layer->lock_dW_const(); for (std::size_t i = 0; i < dW.size(); ++i) { worst = std::max(worst, std::fabs(p[(bb::index_t)i] - dW[i])); } }
    { auto p = layer->lock_db_const(); for (int o = 0; o < outputs; ++o) { worst = std::max(worst, std::fabs(p[o] - db[o])); } }
    check(worst < 1e-5 * frames + 1e-4, "dW, db of two passes", worst);
}

// a dense layer as a convolution's: the same as the layer on every window
static void test_convolution(void)
{
    std::mt19937 mt(3);
    int const frames = 20;
    auto layer = bb::DenseAffine<float, float>::Create((bb::index_t)5, "relu"), alone = bb::DenseAffine<float, float>::Create((bb::index_t)5, "relu");
    auto net = bb::Convolution2d<float, float>::Create(layer, 3, 3);
    bb::FrameBuffer x = random_frames(mt, frames, {2, 6, 7}), y = net->Forward(x), taps(frames * 20, {2, 3, 3}, BB_TYPE_FP32);
    check(y.GetShape() == bb::indices_t({5, 4, 5}) && y.GetFrameSize() == frames, "convolution's shape");
    {
        auto p = x.LockConst<float>(); auto q = taps.Lock<float>();
        for (int f = 0; f < frames; ++f) { for (int at = 0; at < 20; ++at) { for (int c = 0; c < 2; ++c) { for (int v = 0; v < 3; ++v) { for (int h = 0; h < 3; ++h) {
            q.Set(f * 20 + at, c * 9 + v * 3 + h, p.Get(f, c * 42 + (at / 5 + v) * 7 + at % 5 + h)); } } } } }
    }
    bb::FrameBuffer z = alone->Forward(taps);
    auto p = y.LockConst<float>(); auto q = z.LockConst<float>();
    for (int f = 0; f < frames; ++f) { for (int at = 0; at < 20; ++at) { for (int o = 0; o < 5; ++o) { check(p.Get(f, o * 20 + at) == q.Get(f * 20 + at, o), "a window's output"); } } }
    bb::FrameBuffer dx = net->Backward(random_frames(mt, frames, {5, 4, 5}));
    check(dx.GetShape() == x.GetShape() && dx.GetFrameSize() == frames, "convolution's gradient");
}

// two layers, the loss on top of the second, a clipped Adam step
static void test_step(int inputs, int hidden, int channels, int frames)
{
    std::mt19937 mt(5);
    auto first = bb::DenseAffine<float, float>::Create((bb::index_t)hidden, "sigmoid", 2), head = bb::DenseAffine<float, float>::Create((bb::index_t)channels, "none", 3);
    auto loss = bb::LossDenseSoftmaxCrossEntropy<float>::Create(head);
    bb::FrameBuffer x = random_frames(mt, frames, {inputs}), label(frames, {1}, BB_TYPE_INT32);
    { auto p = label.Lock<std::int32_t>(); for (int f = 0; f < frames; ++f) { p.Set(f, 0, f % 5 == 4 ? -1 : (int)(mt() % (unsigned)channels)); } }
    first->SetInputShape({inputs}); head->SetInputShape({hidden});
    bb::Variables params = first->GetParameters(), grads = first->GetGradients();
    params.PushBack(head->GetParameters()); grads.PushBack(head->GetGradients());
    auto value = [&](void) {                        // 64 bits, from the layers' node by node values
        double sum = 0;
        int count = 0;
        auto p = x.LockConst<float>(); auto t = label.LockConst<std::int32_t>();
        for (int f = 0; f < frames; ++f) {
            if (t.Get(f, 0) < 0) { continue; }
            std::vector<double> v, h;
            for (int i = 0; i < inputs; ++i) { v.push_back(p.Get(f, i)); }
            for (int o = 0; o < hidden; ++o) { h.push_back(first->ForwardNode(o, v)[0]); }
            double top = -1e300, s = 0, mine = 0;
            std::vector<double> z;
            for (int c = 0; c < channels; ++c) { z.push_back(head->ForwardNode(c, h)[0]); top = std::max(top, z.back()); }
            for (int c = 0; c < channels; ++c) { s += std::exp(z[(std::size_t)c] - top); }
            mine = z[(std::size_t)t.Get(f, 0)];
            sum += top + std::log(s) - mine;
            ++count;
        }
        return sum / count;
    };
    double const before = value();
    bb::FrameBuffer dh = loss->CalculateLoss(first->Forward(x), label, frames);
    check(std::fabs(loss->GetLoss() - before) < 1e-5 * (1 + before), "the loss", loss->GetLoss(), before);
    (void)first->Backward(dh);
    // the norm against loops, and the loss falls as the gradient tells
    double square = 0;
    std::vector<std::vector<float>> g;
    for (bb::index_t i = 0; i < grads.GetSize(); ++i) {
        auto t = std::dynamic_pointer_cast<bb::Tensor_<float>>(i == 0 ? first->dW() : i == 1 ? first->db() : i == 2 ? head->dW() : head->db());
        auto p = t->LockConst();
        g.emplace_back();
        for (bb::index_t j = 0; j < t->GetSize(); ++j) { g.back().push_back(p[j]); square += (double)p[j] * p[j]; }
    }
    bb::GradientNorm norm(grads);
    check(std::fabs(norm.Calculate() - std::sqrt(square)) < 1e-6 * std::sqrt(square), "the norm", norm.Calculate(), std::sqrt(square));
    // Adam with a clipped gradient: against the formula, from moments of 0
    auto opt = bb::OptimizerAdam<float>::Create(0.001f, 0.875f, 0.9921875f);
    opt->SetVariables(params, grads);
    opt->SetGradientClipping(0.25 * std::sqrt(square));
    std::vector<float> old;
    { auto p = head->lock_W_const(); for (int i = 0; i < channels * hidden; ++i) { old.push_back(p[i]); } }
    opt->Step();
    check(std::fabs(opt->GetGradientNorm() - std::sqrt(square)) < 1e-6 * std::sqrt(square), "the norm of the step");
    double worst = 0;
    {
        auto p = head->lock_W_const();
        double const lr = 0.001f * std::sqrt(1 - 0.9921875) / (1 - 0.875);
        for (int i = 0; i < channels * hidden; ++i) {
            double const c = 0.25 * g[2][(std::size_t)i], m = 0.125 * c, v = 0.0078125 * c * c;
            worst = std::max(worst, std::fabs(p[i] - (old[(std::size_t)i] - lr * m / (std::sqrt(v) + 1e-7))));
        }
    }
    check(worst < 1e-6, "a clipped step", worst);
    // scaled in place, twice: the second time nothing is left to scale
    check(std::fabs(norm.Clip(0.5 * std::sqrt(square)) - std::sqrt(square)) < 1e-6 * std::sqrt(square), "Clip returns the norm that was");
    check(std::fabs(norm.Clip(0.5 * std::sqrt(square)) - 0.5 * std::sqrt(square)) < 1e-6 * std::sqrt(square), "the norm behind Clip");
    { auto p = head->lock_dW_const(); for (std::size_t i = 0; i < g[2].size(); ++i) { check(std::fabs(p[(bb::index_t)i] - 0.5 * g[2][i]) <= 1e-6 * std::fabs(g[2][i]), "scaled"); } }
    opt->ZeroGrad();
    check(norm.Calculate() == 0, "ZeroGrad");
    // the loss alone leaves the gradients as they are; weights of 0 count for nothing
    bb::FrameBuffer weight(frames, {1}, BB_TYPE_FP32);
    { auto p = weight.Lock<float>(); for (int f = 0; f < frames; ++f) { p.Set(f, 0, f < 3 ? 0.0f : 2.0f); } }
    loss->Clear();
    check(loss->CalculateLoss(first->Forward(x, false), label, weight, false).Empty() && loss->GetLoss() > 0 && norm.Calculate() == 0, "evaluation");
}

int main(int argc, char **argv)
{
    try {
        if (argc > 1 && std::strcmp(argv[1], "--rules") == 0) { test_rules(); test_objects(); }
        else {
            if (!bb::Manager::IsDeviceAvailable()) { std::printf("no device available\n"); return 2; }
            test_objects();
            test_layer<float>(20, 30, 33, "none");
            test_layer<float>(70, 40, 66, "sigmoid");
            test_layer<float>(130, 60, 5, "hard_tanh");
            test_layer<bb::Bit>(90, 35, 70, "relu");
            test_layer<bb::Bit>(300, 20, 1, "none");
            test_convolution();
            test_step(12, 20, 10, 64);
            test_step(30, 40, 130, 77);
        }
    }
    catch (std::exception const &e) { std::printf("exception: %s\n", e.what()); return 1; }
    std::printf(g_failures ? "%d checks failed\n" : "all checks passed\n", g_failures);
    return g_failures ? 1 : 0;
}
