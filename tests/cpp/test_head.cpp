// The host classes over the operators at the head of a network: bb::LayerNormalization, TopLogits, LossDistillation, CategoricalSampling.
//   test_head          on the device: values against 64-bit loops, gradients, accumulation, stacked passes, serialization, a chain of all of them
//   test_head --rules  on the CPU: how the column operators divide their work, over many sizes; objects that need no device
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <random>
#include <sstream>
#include <vector>

#include "../../binarybrain_amd/csrc/launch_rules.hpp"
#include "bb/CategoricalSampling.h"
#include "bb/LayerNormalization.h"
#include "bb/LossDistillation.h"
#include "bb/ObjectLoader.h"
#include "bb/OptimizerAdam.h"
#include "bb/Sequential.h"

static int g_failures = 0;
static void check(bool ok, char const *what, double a = 0, double b = 0)
{
    if (!ok) { ++g_failures; std::printf("FAILED %s (%g, %g)\n", what, a, b); }
}

// every row in one slab, every unit in one tile, nothing empty, and the bounds that the kernels rely on
static void test_rules(void)
{
    std::mt19937 mt(1);
    auto pick = [&](int most) { return 1 + (int)(mt() % (unsigned)(mt() % 3 == 0 ? 64 : most)); };
    for (int n = 0; n < 200000; ++n) {
        int const units = pick(n % 2 ? 1 << 20 : 3000), rows = pick(n % 3 ? 70000 : 600), top = 1 + (int)(mt() % 256);
        int log_tx = -1, tiles = 0, slab_rows = 0, slabs = 0;
        for (int wide = 0; wide < 2; ++wide) {
            bbhip::column_split(units, rows, wide != 0, 8, log_tx, tiles, slab_rows, slabs);
            bool ok = log_tx >= 0 && log_tx <= 6 && ((long long)tiles << log_tx) >= units && ((long long)(tiles - 1) << log_tx) < units;
            ok = ok && slabs >= 1 && slabs <= 64 && (long long)slabs * slab_rows >= rows && (long long)(slabs - 1) * slab_rows < rows;
            check(ok, "column_split", units, rows);
            for (int bit = 0; bit < 2; ++bit) {
                bool longer = false;
                if (bbhip::layer_norm_whole(units, rows, wide != 0, bit != 0, log_tx, longer)) {
                    check(log_tx >= 0 && log_tx <= 6 && rows <= (longer ? 16 : 4) * (1024 >> log_tx) && !(bit && longer), "layer_norm_whole", units, rows);
                }
            }
        }
        int const channels = rows < top ? top : rows;
        bbhip::top_split(units, channels, top, log_tx, tiles, slab_rows, slabs);
        bool ok = (log_tx == 0 || log_tx == 2) && ((long long)tiles << log_tx) >= units && ((long long)(tiles - 1) << log_tx) < units;
        ok = ok && slabs >= 1 && (slabs == 1 || slabs * top <= 1024) && (long long)slabs * slab_rows >= channels && (long long)(slabs - 1) * slab_rows < channels;
        check(ok, "top_split", units, channels);
        if (g_failures > 5) { return; }
    }
}

// the variants that the tests of large calls are there for (test_gpu_head_edges.py): a rule that is tuned again must not leave a kernel without them
static void test_variants(void)
{
    // nodes, frames, rows on 16 bytes, one launch with 16 rows per thread
    struct { int nodes, frames; bool wide, longer; } const norms[] = {
        {1025, 4097, true, true}, {1100, 4099, true, true}, {4096, 8190, true, true}, {257, 4097, false, true}, {1024, 8191, false, true},
        {4097, 8190, true, false}, {3000, 8193, true, false}, {1025, 8191, false, false}};
    for (auto const &n : norms) {
        int log_tx = 0;
        bool longer = false;
        bool const whole = bbhip::layer_norm_whole(n.wide ? (n.frames + 3) / 4 : n.frames, n.nodes, n.wide, false, log_tx, longer);
        check(n.longer ? whole && longer : !whole, "layer norm of long columns", n.nodes, n.frames);
    }
    // channels, frames, rows on 16 bytes, k, slabs: all with four units side by side
    struct { int channels, frames; bool wide; int top, slabs; } const tops[] = {
        {3100, 2050, true, 64, 3}, {3100, 2050, true, 200, 3}, {10000, 1030, true, 100, 5}, {2000, 1025, false, 40, 2}, {3200, 2050, false, 120, 1}, {2500, 2050, false, 7, 1}};
    for (auto const &t : tops) {
        int log_tx = 0, tiles = 0, slab_rows = 0, slabs = 0;
        bbhip::top_split(t.wide ? (t.frames + 3) / 4 : t.frames, t.channels, t.top, log_tx, tiles, slab_rows, slabs);
        check(log_tx == 2 && slabs == t.slabs, "selection of large calls", t.channels, slabs);
    }
}

// what a launch cannot hold, no rule asks of it
static void test_launches(void)
{
    check(bbhip::launch_holds((1LL << 24) - 1, 256) && !bbhip::launch_holds(1LL << 24, 256) && !bbhip::launch_holds(0, 64) && !bbhip::launch_holds(1LL << 40, 1024), "launch_holds");
    for (int rows = 1; rows <= 4096; rows = rows < 64 ? rows + 1 : rows * 2) {
        for (int units = 1 << 20; units <= 1 << 28; units *= 2) {
            int log_tx = 0;
            bool longer = false;
            for (int form = 0; form < 4; ++form) {
                if (bbhip::layer_norm_whole(units, rows, (form & 1) != 0, (form & 2) != 0, log_tx, longer)) {
                    check(bbhip::launch_holds((units + (1LL << log_tx) - 1) >> log_tx, 1024), "one launch of layer norm", units, rows);
                }
            }
        }
    }
}

static void test_objects(void)
{
    auto layer = bb::LayerNormalization<float, float>::Create(0.125f);
    layer->SetName("norm");
    layer->SetInputShape({3, 4});
    check(layer->GetOutputShape() == bb::indices_t({3, 4}) && layer->GetParameters().GetSize() == 2 && layer->GetGradients().GetSize() == 2, "shape and parameters");
    { auto g = layer->lock_gamma(); auto b = layer->lock_beta(); for (int i = 0; i < 12; ++i) { check(g[i] == 1.0f && b[i] == 0.0f, "start"); g[i] = (float)i; b[i] = (float)-i; } }
    std::stringstream ss;
    layer->DumpObject(ss);
    auto again = std::dynamic_pointer_cast<bb::LayerNormalization<float, float>>(bb::Object_Load(ss));
    check((bool)again, "loaded by its name");
    if (again) {
        check(again->GetName() == "norm" && again->GetInputShape() == bb::indices_t({3, 4}) && again->GetEps() == 0.125f, "loaded fields");
        auto g = again->lock_gamma_const(); auto b = again->lock_beta_const(); auto d = again->lock_dgamma_const();
        for (int i = 0; i < 12; ++i) { check(g[i] == (float)i && b[i] == (float)-i && d[i] == 0.0f, "loaded weights"); }
    }
    layer->SendCommand("parameter_lock true");
    check(layer->GetParameters().GetSize() == 0 && layer->GetGradients().GetSize() == 0, "parameter_lock");
    bool threw = false;
    try { (void)layer->ForwardNode(0, {1.0}); } catch (bb::Exception const &) { threw = true; }
    check(threw, "ForwardNode refuses");
    auto bits = bb::LayerNormalization<bb::Bit, float>::Create();
    std::stringstream sb;
    bits->DumpObject(sb);
    check((bool)std::dynamic_pointer_cast<bb::LayerNormalization<bb::Bit, float>>(bb::Object_Load(sb)), "bits loaded by its name");
    check(bb::LossDistillation<float>::Create()->GetLoss() == 0 && bb::PixelShape({5, 2, 3}, 0) == bb::indices_t({2, 3}) && bb::PixelShape({5}, 0) == bb::indices_t({1}) &&
          bb::PixelShape({5, 7}, 2) == bb::indices_t({2, 7}), "shapes");
}

static bb::FrameBuffer random_frames(std::mt19937 &mt, int frames, bb::indices_t shape, float scale = 1.0f)
{
    std::normal_distribution<float> dist(0.25f, scale);
    bb::FrameBuffer buf(frames, shape, BB_TYPE_FP32);
    auto p = buf.Lock<float>();
    for (int n = 0; n < buf.GetNodeSize(); ++n) { for (int f = 0; f < frames; ++f) { p.Set(f, n, dist(mt)); } }
    return buf;
}

template <typename BinType>
static void test_layer_norm(int nodes, int frames)
{
    std::mt19937 mt(nodes + frames);
    bool const bit = std::is_same<BinType, bb::Bit>::value;
    auto layer = bb::LayerNormalization<BinType, float>::Create(1.0e-3f);
    layer->SetInputShape({nodes});
    { auto g = layer->lock_gamma(); auto b = layer->lock_beta(); for (int i = 0; i < nodes; ++i) { g[i] = 0.5f + 0.01f * (float)(i % 50); b[i] = 0.1f * (float)(i % 7); } }
    bb::FrameBuffer x[2], dy[2], y[2];
    for (int k = 0; k < 2; ++k) {
        if (bit) {
            x[k] = bb::FrameBuffer(frames, {nodes}, BB_TYPE_BIT);
            auto p = x[k].Lock<bb::Bit>();
            for (int n = 0; n < nodes; ++n) { for (int f = 0; f < frames; ++f) { p.Set(f, n, bb::Bit((mt() >> 7) % 3 == 0)); } }
        }
        else { x[k] = random_frames(mt, frames, {nodes}); }
        dy[k] = random_frames(mt, frames, {nodes});
    }
    // two training passes, then their backward passes in reverse: each finds its own input and statistics; the weights' gradients add up
    for (int k = 0; k < 2; ++k) { y[k] = layer->Forward(x[k]); }
    bb::FrameBuffer dx[2];
    for (int k = 1; k >= 0; --k) { dx[k] = layer->Backward(dy[k]); }
    bb::FrameBuffer const served = layer->Forward(x[0], false);
    std::vector<double> dg(nodes, 0.0), db(nodes, 0.0), g(nodes), b(nodes);
    { auto pg = layer->lock_gamma_const(); auto pb = layer->lock_beta_const(); for (int i = 0; i < nodes; ++i) { g[i] = pg[i]; b[i] = pb[i]; } }
    double worst_y = 0, worst_dx = 0;
    for (int k = 0; k < 2; ++k) {
        auto value = [&](int n, int f) { return bit ? (double)(bool)x[k].template LockConst<bb::Bit>().Get(f, n) : (double)x[k].template LockConst<float>().Get(f, n); };
        auto py = y[k].template LockConst<float>(); auto pd = dy[k].template LockConst<float>(); auto pdx = dx[k].template LockConst<float>(); auto ps = served.template LockConst<float>();
        for (int f = 0; f < frames; ++f) {
            std::vector<double> v(nodes);
            double mean = 0, var = 0, a = 0, c = 0;
            for (int n = 0; n < nodes; ++n) { v[n] = value(n, f); mean += v[n]; }
            mean /= nodes;
            for (int n = 0; n < nodes; ++n) { var += (v[n] - mean) * (v[n] - mean); }
            double const rstd = 1.0 / std::sqrt(var / nodes + (double)1.0e-3f);
            for (int n = 0; n < nodes; ++n) {
                double const xh = (v[n] - mean) * rstd, d = pd.Get(f, n);
                a += d * g[n]; c += d * g[n] * xh; dg[n] += d * xh; db[n] += d;
                worst_y = std::max(worst_y, std::fabs(py.Get(f, n) - (xh * g[n] + b[n])));
                if (k == 0) { check(ps.Get(f, n) == py.Get(f, n), "inference computes the same"); }
            }
            for (int n = 0; n < nodes; ++n) {
                double const xh = (v[n] - mean) * rstd, d = pd.Get(f, n);
                worst_dx = std::max(worst_dx, std::fabs(pdx.Get(f, n) - rstd * (d * g[n] - a / nodes - xh * c / nodes)) / rstd);
            }
        }
    }
    // values of size 5, a hundred roundings of 2^-24 in the statistics
    check(worst_y < 5e-5, "layer norm y", worst_y);
    check(worst_dx < 1e-4, "layer norm dx", worst_dx);
    auto pg = layer->lock_dgamma_const(); auto pb = layer->lock_dbeta_const();
    for (int n = 0; n < nodes; ++n) {
        check(std::fabs(pg[n] - dg[n]) < 1e-4 * std::sqrt(2.0 * frames) + 1e-5 * frames, "dgamma", pg[n], dg[n]);
        check(std::fabs(pb[n] - db[n]) < 1e-4 * std::sqrt(2.0 * frames) + 1e-5 * frames, "dbeta", pb[n], db[n]);
    }
}

// a student with a normalisation in front, a teacher's logits, the loss and its gradient, an Adam step, and categories drawn from the logits
static void test_chain(int ch, int pix, int frames)
{
    std::mt19937 mt(7);
    bb::indices_t const shape = pix > 1 ? bb::indices_t({ch, pix}) : bb::indices_t({ch});
    bb::FrameBuffer x = random_frames(mt, frames, shape), teacher = random_frames(mt, frames, shape, 2.0f);
    auto net = bb::Sequential::Create();
    auto norm = bb::LayerNormalization<float, float>::Create();
    net->Add(norm);
    net->SetInputShape(shape);
    auto loss = bb::LossDistillation<float>::Create(2.0f, 8);
    bb::TopLogits top;
    auto const list = top.Calculate(teacher, std::min(8, ch));
    auto value = [&](bb::FrameBuffer y) {           // 64 bits, from the lists
        auto py = y.LockConst<float>(); auto pi = list.index.LockConst<std::int32_t>(); auto pz = list.logit.LockConst<float>();
        double sum = 0;
        for (int p = 0; p < pix; ++p) {
            for (int f = 0; f < frames; ++f) {
                double s = 0, e = 0, l = 0, top_y = -1e300;
                for (int c = 0; c < ch; ++c) { top_y = std::max(top_y, (double)py.Get(f, c * pix + p) / 2.0); }
                for (int c = 0; c < ch; ++c) { s += std::exp(py.Get(f, c * pix + p) / 2.0 - top_y); }
                int const k = std::min(8, ch);
                double const z0 = pz.Get(f, p);
                for (int j = 0; j < k; ++j) { e += std::exp((pz.Get(f, j * pix + p) - z0) / 2.0); }
                for (int j = 0; j < k; ++j) {
                    double const lq = (pz.Get(f, j * pix + p) - z0) / 2.0 - std::log(e);
                    l += std::exp(lq) * (lq - (py.Get(f, pi.Get(f, j * pix + p) * pix + p) / 2.0 - top_y - std::log(s)));
                    if (j > 0) { check(pz.Get(f, j * pix + p) <= pz.Get(f, (j - 1) * pix + p), "descending"); }
                }
                sum += 4.0 * l;
            }
        }
        return sum / ((double)pix * frames);
    };
    bb::FrameBuffer y = net->Forward(x);
    bb::FrameBuffer dy = loss->CalculateLoss(y, teacher, frames);
    double const want = value(y);
    check(std::fabs(loss->GetLoss() - want) < 1e-5 * (1 + std::fabs(want)) * 20, "distillation loss", loss->GetLoss(), want);
    (void)loss->CalculateLoss(y, list, bb::FrameBuffer());
    check(std::fabs(loss->GetLoss() - want) < 1e-5 * (1 + std::fabs(want)) * 20, "the mean over two equal batches is that of one", loss->GetLoss(), want);
    loss->Clear();
    check(loss->GetLoss() == 0, "Clear");
    // weights: half of the frames count for nothing
    bb::FrameBuffer w(frames, bb::PixelShape(shape, 0), BB_TYPE_FP32);
    { auto p = w.Lock<float>(); for (int n = 0; n < pix; ++n) { for (int f = 0; f < frames; ++f) { p.Set(f, n, f % 2 ? 0.0f : 1.0f); } } }
    bb::FrameBuffer dw = loss->CalculateLoss(y, list, w);
    { auto p = dw.LockConst<float>(); for (int n = 0; n < ch * pix; ++n) { for (int f = 1; f < frames; f += 2) { check(p.Get(f, n) == 0.0f, "a frame without weight"); } } }
    bb::FrameBuffer dx = net->Backward(dy);
    check(dx.GetFrameSize() == frames && dx.GetNodeSize() == ch * pix, "dx");
    // a step against the gradient of gamma and beta lowers the loss by about step * |gradient|^2
    double norm2 = 0;
    {
        auto dg = norm->lock_dgamma_const(); auto db = norm->lock_dbeta_const(); auto g = norm->lock_gamma(); auto b = norm->lock_beta();
        for (int i = 0; i < ch * pix; ++i) { norm2 += (double)dg[i] * dg[i] + (double)db[i] * db[i]; }
        double const step = 1e-3 / std::sqrt(norm2);
        for (int i = 0; i < ch * pix; ++i) { g[i] -= (float)(step * dg[i]); b[i] -= (float)(step * db[i]); }
    }
    double const after = value(net->Forward(x, false)), told = 1e-3 * std::sqrt(norm2);
    check(std::fabs((want - after) - told) < 0.05 * told + 2e-6, "the loss falls as the gradient tells", want - after, told);
    // drawn categories are among the kept, the largest for top_size 1
    bb::CategoricalSampling::create_t cs;
    cs.top_size = 3; cs.temperature = 0.7f;
    bb::FrameBuffer u(frames, bb::PixelShape(shape, 0), BB_TYPE_FP32), share;
    { auto p = u.Lock<float>(); std::uniform_real_distribution<float> d(0, 1); for (int n = 0; n < pix; ++n) { for (int f = 0; f < frames; ++f) { p.Set(f, n, std::min(d(mt), 0.999999f)); } } }
    bb::FrameBuffer const drawn = bb::CategoricalSampling::Create(cs)->Sample(teacher, u, &share);
    cs.top_size = 1;
    bb::FrameBuffer const best = bb::CategoricalSampling::Create(cs)->Sample(teacher, u);
    auto pi = list.index.LockConst<std::int32_t>(); auto pd = drawn.LockConst<std::int32_t>(); auto pb = best.LockConst<std::int32_t>(); auto ps = share.LockConst<float>();
    for (int p = 0; p < pix; ++p) {
        for (int f = 0; f < frames; ++f) {
            bool among = false;
            for (int j = 0; j < std::min(3, ch); ++j) { among = among || pi.Get(f, j * pix + p) == pd.Get(f, p); }
            check(among && ps.Get(f, p) > 0.0f && ps.Get(f, p) <= 1.0f, "drawn among the kept");
            check(pb.Get(f, p) == pi.Get(f, p), "top_size 1 is the largest");
        }
    }
}

int main(int argc, char **argv)
{
    try {
        if (argc > 1 && std::strcmp(argv[1], "--rules") == 0) { test_rules(); test_variants(); test_launches(); test_objects(); }
        else {
            if (!bb::Manager::IsDeviceAvailable()) { std::printf("no device available\n"); return 2; }
            test_objects();
            test_layer_norm<float>(50, 33);
            test_layer_norm<float>(700, 130);
            test_layer_norm<bb::Bit>(90, 70);
            test_layer_norm<bb::Bit>(3000, 40);
            test_chain(10, 1, 64);
            test_chain(12, 6, 33);
            test_chain(300, 1, 50);
        }
    }
    catch (std::exception const &e) { std::printf("exception: %s\n", e.what()); return 1; }
    std::printf(g_failures ? "%d checks failed\n" : "all checks passed\n", g_failures);
    return g_failures ? 1 : 0;
}
