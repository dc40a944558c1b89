// What bb::GradientNorm and OptimizerAdam::SetGradientClipping refuse, and what they say ahead of a first step (no device).
#include <cmath>
#include <cstdio>
#include <string>

#include "bb/DenseAffine.h"
#include "bb/GradientNorm.h"
#include "bb/OptimizerAdam.h"

static int g_failures = 0;
static void check(bool ok, char const *what) { if (!ok) { ++g_failures; std::printf("FAILED %s\n", what); } }

template <class F> static std::string thrown(F const &f)
{
    try { f(); } catch (std::exception const &e) { return e.what(); }
    return "";
}
static bool says(std::string const &text, char const *word) { return text.find(word) != std::string::npos; }

int main()
{
    auto layer = bb::DenseAffine<float, float>::Create((bb::index_t)3);
    layer->SetInputShape({4});
    bb::Variables const params = layer->GetParameters(), grads = layer->GetGradients();
    bb::Variables twice = layer->GetGradients(), copied;
    twice.PushBack(grads);
    auto shallow = std::make_shared<bb::Tensor>(*layer->dW());              // shares its elements
    copied.PushBack(layer->dW()); copied.PushBack(shallow);
    check(twice.HasOneTwice() && copied.HasOneTwice() && !grads.HasOneTwice(), "lists with one twice");
    bb::Variables empty;
    for (int i = 0; i < 2; ++i) { empty.PushBack(std::make_shared<bb::Tensor>()); }
    check(!empty.HasOneTwice(), "tensors without elements");

    check(says(thrown([&] { bb::GradientNorm norm(twice); }), "twice") && says(thrown([&] { bb::GradientNorm norm(copied); }), "twice"), "a norm refuses a tensor twice");

    auto opt = bb::OptimizerAdam<float>::Create();
    check(opt->GetGradientNorm() == 0, "no clipping, no norm");
    check(says(thrown([&] { opt->SetGradientClipping(NAN); }), "not a number"), "NaN is refused");
    opt->SetGradientClipping(1.0);
    check(opt->GetGradientNorm() == 0, "0 ahead of the first step");
    bb::Variables two = params;
    two.PushBack(params);
    check(says(thrown([&] { opt->SetVariables(two, twice); }), "twice"), "clipping refuses a tensor twice");
    bb::Variables both = params, same = params;
    check(says(thrown([&] { opt->SetVariables(both, same); }), "twice"), "clipping refuses parameters as their own gradients");
    // (without a device the rest of the binding throws, of something else; it is not refused for a tensor twice)
    opt->SetGradientClipping(-1.0);
    check(!says(thrown([&] { opt->SetVariables(two, twice); }), "twice"), "without clipping it is as it was");
    check(says(thrown([&] { opt->SetGradientClipping(2.0); }), "twice"), "clipping is not turned on for such lists");
    check(!says(thrown([&] { opt->SetVariables(params, grads); opt->SetGradientClipping(INFINITY); opt->SetGradientClipping(0.0); }), "twice"), "lists as they should be");
    std::printf(g_failures ? "%d checks failed\n" : "all checks passed\n", g_failures);
    return g_failures ? 1 : 0;
}
