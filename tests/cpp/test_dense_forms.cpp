// How the rules divide the products of dense layers and of the loss on top of one, for tests that want a size to take a form (no device).
//   test_dense_forms --rules                                        what the launches rely on, over many sizes
//   test_dense_forms forward  inputs outputs frames                 one line: the form that a call of these sizes takes
//   test_dense_forms backward inputs outputs frames
//   test_dense_forms loss     inputs channels frames
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <random>

#include "../../binarybrain_amd/csrc/dense_rules.hpp"

using namespace bbhip;

static char const *const kSizeNames[] = {"large", "middle", "small"};

static int rules(void)
{
    std::mt19937 mt(2);
    auto pick = [&](int most) { return 1 + (int)(mt() % (unsigned)(mt() % 3 == 0 ? 100 : most)); };
    int failures = 0;
    for (int i = 0; i < 200000; ++i) {
        int const m = pick(i % 5 ? 9000 : kDenseNodesMost), n = pick(i % 7 ? 9000 : kDenseFramesMost), k = pick(i % 2 ? 9000 : 2000000);
        DirectShape a, b;
        direct_shapes(m, n, k, n < 9000 ? n : 9000, k, m, a, b);
        // a kernel of eight, of four and of one wavefront is all there is
        for (DirectShape const &s : {direct_shape(m, n, k), logits_shape(m, n, k), a, b}) {
            if (s.waves != 1 && s.waves != 4 && s.waves != 8) { ++failures; std::printf("%d wavefronts for %d x %d x %d\n", s.waves, m, n, k); }
        }
    }
    return failures;
}

int main(int argc, char **argv)
{
    if (argc == 2 && std::strcmp(argv[1], "--rules") == 0) {
        int const failures = rules();
        std::printf("%d checks failed\n", failures);
        return failures != 0;
    }
    if (argc != 5) { return 2; }
    int const i = std::atoi(argv[2]), o = std::atoi(argv[3]), f = std::atoi(argv[4]);
    auto const packed = [](char const *what, PackedShape const &s, bool wide) { std::printf("%s %s slabs %d %s", what, kSizeNames[s.size], s.slabs, wide ? "wide" : "narrow"); };
    if (std::strcmp(argv[1], "forward") == 0) {
        if (f <= 8)                           { std::printf("few"); }
        else if (!forward_packed(i, o, f))    { DirectShape const s = direct_shape(o, f, i); std::printf("straight waves %d slabs %d", s.waves, s.slabs); }
        else                                  { packed("packed", best_shape(o, f, i), pack_is_wide(i)); }
    }
    else if (std::strcmp(argv[1], "backward") == 0) {
        if (backward_packed(i, o, f)) {
            PackedShape w, x;
            best_shapes(o, i, f, i, f, o, w, x);
            packed("packed", w, pack_is_wide(f > o ? f : o));
            std::printf(" and slabs %d", x.slabs);
        }
        else {
            DirectShape w, x;
            direct_shapes(o, i + 1, f, i, f, o, w, x);
            std::printf("straight waves %d slabs %d and waves %d slabs %d", w.waves, w.slabs, x.waves, x.slabs);
        }
    }
    else {
        LossPlan const p = loss_plan(i, o, f);
        int const pieces = ceil_div(o, p.piece);
        std::printf("%s pieces %d last %d", p.packed ? "packed" : "straight", pieces, o - (pieces - 1) * p.piece);
        if (p.packed) { std::printf(" logits %s slabs %d", kSizeNames[p.logits.size], p.logits.slabs); }
    }
    std::printf("\n");
    return 0;
}
