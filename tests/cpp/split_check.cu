// Host checks of what the paged attention's merge kernels take from a workspace
// (csrc/paged.cuh), built and run by tests/test_paged_cpu.py without a GPU: every
// note that passes note_fits() names parts and rows within the call, whatever
// numbers it holds, and the notes that a call leaves pass.
#include <cstdio>
#include <cstdlib>

#include "paged.cuh"

using namespace nq;

static int fail(const char *what, const SplitNote &n, int cta) {
    std::printf("%s: cta %d, q_row %d, heads0 %d, tokens %d, parts %d\n", what, cta, n.q_row, n.heads0,
                n.tokens, n.parts);
    return 1;
}

int main() {
    const int ctas = 148, tokens = 300, heads = 12, group = 3;
    const int lo = -2147483647 - 1, hi = 2147483647;
    const int values[] = {lo, lo + 1, -1000, -1, 0, 1, 2, 3, 11, 12, 147, 148, 149, 299, 300, 301,
                          1 << 16, 1 << 24, hi - 1, hi};
    for (int cta : {0, 1, 100, 147})
        for (int q_row : values)
            for (int heads0 : values)
                for (int n : values)
                    for (int parts : values) {
                        const SplitNote x{q_row, heads0, n, parts};
                        // in 64 bits, from what the merge does with a note
                        const bool in = parts >= 1 && cta + (int64_t)parts <= ctas && q_row >= 0 &&
                                        n >= 1 && q_row + (int64_t)n <= tokens && heads0 >= 0 &&
                                        heads0 + (int64_t)group <= heads;
                        if (note_fits(x, cta, ctas, tokens, heads, group) != in)
                            return fail("wrong", x, cta);
                    }
    if (note_fits(SplitNote{0, 0, 0, 0}, 0, ctas, tokens, heads, group))
        return fail("an empty note is followed", SplitNote{0, 0, 0, 0}, 0);
    // bytes of any kind in its place
    std::srand(1);
    for (int i = 0; i < 1000000; ++i) {
        const SplitNote x{(int)(std::rand() * 2u), std::rand(), (int)(std::rand() * 2u),
                          (int)(std::rand() * 2u)};
        const int cta = std::rand() % ctas;
        if (note_fits(x, cta, ctas, tokens, heads, group) &&
            (x.parts > ctas - cta || x.q_row + (int64_t)x.tokens > tokens))
            return fail("past the call", x, cta);
    }
    std::puts("ok");
    return 0;
}
