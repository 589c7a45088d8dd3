// The workgroup of a group from the reciprocal in 64 bits (csrc/attn_plan.h owner), on the CPU under sanitizers: the same as
// from the shares' borders, and the same partial result, up to the largest numbers.
#include <cstdio>
#include <cstdlib>
#include <random>

#include "../qwenny_amd/csrc/attn_plan.h"

using namespace qh;

#define CHECK(c)                                               \
    do {                                                       \
        if (!(c)) {                                            \
            std::fprintf(stderr, "line %d: %s\n", __LINE__, #c); \
            std::exit(1);                                      \
        }                                                      \
    } while (0)

int main() {
    std::mt19937_64 rng(12);
    auto in = [&](int64_t lo, int64_t hi) { return (int)std::uniform_int_distribution<int64_t>(lo, hi)(rng); };
    for (int trial = 0; trial < 30000; trial++) {
        const int all = trial % 3 ? in(1, 5000) : trial % 2 ? in(1, 2147483647 - 1) : 2147483647 - in(1, 5000);
        const int used = trial % 5 ? in(1, all < TREE_MAX_WGS ? all : TREE_MAX_WGS) : all < TREE_MAX_WGS ? all : TREE_MAX_WGS;
        const double inv_all = 1.0 / all;
        CHECK(owner(0, used, inv_all) == 0 && owner(all - 1, used, inv_all) == used - 1);
        for (int k = 0; k < 20; k++) {
            const int w = in(0, used - 1), lo = first_group(w, all, used), hi = first_group(w + 1, all, used);
            CHECK(owner(lo, used, inv_all) == w && owner(hi - 1, used, inv_all) == w);
            const int at = in(0, all - 1), of = group_owner(at, all, used);
            CHECK(owner(at, used, inv_all) == of);
            for (int u0 : {at, lo}) {  // the first workgroup of a unit that begins there: has it a part before
                const int first = group_owner(u0, all, used);
                CHECK(2 * first + (owner(u0 - 1, used, inv_all) == first ? 1 : 0) == partial_slot(first, u0, all, used));
            }
        }
    }
    std::puts("ok");
    return 0;
}
