// CPU check of the launch shapes of lucid_amd/csrc/lq_place.h: every workgroup of 1 to 2^31 has exactly one
// place, within what a launch takes.  Built and run by tests/test_launch_shapes.py.
#include <cstdint>
#include <cstdio>
#include <initializer_list>

#include "lq_place.h"

using namespace lq;

int main() {
    const int64_t X = WORKGROUPS_X;
    int fails = 0;
    for (int64_t n : {(int64_t)1, (int64_t)2, (int64_t)65536, X - 1, X, X + 1, 2 * X, ((int64_t)1 << 24) + 5,
                      ((int64_t)1 << 26) + 3, ((int64_t)1 << 31) - 1, (int64_t)65535 * X}) {
        const Workgroups w = workgroups(n);
        const bool fits = (uint64_t)w.x * 512 < ((uint64_t)1 << 32) && w.y <= 65535;
        const bool covers = (int64_t)w.x * w.y >= n && (int64_t)w.x * (w.y - 1) < n;
        // rows of x follow each other without a gap
        const bool line = workgroup_index(0, 0) == 0 && (w.y == 1 || workgroup_index(0, 1) == (int64_t)w.x) &&
                          workgroup_index(w.x - 1, w.y - 1) == (int64_t)w.x * w.y - 1;
        if (!fits || !covers || !line) {
            std::fprintf(stderr, "%lld: %u x %u\n", (long long)n, w.x, w.y);
            ++fails;
        }
    }
    if (fails) return 1;
    std::puts("ok");
    return 0;
}
