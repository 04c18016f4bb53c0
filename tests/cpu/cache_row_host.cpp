// Host-side check of csrc/cache_row.h: rows of small paged and unpaged caches against a plain walk.  Prints "ok" and
// exits 0, or prints what failed and exits 1.  Built and run by tests/test_cache_cpu.py.
#include <climits>
#include <cstdio>
#include <vector>

#include "cache_row.h"

#define CHECK(cond)                                                        \
    do {                                                                   \
        if (!(cond)) { std::printf("FAILED line %d: %s\n", __LINE__, #cond); return 1; } \
    } while (0)

int main() {
    const fa::CacheMap dense{nullptr, 0, -1, 0};
    for (int b : {0, 3, 70000})
        for (int r : {0, 1, 4095, INT_MAX}) {
            const fa::CacheRow at = fa::cache_row(dense, b, r);
            CHECK(at.block == b && at.in_block == r);
        }
    for (int shift : {4, 5, 8, 27, 30}) {
        const int page = 1 << shift;
        const int n_pages = 5, stride = 3;
        // sequence 1 has page numbers that name none: negative, just past the pool, INT_MAX
        const std::vector<int> table = {4, 0, 2, -1, n_pages, INT_MAX, 1, INT_MIN, 3};
        const fa::CacheMap m{table.data(), stride, shift, n_pages};
        for (int b = 0; b < 3; b++)
            for (int p = 0; p < stride; p++)
                for (long long in : {0ll, 1ll, (long long)page - 1}) {
                    const long long row = (long long)p * page + in;
                    if (row > INT_MAX) continue;
                    const fa::CacheRow at = fa::cache_row(m, b, (int)row);
                    const int e = table[b * stride + p];
                    CHECK(at.block == (e >= 0 && e < n_pages ? e : -1));
                    CHECK(at.in_block == in);
                }
    }
    const int lens[] = {-5, 0, 7, 99, INT_MAX};
    CHECK(fa::sequence_length(nullptr, 2, 40) == 40);
    CHECK(fa::sequence_length(lens, 0, 40) == 0 && fa::sequence_length(lens, 1, 40) == 0);
    CHECK(fa::sequence_length(lens, 2, 40) == 7 && fa::sequence_length(lens, 3, 40) == 40);
    CHECK(fa::sequence_length(lens, 4, 40) == 40);
    std::printf("ok\n");
    return 0;
}
