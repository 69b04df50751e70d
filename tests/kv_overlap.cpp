// Host run of the cache's test for rows that share memory (csrc/kv_index.hpp) against sets of bytes: prints "ok".
#include <cstdio>
#include <random>
#include <set>

#include "kv_index.hpp"

using namespace qtts;

static std::set<int64_t> bytes_of(const KvRowsAt& r, int64_t n, int64_t heads, int64_t row) {
    std::set<int64_t> s;
    for (int64_t t = 0; t < n; ++t)
        for (int64_t h = 0; h < heads; ++h)
            for (int64_t i = 0; i < row; ++i) s.insert(r.at + t * r.token + h * r.head + i);
    return s;
}

int main() {
    std::mt19937 rng(3);
    auto in = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
    int shared = 0, apart_inside = 0;
    for (int trial = 0; trial < 30000; ++trial) {
        const int64_t n = in(1, 5), heads = in(1, 4), row = in(1, 4);
        const bool inner_heads = in(0, 1);
        KvRowsAt a{1000, 0, 0};
        if (inner_heads) {
            a.head = in(0, 8);
            a.token = in(0, 30);
        } else {
            a.token = in(0, 8);
            a.head = in(0, 30);
        }
        if (n == 1) a.token = 0;
        if (heads == 1) a.head = 0;
        KvRowsAt b = a;
        b.at += in(-60, 60);
        const bool same = in(0, 4) != 0;
        if (!same && n > 1) b.token = in(0, 30);
        if (!same && heads > 1) b.head = in(0, 30);
        const std::set<int64_t> sa = bytes_of(a, n, heads, row), sb = bytes_of(b, n, heads, row);
        bool truth = false;
        for (int64_t x : sb) truth |= sa.count(x) != 0;
        const bool inside = *sa.begin() <= *sb.rbegin() && *sb.begin() <= *sa.rbegin();
        const bool equal = a.token == b.token && a.head == b.head, got = kv_rows_overlap(a, b, n, heads, row);
        if (got != (equal ? truth : inside) || got != kv_rows_overlap(b, a, n, heads, row)) {
            std::printf("trial %d: n %ld heads %ld row %ld a %ld %ld %ld b %ld %ld %ld: %d, bytes say %d\n", trial, (long)n, (long)heads, (long)row, (long)a.at,
                        (long)a.token, (long)a.head, (long)b.at, (long)b.token, (long)b.head, got, truth);
            return 1;
        }
        shared += truth;
        apart_inside += inside && equal && !truth;
    }
    if (shared < 1000 || apart_inside < 1000) return 1;
    // counts and strides whose product passes 64 bits
    const KvRowsAt far{1 << 20, (int64_t)1 << 42, 256};
    if (!kv_rows_overlap(far, far, 1 << 30, 1 << 16, 256) || kv_rows_overlap(far, KvRowsAt{(1 << 20) - 4096, far.token, 256}, 1 << 30, 16, 256)) return 1;
    std::puts("ok");
    return 0;
}
