// Host run of the cache kernels' index functions (csrc/kv_index.hpp) on arrays that hold anything: prints "ok" when no row, page
// table entry, cache row or part of the workspace that a kernel would touch lies outside its buffer.
#include <cstdlib>
#include <random>
#include <vector>

#include "kv_index.hpp"

using namespace qtts;

#define NEED(c)                                                  \
    do {                                                         \
        if (!(c)) {                                              \
            std::printf("outside: %s (case %d)\n", #c, trial);   \
            return 1;                                            \
        }                                                        \
    } while (0)

template <int TR>
static int tiles(const KvAttendArgs& a, int trial) {
    for (int pair = 0; pair < a.b.n_seq * a.kv.nkv; ++pair)
        for (int tile = 0; tile < a.tiles; ++tile)
            for (int part = 0; part < a.splits; ++part) {
                const KvTile t = kv_tile<TR>(a, pair, tile, part);
                if (!t.live) continue;
                NEED(t.rows <= a.tiles * TR && t.parts >= 1 && t.parts <= a.splits && t.s0 >= 0 && t.s0 % 16 == 0 && t.s1 <= a.b.max_ctx);
                if (part + 1 == t.parts && t.k_end > 0) NEED(t.s1 == t.k_end);
                for (int row = t.row0; row < t.rows && row < t.row0 + TR; ++row)
                    NEED(t.s.t0 + row / t.G >= 0 && t.s.t0 + row / t.G < a.b.n_tokens);
                for (int key = t.s0; key < t.s1; key += 16) {
                    const int p = kv_page16(a, t, key);
                    NEED(p >= -1 && p < a.kv.n_pages);
                    NEED(((long)t.s.row * a.kv.max_pages + (key >> a.kv.page_shift)) < (long)a.b.n_seq * a.kv.max_pages);
                    const size_t r = kv_row(a.kv, p < 0 ? 0 : p, 1, t.g, key) + 15;
                    NEED(r < ((size_t)a.kv.n_pages * 2 * a.kv.nkv << a.kv.page_shift));
                }
                if (t.s0 < t.s1) NEED(kv_page16(a, t, (t.s1 + 15) & ~15) == -1);
            }
    return 0;
}

int main() {
    std::mt19937 rng(7);
    auto in = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
    for (int trial = 0; trial < 4000; ++trial) {
        const int n = in(1, 4), max_pages = in(1, 5), shift = in(4, 6), big = 0x7fffffff;
        KvAttendArgs a{};
        a.kv.nkv = in(1, 3);
        a.kv.d = 64;
        a.kv.page_shift = shift;
        a.kv.n_pages = in(1, 6);
        a.kv.max_pages = max_pages;
        std::vector<int> start(n + 1), ctx(n), table(n * max_pages);
        auto any = [&](int most) { const int k = in(0, 5); return k == 0 ? big : k == 1 ? -big - 1 : k == 2 ? -1 : in(0, most); };
        for (int& x : start) x = any(40);
        for (int& x : ctx) x = any(max_pages << shift);
        for (int& x : table) x = any(a.kv.n_pages);
        a.kv.page_table = table.data();
        a.b = KvBatch{n, in(1, 40), in(1, 40), in(0, max_pages << shift), start.data(), ctx.data(), 1, 0, nullptr};
        a.nh = a.kv.nkv * in(1, 9);
        a.window = in(0, 2) ? 0 : in(1, 100);
        const KvAttendPlan p = kv_attend_plan(a.kv, a.b, a.nh, a.window);
        a.tiles = p.tiles;
        a.splits = p.splits;
        a.split_len = p.split_len;
        NEED(p.split_len % 128 == 0 && p.splits >= 1 && (p.splits == 1 || p.ws_bytes >= (size_t)n * a.kv.nkv * p.tiles * p.splits * p.tile_rows * 66 * 4));
        if (p.tile_rows == 16 ? tiles<16>(a, trial) : p.tile_rows == 32 ? tiles<32>(a, trial) : tiles<128>(a, trial)) return 1;
        // more parts than this small range would get
        a.splits = in(1, 4);
        a.split_len = ((a.b.max_ctx + a.window + 200) / a.splits + 127) / 128 * 128 + 128;
        if (p.tile_rows == 16 ? tiles<16>(a, trial) : p.tile_rows == 32 ? tiles<32>(a, trial) : tiles<128>(a, trial)) return 1;
        for (int s = 0; s < n; ++s) {
            const KvSeq q = kv_seq(a.b, s);
            NEED(q.t0 >= 0 && q.n >= 0 && q.n <= a.b.max_new && q.t0 + q.n <= a.b.n_tokens && q.ctx >= 0 && q.ctx <= a.b.max_ctx);
        }
    }
    std::puts("ok");
    return 0;
}
