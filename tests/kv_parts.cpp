// Host run of the attention's plan and index functions (csrc/kv_index.hpp) over long contexts, windows and many parts: prints "ok" when the
// parts of every tile fit the launch and the workspace, lie one behind the other and cover exactly the keys that its rows see.
#include <cstdio>
#include <random>
#include <vector>

#include "kv_index.hpp"

using namespace qtts;

static int trial, many, many_windowed, planned;

#define NEED(c)                                                \
    do {                                                       \
        if (!(c)) {                                            \
            std::printf("fails: %s (case %d)\n", #c, trial);   \
            return 1;                                          \
        }                                                      \
    } while (0)

template <int TR>
static int tiles(const KvAttendArgs& a) {
    for (int pair = 0; pair < a.b.n_seq * a.kv.nkv; ++pair)
        for (int tile = 0; tile < a.tiles; ++tile) {
            const KvTile first = kv_tile<TR>(a, pair, tile, 0);
            if (first.row0 >= first.rows) {
                NEED(!first.live);
                continue;
            }
            NEED(first.live && first.parts >= 1 && first.parts <= a.splits);
            // what the rows see, from the definition
            int lo = 0x7fffffff, hi = 0;
            for (int row = first.row0; row < first.rows && row < first.row0 + TR; ++row) {
                const int pos = first.s.ctx - first.s.n + row / first.G;
                if (pos < 0) continue;
                lo = kv_min(lo, a.window ? kv_max(0, pos - a.window + 1) : 0);
                hi = kv_max(hi, pos + 1);
            }
            int at = -1;
            for (int part = 0; part < a.splits; ++part) {
                const KvTile t = kv_tile<TR>(a, pair, tile, part);
                NEED(t.live == (part < first.parts));
                if (!t.live) continue;
                NEED(t.parts == first.parts && t.s0 % 64 == 0 && t.s1 <= a.b.max_ctx);
                if (part) NEED(t.s0 == at && t.s0 < t.s1);
                else NEED(hi == 0 || t.s0 <= lo);
                at = t.s1;
                if (t.s0 < t.s1) {
                    NEED(kv_page16(a, t, t.s0) >= -1 && kv_page16(a, t, (t.s1 + 15) & ~15) == -1);
                    const long last = (long)t.s.row * a.kv.max_pages + ((t.s1 - 1) >> a.kv.page_shift);
                    NEED(last < (long)a.b.n_seq * a.kv.max_pages);
                }
                if (part + 1 < first.parts) NEED(t.s1 == t.s0 + a.split_len);
            }
            if (hi > 0) NEED(at == hi);
            many += first.parts >= 3;
            many_windowed += first.parts >= 3 && a.window;
        }
    return 0;
}
static int any_tile(const KvAttendArgs& a, int tile_rows) { return tile_rows == 16 ? tiles<16>(a) : tile_rows == 32 ? tiles<32>(a) : tiles<128>(a); }

int main() {
    std::mt19937 rng(11);
    auto in = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
    for (trial = 0; trial < 3000; ++trial) {
        const int n = in(1, 3), shift = in(4, 7), most = in(1, 12000), max_pages = (most >> shift) + 1;
        KvAttendArgs a{};
        a.kv.nkv = in(1, 3);
        a.kv.d = in(0, 1) ? 64 : 128;
        a.kv.page_shift = shift;
        a.kv.n_pages = in(1, 6);
        a.kv.max_pages = max_pages;
        std::vector<int> start(n + 1, 0), ctx(n), table(n * max_pages);
        int max_new = 0, max_ctx = 0;
        for (int s = 0; s < n; ++s) {
            ctx[s] = in(0, 3) ? in(1, most) : most;
            const int kind = in(0, 2), fresh = kv_min(ctx[s], kind == 0 ? 1 : kind == 1 ? in(0, 40) : in(0, 700));
            start[s + 1] = start[s] + fresh;
            max_new = kv_max(max_new, fresh);
            max_ctx = kv_max(max_ctx, ctx[s]);
        }
        if (max_new == 0) continue;
        for (int& x : table) x = in(-1, a.kv.n_pages);
        a.kv.page_table = table.data();
        a.b = KvBatch{n, start[n], max_new, max_ctx, start.data(), ctx.data(), 1, 0, nullptr};
        a.nh = a.kv.nkv * in(1, 9);
        const int window = in(0, 1) ? in(1, max_ctx) : 0;
        a.window = window >= max_ctx ? 0 : window;
        const KvAttendPlan p = kv_attend_plan(a.kv, a.b, a.nh, a.window);
        a.tiles = p.tiles;
        a.splits = p.splits;
        a.split_len = p.split_len;
        planned += p.splits >= 3;
        NEED(p.split_len % 128 == 0 && p.splits >= 1 && p.splits <= KV_MAX_PARTS);
        NEED(p.splits == 1 || p.ws_bytes == (size_t)n * a.kv.nkv * p.tiles * p.splits * p.tile_rows * (a.kv.d + 2) * sizeof(float));
        if (any_tile(a, p.tile_rows)) return 1;
        // the shortest parts, as many as the same bound on a tile's keys asks for
        const int span = kv_min(a.b.max_new, (p.tile_rows - 1) / (a.nh / a.kv.nkv) + 2);
        const long keys = a.window ? kv_min(max_ctx, a.window + span + 63) : max_ctx;
        a.split_len = 128;
        a.splits = (int)((keys + 127) / 128);
        if (any_tile(a, p.tile_rows)) return 1;
    }
    if (many < 3000 || many_windowed < 1000 || planned < 200) {
        std::printf("too few cases with parts: %d %d %d\n", many, many_windowed, planned);
        return 1;
    }
    std::puts("ok");
    return 0;
}
