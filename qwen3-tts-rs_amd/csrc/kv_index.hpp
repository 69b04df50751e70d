// Where the kernels of the paged cache read and write: lengths, pages and key ranges out of a batch's arrays.  Compiled for the host
// too, so that a test on the CPU can show that nothing these arrays hold leads outside a buffer.
#pragma once
#include "kv.hpp"

#include <algorithm>
#include <cstdint>

#define QTTS_KV_HD __host__ __device__ __forceinline__

namespace qtts {

QTTS_KV_HD int kv_min(int a, int b) { return a < b ? a : b; }
QTTS_KV_HD int kv_max(int a, int b) { return a > b ? a : b; }
QTTS_KV_HD int kv_clamp(int x, int lo, int hi) { return x < lo ? lo : (x > hi ? hi : x); }

// New tokens [t0, t0 + n) and context length of sequence s.  Lengths come from device memory, where the host cannot check
// them: they are cut to the bounds that the launch was checked for, so that no access leaves a buffer whatever they hold.
struct KvSeq {
    int t0, n, ctx, row;
};
QTTS_KV_HD KvSeq kv_seq(const KvBatch& b, int s) {
    KvSeq q;
    int t0 = s, t1 = s + 1;
    if (b.q_start) {
        t0 = b.q_start[s];
        t1 = b.q_start[s + 1];
    }
    q.t0 = kv_clamp(t0, 0, b.n_tokens);
    q.n = kv_clamp(kv_clamp(t1, q.t0, b.n_tokens) - q.t0, 0, b.max_new);
    q.ctx = kv_clamp(b.ctx_len[(long)s * b.ctx_stride] + b.ctx_add, 0, b.max_ctx);
    q.row = b.rows ? b.rows[s] : s;
    return q;
}
// physical page of a position, -1 = hole
QTTS_KV_HD int kv_page(const KvLayer& kv, int row, int pos) {
    const int p = kv.page_table[(long)row * kv.max_pages + (pos >> kv.page_shift)];
    return (unsigned)p < (unsigned)kv.n_pages ? p : -1;
}
// index of a head row within the layer (its elements start at index * d, its scales at index * d / 32)
QTTS_KV_HD size_t kv_row(const KvLayer& kv, int page, int which, int g, int pos) {
    return (((((size_t)page * 2 + which) * kv.nkv + g)) << kv.page_shift) + (pos & ((1 << kv.page_shift) - 1));
}

// What a block works on: tile `tile` of TR rows of sequence and kv head `pair`, part `part` of its keys.
struct KvTile {
    KvSeq s;
    int g, G, rows;         // rows of the sequence and kv head in all
    int row0;               // first row of the tile
    int p0, p1;             // positions of its first and last token
    int k_begin, k_end;     // keys any of its rows can see
    int s0, s1, parts;      // keys of this part; parts with keys
    bool live;
};
template <int TR>
QTTS_KV_HD KvTile kv_tile(const KvAttendArgs& a, int pair, int tile, int part) {
    KvTile t;
    t.live = false;
    const int b = pair / a.kv.nkv;
    t.g = pair - b * a.kv.nkv;
    t.s = kv_seq(a.b, b);
    t.G = a.nh / a.kv.nkv;
    t.rows = t.s.n * t.G;
    t.row0 = tile * TR;
    if (t.row0 >= t.rows) return t;
    const int first = t.s.ctx - t.s.n;  // negative where the caller claims more new tokens than the sequence has: those see nothing
    t.p0 = first + t.row0 / t.G;
    t.p1 = first + kv_min(t.row0 + TR - 1, t.rows - 1) / t.G;
    t.k_begin = a.window ? kv_max(0, t.p0 - a.window + 1) : 0;
    t.k_end = t.p1 + 1;
    const int base = t.k_begin & ~63;
    t.parts = kv_max(1, (t.k_end - base + a.split_len - 1) / a.split_len);
    t.s0 = base + part * a.split_len;
    t.s1 = kv_min(t.s0 + a.split_len, t.k_end);
    t.live = part < t.parts;
    return t;
}
// page of the keys from `key`, a multiple of 16, up to the next one, -1 = hole or past the part.  Only for parts with keys.  The kernels
// load it a step ahead, one lane per group of 16 keys, and hand it out with a lane read: as an ordinary scalar of the loop it is a
// load and a wait for everything in flight.
QTTS_KV_HD int kv_page16(const KvAttendArgs& a, const KvTile& t, int key) {
    const int p = kv_page(a.kv, t.s.row, kv_min(key, t.s1 - 1));
    return key < t.s1 ? p : -1;
}

// ---- host
// Rows [n][heads] of `row` bytes, strides in bytes (0 for a dimension of one).  The two of a question have the same n, heads and row.
struct KvRowsAt {
    int64_t at, token, head;
};
// Do the rows of a and b share a byte?  With equal strides exactly; with others, rows between each other's first and last byte count as
// shared (row i of one may then meet row j of the other in more ways than are worth telling apart).
inline bool kv_rows_overlap(const KvRowsAt& a, const KvRowsAt& b, int64_t n, int64_t heads, int64_t row) {
    typedef __int128 wide;  // strides and counts are the caller's: their product may pass 64 bits
    const auto end = [&](const KvRowsAt& r) { return (wide)r.at + (wide)(n - 1) * r.token + (wide)(heads - 1) * r.head + row; };
    if (b.at >= end(a) || a.at >= end(b)) return false;
    if (a.token != b.token || a.head != b.head) return true;
    // the difference of two rows' addresses is i token + j head with |i| < n, |j| < heads: for each j the two nearest i
    const bool swap = heads > n;  // walk the shorter dimension
    const wide walk = swap ? a.token : a.head, step = swap ? a.head : a.token, delta = (wide)b.at - a.at;
    const int64_t nw = swap ? n : heads, ns = swap ? heads : n;
    for (int64_t j = 1 - nw; j < nw; ++j) {
        const wide r = delta - j * walk;
        wide i = step ? r / step : 0;
        if (step && r < 0 && i * step != r) --i;  // floor
        for (int k = 0; k < 2; ++k, ++i) {
            const wide c = i < 1 - ns ? 1 - ns : (i > ns - 1 ? ns - 1 : i), x = r - c * step;
            if (x < row && -x < row) return true;
        }
    }
    return false;
}

inline KvAttendPlan kv_attend_plan(const KvLayer& kv, const KvBatch& b, int nh, int window) {
    KvAttendPlan p{};
    const long rows = (long)b.max_new * (nh / kv.nkv);
    // Every tile walks, and in 8 bits converts, its keys by itself; a 128-row tile is slow to start and partly empty.  Measured in us (d = 128) with
    // tiles of 16 / 32 / 128 rows: 16 rows of 128 x 8192 int8 keys 57 64 71, bf16 104 105 101, of 512 x 2000 int8 48 59 65, of 8 x 300 bf16
    // 11 12 12; 20 rows 91 65 69, 127 106 102, 86 60 64, 12 12 12; 48 rows 152 114 78, 253 123 105, 123 108 72, 12 14 13.
    p.tile_rows = rows <= 16 ? 16 : rows <= 32 ? 32 : 128;
    p.tiles = (int)std::min<long>((rows + p.tile_rows - 1) / p.tile_rows, 65536);  // the grid's y: callers refuse more than 65535
    // keys the tile with the most of them can see
    const long span_tokens = std::min<long>(b.max_new, (p.tile_rows - 1) / (nh / kv.nkv) + 2);
    const long keys = std::max<long>(1, window ? std::min<long>(b.max_ctx, window + span_tokens + 63) : b.max_ctx);
    const long units = (long)b.n_seq * kv.nkv * p.tiles;
    p.splits = 1;
    if (p.tile_rows != 128) {
        // Two blocks a CU fill it, and a part of fewer than 256 keys is mostly start and join.  Measured with targets of 512 / 768 / 1024
        // blocks: 12 x 30011 int8 keys 130 / 140 / 147 us, 32 x 2047 with five tokens 34.7 / 33.7 / 36.3 us, 7 x 20011 bf16 keys 23.8 / 26.8 /
        // 26.9 us; parts of at least 512 keys: 25.5 us for the last.  The grid keeps a pair on one XCD (launch_kv_attend), so with fewer than
        // eight pairs as many XCDs have these blocks and the others none: 30000 bf16 keys of 1 / 2 / 4 / 8 pairs all take 30 to 34 us.
        const long want = std::max<long>(1, 512 / std::max<long>(units, 1)), most = std::max<long>(1, (keys + 255) / 256);
        p.splits = (int)std::min<long>(std::min(want, most), KV_MAX_PARTS);
    } else {
        // The parts' number with the least time by this account: a CU walks 64 keys with one, two (three at head_dim 64) resident blocks in
        // the microseconds below; a block costs two walks on top; parts cost a launch and their partial results, written and read at 5 TB/s.
        // Measured with 1 / 2 / 4 / 8 parts (d = 128, bf16): 64 tiles of 8192 keys 186 103 66 62 us, 256 of them 233 210 235 279, 384 of them
        // 325 354 359 416, 512 of them 391 429 481 560; 256 tiles of up to 512 keys 20 32 35 35; 512 of up to 4096 110 101 119 134 (the keys a
        // tile of a prompt sees depend on its place, the account takes the most for all).  It takes the blocks as spread over all CUs, which
        // the grid does from eight pairs on: a prompt of 4096 tokens takes 101 / 110 / 114 / 119 us with 1 / 2 / 4 / 8 pairs.
        static constexpr float WALK[2][4] = {{0.f, 1.2f, 1.6f, 2.4f}, {0.f, 1.5f, 2.45f, 0.f}};
        const int most = kv.d == 64 ? 3 : 2;  // resident blocks of a CU
        const float* walk = WALK[kv.d == 64 ? 0 : 1];
        float best = 0.f;
        for (int s = 1; s <= KV_MAX_PARTS; ++s) {
            const long blocks = units * s, full = blocks / (256 * most), rest = blocks % (256 * most);
            if (s > 1 && (keys < 256L * s || blocks > 1024L * most)) break;
            float t = (float)((keys + 64 * s - 1) / (64 * s) + 2) * ((float)full * walk[most] + walk[(rest + 255) / 256]);
            if (s > 1) t += 4.f + (float)blocks * (float)(p.tile_rows * kv.d * 8) / 5e6f;
            if (s == 1 || t < best) {
                best = t;
                p.splits = s;
            }
        }
    }
    p.split_len = (int)(((keys + p.splits - 1) / p.splits + 127) / 128 * 128);
    if (p.splits > 1) p.ws_bytes = (size_t)units * p.splits * p.tile_rows * (kv.d + 2) * sizeof(float);
    return p;
}

}  // namespace qtts
