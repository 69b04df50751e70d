// Key/value cache with a page table, in the model's 16 bits or in 8, and attention of new tokens over it (k_kv.hip, k_kv_attn.hip;
// host side kv.cpp).  Used through qtts_kv_* (include/qtts.h) and by the talker when its cache is held in 8 bits (generate.cpp).
#pragma once
#include "common.hpp"
#include "kernels.hpp"

namespace qtts {

// How a cache holds a head row (the d elements of one token and kv head).
//   KV_BF16: bf16.
//   KV_E4M3, KV_INT8: blocks of KV_BLOCK consecutive elements with one scale 2^e.  With a = max |x| over the block and top = 448
//   (e4m3) or 127 (int8), e is the smallest integer >= KV_MIN_EXP with a <= top 2^e; element x is held as x 2^-e rounded to
//   nearest even.  The scale is a power of two because then x 2^-e is exact, so that holding x costs one rounding and no more, and
//   code 2^e has at most eight significant bits, so that attention multiplies exactly the held values in bf16.  A block with
//   an infinity or a NaN reads back as NaN throughout.
// Scales are biased exponents, one byte each: d / 32 consecutive bytes a row.
enum KvFormat : int { KV_BF16 = 0, KV_E4M3 = 1, KV_INT8 = 2 };
constexpr int KV_BLOCK = 32, KV_MIN_EXP = -100;
inline size_t kv_elem_size(int format) { return format == KV_BF16 ? 2 : 1; }

// One layer of a cache: [page][k|v][kv_head][slot][d] elements, [page][k|v][kv_head][slot][d / 32] scales.
struct KvLayer {
    unsigned char* codes;
    unsigned char* scales;  // null for KV_BF16
    int format, nkv, d;
    int page_shift;         // log2 of the tokens per page: at least 4, so that 16 keys that start at a multiple of 16 share a page
    int n_pages, max_pages;
    const int* page_table;  // [row][max_pages], entries outside [0, n_pages) are holes
};

// The sequences of a call.  Sequence b's new tokens are rows q_start[b] .. q_start[b + 1] - 1 of the call's tensors and, the last
// ones of the ctx_len[b] tokens the cache holds for it, sit at positions ctx_len[b] - n .. ctx_len[b] - 1.
struct KvBatch {
    int n_seq, n_tokens;    // rows of the call's tensors
    int max_new, max_ctx;   // bounds on a sequence's new tokens and on ctx_len; what exceeds them is cut by the kernels
    const int* q_start;     // [n_seq + 1]; null: one new token per sequence
    const int* ctx_len;
    int ctx_stride, ctx_add;  // sequence b's length is ctx_len[b ctx_stride] + ctx_add
    const int* rows;        // page-table row of each sequence, null: sequence b has row b
};

struct KvMoveArgs {         // write: k, v -> cache; read: cache -> k, v
    KvLayer kv;
    KvBatch b;
    const void *k_in, *v_in;
    void *k_out, *v_out;
    long k_token_stride, k_head_stride, v_token_stride, v_head_stride;  // elements
    int head_shift;          // set by the launchers
};
void launch_kv_write(hipStream_t st, int dtype, const KvMoveArgs& a);
void launch_kv_read(hipStream_t st, int dtype, const KvMoveArgs& a);

// q|k|v projection rows -> per-head RMSNorm, RoPE, queries in f32 and keys / values into the cache (the 8-bit counterpart of
// launch_qkv_post; a.toks name row and position of every token)
void launch_kv_qkv_post(hipStream_t st, const QkvPostArgs& a, const KvLayer& kv);

struct KvAttendArgs {
    KvLayer kv;
    KvBatch b;
    const void* q;          // bf16; f32 if wide
    long q_token_stride, q_head_stride;
    void* out;              // bf16
    long out_token_stride, out_head_stride;
    long out_lo;            // element offset of the output's remainder plane (kernels.hpp), 0 = none
    int nh;
    float scale;
    int window;             // a token sees at most this many keys, its own included; 0 = all
    float* ws;              // partial results when plan.splits > 1
    bool wide;              // f32 queries, which enter as two bf16 pieces as the probabilities do (8-bit formats, tiles of 16 or 128 rows: the talker)
    // filled from the plan
    int tiles, splits, split_len;
};
// How a call is cut: row tiles (a row = one query head of one token; the rows of a sequence and kv head in token order), and
// parts of the key range whose partial results a second launch joins.
constexpr int KV_MAX_PARTS = 256;
struct KvAttendPlan {
    int tile_rows;          // 16 or 32: four waves share the rows, each walks keys of its own; 128: four waves of 32 rows share the keys through LDS
    int tiles;              // row tiles a sequence and kv head can have
    int splits, split_len;  // parts, and keys in each (a multiple of 128)
    size_t ws_bytes;
};
void launch_kv_attend(hipStream_t st, KvAttendArgs a, const KvAttendPlan& p);

// The talker's cache in 8 bits (generate.cpp): rows that own consecutive pages, and the batch of the launch at hand.  The plan does not
// depend on what else is in the batch: single tokens in parts of KV_TALKER_PART keys, prompts in tiles with all of their keys, so that
// a row's result is the same whatever rows it shares a launch with.
constexpr int KV_TALKER_PART = 512;
struct KvStack {
    KvLayer base{};
    size_t layer_rows = 0;  // head rows of a layer
    KvBatch batch{};
    KvAttendPlan plan{};
    float* ws = nullptr;
    KvLayer layer(int l) const {
        KvLayer k = base;
        k.codes += (size_t)l * layer_rows * base.d;
        k.scales += (size_t)l * layer_rows * (base.d / KV_BLOCK);
        return k;
    }
};

// one launch with its error as an exception (hipGetLastError would also report what other code left there)
template <typename A>
void kv_launch(void (*kernel)(A), dim3 grid, dim3 block, hipStream_t st, A args) {
    void* p[] = {&args};
    QTTS_HIP(hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, block, p, 0, st));
}

}  // namespace qtts
