// Host side of the key/value cache handle (qtts_kv_*): allocation, and the checks that make every access of the kernels stay in
// bounds whatever the device arrays of a batch hold.
#include "generate.hpp"
#include "kv_index.hpp"


namespace qtts {

struct KvCache {
    Ctx* ctx = nullptr;
    int layers = 0, pages = 0, page_tokens = 0, nkv = 0, d = 0, format = 0;
    DevBuf codes, scales;
    size_t rows() const { return (size_t)pages * 2 * nkv * page_tokens; }  // head rows of a layer
    KvLayer layer(int l, const qtts_kv_batch& b) const {
        KvLayer k{};
        k.codes = codes.as<unsigned char>() + (size_t)l * rows() * d * kv_elem_size(format);
        k.scales = format == KV_BF16 ? nullptr : scales.as<unsigned char>() + (size_t)l * rows() * (d / KV_BLOCK);
        k.format = format;
        k.nkv = nkv;
        k.d = d;
        k.page_shift = __builtin_ctz((unsigned)page_tokens);
        k.n_pages = pages;
        k.max_pages = b.max_pages;
        k.page_table = b.page_table;
        return k;
    }
};

// The calls run on the cache's GPU and leave the caller's current device as it was.
struct DeviceScope {
    int before = 0;
    bool changed = false;
    explicit DeviceScope(int device) {
        QTTS_HIP(hipGetDevice(&before));
        if (before != device) {
            QTTS_HIP(hipSetDevice(device));
            changed = true;
        }
    }
    ~DeviceScope() {
        if (changed) (void)hipSetDevice(before);
    }
};

KvCache* kv_open(Ctx* ctx, const qtts_kv_config& c) {
    QTTS_CHECK(c.format == KV_BF16 || c.format == KV_E4M3 || c.format == KV_INT8, ERR_BAD_ARG, "kv cache: format must be QTTS_KV_BF16, QTTS_KV_E4M3 or QTTS_KV_INT8");
    QTTS_CHECK(c.head_dim == 64 || c.head_dim == 128, ERR_SHAPE, "kv cache: head_dim must be 64 or 128");
    QTTS_CHECK(c.page_tokens >= 16 && c.page_tokens <= 1024 && (c.page_tokens & (c.page_tokens - 1)) == 0, ERR_SHAPE,
               "kv cache: page_tokens must be a power of two from 16 to 1024");
    QTTS_CHECK(c.layers >= 1 && c.pages >= 1 && c.kv_heads >= 1 && c.kv_heads <= 1024, ERR_SHAPE, "kv cache: layers, pages and kv_heads must be positive (at most 1024 kv_heads)");
    QTTS_CHECK((double)c.layers * c.pages * 2 * c.kv_heads * c.page_tokens * c.head_dim < 9e15, ERR_OOM, "kv cache: too large");
    std::unique_ptr<KvCache> k(new KvCache());
    k->ctx = ctx;
    k->layers = c.layers; k->pages = c.pages; k->page_tokens = c.page_tokens; k->nkv = c.kv_heads; k->d = c.head_dim; k->format = c.format;
    DeviceScope dev(ctx->device);
    const size_t n = (size_t)c.layers * k->rows();
    k->codes.alloc(n * c.head_dim * kv_elem_size(c.format));
    QTTS_HIP(hipMemsetAsync(k->codes.p, 0, k->codes.bytes, ctx->stream));
    if (c.format != KV_BF16) {
        k->scales.alloc(n * (c.head_dim / KV_BLOCK));
        QTTS_HIP(hipMemsetAsync(k->scales.p, 0, k->scales.bytes, ctx->stream));
    }
    QTTS_HIP(hipStreamSynchronize(ctx->stream));
    return k.release();
}

void kv_close(KvCache* k) {
    if (!k) return;
    try {
        DeviceScope dev(k->ctx->device);
        delete k;
    } catch (...) {  // the runtime is shutting down
    }
}

int64_t kv_bytes(const KvCache& k) { return (int64_t)(k.codes.bytes + k.scales.bytes); }

static KvBatch check_batch(const KvCache& k, int layer, const qtts_kv_batch& b) {
    QTTS_CHECK(layer >= 0 && layer < k.layers, ERR_BAD_ARG, "kv cache: no such layer");
    QTTS_CHECK(b.n_seq >= 0 && b.n_tokens >= 0 && b.max_new >= 0 && b.max_ctx >= 0 && b.max_pages >= 0, ERR_BAD_ARG, "kv cache: negative size in the batch");
    QTTS_CHECK(b.n_seq == 0 || (b.q_start && b.ctx_len), ERR_BAD_ARG, "kv cache: the batch lacks q_start or ctx_len");
    QTTS_CHECK(b.n_seq == 0 || b.max_pages == 0 || b.page_table, ERR_BAD_ARG, "kv cache: the batch lacks a page table");
    QTTS_CHECK((int64_t)b.max_ctx <= (int64_t)b.max_pages * k.page_tokens, ERR_SHAPE, "kv cache: max_ctx exceeds max_pages pages");
    QTTS_CHECK(b.max_ctx <= 1 << 29 && b.max_new <= 1 << 24 && b.n_tokens <= 1 << 30, ERR_SHAPE, "kv cache: batch too large");
    QTTS_CHECK((int64_t)b.n_seq * k.nkv < 1 << 23, ERR_SHAPE, "kv cache: too many sequences");
    return KvBatch{b.n_seq, b.n_tokens, b.max_new, b.max_ctx, b.q_start, b.ctx_len, 1, 0, nullptr};
}

// `n` rows of `heads` x d elements of `es` bytes: 16-byte accesses; an output's rows may not overlap
static KvRowsAt check_rows(const void* p, int64_t n, int64_t heads, int64_t d, int64_t ts, int64_t hs, int64_t es, bool output, const char* what) {
    const std::string name(what);
    QTTS_CHECK(p, ERR_BAD_ARG, name + ": null tensor");
    if (n <= 1) ts = 0;  // the stride of a single token or head is not used
    if (heads == 1) hs = 0;
    QTTS_CHECK(((uintptr_t)p & 15) == 0 && ts * es % 16 == 0 && hs * es % 16 == 0, ERR_BAD_ARG, name + ": pointer and strides must be multiples of 16 bytes");
    QTTS_CHECK(ts >= 0 && hs >= 0 && ts < (int64_t)1 << 40 && hs < (int64_t)1 << 40, ERR_BAD_ARG, name + ": stride out of range");
    if (output)
        QTTS_CHECK((heads == 1 || hs >= d) && (n <= 1 || ts >= d) && (ts >= (heads - 1) * hs + d || (__int128)hs >= (__int128)(n - 1) * ts + d || n <= 1 || heads == 1), ERR_BAD_ARG,
                   name + ": rows of an output overlap");
    return KvRowsAt{(int64_t)(uintptr_t)p, ts * es, hs * es};
}

static void kv_move(const KvCache& k, int layer, const qtts_kv_batch& b, const qtts_kv_rows& r, hipStream_t st, bool write) {
    KvMoveArgs a{};
    a.b = check_batch(k, layer, b);
    QTTS_CHECK(r.dtype == F32 || r.dtype == BF16, ERR_BAD_ARG, "kv cache: keys and values must be QTTS_F32 or QTTS_BF16");
    if (b.n_seq == 0 || b.n_tokens == 0 || b.max_new == 0) return;
    const int64_t es = (int64_t)dtype_size(r.dtype);
    const KvRowsAt kr = check_rows(r.k, b.n_tokens, k.nkv, k.d, r.k_token_stride, r.k_head_stride, es, !write, "kv cache: k");
    const KvRowsAt vr = check_rows(r.v, b.n_tokens, k.nkv, k.d, r.v_token_stride, r.v_head_stride, es, !write, "kv cache: v");
    QTTS_CHECK(write || r.k != r.v, ERR_BAD_ARG, "kv cache: k and v are read into one tensor");
    QTTS_CHECK(write || !kv_rows_overlap(kr, vr, b.n_tokens, k.nkv, k.d * es), ERR_BAD_ARG, "kv cache: k and v are read into rows that overlap");
    a.kv = k.layer(layer, b);
    a.k_in = r.k; a.v_in = r.v; a.k_out = r.k; a.v_out = r.v;
    a.k_token_stride = r.k_token_stride; a.k_head_stride = r.k_head_stride;
    a.v_token_stride = r.v_token_stride; a.v_head_stride = r.v_head_stride;
    DeviceScope dev(k.ctx->device);
    if (write) launch_kv_write(st, r.dtype, a);
    else launch_kv_read(st, r.dtype, a);
}
void kv_write(const KvCache& k, int layer, const qtts_kv_batch& b, const qtts_kv_rows& r, hipStream_t st) { kv_move(k, layer, b, r, st, true); }
void kv_read(const KvCache& k, int layer, const qtts_kv_batch& b, const qtts_kv_rows& r, hipStream_t st) { kv_move(k, layer, b, r, st, false); }

static KvAttendPlan check_plan(const KvCache& k, const qtts_kv_batch& b, const KvBatch& kb, int n_heads, int window) {
    QTTS_CHECK(n_heads >= 1 && n_heads % k.nkv == 0 && n_heads <= 1 << 16, ERR_SHAPE, "kv attend: query heads must be a multiple of the cache's kv heads");
    QTTS_CHECK(window >= 0, ERR_BAD_ARG, "kv attend: window must be 0 (none) or positive");
    const KvAttendPlan p = kv_attend_plan(k.layer(0, b), kb, n_heads, window >= b.max_ctx ? 0 : window);
    QTTS_CHECK(p.tiles <= 65535, ERR_SHAPE, "kv attend: too many new tokens in one sequence: cut them into several calls");
    return p;
}

int64_t kv_attend_workspace(const KvCache& k, const qtts_kv_batch& b, int n_heads, int window) {
    const KvBatch kb = check_batch(k, 0, b);
    if (b.n_seq == 0 || b.n_tokens == 0 || b.max_new == 0) return 0;
    return (int64_t)check_plan(k, b, kb, n_heads, window).ws_bytes;
}

void kv_attend(const KvCache& k, int layer, const qtts_kv_batch& b, const qtts_kv_attend_args& r, hipStream_t st) {
    KvAttendArgs a{};
    a.b = check_batch(k, layer, b);
    QTTS_CHECK(r.scale > 0.f && r.scale <= 1e30f, ERR_BAD_ARG, "kv attend: scale must be positive and at most 1e30");
    if (b.n_seq == 0 || b.n_tokens == 0 || b.max_new == 0) {
        QTTS_CHECK(r.n_heads >= 1 && r.n_heads % k.nkv == 0, ERR_SHAPE, "kv attend: query heads must be a multiple of the cache's kv heads");
        return;
    }
    const KvAttendPlan p = check_plan(k, b, a.b, r.n_heads, r.window);
    const KvRowsAt qr = check_rows(r.q, b.n_tokens, r.n_heads, k.d, r.q_token_stride, r.q_head_stride, 2, false, "kv attend: q");
    const KvRowsAt outr = check_rows(r.out, b.n_tokens, r.n_heads, k.d, r.out_token_stride, r.out_head_stride, 2, true, "kv attend: out");
    const bool in_place = qr.at == outr.at && qr.token == outr.token && qr.head == outr.head;
    QTTS_CHECK(in_place || !kv_rows_overlap(qr, outr, b.n_tokens, r.n_heads, k.d * 2), ERR_BAD_ARG,
               "kv attend: out overlaps q without being it, with the same strides");
    QTTS_CHECK(p.ws_bytes == 0 || (r.workspace && ((uintptr_t)r.workspace & 15) == 0 && r.workspace_bytes >= (int64_t)p.ws_bytes), ERR_BAD_ARG,
               "kv attend: the workspace is smaller than qtts_kv_attend_workspace asks for, or not aligned to 16 bytes");
    a.kv = k.layer(layer, b);
    a.q = r.q; a.q_token_stride = r.q_token_stride; a.q_head_stride = r.q_head_stride;
    a.out = r.out; a.out_token_stride = r.out_token_stride; a.out_head_stride = r.out_head_stride;
    a.nh = r.n_heads;
    a.scale = r.scale;
    a.window = r.window >= b.max_ctx ? 0 : r.window;
    a.ws = (float*)r.workspace;
    DeviceScope dev(k.ctx->device);
    launch_kv_attend(st, a, p);
}

}  // namespace qtts
