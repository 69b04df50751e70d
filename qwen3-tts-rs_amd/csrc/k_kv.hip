// Writing keys and values into the paged cache and reading them back (gfx950), and the talker's projection pass that ends in it.
//
// A thread owns 16 consecutive elements of a head row, so that 8-bit codes leave and enter in 16-byte accesses; two neighbouring
// lanes hold a block of 32 and share its largest element with one lane swap.  Nothing is reused: both kernels are bound by the
// bytes they move.
#include "kv_device.hpp"

#include <algorithm>

namespace qtts {

__device__ __forceinline__ void load16(const float* p, float (&x)[16]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<float4*>(x + 4 * i) = *reinterpret_cast<const float4*>(p + 4 * i);
}
__device__ __forceinline__ void load16(const bf16_t* p, float (&x)[16]) {
    float a[8], b[8];
    load8(p, a);
    load8(p + 8, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) { x[i] = a[i]; x[8 + i] = b[i]; }
}
template <typename T>
__device__ __forceinline__ void store16(T* p, const float (&x)[16]) {
    float a[8], b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) { a[i] = x[i]; b[i] = x[8 + i]; }
    store8(p, a);
    store8(p + 8, b);
}

// grid: x = sequence, y = pieces of the sequence's rows (strided), z = keys | values
template <typename T, int FMT, int D, bool WRITE>
__global__ __launch_bounds__(256) void kv_move_kernel(KvMoveArgs a) {
    constexpr int LPR = D / 16, RPB = 256 / LPR;  // lanes per row, rows per block
    const KvSeq s = kv_seq(a.b, blockIdx.x);
    const int which = blockIdx.z, sub = threadIdx.x % LPR;
    const long ts = which ? a.v_token_stride : a.k_token_stride, hs = which ? a.v_head_stride : a.k_head_stride;
    const T* src = (const T*)(which ? a.v_in : a.k_in);
    T* dst = (T*)(which ? a.v_out : a.k_out);
    const int nkv = a.kv.nkv;
    const long rows = (long)s.n * nkv;
    for (long r = (long)blockIdx.y * RPB + threadIdx.x / LPR; r < rows; r += (long)gridDim.y * RPB) {
        const int i = (int)(r / nkv), g = (int)(r - (long)i * nkv);
        const int pos = s.ctx - s.n + i;
        const int page = pos >= 0 ? kv_page(a.kv, s.row, pos) : -1;
        const long off = (long)(s.t0 + i) * ts + (long)g * hs + sub * 16;
        if constexpr (WRITE) {
            if (page < 0) continue;  // uniform over the row's lanes
            const size_t row = kv_row(a.kv, page, which, g, pos);
            float x[16];
            load16(src + off, x);
            if constexpr (FMT == KV_BF16) {
                store16((bf16_t*)a.kv.codes + row * D + sub * 16, x);
            } else {
                unsigned m = 0;
#pragma unroll
                for (int e = 0; e < 16; ++e) m = max(m, __float_as_uint(x[e]) & 0x7fffffffu);
                m = max(m, (unsigned)__shfl_xor((int)m, 1, 64));
                const bool bad = m >= 0x7f800000u;
                const int ex = bad ? kv_bad_exp<FMT>() : kv_scale_exp<FMT>(m);
                const float inv = __uint_as_float((unsigned)(254 - (bad ? 127 : ex)) << 23);
                uint4 c;
                c.x = kv_encode4<FMT>(x, inv);
                c.y = kv_encode4<FMT>(x + 4, inv);
                c.z = kv_encode4<FMT>(x + 8, inv);
                c.w = kv_encode4<FMT>(x + 12, inv);
                if (bad) c.x = c.y = c.z = c.w = kv_bad_codes<FMT>();
                *reinterpret_cast<uint4*>(a.kv.codes + row * D + sub * 16) = c;
                if ((sub & 1) == 0) a.kv.scales[row * (D / KV_BLOCK) + (sub >> 1)] = (unsigned char)ex;
            }
        } else {
            float x[16];
            if (page < 0) {
#pragma unroll
                for (int e = 0; e < 16; ++e) x[e] = 0.f;
            } else {
                const size_t row = kv_row(a.kv, page, which, g, pos);
                if constexpr (FMT == KV_BF16) {
                    load16((const bf16_t*)a.kv.codes + row * D + sub * 16, x);
                } else {
                    const uint4 c = *reinterpret_cast<const uint4*>(a.kv.codes + row * D + sub * 16);
                    const float sc = kv_scale(a.kv.scales[row * (D / KV_BLOCK) + (sub >> 1)]);
                    kv_decode4<FMT>(c.x, sc, x);
                    kv_decode4<FMT>(c.y, sc, x + 4);
                    kv_decode4<FMT>(c.z, sc, x + 8);
                    kv_decode4<FMT>(c.w, sc, x + 12);
                }
            }
            store16(dst + off, x);
        }
    }
}

template <bool WRITE>
static void launch_kv_move(hipStream_t st, int dtype, const KvMoveArgs& a) {
    if (a.b.n_seq == 0 || a.b.n_tokens == 0) return;
    const int rpb = 256 / (a.kv.d / 16);
    const long pieces = ((long)a.b.max_new * a.kv.nkv + rpb - 1) / rpb;
    const dim3 grid((unsigned)a.b.n_seq, (unsigned)std::min<long>(pieces, 65535), 2);
#define QTTS_KV_MOVE(T, FMT, DD) \
    if (a.kv.format == FMT && a.kv.d == DD) return kv_launch(kv_move_kernel<T, FMT, DD, WRITE>, grid, dim3(256), st, a);
#define QTTS_KV_MOVE_T(T)           \
    QTTS_KV_MOVE(T, KV_BF16, 64)    \
    QTTS_KV_MOVE(T, KV_E4M3, 64)    \
    QTTS_KV_MOVE(T, KV_INT8, 64)    \
    QTTS_KV_MOVE(T, KV_BF16, 128)   \
    QTTS_KV_MOVE(T, KV_E4M3, 128)   \
    QTTS_KV_MOVE(T, KV_INT8, 128)
    if (dtype == BF16) {
        QTTS_KV_MOVE_T(bf16_t)
    } else {
        QTTS_KV_MOVE_T(float)
    }
#undef QTTS_KV_MOVE_T
#undef QTTS_KV_MOVE
    throw Error(ERR_SHAPE, "kv cache: head_dim must be 64 or 128");
}
void launch_kv_write(hipStream_t st, int dtype, const KvMoveArgs& a) { launch_kv_move<true>(st, dtype, a); }
void launch_kv_read(hipStream_t st, int dtype, const KvMoveArgs& a) { launch_kv_move<false>(st, dtype, a); }

// Split-K combine, bias, per-head RMSNorm and RoPE as in qkv_post_kernel (k_attn.hip), one wave per (token, head); a lane holds
// the rotation pair (i, i + d / 2), so a block of 32 elements lies in 32 neighbouring lanes and its largest element is a reduction
// over half a wave.
struct KvPostArgs {
    QkvPostArgs p;
    KvLayer kv;
    bf16_t* q;
};
__device__ __forceinline__ unsigned half_wave_max(unsigned v) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v = max(v, (unsigned)__shfl_xor((int)v, off, 64));
    return v;
}
template <int FMT>
__device__ __forceinline__ void kv_store_block(const KvLayer& kv, size_t row, int i, float x) {  // lane i % 32 holds element i of its block
    const unsigned mb = half_wave_max(__float_as_uint(x) & 0x7fffffffu);
    const bool bad = mb >= 0x7f800000u;
    const int ex = bad ? kv_bad_exp<FMT>() : kv_scale_exp<FMT>(mb);
    const float v[4] = {x, 0.f, 0.f, 0.f};
    const unsigned c = kv_encode4<FMT>(v, __uint_as_float((unsigned)(254 - (bad ? 127 : ex)) << 23));
    kv.codes[row * kv.d + i] = (unsigned char)(bad ? kv_bad_codes<FMT>() : c);
    if ((i & (KV_BLOCK - 1)) == 0) kv.scales[row * (kv.d / KV_BLOCK) + i / KV_BLOCK] = (unsigned char)ex;
}
template <int FMT>
__global__ __launch_bounds__(64) void kv_qkv_post_kernel(KvPostArgs args) {
    const QkvPostArgs& a = args.p;
    const int m = blockIdx.x, hi = blockIdx.y, lane = threadIdx.x;
    const int d = a.d, half = d >> 1;
    const int ncol = (a.nh + 2 * a.nkv) * d;
    const Tok t = a.toks[m];
    const bool act = lane < half;
    const int i = act ? lane : 0;
    const long col = (long)hi * d + i;
    float x1, x2;
    slab_sum_pair(a.part + (long)m * ncol + col, half, a.KS, a.ks_stride, x1, x2);
    if (a.bias) {
        x1 += a.bias[col];
        x2 += a.bias[col + half];
    }
    const bool is_q = hi < a.nh, is_k = !is_q && hi < a.nh + a.nkv;
    if (is_q || is_k) {
        const float* nw = is_q ? a.q_norm : a.k_norm;
        if (nw) {
            const float ss = wave_sum(act ? x1 * x1 + x2 * x2 : 0.f);
            const float mm = sqrtf(ss / (float)d + a.eps);
            x1 = x1 / mm * nw[i];
            x2 = x2 / mm * nw[i + half];
        }
        const float c = a.cos[(long)t.pos * half + i], s = a.sin[(long)t.pos * half + i];
        const float y1 = x1 * c - x2 * s;
        const float y2 = x1 * s + x2 * c;
        x1 = y1;
        x2 = y2;
    }
    if (!act) return;  // head_dim 64: the upper half of the wave
    if (is_q) {
        bf16_t* q = args.q + (long)m * a.nh * d + (long)hi * d;
        q[i] = from_f32<bf16_t>(x1);
        q[i + half] = from_f32<bf16_t>(x2);
    } else {
        const int g = is_k ? hi - a.nh : hi - a.nh - a.nkv;
        const int page = kv_page(args.kv, t.row, t.pos);
        if (page < 0) return;
        const size_t row = kv_row(args.kv, page, is_k ? 0 : 1, g, t.pos);
        kv_store_block<FMT>(args.kv, row, i, x1);
        kv_store_block<FMT>(args.kv, row, i + half, x2);
    }
}
void launch_kv_qkv_post(hipStream_t st, const QkvPostArgs& a, const KvLayer& kv, void* q_bf16) {
    QTTS_CHECK(a.d == 64 || a.d == 128, ERR_SHAPE, "kv qkv_post: head_dim must be 64 or 128");
    QTTS_CHECK(a.M >= 1 && a.nh >= 1 && a.nkv >= 1 && kv.d == a.d && kv.nkv == a.nkv && a.toks, ERR_SHAPE, "kv qkv_post: bad shape");
    const KvPostArgs args{a, kv, (bf16_t*)q_bf16};
    const dim3 grid((unsigned)a.M, (unsigned)(a.nh + 2 * a.nkv));
    if (kv.format == KV_E4M3) kv_launch(kv_qkv_post_kernel<KV_E4M3>, grid, dim3(64), st, args);
    else if (kv.format == KV_INT8) kv_launch(kv_qkv_post_kernel<KV_INT8>, grid, dim3(64), st, args);
    else throw Error(ERR_BAD_ARG, "kv qkv_post: the cache must be in 8 bits");
}

}  // namespace qtts
