// Writing keys and values into the paged cache and reading them back (gfx950), and the talker's projection pass that ends in it.
//
// Both directions are bound by the bytes they move; nothing is reused.  16 x 8192 tokens of 8 heads (d = 128) between bf16 tensors and int8 pages:
// written in 145 us (4.3 TB/s read + written), read back in 130 us (4.8; a large copy reaches 4.89).  Writing, a lane owns 16 elements: loads may come in pieces (a
// line's other pieces are in the cache by then), stores should not, and 16 codes leave as 16 bytes; two neighbouring lanes hold a
// block of 32 and share its largest element with one lane swap.  Reading back, a lane owns 16 bytes of the caller's row, so that a
// wave's store is contiguous (84 MB of f32: 26 us with 64-byte pieces per lane, 16 us so).  A thread has two or four rows in flight;
// a block of threads covers as many heads as it has rows, so that it stays within neighbouring rows of the caller's tensor.
#include "kv_device.hpp"

#include <algorithm>

namespace qtts {

template <typename T, bool WRITE>
constexpr int kv_move_elems() { return WRITE ? 16 : 16 / (int)sizeof(T); }  // elements a lane owns
template <bool WRITE>
constexpr int kv_move_rows() { return WRITE ? 2 : 4; }                      // rows a thread has in flight

template <int CTRL>
__device__ __forceinline__ unsigned dpp_max(unsigned v) {
    return max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ void load_piece(const bf16_t* p, float (&x)[8]) { load8(p, x); }
__device__ __forceinline__ void load_piece(const float* p, float (&x)[4]) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
}
__device__ __forceinline__ void load_piece(const bf16_t* p, float (&x)[4]) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    x[0] = __uint_as_float(v.x << 16); x[1] = __uint_as_float(v.x & 0xffff0000u);
    x[2] = __uint_as_float(v.y << 16); x[3] = __uint_as_float(v.y & 0xffff0000u);
}
__device__ __forceinline__ void load_piece(const bf16_t* p, float (&x)[16]) {
    float a[8], b[8];
    load8(p, a);
    load8(p + 8, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) { x[i] = a[i]; x[8 + i] = b[i]; }
}
__device__ __forceinline__ void load_piece(const float* p, float (&x)[16]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<float4*>(x + 4 * i) = *reinterpret_cast<const float4*>(p + 4 * i);
}
__device__ __forceinline__ void store_piece(bf16_t* p, const float (&x)[16]) {
#pragma unroll
    for (int i = 0; i < 16; i += 8)
        *reinterpret_cast<u32x4_t*>(p + i) = u32x4_t{pack_bf16(x[i], x[i + 1]), pack_bf16(x[i + 2], x[i + 3]), pack_bf16(x[i + 4], x[i + 5]), pack_bf16(x[i + 6], x[i + 7])};
}
__device__ __forceinline__ void store_piece(bf16_t* p, const float (&x)[8]) {
    *reinterpret_cast<u32x4_t*>(p) = u32x4_t{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7])};
}
__device__ __forceinline__ void store_piece(float* p, const float (&x)[4]) { *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]); }
__device__ __forceinline__ void store_piece(bf16_t* p, const float (&x)[4]) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
}

// grid: x = sequence, y = tokens, z = (keys | values) x heads; a.head_shift: log2 of the heads a block covers
template <typename T, int FMT, int D, bool WRITE>
__global__ __launch_bounds__(256) void kv_move_kernel(KvMoveArgs a) {
    constexpr int EPT = kv_move_elems<T, WRITE>(), LPR = D / EPT, RPB = 256 / LPR, U = kv_move_rows<WRITE>();  // lanes per row, rows per pass
    const KvSeq s = kv_seq(a.b, blockIdx.x);
    const int zh = (int)gridDim.z >> 1, which = (int)blockIdx.z >= zh, sub = threadIdx.x % LPR;
    const int rib = threadIdx.x / LPR, g = (((int)blockIdx.z - (which ? zh : 0)) << a.head_shift) + (rib & ((1 << a.head_shift) - 1));
    const int tpp = RPB >> a.head_shift;  // tokens per pass
    if (g >= a.kv.nkv) return;            // uniform over a row's lanes
    const long ts = which ? a.v_token_stride : a.k_token_stride, hs = which ? a.v_head_stride : a.k_head_stride;
    const T* src = (const T*)(which ? a.v_in : a.k_in) + (long)g * hs + sub * EPT;
    T* dst = (T*)(which ? a.v_out : a.k_out) + (long)g * hs + sub * EPT;
    for (int i0 = (int)blockIdx.y * tpp * U + (rib >> a.head_shift); i0 < s.n; i0 += (int)gridDim.y * tpp * U) {
        int page[U];
        float x[U][EPT];
        size_t row[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int i = i0 + k * tpp, pos = s.ctx - s.n + i;
            page[k] = i < s.n && pos >= 0 ? kv_page(a.kv, s.row, pos) : -1;
            if constexpr (WRITE) load_piece(src + (long)(s.t0 + min(i, s.n - 1)) * ts, x[k]);
        }
        if constexpr (!WRITE) {
#pragma unroll
            for (int k = 0; k < U; ++k) {
                // holes and rows past the end read page 0, which is there, and drop it
                row[k] = kv_row(a.kv, max(page[k], 0), which, g, s.ctx - s.n + i0 + k * tpp);
                if constexpr (FMT == KV_BF16) {
                    load_piece((const bf16_t*)a.kv.codes + row[k] * D + sub * EPT, x[k]);
                } else {
                    const unsigned char* cp = a.kv.codes + row[k] * D + sub * EPT;
                    const float sc = kv_scale(a.kv.scales[row[k] * (D / KV_BLOCK) + sub * EPT / KV_BLOCK]);
                    if constexpr (EPT == 8) {
                        const uint2 c = *reinterpret_cast<const uint2*>(cp);
                        kv_decode4<FMT>(c.x, sc, x[k]);
                        kv_decode4<FMT>(c.y, sc, x[k] + 4);
                    } else {
                        kv_decode4<FMT>(*reinterpret_cast<const unsigned*>(cp), sc, x[k]);
                    }
                }
            }
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int i = i0 + k * tpp;
            if constexpr (WRITE) {
                unsigned m = 0;
#pragma unroll
                for (int e = 0; e < EPT; ++e) m = max(m, __float_as_uint(x[k][e]) & 0x7fffffffu);
                if constexpr (FMT != KV_BF16) m = dpp_max<0xb1>(m);  // the other half of the block: lane ^ 1
                if (page[k] < 0) continue;
                row[k] = kv_row(a.kv, page[k], which, g, s.ctx - s.n + i);
                if constexpr (FMT == KV_BF16) {
                    store_piece((bf16_t*)a.kv.codes + row[k] * D + sub * EPT, x[k]);
                } else {
                    const bool bad = m >= 0x7f800000u;
                    const int ex = bad ? kv_bad_exp<FMT>() : kv_scale_exp<FMT>(m);
                    const float inv = __uint_as_float((unsigned)(254 - (bad ? 127 : ex)) << 23);
                    unsigned char* cp = a.kv.codes + row[k] * D + sub * EPT;
                    u32x4_t c;
#pragma unroll
                    for (int e = 0; e < 4; ++e) c[e] = bad ? kv_bad_codes<FMT>() : kv_encode4<FMT>(x[k] + 4 * e, inv);
                    *reinterpret_cast<u32x4_t*>(cp) = c;
                    if (sub % (KV_BLOCK / EPT) == 0) a.kv.scales[row[k] * (D / KV_BLOCK) + sub * EPT / KV_BLOCK] = (unsigned char)ex;
                }
            } else if (i < s.n) {
                if (page[k] < 0) {
#pragma unroll
                    for (int e = 0; e < EPT; ++e) x[k][e] = 0.f;
                }
                store_piece(dst + (long)(s.t0 + i) * ts, x[k]);
            }
        }
    }
}

template <bool WRITE>
static void launch_kv_move(hipStream_t st, int dtype, KvMoveArgs a) {
    if (a.b.n_seq == 0 || a.b.n_tokens == 0 || a.b.max_new == 0) return;
    const int rpb = 256 / (a.kv.d / (WRITE ? 16 : 16 / (int)dtype_size(dtype)));  // rows per pass
    a.head_shift = 0;
    while ((2 << a.head_shift) <= rpb && (1 << a.head_shift) < a.kv.nkv) ++a.head_shift;
    const long tokens = (long)(rpb >> a.head_shift) * kv_move_rows<WRITE>(), heads = (a.kv.nkv + (1 << a.head_shift) - 1) >> a.head_shift;
    const dim3 grid((unsigned)a.b.n_seq, (unsigned)std::min<long>((a.b.max_new + tokens - 1) / tokens, 65535), (unsigned)(2 * heads));
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
// over half a wave.  Latency, not bytes: 64 tokens of 16 + 2 x 8 heads take 4.8 us (as the same pass over a bf16 cache does), 3264 prompt tokens 31 us.
struct KvPostArgs {
    QkvPostArgs p;
    KvLayer kv;
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
        float* q = a.q_out + (long)m * a.nh * d + (long)hi * d;
        q[i] = x1;
        q[i + half] = x2;
    } else {
        const int g = is_k ? hi - a.nh : hi - a.nh - a.nkv;
        const int page = kv_page(args.kv, t.row, t.pos);
        if (page < 0) return;
        const size_t row = kv_row(args.kv, page, is_k ? 0 : 1, g, t.pos);
        kv_store_block<FMT>(args.kv, row, i, x1);
        kv_store_block<FMT>(args.kv, row, i + half, x2);
    }
}
void launch_kv_qkv_post(hipStream_t st, const QkvPostArgs& a, const KvLayer& kv) {
    QTTS_CHECK(a.d == 64 || a.d == 128, ERR_SHAPE, "kv qkv_post: head_dim must be 64 or 128");
    QTTS_CHECK(a.M >= 1 && a.nh >= 1 && a.nkv >= 1 && kv.d == a.d && kv.nkv == a.nkv && a.toks, ERR_SHAPE, "kv qkv_post: bad shape");
    const KvPostArgs args{a, kv};
    const dim3 grid((unsigned)a.M, (unsigned)(a.nh + 2 * a.nkv));
    if (kv.format == KV_E4M3) kv_launch(kv_qkv_post_kernel<KV_E4M3>, grid, dim3(64), st, args);
    else if (kv.format == KV_INT8) kv_launch(kv_qkv_post_kernel<KV_INT8>, grid, dim3(64), st, args);
    else throw Error(ERR_BAD_ARG, "kv qkv_post: the cache must be in 8 bits");
}

}  // namespace qtts
