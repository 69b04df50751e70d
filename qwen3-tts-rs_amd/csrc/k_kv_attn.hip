// Attention of new tokens over the paged 8- or 16-bit cache (gfx950): prompts, chunks that continue one, drafted tokens, single
// tokens (the talker's decode step: qwen_tts/src/nn/attention/mod.rs:359-472).
//
//   o_ih = sum_j softmax_j(scale q_ih . k_jg) v_jg,   g = h / (heads per kv head),  j <= p_i, j > p_i - window
//
// A row is one query head of one new token; the rows of a sequence and kv head, in token order, are cut into tiles, so any number of
// heads per kv head fills a tile.  Keys are walked once with the running maximum m and sum l of the softmax in f32:
//   S^T = K Q^T   K rows are the A operand, the tile's queries the B operand, so a lane holds scores of one row only and the softmax
//                 needs no more than one or two lane swaps;
//   O^T = V^T P^T the score registers are the B operand as they stand once the keys of a matrix step are numbered in the order in
//                 which the lanes hold them; V^T comes out of a row-major LDS image by transposing reads.
// Rounding: K, V and Q enter exactly (bf16, or codes times a power of two).  P is rounded to bf16 for the second product, at most
// 2^-8 relative per term, as the output itself is afterwards; l is summed from the unrounded f32 values.
// WIDE (the talker over its 8-bit cache): f32 queries and P enter as a bf16 value plus a bf16 remainder, two products each, as over its
// 16-bit cache, so that choosing 8 bits rounds K and V alone; the output has a remainder plane of its own.
// Key ranges are cut into parts where a call has too few tiles to fill the GPU (kv_attend_plan); a second launch joins their (m, l, O).
// A masked key may hold anything: its score is replaced, and its V row meets the products as zero.  Where some rows of a tile see a key
// and others do not, a non-finite V element is taken out of the products and added to the rows that see it one by one.  (An infinity whose
// weight f32 takes for zero, below 2^-126 of the row's largest, may come out as NaN: 0 * infinity.)
#include "kv_device.hpp"

#include <algorithm>

namespace qtts {

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));

template <typename F>
__device__ __forceinline__ float kv_quad_rows(float v, F op) {  // over lanes r, r + 16, r + 32, r + 48, left in all of them
    return fold_rows(fold_halves(v, op), op);
}
__device__ __forceinline__ float fmax2(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ float fadd2(float a, float b) { return a + b; }

// four V rows x 16 columns, transposed: lane 4 q + p of a 16-lane group points at row q, columns 4 p ..; it receives column
// (lane & 15) of the four rows
__device__ __forceinline__ s16x4_t read_tr4(const u16* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)p);
}
__device__ __forceinline__ bf16x8_t join8(s16x4_t a, s16x4_t b) {
    return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}
__device__ __forceinline__ bool bf16_pair_bad(unsigned w) { return ((w & 0x7f80u) == 0x7f80u) | ((w & 0x7f800000u) == 0x7f800000u); }
__device__ __forceinline__ bool bf16x8_bad(u32x4_t w) { return bf16_pair_bad(w.x) | bf16_pair_bad(w.y) | bf16_pair_bad(w.z) | bf16_pair_bad(w.w); }
__device__ __forceinline__ unsigned bf16_pair_clean(unsigned w) {
    if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
    if ((w & 0x7f800000u) == 0x7f800000u) w &= 0xffffu;
    return w;
}
__device__ __forceinline__ u32x4_t bf16x8_clean(u32x4_t w) {
    return u32x4_t{bf16_pair_clean(w.x), bf16_pair_clean(w.y), bf16_pair_clean(w.z), bf16_pair_clean(w.w)};
}
__device__ __forceinline__ u32x4_t keep(u32x4_t w, bool in) { return in ? w : u32x4_t{0u, 0u, 0u, 0u}; }
// eight f32 as bf16 plus bf16 remainder
__device__ __forceinline__ bf16x8_t pack8(const float* f) {
    return __builtin_bit_cast(bf16x8_t, u32x4_t{pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7])});
}
__device__ __forceinline__ bf16x8_t rest8(const float* f, bf16x8_t hi) {
    const u32x4_t w = __builtin_bit_cast(u32x4_t, hi);
    float r[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        r[2 * i] = f[2 * i] - __uint_as_float(w[i] << 16);
        r[2 * i + 1] = f[2 * i + 1] - __uint_as_float(w[i] & 0xffff0000u);
    }
    return pack8(r);
}
// value added to a row that sees a V element: the element if it is not finite (it was taken out of the products), else nothing
__device__ __forceinline__ float bad_only(u16 b) { return (b & 0x7f80u) == 0x7f80u ? bf16_bits_to_f32(b) : 0.f; }

// ---------------------------------------------------------------------------------------------- 16 or 32 rows a tile
// Single tokens and drafts: bound by the bytes of the cache, so keys go from the cache into registers in operand order (a lane's 16 bytes
// of a K row are its share of the A operand), only V passes through LDS for its transpose, and no wave waits for another before the end:
// each walks every fourth group of 32 keys with the next group's loads in flight, and the four results are joined in LDS.  32 rows share
// one walk (and one conversion of 8-bit keys) instead of walking twice.  Measured (d = 128): 12 x 30011 int8 keys of 8 kv heads 124 us with the join = 4.8 TB/s
// (a large copy: 4.89), 64 x 500 e4m3 keys 13 us = 3.9 TB/s, 32 x 2047 int8 keys with five tokens 27 us (+ 5 us of joining), 113 keys of one sequence 6 us,
// of which all is latency; the talker's step (WIDE, 64 x 51 .. 91 e4m3 keys) 8.2 us, 7.7 without the second pieces.  Four waves a SIMD instead of
// three spilled registers and were slower.
template <int FMT, int D, int RG, bool WIDE>
__global__ __launch_bounds__(256, RG == 1 ? 3 : 2) void kv_attend_few_kernel(KvAttendArgs a) {
    constexpr bool Q8 = FMT != KV_BF16;
    constexpr int TR = 16 * RG;                        // a lane holds scores of RG rows, 16 apart
    constexpr int NJ = D / 32, NDT = D / 16;
    constexpr int KLD = Q8 ? D / 64 : D / 32;          // 16-byte loads of a K row per lane
    constexpr int EPP = Q8 ? 16 : 8, PPR = D / EPP;    // V: elements per 16-byte piece, pieces per row
    constexpr int RPI = 64 / PPR, NV = 32 / RPI;       // rows a wave loads at once, loads per 32 rows
    constexpr int LDV = D + 16;                        // rows of the V image 8 banks apart (modulo 64): its reads hit every bank once
    constexpr int LDO = D + 4;
    constexpr int VBYTES = 4 * 32 * LDV * 2, OBYTES = 4 * 16 * LDO * 4;
    __shared__ __attribute__((aligned(16))) unsigned char smem[VBYTES > OBYTES ? VBYTES : OBYTES];
    __shared__ float pm[4][TR], pl[4][TR];

    const int pair = blockIdx.x;
    if (pair >= a.b.n_seq * a.kv.nkv) return;
    const KvTile t = kv_tile<TR>(a, pair, blockIdx.y, blockIdx.z);
    if (!t.live) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, gq = lane >> 4;
    u16* Vs = reinterpret_cast<u16*>(smem) + wave * 32 * LDV;

    // this lane's rows: their key ranges and queries
    int pos[RG], klo[RG];
    bool has[RG];
    bf16x8_t q[RG][NJ], ql[RG][WIDE ? NJ : 1];
#pragma unroll
    for (int rg = 0; rg < RG; ++rg) {
        const int row = t.row0 + 16 * rg + r;
        has[rg] = row < t.rows;
        const int rr = has[rg] ? row : t.row0, tok = rr / t.G, head = t.g * t.G + rr - tok * t.G;
        pos[rg] = t.s.ctx - t.s.n + tok;
        klo[rg] = has[rg] ? (a.window ? pos[rg] - a.window + 1 : 0) : 0x7fffffff;
        const long qat = (long)(t.s.t0 + tok) * a.q_token_stride + (long)head * a.q_head_stride;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int d0 = Q8 ? 64 * (j >> 1) + 16 * gq + 8 * (j & 1) : 32 * j + 8 * gq;
            if constexpr (WIDE) {
                float f[8];
                load8((const float*)a.q + qat + d0, f);
                q[rg][j] = pack8(f);
                ql[rg][j] = rest8(f, q[rg][j]);
            } else {
                q[rg][j] = *reinterpret_cast<const bf16x8_t*>((const u16*)a.q + qat + d0);
            }
        }
    }

    f32x4_t acc[RG][NDT];
    float m[RG], l[RG];
#pragma unroll
    for (int rg = 0; rg < RG; ++rg) {
        m[rg] = -INFINITY;
        l[rg] = 0.f;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) acc[rg][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    const float sc = a.scale * 1.4426950408889634f;  // exponentials to base 2

    u32x4_t kreg[2][KLD], vreg[NV];
    unsigned ksc[2], vsc[NV];
    // a page is the same for all lanes: scalar base, constant lane offsets
    constexpr unsigned ROWB = Q8 ? D : 2 * D;  // bytes of a head row
    const unsigned koff = r * ROWB + gq * 16, voff = (lane / PPR) * ROWB + (lane % PPR) * 16, vsoff = (lane / PPR) * (D / KV_BLOCK) + (lane % PPR) / 2;
    auto load = [&](int kb, const int (&pg)[2]) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            // a hole is read as page 0: in bounds, and what it holds is masked
            const size_t kr = kv_row(a.kv, max(pg[kt], 0), 0, t.g, kb + 16 * kt);
            const unsigned char* kp = a.kv.codes + kr * ROWB;
#pragma unroll
            for (int j = 0; j < KLD; ++j) kreg[kt][j] = *reinterpret_cast<const u32x4_t*>(kp + (koff + 64 * j));
            if constexpr (Q8) {
                const unsigned char* sp = a.kv.scales + kr * (D / KV_BLOCK);
                ksc[kt] = D == 128 ? *reinterpret_cast<const unsigned*>(sp + (unsigned)r * 4) : *reinterpret_cast<const u16*>(sp + (unsigned)r * 2);
            }
        }
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int k0 = n * RPI;  // the wave's first row of this load; all of them in one group of 16
            const size_t vr = kv_row(a.kv, max(pg[k0 >> 4], 0), 1, t.g, kb + k0);
            vreg[n] = *reinterpret_cast<const u32x4_t*>(a.kv.codes + vr * ROWB + voff);
            if constexpr (Q8) vsc[n] = (a.kv.scales + vr * (D / KV_BLOCK))[vsoff];
        }
    };

    // this lane's page of a step ahead: lanes 0 and 1 (modulo 2) have those of the step's two groups of 16 keys
    int kb = t.s0 + wave * 32, pv = -1;
    int pg[2] = {-1, -1};
    auto take = [&]() {
        pg[0] = __builtin_amdgcn_readlane(pv, 0);
        pg[1] = __builtin_amdgcn_readlane(pv, 1);
    };
    if (t.s0 < t.s1) {
        pv = kv_page16(a, t, kb + 16 * (lane & 1));
        take();
        load(kb, pg);
        pv = kv_page16(a, t, kb + 128 + 16 * (lane & 1));
    }
    for (; kb < t.s1; kb += 128) {
        // V rows into this wave's image: rows outside the tile's range and holes as zeros
        const bool mixed = t.p0 != t.p1 && (kb + 31 > t.p0 || (a.window && kb <= t.p1 - a.window));
        const bool edge = mixed || kb < t.k_begin || kb + 32 > t.s1 || pg[0] < 0 || pg[1] < 0;
        bool bad = false;
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            u32x4_t w[Q8 ? 2 : 1];
            if constexpr (Q8) {
                const float f = kv_scale(vsc[n]);
                w[0] = kv_decode8<FMT>(vreg[n].x, vreg[n].y, f);
                w[1] = kv_decode8<FMT>(vreg[n].z, vreg[n].w, f);
            } else {
                w[0] = vreg[n];
            }
            if (edge) {
                const int key = kb + n * RPI + lane / PPR;
                const bool in = key >= t.k_begin && key < t.s1 && pg[(n * RPI) >> 4] >= 0;
#pragma unroll
                for (int h = 0; h < (Q8 ? 2 : 1); ++h) {
                    w[h] = keep(w[h], in);
                    bad |= mixed && bf16x8_bad(w[h]);
                }
            }
#pragma unroll
            for (int h = 0; h < (Q8 ? 2 : 1); ++h)
                *reinterpret_cast<u32x4_t*>(Vs + (n * RPI + lane / PPR) * LDV + (lane % PPR) * EPP + 8 * h) = w[h];
        }
        // scores of 2 x 16 keys: s[rg][kt][i] = key kb + 16 kt + 4 gq + i
        f32x4_t s[RG][2];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
            for (int rg = 0; rg < RG; ++rg) s[rg][kt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
            if constexpr (Q8) {
#pragma unroll
                for (int j = 0; j < KLD; ++j) {
                    const float f = kv_scale((ksc[kt] >> (8 * (2 * j + (gq >> 1)))) & 0xffu);
                    const u32x4_t c = kreg[kt][j];
                    const bf16x8_t k0 = __builtin_bit_cast(bf16x8_t, kv_decode8<FMT>(c.x, c.y, f)), k1 = __builtin_bit_cast(bf16x8_t, kv_decode8<FMT>(c.z, c.w, f));
#pragma unroll
                    for (int rg = 0; rg < RG; ++rg) {
                        s[rg][kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k0, q[rg][2 * j], s[rg][kt], 0, 0, 0);
                        s[rg][kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k1, q[rg][2 * j + 1], s[rg][kt], 0, 0, 0);
                        if constexpr (WIDE) {
                            s[rg][kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k0, ql[rg][2 * j], s[rg][kt], 0, 0, 0);
                            s[rg][kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k1, ql[rg][2 * j + 1], s[rg][kt], 0, 0, 0);
                        }
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < KLD; ++j)
#pragma unroll
                    for (int rg = 0; rg < RG; ++rg)
                        s[rg][kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, kreg[kt][j]), q[rg][j], s[rg][kt], 0, 0, 0);
            }
        }
        // the next rows travel while these go through the softmax
        const int pc[2] = {pg[0], pg[1]};
        take();
        load(kb + 128, pg);  // behind the part: page 0, not used
        pv = kv_page16(a, t, kb + 256 + 16 * (lane & 1));

        bf16x8_t ph[RG], pr[RG];  // pr: the remainders
#pragma unroll
        for (int rg = 0; rg < RG; ++rg) {
            float p[8], mx = -INFINITY;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int key = kb + 16 * (e >> 2) + 4 * gq + (e & 3);
                const bool see = key >= klo[rg] && key <= pos[rg] && key < t.s1 && pc[e >> 2] >= 0;
                p[e] = see ? s[rg][e >> 2][e & 3] * sc : -INFINITY;
                mx = fmaxf(mx, p[e]);
            }
            const float mn = fmaxf(m[rg], kv_quad_rows(mx, fmax2));
            const float ref = mn == -INFINITY ? 0.f : mn;  // nothing seen yet: every exponential below is 0
            const float alpha = __builtin_amdgcn_exp2f(m[rg] - ref);
            m[rg] = mn;
            float ps = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                p[e] = __builtin_amdgcn_exp2f(p[e] - ref);
                ps += p[e];
            }
            l[rg] = l[rg] * alpha + ps;
            ph[rg] = pack8(p);
            if constexpr (WIDE) pr[rg] = rest8(p, ph[rg]);
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) acc[rg][dt] *= alpha;
        }
        __builtin_amdgcn_wave_barrier();  // the image is this wave's own: its LDS accesses are served in order
        if (mixed && __any(bad)) {
            for (int j = 0; j < 32; ++j) {
                const int key = kb + j;
#pragma unroll
                for (int rg = 0; rg < RG; ++rg)
                    if (key >= klo[rg] && key <= pos[rg] && has[rg]) {
#pragma unroll
                        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                            for (int i = 0; i < 4; ++i) acc[rg][dt][i] += bad_only(Vs[j * LDV + 16 * dt + 4 * gq + i]);
                    }
            }
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int n = 0; n < NV; ++n)
#pragma unroll
                for (int h = 0; h < (Q8 ? 2 : 1); ++h) {
                    u32x4_t* p = reinterpret_cast<u32x4_t*>(Vs + (n * RPI + lane / PPR) * LDV + (lane % PPR) * EPP + 8 * h);
                    *p = bf16x8_clean(*p);
                }
            __builtin_amdgcn_wave_barrier();
        }
        const u16* vrow = Vs + (4 * gq + (r >> 2)) * LDV + 4 * (r & 3);
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
            const bf16x8_t vt = join8(read_tr4(vrow + 16 * dt), read_tr4(vrow + 16 * LDV + 16 * dt));
#pragma unroll
            for (int rg = 0; rg < RG; ++rg) {
                acc[rg][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vt, ph[rg], acc[rg][dt], 0, 0, 0);
                if constexpr (WIDE) acc[rg][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vt, pr[rg], acc[rg][dt], 0, 0, 0);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }

    // join the four waves, 16 rows at a time
    float* Os = reinterpret_cast<float*>(smem);
    constexpr int EPT = D / 16;
    const int orow = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * EPT;
#pragma unroll
    for (int rg = 0; rg < RG; ++rg) {
        const float lr = kv_quad_rows(l[rg], fadd2);
        __syncthreads();
        if (gq == 0) {
            pm[wave][16 * rg + r] = m[rg];
            pl[wave][16 * rg + r] = lr;
        }
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) *reinterpret_cast<f32x4_t*>(Os + (wave * 16 + r) * LDO + 16 * dt + 4 * gq) = acc[rg][dt];
        __syncthreads();
        const int trow = 16 * rg + orow, rr = t.row0 + trow;
        if (rr >= t.rows) continue;
        float M = pm[0][trow];
#pragma unroll
        for (int w = 1; w < 4; ++w) M = fmaxf(M, pm[w][trow]);
        float L = 0.f, o[EPT];
#pragma unroll
        for (int e = 0; e < EPT; ++e) o[e] = 0.f;
        const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float wt = __builtin_amdgcn_exp2f(pm[w][trow] - ref);
            L += wt * pl[w][trow];
#pragma unroll
            for (int e = 0; e < EPT; ++e) o[e] += wt * Os[(w * 16 + orow) * LDO + d0 + e];
        }
        if (t.parts > 1) {
            const size_t u = ((size_t)(pair * a.tiles + blockIdx.y) * a.splits + blockIdx.z) * TR + trow;  // slot
            float* po = a.ws + u * D + d0;
#pragma unroll
            for (int e = 0; e < EPT; e += 4) *reinterpret_cast<float4*>(po + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            if ((threadIdx.x & 15) == 0) {
                float* ml = a.ws + (size_t)a.b.n_seq * a.kv.nkv * a.tiles * a.splits * TR * D + u * 2;
                ml[0] = M;
                ml[1] = L;
            }
            continue;
        }
        const int tk = rr / t.G, hd = t.g * t.G + rr - tk * t.G;
        bf16_t* op = (bf16_t*)a.out + (long)(t.s.t0 + tk) * a.out_token_stride + (long)hd * a.out_head_stride + d0;
        const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
        for (int e = 0; e < EPT; e += 4) {
            const float v[4] = {o[e] * inv, o[e + 1] * inv, o[e + 2] * inv, o[e + 3] * inv};
            store4_split(op + e, a.out_lo, v);
        }
    }
}

// ------------------------------------------------------------------------------------------------------ 128 rows a tile
// Prompts and chunks: bound by the matrix and vector instructions, so 128 rows share one staging (and conversion) of 64 keys: four waves of 32
// rows, the K and V images in LDS, the next block of keys travelling in registers, two blocks of threads a CU (three at d = 64) that fill each
// other's waits.  Measured (d = 128): 512 equal tiles of 8192 keys 847 TFLOP/s in bf16, 953 in e4m3 (half the bytes), 852 in int8 (byte conversions);
// 1024 of them 814, 892, 822; a large library product 1257.  Prompts of 4096 and 2912 tokens 131 us = 788 TFLOP/s: the longest tile walks 64 blocks of
// keys at 2 us; 509 new tokens behind 3 x 15013 e4m3 keys 354 us = 820 (the same in int8: 391).  The talker's prompts of 64 x 51 tokens (WIDE) take 22 us a
// layer, 19 without the second pieces.  Counters of the prompts before the reads went ahead and the priorities: matrix pipe busy 35 % of the CUs' time, vector
// pipe 37 %, LDS 26 % without a conflict: none was full, a wave's chain S -> softmax -> P V was what waited.  Tried, not faster: S of the next block issued before the softmax of
// this one over double images; 256 rows with eight waves (prompts 7 % faster, chunks and windows slower); longest tiles at a higher wave
// priority from end to end; blocks of keys dealt evenly to the CUs (the tiles of a head no longer walk in step and miss the L2).
template <int FMT, int D, bool WIDE>
__global__ __launch_bounds__(256, 2) void kv_attend_tile_kernel(KvAttendArgs a) {
    constexpr bool Q8 = FMT != KV_BF16;
    constexpr int KB = 64;
    constexpr int LDK = D + 8;    // K rows 4 banks apart: 16 lanes' 16-byte reads hit every bank once
    constexpr int LDV = D + 32;   // V rows 16 banks apart (modulo 64): the four rows of a transposing read share no bank
    constexpr int NS = D / 16, NDT = D / 32;          // contraction steps of K Q^T; 32-column tiles of the output
    constexpr int EPP = Q8 ? 16 : 8, PPR = D / EPP;   // elements per 16-byte piece of the cache, pieces per row
    constexpr int KPW = 64 / PPR, NP = KB / (4 * KPW);  // keys a wave stages at once, passes per block of keys
    __shared__ __attribute__((aligned(16))) u16 Ks[KB * LDK];
    __shared__ __attribute__((aligned(16))) u16 Vs[KB * LDV];
    __shared__ int sh_bad;  // a V element that some rows see and others do not was not finite

    const int pair = blockIdx.x;
    if (pair >= a.b.n_seq * a.kv.nkv) return;
    const int tile = (int)gridDim.y - 1 - (int)blockIdx.y;  // the last tiles see the most keys: they start first
    const KvTile t = kv_tile<128>(a, pair, tile, blockIdx.z);
    if (!t.live) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 31, hf = lane >> 5;
    const int wrow0 = t.row0 + wave * 32;
    const bool wlive = wrow0 < t.rows;
    const int first = t.s.ctx - t.s.n;
    const int wp0 = first + min(wrow0, t.rows - 1) / t.G, wp1 = first + min(wrow0 + 31, t.rows - 1) / t.G;

    const int row = wrow0 + r;
    const bool has = row < t.rows;
    const int rr = has ? row : t.rows - 1;
    const int tok = rr / t.G, head = t.g * t.G + rr - tok * t.G;
    const int pos = first + tok;
    const int klo = has ? (a.window ? pos - a.window + 1 : 0) : 0x7fffffff;
    bf16x8_t q[NS], ql[WIDE ? NS : 1];
    {
        const long qat = (long)(t.s.t0 + tok) * a.q_token_stride + (long)head * a.q_head_stride + 8 * hf;
#pragma unroll
        for (int j = 0; j < NS; ++j) {
            if constexpr (WIDE) {
                float f[8];
                load8((const float*)a.q + qat + 16 * j, f);
                q[j] = pack8(f);
                ql[j] = rest8(f, q[j]);
            } else {
                q[j] = *reinterpret_cast<const bf16x8_t*>((const u16*)a.q + qat + 16 * j);
            }
        }
    }
    f32x16_t acc[NDT];
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[dt][i] = 0.f;
    float m = -INFINITY, l = 0.f;
    const float sc = a.scale * 1.4426950408889634f;

    u32x4_t kreg[NP], vreg[NP];
    unsigned ksc[NP], vsc[NP];
    const int krow = lane / PPR, pc = lane % PPR;
    constexpr unsigned ROWB = Q8 ? D : 2 * D;  // bytes of a head row
    // Lanes 0 .. 3 (modulo 4) work out where a block's four groups of 16 keys start and hand it round: as scalars of the loop these are a
    // hundred instructions a block.  A hole is read as page 0: in bounds, and what it holds is masked.
    const unsigned long page_bytes = ((unsigned long)a.kv.nkv << a.kv.page_shift) * (2 * ROWB);
    const unsigned head_bytes = ((unsigned)t.g << a.kv.page_shift) * ROWB;
    const unsigned koff = ((wave * KPW) & 15) * ROWB + krow * ROWB + pc * 16, voff = koff + (unsigned)(page_bytes >> 1);
    int pv = -1;
    unsigned holes = 0, hole = 0;  // bit i: group i of the block that travels, of the block in the images
    auto load = [&](int kb) {      // pv: the block's pages
        holes = (unsigned)__ballot(pv < 0) & 15u;
        const unsigned long ga = (unsigned long)max(pv, 0) * page_bytes + head_bytes + ((kb + 16 * (lane & 3)) & ((1 << a.kv.page_shift) - 1)) * ROWB;
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            const int gi = ((n * 4 + wave) * KPW) >> 4;  // group of the wave's keys in this pass
            const unsigned long at = ((unsigned long)(unsigned)__builtin_amdgcn_readlane((int)(ga >> 32), gi) << 32) | (unsigned)__builtin_amdgcn_readlane((int)ga, gi);
            kreg[n] = *reinterpret_cast<const u32x4_t*>(a.kv.codes + at + koff);
            vreg[n] = *reinterpret_cast<const u32x4_t*>(a.kv.codes + at + voff);
            if constexpr (Q8) {  // a scale byte per 32 code bytes
                ksc[n] = (a.kv.scales + (at >> 5))[koff / KV_BLOCK];
                vsc[n] = (a.kv.scales + (at >> 5))[voff / KV_BLOCK];
            }
        }
    };
    if (t.s0 < t.s1) {
        pv = kv_page16(a, t, t.s0 + 16 * (lane & 3));
        load(t.s0);
        pv = kv_page16(a, t, t.s0 + KB + 16 * (lane & 3));
    }
    if (threadIdx.x == 0) sh_bad = 0;
    for (int kb = t.s0; kb < t.s1; kb += KB) {
        const bool mixed = kb + KB - 1 > t.p0 || (a.window && kb <= t.p1 - a.window);
        const bool edge = mixed || kb < t.k_begin || kb + KB > t.s1 || holes;
        __syncthreads();  // every wave is done with the previous image
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            const int k0 = (n * 4 + wave) * KPW;
            const int key = k0 + krow;
            u32x4_t w[Q8 ? 2 : 1];
            if constexpr (Q8) {
                const float fk = kv_scale(ksc[n]), fv = kv_scale(vsc[n]);
                *reinterpret_cast<u32x4_t*>(Ks + key * LDK + pc * 16) = kv_decode8<FMT>(kreg[n].x, kreg[n].y, fk);
                *reinterpret_cast<u32x4_t*>(Ks + key * LDK + pc * 16 + 8) = kv_decode8<FMT>(kreg[n].z, kreg[n].w, fk);
                w[0] = kv_decode8<FMT>(vreg[n].x, vreg[n].y, fv);
                w[1] = kv_decode8<FMT>(vreg[n].z, vreg[n].w, fv);
            } else {
                *reinterpret_cast<u32x4_t*>(Ks + key * LDK + pc * 8) = kreg[n];
                w[0] = vreg[n];
            }
            if (edge) {
                const bool in = kb + key >= t.k_begin && kb + key < t.s1 && !((holes >> (k0 >> 4)) & 1u);
#pragma unroll
                for (int h = 0; h < (Q8 ? 2 : 1); ++h) {
                    w[h] = keep(w[h], in);
                    if (mixed && bf16x8_bad(w[h])) {
                        sh_bad = 1;  // read behind the loop, and so behind a barrier
                        w[h] = bf16x8_clean(w[h]);
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < (Q8 ? 2 : 1); ++h) *reinterpret_cast<u32x4_t*>(Vs + key * LDV + pc * EPP + 8 * h) = w[h];
        }
        hole = holes;
        load(kb + KB);  // behind the part: page 0, not used
        pv = kv_page16(a, t, kb + 2 * KB + 16 * (lane & 3));
        __syncthreads();
        // wave-uniform: no row of this wave sees the block
        if (!wlive || kb > wp1 || (a.window && kb + KB <= wp0 - a.window + 1)) continue;

        f32x16_t s[2];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[kt][i] = 0.f;
        // A wave at its products goes before one that stages or waits, one further on before one at its start: the two blocks of a CU, which
        // start in step, come apart (prompts 155 -> 133 us, equal tiles 3 to 6 % faster; at d = 64 no gain, the window's case 5 % slower).
        if constexpr (D == 128) __builtin_amdgcn_s_setprio(1);
        const u16* kp = Ks + r * LDK + 8 * hf;
        constexpr int AHEAD = 3;
        bf16x8_t kf[AHEAD][2];
        auto read_k = [&](int j) {
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) kf[j % AHEAD][kt] = *reinterpret_cast<const bf16x8_t*>(kp + kt * 32 * LDK + 16 * j);
        };
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) read_k(j);
#pragma unroll
        for (int j = 0; j < NS; ++j) {
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) s[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[j % AHEAD][kt], q[j], s[kt], 0, 0, 0);
            if constexpr (WIDE) {
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) s[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[j % AHEAD][kt], ql[j], s[kt], 0, 0, 0);
            }
            if (j + AHEAD < NS) read_k(j + AHEAD);
        }
        // in this order: the compiler would read each operand right before its product
        __builtin_amdgcn_sched_group_barrier(0x100, 2 * AHEAD, 0);  // LDS reads
#pragma unroll
        for (int j = 0; j < NS; ++j) {
            __builtin_amdgcn_sched_group_barrier(0x8, WIDE ? 4 : 2, 0);  // products
            if (j + AHEAD < NS) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
        const u16* vp = Vs + (4 * hf + ((lane & 15) >> 2)) * LDV + (lane & 16) + 4 * (lane & 3);
        bf16x8_t vf[2][NDT];
        auto read_v = [&](int g) {  // V^T of 16 keys
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) vf[g & 1][dt] = join8(read_tr4(vp + 16 * g * LDV + 32 * dt), read_tr4(vp + (16 * g + 8) * LDV + 32 * dt));
            asm volatile("" ::: "memory");
        };
        read_v(0);
        // s[kt][i] = key kb + 32 kt + 8 (i / 4) + 4 hf + i % 4 of this lane's row
        const bool whole = kb + KB - 1 <= wp0 && !(a.window && kb <= wp1 - a.window) && kb + KB <= t.s1 && !hole;
        if (!whole) {
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int key = kb + 32 * kt + 8 * (i >> 2) + 4 * hf + (i & 3);
                    const bool see = key >= klo && key <= pos && key < t.s1 && !((hole >> (2 * kt + (i >> 3))) & 1u);
                    s[kt][i] = see ? s[kt][i] : -INFINITY;
                }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[kt][i]);
        mx = fold_halves(mx, fmax2) * sc;
        // The reference m of the exponentials need not be the maximum, only near it: it moves when a row's maximum has left it by more than
        // 2^8 (p and l stay far from overflow, their relative precision is the same).  Moved at every new maximum, which some row of 32 has in
        // most blocks, acc's scaling was a fifth of the vector instructions.  Each row decides for itself: a row's result does not depend on what
        // shares its wave.
        if (__any(mx - m > 8.f)) {
            const float mn = mx - m > 8.f ? mx : m;
            const float alpha = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
            l *= alpha;
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) acc[dt] *= alpha;
            m = mn;
        }
        // m is a rounded product; the exponents below are s sc - m with one rounding at the end.  The rounding that m had is a factor common to
        // the row, at most 2^(1/16) while m is below 2^20.  Above, it would drive weights out of f32's range (by 2^64 at 2^30): there the
        // products are rounded as m was, so that the largest weight is at most 2^8 again.
        float ref = m == -INFINITY ? 0.f : m, fac = sc;
        const bool far = fabsf(ref) >= 1048576.f;
        if (__any(far)) {
#pragma clang fp contract(off)  // two roundings
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float x = s[kt][i] * sc;
                    s[kt][i] = far ? x - ref : s[kt][i];
                }
            fac = far ? 1.f : sc;
            ref = far ? 0.f : ref;
        }
        if constexpr (D == 128) __builtin_amdgcn_s_setprio(2);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            float p[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[g >> 1][8 * (g & 1) + e], fac, -ref));
                l += p[e];
            }
            const bf16x8_t ph = pack8(p);
            if (g < 3) read_v(g + 1);
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[g & 1][dt], ph, acc[dt], 0, 0, 0);
            if constexpr (WIDE) {
                const bf16x8_t pr = rest8(p, ph);
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt) acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[g & 1][dt], pr, acc[dt], 0, 0, 0);
            }
        }
        if constexpr (D == 128) __builtin_amdgcn_s_setprio(0);
    }

    // What was taken out of the products, added to the rows that see it: here, behind the last scaling of acc, and not in the loop, where a
    // factor of 0 (a row's first block, a maximum that rises by 2^7 or more) would make NaN of an infinity.
    if (t.s0 < t.s1 && sh_bad) {
        for (int key = t.s0; key < t.s1; ++key) {
            const int kb = key & ~(KB - 1);
            if (!(kb + KB - 1 > t.p0 || (a.window && kb <= t.p1 - a.window)) || key < klo || key > pos) continue;
            const int page = kv_page(a.kv, t.s.row, key);
            if (page < 0) continue;
            const size_t vr = kv_row(a.kv, page, 1, t.g, key);
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const size_t at = vr * D + 32 * dt + 2 * i + 4 * hf;
                    float v[4];
                    if constexpr (Q8) {
                        kv_decode4<FMT>(*reinterpret_cast<const unsigned*>(a.kv.codes + at), kv_scale(a.kv.scales[at / KV_BLOCK]), v);
                    } else {
                        const uint2 w = *reinterpret_cast<const uint2*>((const u16*)a.kv.codes + at);
                        v[0] = __uint_as_float(w.x << 16);
                        v[1] = __uint_as_float(w.x & 0xffff0000u);
                        v[2] = __uint_as_float(w.y << 16);
                        v[3] = __uint_as_float(w.y & 0xffff0000u);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!__builtin_isfinite(v[e])) acc[dt][i + e] += v[e];
                }
        }
    }

    l = fold_halves(l, fadd2);
    if (!has) return;
    if (t.parts > 1) {
        const size_t u = ((size_t)(pair * a.tiles + tile) * a.splits + blockIdx.z) * 128 + wave * 32 + r;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *reinterpret_cast<float4*>(a.ws + u * D + 32 * dt + 2 * i + 4 * hf) = make_float4(acc[dt][i], acc[dt][i + 1], acc[dt][i + 2], acc[dt][i + 3]);
        if (hf == 0) {
            float* ml = a.ws + (size_t)a.b.n_seq * a.kv.nkv * a.tiles * a.splits * 128 * D + u * 2;
            ml[0] = m;
            ml[1] = l;
        }
        return;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    bf16_t* op = (bf16_t*)a.out + (long)(t.s.t0 + tok) * a.out_token_stride + (long)head * a.out_head_stride + 4 * hf;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const float v[4] = {acc[dt][i] * inv, acc[dt][i + 1] * inv, acc[dt][i + 2] * inv, acc[dt][i + 3] * inv};
            store4_split(op + 32 * dt + 2 * i, a.out_lo, v);
        }
}

// ------------------------------------------------------------------------------------------------ joining the parts
// One wave per row: its lanes take the parts' maxima and sums (64 at a time) and turn them into weights; then each lane adds up its
// D / 64 columns of the parts' outputs with eight loads in flight: 5 us for 73 parts of 56 rows, where one thread an element and all parts in a
// row of loads took 19 us and the kernel below takes 11 us.
template <int D, int TR>
__global__ __launch_bounds__(256) void kv_attend_join_few_kernel(KvAttendArgs a) {
    constexpr int EPL = D / 64;
    typedef float vec_t __attribute__((ext_vector_type(EPL)));
    const int unit = blockIdx.x, pair = unit / a.tiles, tile = unit - pair * a.tiles;
    const KvTile t = kv_tile<TR>(a, pair, tile, 0);
    const int lane = threadIdx.x & 63, trow = (int)blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rr = t.row0 + trow;
    if (!t.live || t.parts == 1 || rr >= t.rows) return;
    const size_t u = (size_t)unit * a.splits * TR + trow;
    const float* ml = a.ws + (size_t)a.b.n_seq * a.kv.nkv * a.tiles * a.splits * TR * D + u * 2;
    const float* po = a.ws + u * D + lane * EPL;
    float M = -INFINITY;
    for (int s = lane; s < t.parts; s += 64) M = fmaxf(M, ml[(size_t)s * TR * 2]);
    M = wave_max(M);
    const float ref = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    vec_t o;
#pragma unroll
    for (int e = 0; e < EPL; ++e) o[e] = 0.f;
    for (int s0 = 0; s0 < t.parts; s0 += 64) {
        const int n = min(t.parts - s0, 64);
        float w = 0.f;  // weight of part s0 + lane
        if (lane < n) {
            w = __builtin_amdgcn_exp2f(ml[(size_t)(s0 + lane) * TR * 2] - ref);
            L += w * ml[(size_t)(s0 + lane) * TR * 2 + 1];
        }
        for (int s = 0; s < n; s += 8) {
            vec_t v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = *reinterpret_cast<const vec_t*>(po + (size_t)(s0 + min(s + k, n - 1)) * TR * D);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float wk = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), min(s + k, n - 1)));
#pragma unroll
                for (int e = 0; e < EPL; ++e) o[e] += s + k < n ? wk * v[k][e] : 0.f;
            }
        }
    }
    L = wave_sum(L);
    const int tk = rr / t.G, hd = t.g * t.G + rr - tk * t.G;
    bf16_t* op = (bf16_t*)a.out + (long)(t.s.t0 + tk) * a.out_token_stride + (long)hd * a.out_head_stride + lane * EPL;
    const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int e = 0; e < EPL; ++e) store_split(op + e, a.out_lo, o[e] * inv);
}

// Tiles of 128 rows have few parts and many rows: D / 4 lanes a row, each with 16 bytes of it, O = sum_s 2^(m_s - M) O_s over
// sum_s 2^(m_s - M) l_s, four parts' loads in flight.  Bound by the partial results' bytes (20 us for 60 MB; a wave per row 34 us).
template <int D>
__global__ __launch_bounds__(256) void kv_attend_join_tile_kernel(KvAttendArgs a) {
    constexpr int TR = 128, LPR = D / 4, RPB = 256 / LPR;
    const int unit = blockIdx.x, pair = unit / a.tiles, tile = unit - pair * a.tiles;
    const KvTile t = kv_tile<TR>(a, pair, tile, 0);
    const int trow = (int)blockIdx.y * RPB + threadIdx.x / LPR, rr = t.row0 + trow, d0 = threadIdx.x % LPR * 4;
    if (!t.live || t.parts == 1 || rr >= t.rows) return;
    const size_t u = (size_t)unit * a.splits * TR + trow;
    const float* ml = a.ws + (size_t)a.b.n_seq * a.kv.nkv * a.tiles * a.splits * TR * D + u * 2;
    const float* po = a.ws + u * D + d0;
    float M = -INFINITY, L = 0.f;
    f32x4_t o = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < t.parts; s += 4) {
        float m[4], l[4];
        f32x4_t v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const size_t q = (size_t)min(s + k, t.parts - 1) * TR;
            const float2 x = *reinterpret_cast<const float2*>(ml + q * 2);
            m[k] = s + k < t.parts ? x.x : -INFINITY;  // a part that is not there weighs nothing
            l[k] = x.y;
            v[k] = *reinterpret_cast<const f32x4_t*>(po + q * D);
        }
        const float mn = fmaxf(M, fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])));
        const float ref = mn == -INFINITY ? 0.f : mn;
        const float alpha = __builtin_amdgcn_exp2f(M - ref);
        L *= alpha;
        o *= alpha;
        M = mn;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float w = __builtin_amdgcn_exp2f(m[k] - ref);
            L += s + k < t.parts ? w * l[k] : 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] += s + k < t.parts ? w * v[k][e] : 0.f;
        }
    }
    const int tk = rr / t.G, hd = t.g * t.G + rr - tk * t.G;
    bf16_t* op = (bf16_t*)a.out + (long)(t.s.t0 + tk) * a.out_token_stride + (long)hd * a.out_head_stride + d0;
    const float inv = L == 0.f ? 0.f : 1.f / L;
    const float r[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
    store4_split(op, a.out_lo, r);
}

// ---------------------------------------------------------------------------------------------------------- host side
void launch_kv_attend(hipStream_t st, KvAttendArgs a, const KvAttendPlan& p) {
    if (a.b.n_seq == 0 || a.b.n_tokens == 0) return;
    QTTS_CHECK(p.splits == 1 || a.ws, ERR_BAD_ARG, "kv attend: workspace missing");
    a.tiles = p.tiles;
    a.splits = p.splits;
    a.split_len = p.split_len;
    const unsigned pairs = (unsigned)(a.b.n_seq * a.kv.nkv);
    // pairs vary fastest and are padded to the number of XCDs: all tiles and parts of a pair run on one XCD and share its L2 (fewer than eight
    // pairs leave XCDs idle)
    const dim3 grid((pairs + 7) / 8 * 8, (unsigned)p.tiles, (unsigned)p.splits);
    const dim3 join(pairs * (unsigned)p.tiles, p.tile_rows == 128 ? (unsigned)a.kv.d / 8u : (unsigned)p.tile_rows / 4u);
#define QTTS_KV_ATTEND(FMT, DD, WIDE)                                                                   \
    if (a.kv.format == FMT && a.kv.d == DD && a.wide == WIDE) {                                         \
        if (p.tile_rows == 16) {                                                                        \
            kv_launch(kv_attend_few_kernel<FMT, DD, 1, WIDE>, grid, dim3(256), st, a);                  \
            if (p.splits > 1) kv_launch(kv_attend_join_few_kernel<DD, 16>, join, dim3(256), st, a);     \
            return;                                                                                     \
        }                                                                                               \
        if constexpr (!WIDE) {                                                                          \
            if (p.tile_rows == 32) {                                                                    \
                kv_launch(kv_attend_few_kernel<FMT, DD, 2, WIDE>, grid, dim3(256), st, a);              \
                if (p.splits > 1) kv_launch(kv_attend_join_few_kernel<DD, 32>, join, dim3(256), st, a); \
                return;                                                                                 \
            }                                                                                           \
        }                                                                                               \
        if (p.tile_rows == 128) {                                                                       \
            kv_launch(kv_attend_tile_kernel<FMT, DD, WIDE>, grid, dim3(256), st, a);                    \
            if (p.splits > 1) kv_launch(kv_attend_join_tile_kernel<DD>, join, dim3(256), st, a);        \
            return;                                                                                     \
        }                                                                                               \
    }
    QTTS_KV_ATTEND(KV_BF16, 64, false)
    QTTS_KV_ATTEND(KV_E4M3, 64, false)
    QTTS_KV_ATTEND(KV_INT8, 64, false)
    QTTS_KV_ATTEND(KV_BF16, 128, false)
    QTTS_KV_ATTEND(KV_E4M3, 128, false)
    QTTS_KV_ATTEND(KV_INT8, 128, false)
    QTTS_KV_ATTEND(KV_E4M3, 64, true)
    QTTS_KV_ATTEND(KV_INT8, 64, true)
    QTTS_KV_ATTEND(KV_E4M3, 128, true)
    QTTS_KV_ATTEND(KV_INT8, 128, true)
#undef QTTS_KV_ATTEND
    throw Error(ERR_SHAPE, "kv attend: no kernel for this head_dim, format and tile");
}

}  // namespace qtts
