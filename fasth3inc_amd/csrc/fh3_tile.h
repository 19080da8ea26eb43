// fh3_tile.h -- one wavefront's 32 query rows against 64-key tiles in LDS, for
// the kernels over packed sequences (fh3_seqs.hip) and the 8-bit cache (fh3_kv.hip).
//
// S^T = K Q^T and O^T = V^T P^T on 32x32x16 matrix products: a lane holds one row
// (lane & 31) and, of each 32 keys, those with (key >> 2) & 1 == lane >> 5, so the
// softmax needs no exchange between lanes but the last sums, and the weights go
// from the first product's registers straight into the second's operand.  The
// rows of a tile are (token, query head of the group) pairs of one key head, so
// shared key heads fill the tile.
#ifndef FH3_TILE_H
#define FH3_TILE_H

#include "fh3_seqs.h"

namespace {

constexpr int TILE_K = 64;   // keys per tile
constexpr int WAVE_R = 32;   // rows per wavefront
// Weights are exp2(t - m) where m is raised, to OFFSET below a tile's largest t, only when
// that exceeds it by more than RAISE: the largest weight is from 2^OFFSET to 2^RAISE
// and most tiles need no rescale of the sums.  In fp16 6 and 14 keep small weights out of
// the subnormal range (2^14 < 65504).  bf16 weights have fp32's range, and so has V
// then: with -18 and -10 the sums of 1024 keys stay below V's largest (at 2^14 those
// of 10^34 passed it), and V's least normal numbers times 2^-18 are still held.
// From |t| = FAR on, m alone could not stand OFFSET below the largest t (half a step of fp32
// is 8 and more from 2^27), nor is t = c s itself exact enough: there m is the rounded largest
// t and a second term lo what the exact product is off it by, and the weights' arguments
// (c s - m) - lo are small numbers made by one multiply-add from the products s.  Below, lo
// is 0 and arguments are c s - m.
constexpr float FAR = 0x1p20f;
constexpr float M_NONE = -3.402823466e38f;  // no key seen yet: finite, so that masked t = -inf gives 0
// Parts of a row with offsets (m, lo) and (m2, lo2): what the larger offset leaves of each; m, lo become the larger.
__device__ __forceinline__ void join_offsets(float &m, float &lo, float m2, float lo2, float &keep, float &add) {
    const float d = (m2 - m) + (lo2 - lo), e = __builtin_amdgcn_exp2f(-fabsf(d));
    keep = d > 0.f ? e : 1.f;
    add = d > 0.f ? 1.f : e;
    m = d > 0.f ? m2 : m, lo = d > 0.f ? lo2 : lo;
}

template <class T> struct Vec;
template <> struct Vec<_Float16> {
    typedef half8 v8;
    static constexpr float OFFSET = 6.f, RAISE = 14.f;
    static __device__ __forceinline__ uint32_t pair(float a, float b) {
        uint32_t w = __builtin_bit_cast(uint32_t, half2v{(_Float16)a, (_Float16)b});
        asm("" : "+v"(w));  // one pair, not converted once for each use
        return w;
    }
    static __device__ __forceinline__ float sum(uint32_t w, float c) {
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(half2v, w), half2v{1, 1}, c, false);
    }
};
template <> struct Vec<__bf16> {
    typedef bf8 v8;
    static constexpr float OFFSET = -18.f, RAISE = -10.f;
    static __device__ __forceinline__ uint32_t pair(float a, float b) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf2));
    }
    static __device__ __forceinline__ float sum(uint32_t w, float c) {
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf2, w), bf2{1.f, 1.f}, c, false);
    }
};

__device__ __forceinline__ f32x16 mfma32(half8 a, half8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(bf8 a, bf8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// What every row of a call shares.
struct Score {
    float f;        // product sum -> t (log2 units), or -> 2 log2(e) x / cap before the tanh
    float cap2;     // cap * log2(e), or 0
    bool fine;      // the cap's tanh to fp32's last bits
    bool bias;
};
__device__ __forceinline__ Score score_of(const Fh3kAttn &a) {
    Score sc;
    sc.cap2 = a.softcap > 0.f ? a.softcap * LOG2E : 0.f;
    sc.f = a.softcap > 0.f ? 2.f * LOG2E * (a.scale / a.softcap) : a.scale * LOG2E;
    sc.fine = a.type == FH3K_F32 || a.softcap > 64.f;
    sc.bias = a.slopes != nullptr;
    return sc;
}
// A factor of the products, kept positive and finite: a product of 0 and a masked -inf are then
// what they should be (0 or an infinite factor would make a NaN of them).
__device__ __forceinline__ float factor(float x) { return __builtin_amdgcn_fmed3f(x, 0x1p-149f, 3.402823466e38f); }
// cap tanh(z), z = x / cap, from y = 2 log2(e) z: tanh = 1 - 2 / (1 + e^2z).  Its error is
// 10^-7 of the cap, whatever x is: enough for 16-bit rows and caps to 64 (10^-5).
__device__ __forceinline__ float capped(float y, float cap2) {
    return cap2 - 2.f * cap2 * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(y));
}
// Otherwise up to |z| = 1 by the continued fraction z / (1 + z^2 / (3 + z^2 / (5 + ..)))
// cut after 9, z (945 + 105 z^2 + z^4) / (945 + 420 z^2 + 15 z^4), which is off by 6 10^-8 of
// itself at most; the reciprocal by one Newton step.
__device__ __forceinline__ float capped_fine(float y, float cap2) {
    const float z = y * 0.34657359f, z2 = z * z;
    const float num = fmaf(z2, z2 + 105.f, 945.f), den = fmaf(z2, fmaf(15.f, z2, 420.f), 945.f);
    float r = __builtin_amdgcn_rcpf(den);
    r = fmaf(fmaf(-den, r, 1.f), r, r);
    return fabsf(z) < 1.f ? cap2 * z * (num * r) : capped(y, cap2);
}

// 2^e such that amax * 2^e lies in [2^13, 2^14); 1 for zeros and values that are not finite.
__device__ __forceinline__ float pow2_to_14(float amax) {
    int e = 13 - ((int)(__builtin_bit_cast(uint32_t, amax) >> 23) - 127);
    e = e > 126 ? 126 : e;
    return amax > 0.f && amax <= 3.402823466e38f ? __builtin_bit_cast(float, (uint32_t)(e + 127) << 23) : 1.f;
}

// Eight consecutive values of a row: as they stand in memory (so that the load can
// be on its way while other work is done), and as fp32.
struct Raw8 {
    u32x4 a, b;  // b: fp32 only
};
__device__ __forceinline__ Raw8 load8(const void *p, int type, int64_t at) {
    Raw8 r = {};
    if (type == FH3K_F32) {
        const u32x4 *q = (const u32x4 *)((const float *)p + at);
        r.a = q[0], r.b = q[1];
    } else {
        r.a = *(const u32x4 *)((const uint16_t *)p + at);
    }
    return r;
}
__device__ __forceinline__ void values8(const Raw8 &r, int type, float (&x)[8]) {
    if (type == FH3K_F32) {
        const f32x4 a = __builtin_bit_cast(f32x4, r.a), b = __builtin_bit_cast(f32x4, r.b);
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = a[i], x[4 + i] = b[i];
    } else if (type == FH3K_F16) {
        const half8 a = __builtin_bit_cast(half8, r.a);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = (float)a[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            x[i] = __builtin_bit_cast(float, i & 1 ? r.a[i >> 1] & 0xFFFF0000u : r.a[i >> 1] << 16);
    }
}
// four consecutive values of an output row
__device__ __forceinline__ void store4(void *p, int type, int64_t at, f32x4 x) {
    if (type == FH3K_F32) *(f32x4 *)((float *)p + at) = x;
    else if (type == FH3K_F16) {
        half4 h;
#pragma unroll
        for (int i = 0; i < 4; i++) h[i] = (_Float16)x[i];
        *(half4 *)((_Float16 *)p + at) = h;
    } else {
        const u32x2 h = {__builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x[0], x[1]}, bf2)),
                         __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x[2], x[3]}, bf2))};
        *(u32x2 *)((uint16_t *)p + at) = h;
    }
}

// Two values times a power of two as two fp16 terms each, x ~ hi + lo, all rounded to nearest.
__device__ __forceinline__ void split2(float a, float b, float scale, uint32_t &hi, uint32_t &lo) {
    const half2v h = __builtin_convertvector(f32x2{a * scale, b * scale}, half2v);
    const f32x2 l = {fmaf(a, scale, -(float)h[0]), fmaf(b, scale, -(float)h[1])};
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, __builtin_convertvector(l, half2v));
}
// The lanes 32 (16) apart: the larger value, the sum, in both.
__device__ __forceinline__ f32x2 swap32(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    const uint32_t lo = r[0], hi = r[1];
    return {__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi)};
}
__device__ __forceinline__ f32x2 swap16(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    const uint32_t lo = r[0], hi = r[1];
    return {__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi)};
}
__device__ __forceinline__ float max32(float x) {
    const f32x2 r = swap32(x);
    return fmaxf(r[0], r[1]);
}
__device__ __forceinline__ float sum32(float x) {
    const f32x2 r = swap32(x);
    return r[0] + r[1];
}
__device__ __forceinline__ float max16(float x) {
    const f32x2 r = swap16(x);
    return fmaxf(r[0], r[1]);
}
__device__ __forceinline__ float sum16(float x) {
    const f32x2 r = swap16(x);
    return r[0] + r[1];
}
// TQ: element of the first product's operands, TP: of the second's.  QT: terms of
// q and of the weights.
template <int HD, class TQ, class TP, int QT> struct Rows {
    static constexpr int KS = HD / 16, DB = HD / 32;
    static constexpr int KROW = HD + 8;  // LDS row of K
    static constexpr float OFFSET = Vec<TP>::OFFSET, RAISE = Vec<TP>::RAISE;
    typedef typename Vec<TQ>::v8 q8;
    typedef typename Vec<TP>::v8 p8;

    q8 q[QT][KS];
    f32x16 o[DB];
    float m, lo, l;  // of the row: the weights' offset in two terms, the sum over this lane's keys
    uint64_t far;    // rows of the wavefront that have an offset of FAR and more
    float f;         // Score::f over the row's own power of two
    float slope2;
    int pos, lim;    // the row sees keys 0 .. lim - 1

    // q's fragments: lane holds row lane & 31, channels 16 kk + 8 (lane >> 5) ..
    // SCALED: by the row's power of two (fp32 or the cache's fp16 products), its largest to [2^13, 2^14) times `less`
    template <bool SCALED>
    __device__ __forceinline__ void load_q(const void *qp, int type, int64_t at, const Score &sc, float less = 1.f) {
        const int hf = (threadIdx.x >> 5) & 1;
        f = sc.f;
        if constexpr (!SCALED) {
#pragma unroll
            for (int kk = 0; kk < KS; kk++) q[0][kk] = *(const q8 *)((const TQ *)qp + at + 16 * kk + 8 * hf);
        } else {
            float x[KS][8], top = 0.f;
#pragma unroll
            for (int kk = 0; kk < KS; kk++) {
                values8(load8(qp, type, at + 16 * kk + 8 * hf), type, x[kk]);
#pragma unroll
                for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf(x[kk][i]));
            }
            top = max32(top);
            const float up = pow2_to_14(top) * less;
            f = sc.f / up;
#pragma unroll
            for (int kk = 0; kk < KS; kk++) {
                if constexpr (QT == 2) {
                    u32x4 h, l4;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        uint32_t hi, lo;
                        split2(x[kk][2 * i], x[kk][2 * i + 1], up, hi, lo);
                        h[i] = hi, l4[i] = lo;
                    }
                    q[0][kk] = __builtin_bit_cast(q8, h), q[QT - 1][kk] = __builtin_bit_cast(q8, l4);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i++) q[0][kk][i] = (TQ)(x[kk][i] * up);
                }
            }
        }
    }

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < DB; i++) o[i] = f32x16{};
        m = M_NONE;
        lo = l = 0.f;
        far = 0;
    }

    // S^T of the 64 keys whose rows sk holds.
    __device__ __forceinline__ void products(const TQ *sk, f32x16 (&s)[2]) {
        const int l32 = threadIdx.x & 31, hf = (threadIdx.x >> 5) & 1;
        s[0] = s[1] = f32x16{};
#pragma unroll
        for (int kk = 0; kk < KS; kk++)
#pragma unroll
            for (int st = 0; st < 2; st++) {
                const TQ *row = sk + (32 * st + l32) * KROW + 16 * kk + 8 * hf;
                const q8 a = *(const q8 *)row;
                if constexpr (QT == 2) s[st] = mfma32(a, q[1][kk], s[st]);
                s[st] = mfma32(a, q[0][kk], s[st]);
            }
    }

    // From the products to weights exp2(c s + nm) (c is returned), the offset raised
    // where one asks for it.  The 32 NS keys are those from position j0 on; kscale: one
    // scale for the tile, or (PER_KEY) sks[key]; cut: keys from `seen` on are not seen.
    template <bool PER_KEY, int NS>
    __device__ __forceinline__ float scores(f32x16 (&s)[NS], const Score &sc, float kscale, const float *sks, int j0,
                                            bool cut, int seen, float &nm) {
        const int hf = (threadIdx.x >> 5) & 1;
        if constexpr (PER_KEY) {
#pragma unroll
            for (int st = 0; st < NS; st++)
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    const f32x4 ks = *(const f32x4 *)(sks + 32 * st + 8 * g + 4 * hf);
#pragma unroll
                    for (int v = 0; v < 4; v++) s[st][4 * g + v] *= ks[v];
                }
        }
        float c = factor(f * kscale);  // t = c s, unless there is more to do
        // (two loops and two branches: in one loop both would be computed and selected)
        if (sc.cap2) {
            if (sc.fine) {
#pragma unroll
                for (int st = 0; st < NS; st++)
#pragma unroll
                    for (int v = 0; v < 16; v++) s[st][v] = capped_fine(s[st][v] * c, sc.cap2);
            } else {
#pragma unroll
                for (int st = 0; st < NS; st++)
#pragma unroll
                    for (int v = 0; v < 16; v++) s[st][v] = capped(s[st][v] * c, sc.cap2);
            }
            c = 1.f;
        }
        if (sc.bias) {
            const float far = (float)(pos - j0 - 4 * hf);
            if (!__ballot(pos < j0 + 32 * NS - 1)) {  // no row has a key behind it
                const float at = -slope2 * far;
#pragma unroll
                for (int st = 0; st < NS; st++)
#pragma unroll
                    for (int v = 0; v < 16; v++)
                        s[st][v] = fmaf(s[st][v], c, fmaf(slope2, (float)(32 * st + 8 * (v >> 2) + (v & 3)), at));
            } else {
#pragma unroll
                for (int st = 0; st < NS; st++)
#pragma unroll
                    for (int v = 0; v < 16; v++)
                        s[st][v] = fmaf(-slope2, fabsf(far - (float)(32 * st + 8 * (v >> 2) + (v & 3))), s[st][v] * c);
            }
            c = 1.f;
        }
        if (cut) {
            const int left = seen - j0 - 4 * hf;
#pragma unroll
            for (int st = 0; st < NS; st++)
#pragma unroll
                for (int v = 0; v < 16; v++) s[st][v] = left > 32 * st + 8 * (v >> 2) + (v & 3) ? s[st][v] : -INFINITY;
        }
        float mt = fmaxf(s[0][0], s[NS - 1][15]);
#pragma unroll
        for (int i = 1; i < 16 * NS - 1; i += 2) mt = fmaxf(fmaxf(mt, s[i >> 4][i & 15]), s[(i + 1) >> 4][(i + 1) & 15]);
        nm = -m;
        const uint64_t up = __ballot(fmaf(mt, c, -m) - lo > RAISE);
        if (up | far) {  // wave-uniform
            if (up) {
                mt = max32(mt);
                const float t = mt * c, off = fmaf(mt, c, -t) - OFFSET;
                const bool raise = fmaf(mt, c, -m) - lo > RAISE, two = fabsf(t) >= FAR;
                const float now = two ? t : t - OFFSET, rest = two ? off : 0.f;
                const float keep = raise ? __builtin_amdgcn_exp2f((m - now) + (lo - rest)) : 1.f;
                m = raise ? now : m;
                lo = raise ? rest : lo;
                nm = -m;
                far = __ballot(fabsf(m) >= FAR && m != M_NONE);
                l *= keep;
#pragma unroll
                for (int i = 0; i < DB; i++) o[i] *= keep;
            }
            if (far) {
#pragma unroll
                for (int st = 0; st < NS; st++)
#pragma unroll
                    for (int v = 0; v < 16; v++) s[st][v] = fmaf(s[st][v], c, -m) - lo;
                c = 1.f, nm = 0.f;
            }
        }
        return c;
    }

    // The weights exp2(c s + nm) as the second product's operand, and their sum.  16-bit V takes
    // weights of its own type, one term: a second one would double that product, and the
    // rounding (half a step of the type, r.m.s. a tenth to a third more error than fp32 weights
    // leave after the output's own rounding) is the caller's choice of type.
    __device__ __forceinline__ void weights(const f32x16 (&s)[2], float c, float nm, p8 (&pf)[QT][4]) {
        float sum[2] = {};
#pragma unroll
        for (int tt = 0; tt < 4; tt++) {
            float p[8];
#pragma unroll
            for (int e = 0; e < 8; e++) p[e] = __builtin_amdgcn_exp2f(fmaf(s[tt >> 1][8 * (tt & 1) + e], c, nm));
            if constexpr (QT == 2) {
                u32x4 h, l4;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    uint32_t hi, lo;
                    split2(p[2 * e], p[2 * e + 1], 1.f, hi, lo);
                    h[e] = hi, l4[e] = lo;
                    sum[0] += p[2 * e], sum[1] += p[2 * e + 1];
                }
                pf[0][tt] = __builtin_bit_cast(p8, h), pf[QT - 1][tt] = __builtin_bit_cast(p8, l4);
            } else {  // the sum is of the rounded weights, which the product takes
                u32x4 w;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    w[e] = Vec<TP>::pair(p[2 * e], p[2 * e + 1]);
                    sum[e & 1] = Vec<TP>::sum(w[e], sum[e & 1]);
                }
                pf[0][tt] = __builtin_bit_cast(p8, w);
            }
        }
        l += sum[0] + sum[1];
    }
};

}  // namespace

#endif
