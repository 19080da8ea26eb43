// fh3_seqs.hip -- attention within packed sequences (fh3_hip_attention_seqs_dev).
#include "fh3_tile.h"

namespace {

// How the three value types enter the matrix products.
template <int TY> struct Operand;
template <> struct Operand<0> { typedef _Float16 TQ, TP; static constexpr int T = 1, NW = 4, TYPE = FH3K_F16; };
template <> struct Operand<1> { typedef __bf16 TQ, TP; static constexpr int T = 1, NW = 4, TYPE = FH3K_BF16; };
// fp32 as two 16-bit terms: q and k fp16 after a power of two for each row (22
// bits), v and the weights bf16 (16 bits, any exponent); three products each
template <> struct Operand<2> {
    typedef _Float16 TQ;
    typedef __bf16 TP;
    static constexpr int T = 2, NW = 8, TYPE = FH3K_F32;
};

// A tile of K and V in LDS: T planes of K [64][HD + 8], of V [64][HD + 32] (the
// transposing reads take 4 rows x 64 bytes at once: rows 64 bytes apart modulo the
// banks), and for fp32 one factor per key.
template <int HD, int TY> struct TileLds {
    static constexpr int T = Operand<TY>::T, KROW = HD + 8, VROW = HD + 32;
    uint16_t k[T][TILE_K][KROW];
    uint16_t v[T][TILE_K][VROW];
    float ks[T == 2 ? TILE_K : 4];
};

// V^T operand of channels 32 db .. and keys 16 tt ..: two transposing reads of
// four keys each; lane gets channel 32 db + (lane & 31), keys 16 tt + 4 hf + 0..3
// and 16 tt + 8 + 4 hf + 0..3, the order of the first product's accumulator.
template <class V8, int VROW> __device__ __forceinline__ V8 v_frag(const uint16_t *sv, int db, int tt) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s4 *lds4;
    const int lane = threadIdx.x & 63, i = lane & 15, hf = lane >> 5;
    const uint16_t *at = sv + (16 * tt + 4 * hf + (i >> 2)) * VROW + 32 * db + 16 * ((lane >> 4) & 1) + 4 * (i & 3);
    struct { s4 a, b; } w;
    w.a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(at));
    w.b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(at + 8 * VROW));
    return __builtin_bit_cast(V8, w);
}

template <int CTRL> __device__ __forceinline__ float dpp_max(float x) {
    const int y = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xF, 0xF, true);
    return fmaxf(x, __builtin_bit_cast(float, y));
}
// The largest of N = 16 or 32 neighbouring lanes' values, in all of them.
template <int N> __device__ __forceinline__ float row_max(float x) {
    x = dpp_max<0xB1>(x);   // quad_perm 1 0 3 2
    x = dpp_max<0x4E>(x);   // quad_perm 2 3 0 1
    x = dpp_max<0x141>(x);  // row_half_mirror
    x = dpp_max<0x140>(x);  // row_mirror
    return N == 32 ? fmaxf(x, __shfl_xor(x, 16)) : x;
}

// Whether any of 16 bytes of values is infinite or NaN (all exponent bits set);
// those become 0.
template <int TYPE> __device__ __forceinline__ bool not_finite(u32x4 &w) {
    bool any = false;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (TYPE == FH3K_F32) {
            const bool b = (w[i] & 0x7F800000u) == 0x7F800000u;
            w[i] = b ? 0 : w[i];
            any = any || b;
        } else {
            constexpr uint32_t E = TYPE == FH3K_BF16 ? 0x7F80u : 0x7C00u;
            const bool a = (w[i] & E) == E, b = (w[i] >> 16 & E) == E;
            w[i] &= (a ? 0xFFFF0000u : ~0u) & (b ? 0xFFFFu : ~0u);
            any = any || a || b;
        }
    }
    return any;
}

template <int HD, int TY>
__global__ __launch_bounds__(64 * Operand<TY>::NW, 2) void k_attn_seqs(
    Fh3kAttn a, const void *__restrict__ q, int64_t ldq, const void *__restrict__ k, int64_t ldk,
    const void *__restrict__ v, int64_t ldv, void *__restrict__ o, int64_t ldo, Fh3kSeqs s,
    const int *__restrict__ prefix, int tiles) {
    typedef Operand<TY> Op;
    typedef typename Op::TQ TQ;
    typedef typename Op::TP TP;
    constexpr int T = Op::T, NT = 64 * Op::NW, ROWS = WAVE_R * Op::NW;
    typedef Rows<HD, TQ, TP, T, T> R;
    typedef typename R::p8 p8;
    typedef TileLds<HD, TY> Lds;
    __shared__ __align__(16) Lds lds[2];
    __shared__ int lost;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, hf = lane >> 5;
    // workgroups next to each other run on different XCDs: with the key head as
    // the fastest index an XCD keeps to few heads' K and V.  The last rows of a
    // sequence see most keys and go first.
    const int kvh = blockIdx.x % a.kv_heads, G = a.heads / a.kv_heads;
    int seq, first, cnt;
    int at;
    if (!find_unit(tiles - 1 - (int)blockIdx.x / a.kv_heads, s.n_seq, [&](int i) {
            int b, n;
            seq_rows(s, i, b, n);
            return (n * G + ROWS - 1) / ROWS;
        }, seq, at))
        return;
    seq_rows(s, seq, first, cnt);
    const int rows = cnt * G, r0 = at * ROWS;
    int pre = a.causal ? (prefix ? prefix[seq] : 0) : cnt;
    pre = pre < cnt ? pre : cnt;
    auto limit = [&](int i) { return i + 1 > pre ? i + 1 : pre; };  // keys that token i sees

    const int row = r0 + WAVE_R * wave + l32, rc = row < rows ? row : rows - 1;
    const int tok = rc / G, head = kvh * G + rc % G;
    const Score sc = score_of(a);
    R w;
    w.template load_q<TY == 2>(q, Op::TYPE, (int64_t)(first + tok) * ldq + head * HD, sc);
    w.clear();
    w.pos = tok;
    w.lim = limit(tok);
    w.slope2 = sc.bias ? a.slopes[head] * LOG2E : 0.f;
    const bool active = r0 + WAVE_R * wave < rows;
    const int lo = __builtin_amdgcn_readfirstlane(w.lim), hi = __builtin_amdgcn_readlane(w.lim, 31);
    const int last = r0 + ROWS < rows ? r0 + ROWS - 1 : rows - 1;
    const int end = limit(last / G);
    const int n_tiles = (end + TILE_K - 1) / TILE_K;

    // The next tile's rows, on their way from memory while this one is in work.
    constexpr int VAL = TY == 2 ? 4 : 8, CPR = HD / VAL, CH = TILE_K * CPR / NT;  // 16-byte pieces
    u32x4 rk[CH], rv[CH];
    const char *kp = (const char *)k + ((int64_t)first * ldk + kvh * HD) * (16 / VAL);
    const char *vp = (const char *)v + ((int64_t)first * ldv + kvh * HD) * (16 / VAL);
    uint32_t ko[CH], vo[CH];  // of this thread's pieces in a tile
#pragma unroll
    for (int i = 0; i < CH; i++) {
        const int c = tid + i * NT;
        ko[i] = ((uint32_t)(c / CPR) * (uint32_t)ldk + c % CPR * VAL) * (16 / VAL);
        vo[i] = ((uint32_t)(c / CPR) * (uint32_t)ldv + c % CPR * VAL) * (16 / VAL);
    }
    auto load = [&](int j0) {
        const char *kt = kp + j0 * ldk * (16 / VAL), *vt = vp + j0 * ldv * (16 / VAL);
        if (j0 + TILE_K <= cnt) {
#pragma unroll
            for (int i = 0; i < CH; i++) rk[i] = *(const u32x4 *)(kt + ko[i]), rv[i] = *(const u32x4 *)(vt + vo[i]);
        } else {  // past the sequence its last row again: no row sees those keys
#pragma unroll
            for (int i = 0; i < CH; i++) {
                const int c = tid + i * NT, key = j0 + c / CPR < cnt ? c / CPR : cnt - 1 - j0;
                rk[i] = *(const u32x4 *)(kt + (key * ldk + c % CPR * VAL) * (16 / VAL));
                rv[i] = *(const u32x4 *)(vt + (key * ldv + c % CPR * VAL) * (16 / VAL));
            }
        }
    };
    // A value that is not finite must not reach rows that do not see it (their
    // weight of 0 would make it NaN): in tiles that some row sees in part it enters
    // as 0, and the rows that do see it are put right at the end.
    const int whole = limit(r0 / G);  // keys that every row of the workgroup sees
    auto store = [&](Lds &t, int j0) {
        if (j0 + TILE_K > whole) {
            bool any = false;
#pragma unroll
            for (int i = 0; i < CH; i++) any = not_finite<Op::TYPE>(rv[i]) || any;
            if (any) lost = 1;
        }
#pragma unroll
        for (int i = 0; i < CH; i++) {
            const int c = tid + i * NT, key = c / CPR, d = c % CPR * VAL;
            if constexpr (TY != 2) {
                *(u32x4 *)&t.k[0][key][d] = rk[i];
                *(u32x4 *)&t.v[0][key][d] = rv[i];
            } else {
                const f32x4 x = __builtin_bit_cast(f32x4, rk[i]), y = __builtin_bit_cast(f32x4, rv[i]);
                float top = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
                top = row_max<CPR>(top);
                const float up = pow2_to_14(top);
                if (c % CPR == 0) t.ks[key] = 1.f / up;
                TQ kh[4], kl[4];
                TP vh[4], vl[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const Two<TQ> kt = split<TQ>(x[e] * up);
                    const Two<TP> vt = split<TP>(y[e]);
                    kh[e] = kt.hi, kl[e] = kt.lo, vh[e] = vt.hi, vl[e] = vt.lo;
                }
                *(u32x2 *)&t.k[0][key][d] = *(const u32x2 *)kh;
                *(u32x2 *)&t.k[T - 1][key][d] = *(const u32x2 *)kl;
                *(u32x2 *)&t.v[0][key][d] = *(const u32x2 *)vh;
                *(u32x2 *)&t.v[T - 1][key][d] = *(const u32x2 *)vl;
            }
        }
    };

    if (tid == 0) lost = 0;
    load(0);
    __syncthreads();
    store(lds[0], 0);
    __syncthreads();
    for (int e = 0; e < n_tiles; e++) {
        const Lds &t = lds[e & 1];
        const int j0 = e * TILE_K;
        if (e + 1 < n_tiles) load(j0 + TILE_K);
        if (active && j0 < hi) {
            const bool cut = j0 + TILE_K > lo;  // some row does not see all of it
            p8 pf[T][4];
            w.template weigh<TY == 2>((const TQ *)&t.k[0][0][0], sc, 1.f, t.ks, j0, cut, w.lim, pf);
#pragma unroll
            for (int db = 0; db < R::DB; db++)
#pragma unroll
                for (int tt = 0; tt < 4; tt++) {
                    const p8 x = v_frag<p8, Lds::VROW>(&t.v[0][0][0], db, tt);
                    if constexpr (T == 2) {
                        w.o[db] = mfma32(v_frag<p8, Lds::VROW>(&t.v[T - 1][0][0], db, tt), pf[0][tt], w.o[db]);
                        w.o[db] = mfma32(x, pf[T - 1][tt], w.o[db]);
                    }
                    w.o[db] = mfma32(x, pf[0][tt], w.o[db]);
                }
        }
        if (e + 1 < n_tiles) store(lds[(e & 1) ^ 1], j0 + TILE_K);
        __syncthreads();
    }

    if (lost) {
        for (int j = whole & ~(TILE_K - 1); j < end; j++)
            if (j < w.lim)
#pragma unroll
                for (int db = 0; db < R::DB; db++)
#pragma unroll
                    for (int g = 0; g < 4; g++) {
                        const int64_t at_v = (first + j) * ldv + kvh * HD + 32 * db + 8 * g + 4 * hf;
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const float x = value_at(v, Op::TYPE, at_v + i);
                            if (!(fabsf(x) <= 3.402823466e38f)) w.o[db][4 * g + i] = __builtin_nanf("");
                        }
                    }
    }
    const float l = w.l + half_swap(w.l), inv = l == 0.f ? 0.f : 1.f / l;
    if (row < rows) {
        const int64_t at_o = (int64_t)(first + tok) * ldo + head * HD;
#pragma unroll
        for (int db = 0; db < R::DB; db++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                f32x4 x;
#pragma unroll
                for (int i = 0; i < 4; i++) x[i] = w.o[db][4 * g + i] * inv;
                store4(o, Op::TYPE, at_o + 32 * db + 8 * g + 4 * hf, x);
            }
    }
}

template <int HD, int TY>
hipError_t launch_seqs(const Fh3kAttn &a, const void *q, int64_t ldq, const void *k, int64_t ldk, const void *v,
                       int64_t ldv, void *o, int64_t ldo, const Fh3kSeqs &s, const int *prefix, hipStream_t st) {
    constexpr int NW = Operand<TY>::NW, ROWS = WAVE_R * NW;
    const int64_t G = a.heads / a.kv_heads;
    // tiles of all sequences at most: each may have one that is not full
    const int64_t tiles = s.first ? s.n_tok * G / ROWS + (s.n_seq < s.n_tok ? s.n_seq : s.n_tok)
                                  : (int64_t)s.n_seq * ((s.n_tok / s.n_seq * G + ROWS - 1) / ROWS);
    if (tiles * a.kv_heads > 0x7FFFFF) return hipErrorInvalidValue;
    hipLaunchKernelGGL((k_attn_seqs<HD, TY>), dim3((unsigned)(tiles * a.kv_heads)), dim3(64 * NW), 0, st, a, q, ldq, k,
                       ldk, v, ldv, o, ldo, s, prefix, (int)tiles);
    return hipGetLastError();
}

}  // namespace

extern "C" hipError_t fh3k_attn_seqs(const Fh3kAttn *a, const void *q, int64_t ldq, const void *k, int64_t ldk,
                                     const void *v, int64_t ldv, void *o, int64_t ldo, Fh3kSeqs s, const int *prefix,
                                     hipStream_t st) {
#define FH3K_SEQS(HD, TY) launch_seqs<HD, TY>(*a, q, ldq, k, ldk, v, ldv, o, ldo, s, prefix, st)
    if (a->hd == 128)
        return a->type == FH3K_F16 ? FH3K_SEQS(128, 0) : a->type == FH3K_BF16 ? FH3K_SEQS(128, 1) : FH3K_SEQS(128, 2);
    return a->type == FH3K_F16 ? FH3K_SEQS(64, 0) : a->type == FH3K_BF16 ? FH3K_SEQS(64, 1) : FH3K_SEQS(64, 2);
#undef FH3K_SEQS
}
