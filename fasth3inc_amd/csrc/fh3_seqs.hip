// fh3_seqs.hip -- attention within packed sequences (fh3_hip_attention_seqs_dev).
#include "fh3_tile.h"

namespace {

// How the three value types enter the matrix products.
template <int TY> struct Operand;
template <> struct Operand<0> { typedef _Float16 TQ, TP; static constexpr int TYPE = FH3K_F16; };
template <> struct Operand<1> { typedef __bf16 TQ, TP; static constexpr int TYPE = FH3K_BF16; };
// fp32 as two fp16 terms (22 bits) after a power of two for each row of q, k and
// v; three products each
template <> struct Operand<2> { typedef _Float16 TQ, TP; static constexpr int TYPE = FH3K_F32; };

// Tiles of fp32 K and V in LDS: two planes of K [32][HD + 8], of V [32][HD + 32] (the
// transposing reads take 4 rows x 64 bytes at once: rows 64 bytes apart modulo the
// banks).
constexpr int TILE_32 = 32;
template <int HD> struct KLds {
    static constexpr int ROW = HD + 8;
    uint16_t x[2][TILE_32][ROW];
};
template <int HD> struct VLds {
    static constexpr int ROW = HD + 32;
    uint16_t x[2][TILE_32][ROW];
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
    return N == 32 ? max16(x) : x;
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

struct SeqsArgs {
    Fh3kAttn a;
    const void *q, *k, *v;
    void *o;
    int64_t ldq, ldk, ldv, ldo;
    Fh3kSeqs s;
    const int *prefix;
    int tiles;  // of all sequences at most
};

// A workgroup's tile of rows.
struct Place {
    int kvh, G, first, cnt, rows, r0;
    int pre;  // tokens that every row sees
    __device__ __forceinline__ int limit(int tok) const { return tok + 1 > pre ? tok + 1 : pre; }  // keys that it sees
};
// Workgroups next to each other run on different XCDs: with the key head as the
// fastest index an XCD keeps to few heads' K and V.  The last rows of a sequence see
// most keys and go first.
template <int ROWS> __device__ __forceinline__ bool place(const SeqsArgs &g, Place &p) {
    p.kvh = blockIdx.x % g.a.kv_heads;
    p.G = g.a.heads / g.a.kv_heads;
    int seq, at, b = 0, n = 0, pre = 0;
    if (!find_unit(g.tiles - 1 - (int)blockIdx.x / g.a.kv_heads, g.s.n_seq, [&](int i) {
            if (g.a.causal && g.prefix) pre = g.prefix[i];
            seq_rows(g.s, i, b, n);
            return (n * p.G + ROWS - 1) / ROWS;
        }, seq, at))
        return false;
    p.first = of_lane(b, seq);
    p.cnt = of_lane(n, seq);
    pre = g.a.causal ? of_lane(pre, seq) : p.cnt;
    p.rows = p.cnt * p.G;
    p.r0 = at * ROWS;
    p.pre = pre < p.cnt ? pre : p.cnt;
    return true;
}

// A value that is not finite must not reach rows that do not see it (their weight
// of 0 would make it NaN): in tiles that some row of the workgroup sees only in part
// it enters as 0, and here the channels of the rows that do see it are lost.
template <int HD, int TYPE, class R>
__device__ __forceinline__ void lose(R &w, const SeqsArgs &g, const Place &p, int from, int to) {
    const int hf = (threadIdx.x >> 5) & 1;
    uint64_t gone = 0;
    for (int j = from; j < to; j++)
        if (j < w.lim)
#pragma unroll 1
            for (int c = 0; c < HD / 8; c++)
                for (int i = 0; i < 4; i++) {
                    const float x = value_at(g.v, TYPE, (p.first + j) * g.ldv + p.kvh * HD + 8 * c + 4 * hf + i);
                    gone |= (uint64_t)!(fabsf(x) <= 3.402823466e38f) << (4 * c + i);
                }
    if (__ballot(gone != 0)) {
#pragma unroll
        for (int db = 0; db < R::DB; db++)
#pragma unroll
            for (int v = 0; v < 16; v++) w.o[db][v] = gone >> (16 * db + v) & 1 ? __builtin_nanf("") : w.o[db][v];
    }
}

template <int HD, int TYPE, class R>
__device__ __forceinline__ void put_rows(const R &w, const SeqsArgs &g, const Place &p, int row, int head, float unit) {
    const int hf = (threadIdx.x >> 5) & 1;
    const float l = sum32(w.l), inv = l == 0.f ? 0.f : 1.f / l;
    if (row >= p.rows) return;
    const int64_t at = (int64_t)(p.first + w.pos) * g.ldo + head * HD + 4 * hf;
#pragma unroll
    for (int db = 0; db < R::DB; db++)
#pragma unroll
        for (int c = 0; c < 4; c++) {
            f32x4 x;
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = w.o[db][4 * c + i] * inv * unit;  // (unit / l could leave fp32's range)
            store4(g.o, TYPE, at + 32 * db + 8 * c, x);
        }
}

// Two halves of the workgroup that took every other tile of keys: the second's sums
// go through LDS (in a and b, DB / 2 blocks of 16 KB each; offsets, sums of weights
// and units in c) to the first.
template <class R>
__device__ __forceinline__ void join_halves(R &w, float &unit, float first, int half, int wave, char *a, char *b, char *c) {
    const int lane = threadIdx.x & 63;
    float *ml = (float *)c + wave * 64 + lane;
    auto at = [&](int db, int q) {
        return (f32x4 *)((db < R::DB / 2 ? a : b) + db % (R::DB / 2) * 16384) + (q * 4 + wave) * 64 + lane;
    };
    __syncthreads();
    if (half) {
        ml[0] = w.m, ml[256] = w.l, ml[512] = unit, ml[768] = w.lo;
#pragma unroll
        for (int db = 0; db < R::DB; db++)
#pragma unroll
            for (int q = 0; q < 4; q++) *at(db, q) = f32x4{w.o[db][4 * q], w.o[db][4 * q + 1], w.o[db][4 * q + 2], w.o[db][4 * q + 3]};
    }
    __syncthreads();
    if (half) return;
    const float other = ml[512];
    float x, y;
    join_offsets(w.m, w.lo, ml[0], ml[768], x, y);
    // (a half that saw nothing has no say in the unit)
    const float mine = unit >= 0.f ? unit : max32(w.l) > 0.f ? first : 0.f, its = other >= 0.f ? other : max32(ml[256]) > 0.f ? first : 0.f;
    const float u = fmaxf(mine, its), ox = u > 0.f ? x * (mine / u) : 0.f, oy = u > 0.f ? y * (its / u) : 0.f;
    unit = u;
    w.l = w.l * x + ml[256] * y;
#pragma unroll
    for (int db = 0; db < R::DB; db++)
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const f32x4 z = *at(db, q);
#pragma unroll
            for (int i = 0; i < 4; i++) w.o[db][4 * q + i] = w.o[db][4 * q + i] * ox + z[i] * oy;
        }
}

// F16 and BF16.  K and V go from memory to LDS without registers (16 bytes a lane),
// rows unpadded, their 16-byte (K) or 64-byte (V) pieces permuted by the row
// so that the reads meet no bank twice.  The next tile's scores are computed
// while this one's weights are (matrix and vector instructions alternate), so K
// is a tile ahead of V.  Bound by the matrix cores at the clock that the power
// limit leaves: 8192 tokens x 64 heads bf16 1.03-1.11 ms, 1.0 PFLOP/s, where the
// library's large product reaches 1.2 (through registers and one product after
// the other 1.28 ms); capped scores and hd 64 by vector instructions: 5.8 to a matrix
// instruction there, 14 with the tanh (a fifth of them exponentials and reciprocals; 24
// documents 109 us), 21 at hd 64 with the distance bias (half the matrix work for the same
// softmax; 48 us).
template <int HD, int TY>
__global__ __launch_bounds__(256, 2) void k_attn_seqs16(SeqsArgs g) {
    typedef Operand<TY> Op;
    typedef typename Op::TQ T;
    constexpr int NW = 4, ROWS = WAVE_R * NW, RB = HD * 2, TILE_B = TILE_K * RB, PPR = RB / 16;  // pieces per row
    constexpr int CH = TILE_B / (1024 * NW);  // a wavefront's loads of a tile
    typedef Rows<HD, T, T, 1> R;
    typedef typename R::q8 v8;
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s4 *lds4;
    typedef __attribute__((address_space(3))) void lds_void;
    // Four arrays, not one: reads of one then need not wait for the loads into another.
    __shared__ __align__(16) char sk0[TILE_B], sk1[TILE_B], sv0[TILE_B], sv1[TILE_B];
    __shared__ int lost;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, hf = lane >> 5;
    Place p;
    if (!place<ROWS>(g, p)) return;
    if (tid == 0) lost = 0;
    __syncthreads();

    // DMA: lane's piece of the wavefront's 1024 bytes i: row (CH wave + i) (64 / PPR) + lane / PPR
    int ko[CH], vo[CH];  // its offset in a tile of K and V
#pragma unroll
    for (int i = 0; i < CH; i++) {
        const int r = (CH * wave + i) * (64 / PPR) + lane / PPR, at = lane % PPR;
        ko[i] = (r * (int)g.ldk + 8 * (HD == 128 ? at ^ (r & 15) : at ^ ((r >> 1) & 7))) * 2;
        vo[i] = (r * (int)g.ldv + 8 * (HD == 128 ? at ^ ((r & 3) << 2) : at ^ ((r & 2) << 1))) * 2;
    }
    auto dma = [&](const void *x, int64_t ld, const int (&o)[CH], int j0, char *to) {
        const char *base = (const char *)x + ((p.first + j0) * ld + p.kvh * HD) * 2;
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, 0xFFFFFFFF, 0x00020000);
        const int rows = p.cnt - j0;
        auto get = [&](int i, int at) {
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void *)(to + (CH * wave + i) * 1024), 16, at, 0, 0, 0);
        };
        if (rows >= TILE_K) {
#pragma unroll
            for (int i = 0; i < CH; i++) get(i, o[i]);
        } else {  // past the sequence its last row again: no row sees those keys
#pragma unroll
            for (int i = 0; i < CH; i++) {
                const int over = (CH * wave + i) * (64 / PPR) + lane / PPR - rows + 1;
                get(i, o[i] - (over > 0 ? over * (int)ld * 2 : 0));
            }
        }
    };
    auto load_k = [&](int e, char *to) { dma(g.k, g.ldk, ko, e * TILE_K, to); };
    auto load_v = [&](int e, char *to) { dma(g.v, g.ldv, vo, e * TILE_K, to); };
    const int whole = p.limit(p.r0 / p.G);  // keys that every row sees
    const int last = p.r0 + ROWS < p.rows ? p.r0 + ROWS - 1 : p.rows - 1;
    const int end = p.limit(last / p.G), n_tiles = (end + TILE_K - 1) / TILE_K;
    load_k(0, sk0);
    load_v(0, sv0);
    if (n_tiles > 1) load_k(1, sk1);

    const int row = p.r0 + WAVE_R * wave + l32, rc = row < p.rows ? row : p.rows - 1;
    const int tok = rc / p.G, head = p.kvh * p.G + rc % p.G;
    const Score sc = score_of(g.a);
    R w;
    w.template load_q<false>(g.q, Op::TYPE, (int64_t)(p.first + tok) * g.ldq + head * HD, sc);
    w.clear();
    w.pos = tok;
    w.lim = p.limit(tok);
    w.slope2 = sc.bias ? g.a.slopes[head] * LOG2E : 0.f;
    const bool active = p.r0 + WAVE_R * wave < p.rows;
    const int lo = __builtin_amdgcn_readfirstlane(w.lim);
    const int hi = active ? __builtin_amdgcn_readlane(w.lim, 31) : 0;

    const int k_at = l32 * RB + ((hf ^ (HD == 128 ? l32 & 15 : (l32 >> 1) & 7)) << 4);
    auto products = [&](const char *b, f32x16 (&s)[2]) {
        s[0] = s[1] = f32x16{};
#pragma unroll
        for (int kk = 0; kk < R::KS; kk++) {
            const char *at = b + (k_at ^ (kk << 5));
#pragma unroll
            for (int st = 0; st < 2; st++) s[st] = mfma32(*(const v8 *)(at + 32 * st * RB), w.q[0][kk], s[st]);
        }
    };
    // V^T operand of channels 32 db .. and keys 16 tt ..: two transposing reads of
    // four keys each; the lane gets channel 32 db + l32, keys 16 tt + 4 hf + 0..3
    // and 16 tt + 8 + 4 hf + 0..3, the order of the first product's accumulator.
    const int v_at = (4 * hf + ((lane & 15) >> 2)) * RB + ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
    const int v_x = HD == 128 ? (lane & 15) >> 2 : (lane >> 3) & 1;
    auto product2 = [&](const char *b, const v8 (&pf)[1][4]) {
#pragma unroll
        for (int db = 0; db < R::DB; db++) {
            const char *at = b + v_at + ((db ^ v_x) << 6);
#pragma unroll
            for (int tt = 0; tt < 4; tt++) {
                struct { s4 a, b; } x;
                x.a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(at + 16 * tt * RB));
                x.b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(at + (16 * tt + 8) * RB));
                w.o[db] = mfma32(__builtin_bit_cast(v8, x), pf[0][tt], w.o[db]);
            }
        }
    };
    // a wavefront's own pieces of V's tile e, once they are there
    auto clean_v = [&](int e, char *b) {
        if ((e + 1) * TILE_K <= whole) return;
        bool any = false;
#pragma unroll 1
        for (int i = 0; i < CH; i++) {
            u32x4 *at = (u32x4 *)(b + (CH * wave + i) * 1024 + 16 * lane);
            u32x4 x = *at;
            if (not_finite<Op::TYPE>(x)) *at = x, any = true;
        }
        if (any) lost = 1;
    };
    auto wait = [&](int e, char *b) {  // for tile e of V and e + 1 of K
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
        clean_v(e, b);
        __syncthreads();
    };

    f32x16 s0[2], s1[2];
    auto step = [&](int e, f32x16 (&s)[2], f32x16 (&next)[2], char *ke, char *kn, char *ve, char *vn) {
        const int j0 = e * TILE_K;
        if (e + 2 < n_tiles) load_k(e + 2, ke);
        if (e + 1 < n_tiles) load_v(e + 1, vn);
        if (j0 < hi) {
            v8 pf[1][4];
            float nm;
            const float c = w.template scores<false>(s, sc, 1.f, nullptr, j0, j0 + TILE_K > lo, w.lim, nm);
            products(kn, next);  // past the last tile: what is there, not used
            w.weights(s, c, nm, pf);
            product2(ve, pf);
            constexpr int M1 = 2 * R::KS, M2 = 4 * R::DB;  // matrix instructions of the two products
            __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);  // LDS reads, four ahead
#pragma unroll
            for (int i = 0; i < M1; i++) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);        // matrix
                __builtin_amdgcn_sched_group_barrier(0x402, 96 / M1, 0);  // vector
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                if (i >= M1 - 4) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
#pragma unroll
            for (int i = 0; i < M2; i++) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
            }
        }
        if (e + 1 < n_tiles) wait(e + 1, vn);
    };
    wait(0, sv0);
    if (hi > 0) products(sk0, s0);
    __syncthreads();  // before the third tile's K takes the first's place
    for (int e = 0; e < n_tiles; e += 2) {
        step(e, s0, s1, sk0, sk1, sv0, sv1);
        if (e + 1 < n_tiles) step(e + 1, s1, s0, sk1, sk0, sv1, sv0);
    }
    if (lost) lose<HD, Op::TYPE>(w, g, p, whole & ~(TILE_K - 1), end);
    put_rows<HD, Op::TYPE>(w, g, p, row, head, 1.f);
}

// F32: every operand is two fp16 terms, made on the way to LDS: the terms of the
// next V beside the first product, the weights and the terms of the next K beside
// the second.  (V and weights as two bf16 terms, which need no power of two, took 46 us at
// 600 tokens where fp16 took 49-51, but are 4e-6 off for 3e-7.)  Tiles of 32 keys, so that two
// workgroups fit a CU and nothing has to be moved to accumulation registers (64 keys,
// one workgroup: 600 tokens x 64 heads 52.6 us; a third of the instructions were such
// moves).  KH = 2: eight wavefronts, two to a SIMD, each four with every other tile of keys.
// 600 tokens x 64 heads 48.5 us: 12 vector instructions to a matrix instruction, the terms
// for the most part, made anew for each of 38 tiles of rows; matrix pipe busy 14 %.  At hd
// 128 24 to 26 registers spill (LDS addresses, read back once a step).
template <int HD, int KH>
__global__ __launch_bounds__(256 * KH, 2) void k_attn_seqs32(SeqsArgs g) {
    typedef Operand<2> Op;
    typedef Op::TQ TQ;
    typedef Op::TP TP;
    constexpr int NT = 256, ROWS = WAVE_R * 4;
    typedef Rows<HD, TQ, TP, 2> R;
    typedef typename R::p8 p8;
    typedef KLds<HD> LK;
    typedef VLds<HD> LV;
    // (arrays of their own, so that writes to one need not wait for reads of another)
    __shared__ __align__(16) LK lk0[KH], lk1[KH];
    __shared__ __align__(16) LV lv0[KH], lv1[KH];
    __shared__ __align__(16) float ks0[KH][2 * TILE_32], ks1[KH][2 * TILE_32];  // each key's factor; the other half is not read
    __shared__ __align__(16) float vs0[KH][2 * TILE_32], vs1[KH][2 * TILE_32];
    __shared__ int lost, odd;  // odd: some factor of V so far is not 1 / V_UP

    const int tid = threadIdx.x % NT, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int half = KH == 2 ? __builtin_amdgcn_readfirstlane(threadIdx.x / NT) : 0;
    const int l32 = lane & 31;
    Place p;
    if (!place<ROWS>(g, p)) return;
    if (tid == 0) lost = odd = 0;

    constexpr int CPR = HD / 4, CH = TILE_32 * CPR / NT;  // 16-byte pieces of a row; of a tile, to a thread
    const int key0 = tid / CPR, d0 = tid % CPR * 4;      // the first; the others NT / CPR keys on
    const int whole = p.limit(p.r0 / p.G);               // keys that every row sees
    const int last = p.r0 + ROWS < p.rows ? p.r0 + ROWS - 1 : p.rows - 1;
    const int end = p.limit(last / p.G), n_tiles = (end + TILE_32 - 1) / TILE_32;
    auto load = [&](const void *x, int64_t ld, int e, u32x4 (&r)[CH]) {
        const float *base = (const float *)x + (p.first + e * TILE_32) * ld + p.kvh * HD;
        const int keys = p.cnt - e * TILE_32;  // past the sequence its last row again: no row sees those keys
#pragma unroll
        for (int i = 0; i < CH; i++) {
            int key = key0 + i * (NT / CPR);
            if (keys < TILE_32) key = key < keys ? key : keys - 1;
            r[i] = *(const u32x4 *)(base + (uint32_t)((uint32_t)key * (uint32_t)ld + d0));
        }
    };
    auto largest = [&](const u32x4 &r) {
        const f32x4 x = __builtin_bit_cast(f32x4, r);
        return fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
    };
    // 0 where each row of a piece has a value of 2^-5 at least and none of `limit` or more.
    auto rows_odd = [&](float top, float limit) {
        uint64_t some = __ballot(top >= 0.03125f);  // any lane of a row
#pragma unroll
        for (int e = 1; e < CPR; e <<= 1) some |= some >> e;
        constexpr uint64_t FIRST = CPR == 32 ? 0x0000000100000001ull : 0x0001000100010001ull;
        return (~some & FIRST) | __ballot(!(top < limit));
    };
    // Powers of two for this thread's pieces of K: 64 for rows from 2^-5 to 512 (the
    // largest comes to 2 at least, and the second term's rounding, 2^-25, is 2^-26 of
    // that; with 1 in place of 64 rows of about 0.03 were 2^-20 off, and outputs 1.5e-6);
    // otherwise the row's largest gives it.
    constexpr float K_UP = 64.f;
    auto scales = [&](const u32x4 (&r)[CH], float (&up)[CH]) {
        float top[CH];
        uint64_t other = 0;
#pragma unroll
        for (int i = 0; i < CH; i++) top[i] = largest(r[i]), up[i] = K_UP, other |= rows_odd(top[i], 512.f);
        if (other) {
#pragma unroll
            for (int i = 0; i < CH; i++) {
                const float m = row_max<CPR>(top[i]);  // each row for itself
                up[i] = m >= 0.03125f && m < 512.f ? K_UP : pow2_to_14(m);
            }
        }
    };
    // a piece of K, of V, as two terms
    auto put_k = [&](const u32x4 &r, float up, int i, LK &to, float *ks) {
        const int key = key0 + i * (NT / CPR);
        const f32x4 x = __builtin_bit_cast(f32x4, r);
        uint32_t h0, h1, l0, l1;
        split2(x[0], x[1], up, h0, l0);
        split2(x[2], x[3], up, h1, l1);
        *(u32x2 *)&to.x[0][key][d0] = u32x2{h0, h1};
        *(u32x2 *)&to.x[1][key][d0] = u32x2{l0, l1};
        ks[d0 ? TILE_32 + key : key] = __builtin_bit_cast(float, 0x7F000000u - __builtin_bit_cast(uint32_t, up));  // 1 / up
    };
    // V's rows enter times V_UP (down to 2^-29 of the row's largest).  Where one is not
    // as above put_v says so, and again_v gives each row of the pieces, written once
    // more, a power of two of its own where it needs one: the largest of a small row
    // comes to 2^3 .. 2^4 and of a large one to 2^14 .. 2^15, next to the least and the
    // greatest that the rows left alone have, so that the weights' least step in the
    // other's units is 2^-25 of the larger row's.  The way back is the key's factor; 0
    // for a row of zeros.
    constexpr float V_UP = 512.f;
    auto v_terms = [&](const u32x4 &r, float up, float back, int i, LV &to, float *vs) {
        const int key = key0 + i * (NT / CPR);
        const f32x4 x = __builtin_bit_cast(f32x4, r);
        uint32_t h0, h1, l0, l1;
        split2(x[0], x[1], up, h0, l0);
        split2(x[2], x[3], up, h1, l1);
        *(u32x2 *)&to.x[0][key][d0] = u32x2{h0, h1};
        *(u32x2 *)&to.x[1][key][d0] = u32x2{l0, l1};
        vs[d0 ? TILE_32 + key : key] = back;
    };
    auto put_v = [&](const u32x4 &r, int i, LV &to, float *vs) {
        v_terms(r, V_UP, 1.f / V_UP, i, to, vs);
        return rows_odd(largest(r), 64.f);
    };
    auto again_v = [&](const u32x4 (&r)[CH], LV &to, float *vs) {
#pragma unroll
        for (int i = 0; i < CH; i++) {
            const float m = row_max<CPR>(largest(r[i]));
            const bool leave = (m >= 0.03125f && m < 64.f) || !(m <= 3.402823466e38f);
            const float up = leave ? V_UP : pow2_to_14(m) * (m < 1.f ? 0x1p-10f : 2.f);
            v_terms(r[i], up, m == 0.f ? 0.f : __builtin_bit_cast(float, 0x7F000000u - __builtin_bit_cast(uint32_t, up)), i, to, vs);
        }
        odd = 1;
    };
    auto clean = [&](u32x4 (&r)[CH], int e) {
        if ((e + 1) * TILE_32 <= whole) return;
        bool any = false;
#pragma unroll
        for (int i = 0; i < CH; i++) any = not_finite<FH3K_F32>(r[i]) || any;
        if (any) lost = 1;
    };
    const int steps = (n_tiles + KH - 1) / KH;
    auto tile = [&](int e) { return e * KH + half; };  // of this half's step e
    auto there = [&](int t) { return t < n_tiles ? t : n_tiles - 1; };  // past the last tile that one again, all cut
    u32x4 rk[CH], rv[CH];
    load(g.k, g.ldk, there(tile(0)), rk);
    load(g.v, g.ldv, there(tile(0)), rv);

    const int row = p.r0 + WAVE_R * wave + l32, rc = row < p.rows ? row : p.rows - 1;
    const int tok = rc / p.G, head = p.kvh * p.G + rc % p.G;
    const Score sc = score_of(g.a);
    R w;
    // (q's largest to 2^2 .. 2^3, not 2^13: its products with K at its own size, 2^10 times that
    // at most, stay in fp32's range for K up to 2^117; the second term's rounding, 2^-25, is
    // 2^-27 of the largest)
    w.template load_q<true>(g.q, Op::TYPE, (int64_t)(p.first + tok) * g.ldq + head * HD, sc, 0x1p-11f);
    w.clear();
    w.pos = tok;
    w.lim = p.limit(tok);
    w.slope2 = sc.bias ? g.a.slopes[head] * LOG2E : 0.f;
    const int lo = __builtin_amdgcn_readfirstlane(w.lim);

    float up[CH], unit = -1.f;  // the row's sums of weighted V are in units of this (-1: of 1 / V_UP until a key has another factor)
    __syncthreads();
    clean(rv, tile(0));
    scales(rk, up);
    uint64_t other = 0;
#pragma unroll
    for (int i = 0; i < CH; i++) {
        put_k(rk[i], up[i], i, lk0[half], ks0[half]);
        other |= put_v(rv[i], i, lv0[half], vs0[half]);
    }
    if (other) again_v(rv, lv0[half], vs0[half]);
    load(g.k, g.ldk, there(tile(1)), rk);
    load(g.v, g.ldv, there(tile(1)), rv);
    __syncthreads();
    // Keys whose V stands there by a factor: it goes to the weight, in units of the
    // largest one that a key with a weight has had (2^-25 of that one's weights is
    // the least that fp16 holds).  s becomes the weights' arguments themselves.
    auto units = [&](f32x16 &s, float &c, float &nm, const float *vs) {
        vs += 4 * (lane >> 5);
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            s[i] = fmaf(s[i], c, nm);
            if (s[i] > -25.f) top = fmaxf(top, vs[8 * (i >> 2) + (i & 3)]);
        }
        c = 1.f, nm = 0.f;
        top = max32(top);
        const float was = unit >= 0.f ? unit : max32(w.l) > 0.f ? 1.f / V_UP : 0.f;
        unit = fmaxf(was, top);
        if (was < unit) {
            const float down = was / unit;
#pragma unroll
            for (int db = 0; db < R::DB; db++) w.o[db] *= down;
        }
        float full = 0.f, left = 0.f;  // the weights' sum, and the one that the second product's will give
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float r = fminf(vs[8 * (i >> 2) + (i & 3)] / unit, 1.f);
            full += __builtin_amdgcn_exp2f(s[i]);
            s[i] = r > 0.f ? s[i] + __builtin_amdgcn_logf(r) : -INFINITY;  // (0: zeros, or too small beside the unit)
            left += __builtin_amdgcn_exp2f(s[i]);
        }
        w.l += full - left;
    };
    // Rows that see nothing of a tile have weights of 0: the workgroup waits for
    // those that do either way.  Past the last tile that one is made again, not read.
    auto step = [&](int e, const LK &k_now, LK &k_next, const LV &v_now, LV &v_next, const float *ks, float *ks_next,
                    const float *vs, float *vs_next) {
        const int j0 = tile(e) * TILE_32;
        const int some_odd = odd;
        clean(rv, tile(e + 1));
        uint64_t other = 0;
        f32x16 s[1] = {};
        constexpr int N1 = R::KS, N2 = 2 * R::DB;
        typedef typename R::q8 q8;
        auto k_frag = [&](int i, int plane) {
            return *(const q8 *)&k_now.x[plane][l32][16 * i + 8 * (lane >> 5)];
        };
        q8 a0 = k_frag(0, 0), a1 = k_frag(0, 1);
#pragma unroll
        for (int i = 0; i < N1; i++) {
            const q8 c0 = a0, c1 = a1;
            if (i + 1 < N1) a0 = k_frag(i + 1, 0), a1 = k_frag(i + 1, 1);
            s[0] = mfma32(c1, w.q[0][i], s[0]);
            s[0] = mfma32(c0, w.q[1][i], s[0]);
            s[0] = mfma32(c0, w.q[0][i], s[0]);
            if (i * CH % N1 < CH) other |= put_v(rv[i * CH / N1], i * CH / N1, v_next, vs_next);
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);  // LDS reads
#pragma unroll
            for (int x = 0; x < 3; x++) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // matrix
                __builtin_amdgcn_sched_group_barrier(0x002, 5, 0);  // vector
            }
            __builtin_amdgcn_sched_group_barrier(0x200, 2, 0);  // LDS writes
        }
        if (other) again_v(rv, v_next, vs_next);
        load(g.v, g.ldv, there(tile(e + 2)), rv);
        float nm, c = w.template scores<true>(s, sc, 1.f, ks, j0, j0 + TILE_32 > lo, w.lim, nm);
        if (__builtin_amdgcn_readfirstlane(some_odd)) units(s[0], c, nm, vs);
        scales(rk, up);
        float sum[2] = {};
        u32x4 ph[2], pl[2];
        auto weigh = [&](int tt, int x) {  // two keys' weights
            const float p0 = __builtin_amdgcn_exp2f(fmaf(s[0][8 * tt + 2 * x], c, nm));
            const float p1 = __builtin_amdgcn_exp2f(fmaf(s[0][8 * tt + 2 * x + 1], c, nm));
            uint32_t hi, lw;
            split2(p0, p1, 1.f, hi, lw);
            ph[tt][x] = hi, pl[tt][x] = lw;
            sum[0] += p0, sum[1] += p1;
        };
#pragma unroll
        for (int x = 0; x < 4; x++) weigh(0, x);
        p8 y0 = v_frag<p8, LV::ROW>(&v_now.x[0][0][0], 0, 0), y1 = v_frag<p8, LV::ROW>(&v_now.x[1][0][0], 0, 0);
#pragma unroll
        for (int i = 0; i < N2; i++) {
            const int tt = i / R::DB, db = i % R::DB, n = i + 1;
            const p8 c0 = y0, c1 = y1;
            if (n < N2) {
                y0 = v_frag<p8, LV::ROW>(&v_now.x[0][0][0], n % R::DB, n / R::DB);
                y1 = v_frag<p8, LV::ROW>(&v_now.x[1][0][0], n % R::DB, n / R::DB);
            }
            const p8 p0 = __builtin_bit_cast(p8, ph[tt]), p1 = __builtin_bit_cast(p8, pl[tt]);
            w.o[db] = mfma32(c1, p0, w.o[db]);
            w.o[db] = mfma32(c0, p1, w.o[db]);
            w.o[db] = mfma32(c0, p0, w.o[db]);
            if (tt < 1)
#pragma unroll
                for (int x = db * 4 / R::DB; x < (db + 1) * 4 / R::DB; x++) weigh(tt + 1, x);
            if (i * CH % N2 < CH) put_k(rk[i * CH / N2], up[i * CH / N2], i * CH / N2, k_next, ks_next);
            __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
            for (int x = 0; x < 3; x++) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x402, 10, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x200, 3, 0);
        }
        w.l += sum[0] + sum[1];
        load(g.k, g.ldk, there(tile(e + 2)), rk);
        __syncthreads();
    };
#pragma unroll 1
    for (int e = 0; e < steps; e += 2) {
        step(e, lk0[half], lk1[half], lv0[half], lv1[half], ks0[half], ks1[half], vs0[half], vs1[half]);
        if (e + 1 < steps) step(e + 1, lk1[half], lk0[half], lv1[half], lv0[half], ks1[half], ks0[half], vs1[half], vs0[half]);
    }
    if constexpr (KH == 2) {
        static_assert(sizeof lk0 >= R::DB / 2 * 16384 && sizeof lv0 >= 4 * 1024, "");
        join_halves(w, unit, 1.f / V_UP, half, wave, (char *)lk0, (char *)lk1, (char *)lv0);
        if (half) return;
    }
    if (lost) lose<HD, Op::TYPE>(w, g, p, whole & ~(TILE_32 - 1), end);
    put_rows<HD, Op::TYPE>(w, g, p, row, head, unit < 0.f ? 1.f / V_UP : unit);
}

// F32 with every other tile of keys to four more wavefronts, against four wavefronts
// alone, us.  64 heads over 8, hd 128 (one workgroup of eight to a CU, two of four): one
// sequence of 37 tokens 16.8 / 12.1, 100 20.5 / 17.2, 150 23.5 / 22.3, 200 25.0 / 25.8, 300
// 31.1 / 34.7, 600 50.0 / 61.9, 1000 (504 workgroups) 90.2 / 100, 1200 (600) 128 / 122;
// several sequences, which leave no short tiles for the second round: 2 x 250 (256 workgroups)
// 30.3 / 32.5, 2 x 300 (304) 42.0 / 39.8, 3 x 200 (312) 40.7 / 32.0, 4 x 200 (416) 48.6 / 36.5.
// 16 heads over 16, hd 64: 150 tokens 12.0 / 12.0, 250 15.2 / 17.1, 500 21.8 / 27.6, 2000 63 /
// 90, 4000 (512) 137 / 174, 4600 (576) 181 / 207; 2 x 1000 (256) 37.1 / 49.7, 4 x 1000 (512)
// 64.1 / 65.2, 2 x 3000 (768) 164 / 165.
// (16 bits: 0.7 to 0.9 as fast at hd 128, 0.8 to 1.1 at hd 64, so not there.)
constexpr int SPLIT_FROM = 192;
constexpr int split_to(int hd, int n_seq) { return hd == 128 && n_seq > 1 ? 256 : 512; }

// Tiles of all sequences at most: each may have one that is not full.
int64_t most_tiles(const Fh3kAttn &a, const Fh3kSeqs &s) {
    constexpr int ROWS = WAVE_R * 4;
    const int64_t G = a.heads / a.kv_heads;
    return s.first ? s.n_tok * G / ROWS + (s.n_seq < s.n_tok ? s.n_seq : s.n_tok)
                   : (int64_t)s.n_seq * ((s.n_tok / s.n_seq * G + ROWS - 1) / ROWS);
}

template <int HD, int TY>
hipError_t launch_seqs(const Fh3kAttn &a, const void *q, int64_t ldq, const void *k, int64_t ldk, const void *v,
                       int64_t ldv, void *o, int64_t ldo, const Fh3kSeqs &s, const int *prefix, hipStream_t st) {
    const int64_t tiles = most_tiles(a, s);
    const SeqsArgs g = {a, q, k, v, o, ldq, ldk, ldv, ldo, s, prefix, (int)tiles};
    const dim3 grid((unsigned)(tiles * a.kv_heads));
    if constexpr (TY == 2) {
        // Few workgroups with more than a few tiles of keys: eight wavefronts each, so
        // that a SIMD has two and a row half as many steps.
        if (tiles * a.kv_heads <= split_to(HD, s.n_seq) && (int64_t)s.n_tok >= (int64_t)SPLIT_FROM * s.n_seq)
            hipLaunchKernelGGL((k_attn_seqs32<HD, 2>), grid, dim3(512), 0, st, g);
        else
            hipLaunchKernelGGL((k_attn_seqs32<HD, 1>), grid, dim3(256), 0, st, g);
    } else
        hipLaunchKernelGGL((k_attn_seqs16<HD, TY>), grid, dim3(256), 0, st, g);
    return hipGetLastError();
}

}  // namespace

extern "C" int fh3k_attn_seqs_fits(const Fh3kAttn *a, Fh3kSeqs s) { return most_tiles(*a, s) * a->kv_heads <= 0x7FFFFF; }

extern "C" hipError_t fh3k_attn_seqs(const Fh3kAttn *a, const void *q, int64_t ldq, const void *k, int64_t ldk,
                                     const void *v, int64_t ldv, void *o, int64_t ldo, Fh3kSeqs s, const int *prefix,
                                     hipStream_t st) {
#define FH3K_SEQS(HD, TY) launch_seqs<HD, TY>(*a, q, ldq, k, ldk, v, ldv, o, ldo, s, prefix, st)
    if (a->hd == 128)
        return a->type == FH3K_F16 ? FH3K_SEQS(128, 0) : a->type == FH3K_BF16 ? FH3K_SEQS(128, 1) : FH3K_SEQS(128, 2);
    return a->type == FH3K_F16 ? FH3K_SEQS(64, 0) : a->type == FH3K_BF16 ? FH3K_SEQS(64, 1) : FH3K_SEQS(64, 2);
#undef FH3K_SEQS
}
