// fh3_kv.hip -- the 8-bit key/value cache: new rows written to it
// (fh3_hip_kv_append_dev), read back (fh3_hip_kv_read_dev), lengths moved on
// (fh3_hip_kv_extend_dev) and attention over it (fh3_hip_kv_attention_dev).
#include "fh3_tile.h"

namespace {

// Pages that a sequence's cnt rows touch at most.
int64_t most_pages(int64_t cnt) { return cnt > 0 ? (cnt + 62) / 64 + 1 : 0; }
int64_t touched_most(Fh3kSeqs s) {  // over all sequences: at least one row to a page
    if (!s.first) return s.n_seq * most_pages(s.n_tok / s.n_seq);
    const int64_t n = (int64_t)s.n_tok / 64 + 2 * (int64_t)s.n_seq;
    return n < s.n_tok ? n : s.n_tok;
}

// The exponent of the least power of two s >= 2^-100 with amax <= 127 s.
__device__ __forceinline__ float page_scale(float amax) {
    int x;
    const float m = frexpf(amax, &x);
    int e = m <= 127.f / 128.f ? x - 7 : x - 6;
    e = amax > 0.f && e > -100 ? e : -100;
    return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23);
}
__device__ __forceinline__ float finite_abs(float x) {
    const float y = fabsf(x);
    return y <= 3.402823466e38f ? y : 0.f;
}
// x / s as a stored byte in the low eight bits: 1.5 * 2^23 + 128 leaves the integer
// nearest (ties to even) there; the clamp takes infinities, a NaN becomes 0.
__device__ __forceinline__ uint32_t to_byte(float x, float inv) {
    const float y = x == x ? fminf(fmaxf(x * inv, -127.f), 127.f) : 0.f;
    return __builtin_bit_cast(uint32_t, y + 12583040.f);
}
// the low bytes of four words
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0C0C0400u), __builtin_amdgcn_perm(b, a, 0x0C0C0400u), 0x05040100u);
}
__device__ __forceinline__ float byte_value(uint32_t w, int e) { return (float)(w >> (8 * e) & 255) - 128.f; }
// Four stored bytes at a new scale: ratio = old / new <= 1, exactly a power of two.
__device__ __forceinline__ uint32_t again4(uint32_t w, float ratio) {
    return pack4(to_byte(byte_value(w, 0), ratio), to_byte(byte_value(w, 1), ratio), to_byte(byte_value(w, 2), ratio),
                 to_byte(byte_value(w, 3), ratio));
}

constexpr int ROW_T = 256;  // threads of the kernels that move rows

// A page that new rows touch (work unit), of a head, K or V: blockIdx.y.
struct RowPage {
    int h, which, seq, id;
    int64_t row0;  // the row of slot 0, were it one
    int lo, hi;    // its rows are slots lo .. hi - 1
};
__device__ __forceinline__ bool row_page(const Fh3kKv &c, const Fh3kSeqs &s, RowPage &r) {
    int a = 0, cnt = 0, len, base = 0, at;
    r.h = blockIdx.y >> 1, r.which = blockIdx.y & 1;
    if (!find_unit(blockIdx.x, s.n_seq, [&](int i) {
            seq_rows(s, i, a, cnt);
            kv_len(c, i, cnt, len, base);
            // base may be negative: rows that no page holds
            return cnt > 0 ? ((base + cnt - 1) >> 6) - (base >> 6) + 1 : 0;
        }, r.seq, at))
        return false;
    a = of_lane(a, r.seq), cnt = of_lane(cnt, r.seq), base = of_lane(base, r.seq);
    const int p = (base >> 6) + at;
    r.id = kv_page(c, r.seq, p);
    const int64_t pos0 = (int64_t)p * KV_PAGE;
    r.row0 = a + (pos0 - base);
    r.lo = (int)(base > pos0 ? base - pos0 : 0);
    r.hi = (int)(base + cnt < pos0 + KV_PAGE ? base + cnt - pos0 : KV_PAGE);
    return r.lo < r.hi;
}

// The rows go through LDS as fp32: their largest finite value gives the scale, then
// a whole page is made in 16-byte pieces, part of one in the smallest that its
// rows fill (K: 16 channels of a slot; V: four slots of a channel).  Prompts: 55 MB in 15 us,
// 3.6 TB/s where a copy reaches 4.8; wavefronts wait half of their time (rows, then the
// barrier before the scale) and half of the LDS cycles are V's bank conflicts.  One token of
// 64 sequences is bound by the loads that wait for each other: length, page, rows (4 us).
template <int HD>
__global__ __launch_bounds__(ROW_T) void k_kv_append(Fh3kKv c, int type, const void *__restrict__ k, int64_t ldk,
                                                     const void *__restrict__ v, int64_t ldv, Fh3kSeqs s) {
    constexpr int LD = HD + 4, PPR = HD / 8, PIECES = KV_PAGE * PPR / ROW_T;
    __shared__ __align__(16) float sx[KV_PAGE * LD];
    __shared__ float smax[ROW_T / 64];
    const int t = threadIdx.x;
    RowPage r;
    if (!row_page(c, s, r) || r.id < 0) return;
    const int lo = r.lo, hi = r.hi;
    const void *x = r.which ? v : k;
    const int64_t ld = r.which ? ldv : ldk, at0 = r.row0 * ld + r.h * HD;
    const int64_t blk = ((int64_t)r.id * c.kv_heads + r.h) * 2 + r.which;
    const float before = c.scales[blk];
    Raw8 raw[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; i++) {
        const int e = t + ROW_T * i, slot = lo + e / PPR, d = e % PPR * 8;
        if (slot < hi) raw[i] = load8(x, type, at0 + slot * ld + d);
    }
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < PIECES; i++) {
        const int e = t + ROW_T * i, slot = lo + e / PPR, d = e % PPR * 8;
        if (slot < hi) {
            float y[8];
            values8(raw[i], type, y);
#pragma unroll
            for (int j = 0; j < 8; j++) m = fmaxf(m, finite_abs(y[j]));
            *(f32x4 *)&sx[slot * LD + d] = f32x4{y[0], y[1], y[2], y[3]};
            *(f32x4 *)&sx[slot * LD + d + 4] = f32x4{y[4], y[5], y[6], y[7]};
        }
    }
#pragma unroll
    for (int w = 1; w < 64; w <<= 1) m = fmaxf(m, __shfl_xor(m, w));
    if ((t & 63) == 0) smax[t >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(smax[0], smax[1]), fmaxf(smax[2], smax[3]));
    float now = page_scale(m);
    if (lo > 0) now = fmaxf(now, before);
    const float inv = 1.f / now, ratio = before * inv;
    const bool redo = lo > 0 && before != now;
    if (t == 0) c.scales[blk] = now;
    uint8_t *page = c.pool + blk * KV_PAGE * HD;
    if (lo == 0 && hi == KV_PAGE) {
#pragma unroll
        for (int u = 0; u < KV_PAGE * HD / 16 / ROW_T; u++) {
            const int p = t + ROW_T * u, i = p & 15, g = (p >> 4) & 3, b = p >> 6;
            const float *at = r.which ? &sx[4 * g * LD + 16 * b + i] : &sx[(16 * (b / (HD / 64)) + i) * LD + 64 * (b % (HD / 64)) + 16 * g];
            u32x4 w;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int o = r.which ? 16 * e * LD : 4 * e, n = r.which ? LD : 1;
                w[e] = pack4(to_byte(at[o], inv), to_byte(at[o + n], inv), to_byte(at[o + 2 * n], inv), to_byte(at[o + 3 * n], inv));
            }
            *(u32x4 *)(page + 16 * p) = w;
        }
    } else if (r.which == 0) {
        const int from = redo ? 0 : lo;
        for (int e = t; e < (hi - from) * (HD / 16); e += ROW_T) {
            const int slot = from + e / (HD / 16), d = e % (HD / 16) * 16;
            u32x4 *at = (u32x4 *)(page + k_byte<HD>(slot, d)), w;
            if (slot < lo) {
                w = *at;
                for (int i = 0; i < 4; i++) w[i] = again4(w[i], ratio);
            } else {
                const float *y = &sx[slot * LD + d];
                for (int i = 0; i < 4; i++)
                    w[i] = pack4(to_byte(y[4 * i], inv), to_byte(y[4 * i + 1], inv), to_byte(y[4 * i + 2], inv), to_byte(y[4 * i + 3], inv));
            }
            *at = w;
        }
    } else {
        const int from = redo ? 0 : lo >> 2, to = (hi + 3) >> 2;  // fours of slots
        for (int e = t; e < (to - from) * HD; e += ROW_T) {
            const int slot = 4 * (from + e / HD), d = e % HD;
            uint32_t *at = (uint32_t *)(page + v_byte<HD>(slot, d)), w = 0;
            if (slot < lo || slot + 4 > hi) w = *at;
            if (redo && slot < lo) {  // (bytes from lo on are new, or behind the length: those stay, as K's do)
                const uint32_t held = slot + 4 <= lo ? ~0u : (1u << 8 * (lo - slot)) - 1;
                w = (again4(w, ratio) & held) | (w & ~held);
            }
            for (int i = 0; i < 4; i++)
                if (slot + i >= lo && slot + i < hi)
                    w = (w & ~(255u << 8 * i)) | (to_byte(sx[(slot + i) * LD + d], inv) & 255) << 8 * i;
            *at = w;
        }
    }
}

// The same pages read back as rows; rows that no page holds become zeros.  A thread
// takes four slots x four channels, so that rows are written in order.  4-byte loads 16
// bytes apart and none ahead: 10 us for the pages that one token of 64 sequences touches,
// 14 for 5400 fp32 tokens (55 MB).
template <int HD>
__global__ __launch_bounds__(ROW_T) void k_kv_read(Fh3kKv c, int type, void *__restrict__ k, int64_t ldk,
                                                   void *__restrict__ v, int64_t ldv, Fh3kSeqs s) {
    void *x = blockIdx.y & 1 ? v : k;
    RowPage r;
    if (!x || !row_page(c, s, r)) return;
    const int64_t ld = r.which ? ldv : ldk, at0 = r.row0 * ld + r.h * HD;
    const int64_t blk = ((int64_t)(r.id < 0 ? 0 : r.id) * c.kv_heads + r.h) * 2 + r.which;
    const float scale = r.id < 0 ? 0.f : c.scales[blk];
    const uint8_t *page = c.pool + blk * KV_PAGE * HD;
    const int from = r.lo >> 2, to = (r.hi + 3) >> 2;
    for (int e = threadIdx.x; e < (to - from) * (HD / 4); e += ROW_T) {
        const int slot = 4 * (from + e / (HD / 4)), d = e % (HD / 4) * 4;
        uint32_t w[4];  // K: of a slot; V: of a channel
#pragma unroll
        for (int i = 0; i < 4; i++)
            w[i] = *(const uint32_t *)(page + (r.which ? v_byte<HD>(slot, d + i) : k_byte<HD>(slot + i, d)));
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (slot + i < r.lo || slot + i >= r.hi) continue;
            f32x4 y;
#pragma unroll
            for (int j = 0; j < 4; j++) y[j] = byte_value(r.which ? w[j] : w[i], r.which ? i : j) * scale;
            if (r.id < 0) y = f32x4{};
            store4(x, type, at0 + (slot + i) * ld + d, y);
        }
    }
}

__global__ __launch_bounds__(ROW_T) void k_kv_extend(int *len, Fh3kSeqs s) {
    const int i = blockIdx.x * ROW_T + threadIdx.x;
    if (i >= s.n_seq) return;
    int a, cnt;
    seq_rows(s, i, a, cnt);
    const int l = len[i] > 0 ? len[i] : 0;
    len[i] = l < 0x7FFFFFFF - cnt ? l + cnt : 0x7FFFFFFF;
}

// ---------------------------------------------------------------------------
// Attention over the cache.  The work is the pages that each tile of rows looks
// through, one after the other over all sequences ("units", the same for every
// key head); a key head's workgroups take equal runs of units, whatever the
// lengths are, so a run may end inside a tile: the parts then go to the workspace
// and k_kv_join adds them in order.  Tiles of at most WHOLE pages are not divided:
// the workgroup of their first page takes them.
// ---------------------------------------------------------------------------
constexpr int WHOLE = 8;

struct KvWork {
    int G;      // query heads of a key head
    int shift;  // tiles of 2^shift rows
    int wgs;    // workgroups of a key head
};
// A sequence: its rows first .. first + cnt - 1, tokens held, position of the first
// row, tiles, and pages (units) of each; a tile that sees no key has one unit.
struct KvSeq {
    int first, cnt, len, base, tiles, pages;
};
__device__ __forceinline__ KvSeq kv_seq(const Fh3kKv &c, const Fh3kSeqs &s, const KvWork &w, int i) {
    KvSeq q;
    seq_rows(s, i, q.first, q.cnt);
    kv_len(c, i, q.cnt, q.len, q.base);
    q.pages = q.len > 0 ? (q.len + KV_PAGE - 1) / KV_PAGE : 1;
    q.tiles = (q.cnt * w.G + (1 << w.shift) - 1) >> w.shift;
    return q;
}
// A workgroup's run of units u .. end - 1 and the sequence, tile and page of the first.
struct KvRun {
    int size, u, end, seq, tile, page;
    KvSeq q;
    __device__ __forceinline__ int ends(int pages, int wgs) const {  // the workgroup that ends a tile begun at u
        const int w = (u + pages - 1) / size;
        return w < wgs ? w : wgs - 1;
    }
};
__device__ __forceinline__ bool kv_run(const Fh3kKv &c, const Fh3kSeqs &s, const KvWork &w, int wg, KvRun &r) {
    KvSeq q = {};
    auto units = [&](int i) {
        q = kv_seq(c, s, w, i);
        return q.tiles * q.pages;
    };
    const int lane = threadIdx.x & 63;
    int all = 0, mine = 0, end = 0;
    for (int s0 = 0; s0 < s.n_seq; s0 += 64) {
        mine = s0 + lane < s.n_seq ? units(s0 + lane) : 0;
        end = wave_scan(mine);
        all += __builtin_amdgcn_readlane(end, 63);
    }
    const int even = (all + w.wgs - 1) / w.wgs;
    r.size = __builtin_amdgcn_readfirstlane(even > WHOLE ? even : WHOLE);
    // wg * size may pass 2^31 only where it also passes all
    if ((int64_t)wg * r.size >= all) return false;
    r.u = wg * r.size;
    r.end = all - r.u < r.size ? all : r.u + r.size;
    int at = 0;
    if (s.n_seq <= 64) {
        r.seq = __builtin_ctzll(__ballot(end > r.u));
        at = r.u - (of_lane(end, r.seq) - of_lane(mine, r.seq));
    } else {
        if (!find_unit(r.u, s.n_seq, units, r.seq, at)) return false;
    }
    r.q = {of_lane(q.first, r.seq), of_lane(q.cnt, r.seq), of_lane(q.len, r.seq), of_lane(q.base, r.seq),
           of_lane(q.tiles, r.seq), of_lane(q.pages, r.seq)};
    r.tile = at / r.q.pages;
    r.page = at - r.tile * r.q.pages;
    return true;
}
// The next tile after r.tile is done; false behind the last.
__device__ __forceinline__ bool kv_next(const Fh3kKv &c, const Fh3kSeqs &s, const KvWork &w, KvRun &r) {
    r.page = 0;
    if (++r.tile < r.q.tiles) return true;
    r.tile = 0;
    do {
        if (++r.seq >= s.n_seq) return false;
        r.q = kv_seq(c, s, w, r.seq);
    } while (r.q.tiles == 0);
    return true;
}

// Where the parts of a divided tile stand: of each workgroup two, the end of a
// tile begun before its run (0) and the beginning of one that goes on behind it
// (1); rows x HD sums, then the rows' sums of weights and their offsets' two terms.  What k_kv_join
// has to know of the second, the workgroup that begins the tile writes down.
struct Begun {
    int last;               // the workgroup that ends it, or 0: there is none
    int first, r0, rows;    // the sequence's first row in q and o, the tile's row in it, its rows
};
template <int HD> struct Parts {
    float *p;
    int rows, kv_heads, wgs;
    __device__ __forceinline__ float *of(int kvh, int wg, int which) const {
        return p + (((int64_t)kvh * wgs + wg) * 2 + which) * rows * (HD + 3);
    }
    __device__ __forceinline__ Begun *begun(int kvh, int wg) const {
        return (Begun *)(p + (int64_t)kv_heads * wgs * 2 * rows * (HD + 3)) + (kvh * wgs + wg);
    }
};
__host__ __device__ constexpr int64_t parts_bytes(int hd, int rows, int kv_heads, int wgs) {
    return (int64_t)kv_heads * wgs * (2 * rows * (hd + 3) * (int)sizeof(float) + (int)sizeof(Begun));
}

// Weighted sums of V, V's page scale (2^-100 to 2^121) in them, are held times DOWN: 2^17
// keys of the largest value with weights of 2^14 each (2^25 with 2^6) stay below fp32's
// largest number, and the least scale times 2^6 is still fp32's least normal one.
constexpr float DOWN = 0x1p-32f, BACK = 0x1p32f;

__device__ __forceinline__ f32x4 mfma16(half8 a, half8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float lane_value(float x, int n) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), n & 63));
}
// Eight stored bytes -> fp16 integers: 0x64 before a byte makes 1024 + it.
__device__ __forceinline__ half8 to_half(uint32_t a, uint32_t b) {
    u32x4 w = {__builtin_amdgcn_perm(0x64646464u, a, 0x04010400u), __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u),
               __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u), __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)};
    return __builtin_bit_cast(half8, w) - (half8)(_Float16)1152.f;
}

// Few rows to a sequence: tiles of 16 R rows; each of four wavefronts takes every
// fourth page of a tile with all its rows, straight from memory into the
// operands of 16x16x32 products (S^T = K Q^T, O^T = V^T P^T), and the four are
// joined in LDS.  NT: 16-bit terms of q and of the weights (fp32: two).  16 KB are on
// their way to each wavefront, 128 KB to a CU, so that memory bounds it: 0.5 GB of cache
// in 96 us and 103 with the join (5.0 TB/s; a device copy moves 4.8), 140 MB in 40 with the
// join.  One token of one sequence takes 8.5 us, launch and latencies.  The form of 32 16-bit
// rows at hd 128 spills one register.
constexpr int FEW_W = 4;
constexpr float OFFSET = Vec<_Float16>::OFFSET, RAISE = Vec<_Float16>::RAISE;
template <int HD, int R, int NT>
__global__ __launch_bounds__(64 * FEW_W, 2) void k_kv_few(Fh3kAttn a, Fh3kKv c, const void *__restrict__ q, int64_t ldq,
                                                          void *__restrict__ o, int64_t ldo, Fh3kSeqs s, KvWork work,
                                                          float *__restrict__ ws) {
    constexpr int ROWS = 16 * R, KU = HD / 64, DT = HD / 16, OROW = HD + 4;
    __shared__ __align__(16) float so[FEW_W][ROWS][OROW];
    __shared__ float sm[FEW_W][ROWS], slo[FEW_W][ROWS], sl[FEW_W][ROWS];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, g = lane >> 4;
    const int kvh = blockIdx.x % c.kv_heads, wg = blockIdx.x / c.kv_heads, G = work.G;
    const Score sc = score_of(a);
    const Parts<HD> parts = {ws, ROWS, c.kv_heads, work.wgs};
    KvRun run;
    const bool any = kv_run(c, s, work, wg, run);
    if (ws && tid == 0) parts.begun(kvh, wg)->last = 0;
    if (!any) return;
    do {
        const int page0 = run.page, pages = run.q.pages;
        const bool whole = pages <= WHOLE;
        if (!(whole && page0)) {
            const int page1 = whole || pages - page0 <= run.end - run.u ? pages : page0 + run.end - run.u;
            const int seq = run.seq, first = run.q.first, cnt = run.q.cnt, len = run.q.len, base = run.q.base;
            const int rows = cnt * G, r0 = run.tile * ROWS;
            auto limit = [&](int tok) { return a.causal && base + tok + 1 < len ? base + tok + 1 : len; };
            const int lo = limit(r0 / G);  // keys that all rows see
            // 64 of this wavefront's pages at a time, one to a lane: page and scales
            int ids = -1;
            f32x2 scs = {};
            auto load_ids = [&](int n) {
                const int p = page0 + wave + FEW_W * (n + lane);
                ids = p < page1 ? kv_page(c, seq, p) : -1;
                scs = f32x2{};
                if (ids >= 0) scs = *(const f32x2 *)(c.scales + ((int64_t)ids * c.kv_heads + kvh) * 2);
            };
            u32x4 kr[4 * KU], vr[DT];
            auto block = [&](int n) {  // a page that is not there: page 0, whose keys are then all cut
                const int id = __builtin_amdgcn_readlane(ids, n & 63);
                return (const u32x4 *)(c.pool + ((int64_t)(id < 0 ? 0 : id) * c.kv_heads + kvh) * 2 * KV_PAGE * HD) + lane;
            };
            const int n_pages = (page1 - page0 - wave + FEW_W - 1) / FEW_W;
            // rows of this lane: R times l16; q's fragments, 16 channels of each 64.
            // q, the first pages and their K are on their way before any is used.
            Raw8 raw[R][2 * KU];
            float f[R], m[R], l[R], slope2[R];  // m: the weights' offset, its second term in slo
            int pos[R], lim[R];
#pragma unroll
            for (int r = 0; r < R; r++) {
                const int row = r0 + 16 * r + l16, rc = row < rows ? row : rows - 1;
                const int tok = rc / G, head = kvh * G + rc % G;
                const int64_t at_q = (int64_t)(first + tok) * ldq + head * HD + 16 * g;
#pragma unroll
                for (int i = 0; i < 2 * KU; i++) raw[r][i] = load8(q, a.type, at_q + 64 * (i >> 1) + 8 * (i & 1));
                pos[r] = base + tok;
                lim[r] = limit(tok);
                slope2[r] = sc.bias ? a.slopes[head] * LOG2E : 0.f;
            }
            if (n_pages > 0) {
                load_ids(0);
                const u32x4 *b = block(0);
#pragma unroll
                for (int i = 0; i < 4 * KU; i++) kr[i] = b[64 * i];
            }
            half8 qf[R][NT][2 * KU];
            f32x4 acc[R][DT];
            int far = 0;  // bit r: some row of sixteen r has an offset of FAR and more; otherwise slo is 0 and is not read
#pragma unroll
            for (int r = 0; r < R; r++) {
                float x[2 * KU][8], top = 0.f;
#pragma unroll
                for (int i = 0; i < 2 * KU; i++) {
                    values8(raw[r][i], a.type, x[i]);
#pragma unroll
                    for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[i][e]));
                }
                top = max32(max16(top));
                const float up = pow2_to_14(top);
                f[r] = sc.f / up;
#pragma unroll
                for (int i = 0; i < 2 * KU; i++) {
                    u32x4 h, l4;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        uint32_t hi, lo;
                        split2(x[i][2 * e], x[i][2 * e + 1], up, hi, lo);
                        h[e] = hi, l4[e] = lo;
                    }
                    qf[r][0][i] = __builtin_bit_cast(half8, h);
                    if constexpr (NT == 2) qf[r][NT - 1][i] = __builtin_bit_cast(half8, l4);
                }
                m[r] = M_NONE;
                l[r] = 0.f;
                slo[wave][16 * r + l16] = 0.f;
#pragma unroll
                for (int d = 0; d < DT; d++) acc[r][d] = f32x4{};
            }
            for (int n = 0; n < n_pages; n++) {
                const u32x4 *b = block(n);
#pragma unroll
                for (int i = 0; i < DT; i++) vr[i] = b[64 * (4 * KU + i)];
                const bool there = __builtin_amdgcn_readlane(ids, n & 63) >= 0;
                const float ks = lane_value(scs[0], n);
                const float vs = lane_value(scs[1], n) * DOWN;
                const int j0 = (page0 + wave + FEW_W * n) * KV_PAGE;
                f32x4 t[R][4] = {};
#pragma unroll
                for (int h = 0; h < KU; h++)
#pragma unroll
                    for (int tt = 0; tt < 4; tt++) {
                        const u32x4 w = kr[tt * KU + h];
                        const half8 k0 = to_half(w[0], w[1]), k1 = to_half(w[2], w[3]);
#pragma unroll
                        for (int r = 0; r < R; r++) {
#pragma unroll
                            for (int e = NT - 1; e >= 0; e--) {
                                t[r][tt] = mfma16(k0, qf[r][e][2 * h], t[r][tt]);
                                t[r][tt] = mfma16(k1, qf[r][e][2 * h + 1], t[r][tt]);
                            }
                        }
                    }
                if (n + 1 < n_pages) {
                    if (((n + 1) & 63) == 0) load_ids(n + 1);
                    const u32x4 *nb = block(n + 1);
#pragma unroll
                    for (int i = 0; i < 4 * KU; i++) kr[i] = nb[64 * i];
                }
                // lane holds keys 16 tt + 4 g + v of row l16
                const bool cut = !there || j0 + KV_PAGE > lo;
                half8 pf[R][NT][2];
#pragma unroll
                for (int r = 0; r < R; r++) {
                    float x = factor(f[r] * ks);  // scores are x t, unless there is more to do
                    const float ahead = (float)(pos[r] - j0 - 4 * g);
                    const int left = there ? lim[r] - j0 - 4 * g : 0x80000000;
                    if (sc.cap2 && sc.fine) {
#pragma unroll
                        for (int i = 0; i < 16; i++) t[r][i >> 2][i & 3] = capped_fine(t[r][i >> 2][i & 3] * x, sc.cap2);
                        x = 1.f;
                    } else if (sc.cap2) {
#pragma unroll
                        for (int i = 0; i < 16; i++) t[r][i >> 2][i & 3] = capped(t[r][i >> 2][i & 3] * x, sc.cap2);
                        x = 1.f;
                    }
                    if (sc.bias) {
#pragma unroll
                        for (int i = 0; i < 16; i++)
                            t[r][i >> 2][i & 3] = fmaf(-slope2[r], fabsf(ahead - (float)(16 * (i >> 2) + (i & 3))), t[r][i >> 2][i & 3] * x);
                        x = 1.f;
                    }
                    if (cut) {
#pragma unroll
                        for (int tt = 0; tt < 4; tt++)
#pragma unroll
                            for (int v = 0; v < 4; v++) t[r][tt][v] = left > 16 * tt + v ? t[r][tt][v] : -INFINITY;
                    }
                    float mt = t[r][0][0];
#pragma unroll
                    for (int i = 1; i < 16; i++) mt = fmaxf(mt, t[r][i >> 2][i & 3]);
                    float nm = -m[r];
                    const bool was = far >> r & 1;
                    if (was || __ballot(fmaf(mt, x, nm) > RAISE)) {
                        float lo2 = was ? slo[wave][16 * r + l16] : 0.f;
                        mt = max32(max16(mt));
                        const float y = mt * x, off = fmaf(mt, x, -y) - OFFSET;
                        const bool raise = fmaf(mt, x, nm) - lo2 > RAISE, two = fabsf(y) >= FAR;
                        const float now = two ? y : y - OFFSET, rest = two ? off : 0.f;
                        const float keep = raise ? __builtin_amdgcn_exp2f((m[r] - now) + (lo2 - rest)) : 1.f;
                        m[r] = raise ? now : m[r];
                        lo2 = raise ? rest : lo2;
                        nm = -m[r];
                        l[r] *= keep;
#pragma unroll
                        for (int d = 0; d < DT; d++) acc[r][d] *= keep;
                        const bool is = __ballot(fabsf(m[r]) >= FAR && m[r] != M_NONE);
                        if (was || is) {
                            far = is ? far | 1 << r : far & ~(1 << r);
                            slo[wave][16 * r + l16] = lo2;
                        }
                        if (is) {
#pragma unroll
                            for (int i = 0; i < 16; i++) t[r][i >> 2][i & 3] = fmaf(t[r][i >> 2][i & 3], x, nm) - lo2;
                            x = 1.f, nm = 0.f;
                        }
                    }
                    float sum = 0.f;
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        u32x4 h, l4;
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int i = 8 * u + 2 * e;
                            const float p0 = __builtin_amdgcn_exp2f(fmaf(t[r][i >> 2][i & 3], x, nm));
                            const float p1 = __builtin_amdgcn_exp2f(fmaf(t[r][i >> 2][(i & 3) + 1], x, nm));
                            if constexpr (NT == 2) {
                                uint32_t hi, lo;
                                split2(p0, p1, 1.f, hi, lo);
                                h[e] = hi, l4[e] = lo;
                                sum += p0 + p1;
                            } else {  // the sum is of the rounded weights, which the product takes
                                h[e] = Vec<_Float16>::pair(p0, p1);
                                sum = Vec<_Float16>::sum(h[e], sum);
                            }
                        }
                        pf[r][0][u] = __builtin_bit_cast(half8, h);
                        if constexpr (NT == 2) pf[r][NT - 1][u] = __builtin_bit_cast(half8, l4);
                    }
                    l[r] += sum;
                }
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    const half8 v0 = to_half(vr[d][0], vr[d][1]), v1 = to_half(vr[d][2], vr[d][3]);
#pragma unroll
                    for (int r = 0; r < R; r++) {
                        f32x4 y = {};
#pragma unroll
                        for (int e = NT - 1; e >= 0; e--) {
                            y = mfma16(v0, pf[r][e][0], y);
                            y = mfma16(v1, pf[r][e][1], y);
                        }
#pragma unroll
                        for (int v = 0; v < 4; v++) acc[r][d][v] = fmaf(y[v], vs, acc[r][d][v]);
                    }
                }
            }

            // the four wavefronts' parts, in order
#pragma unroll
            for (int r = 0; r < R; r++) {
                l[r] = sum32(sum16(l[r]));
                const int row = 16 * r + l16;
                if (g == 0) sm[wave][row] = m[r], sl[wave][row] = l[r];
#pragma unroll
                for (int d = 0; d < DT; d++) *(f32x4 *)&so[wave][row][16 * d + 4 * g] = acc[r][d];
            }
            __syncthreads();
            const bool done = page0 == 0 && page1 == pages;
            float *part = done ? nullptr : parts.of(kvh, wg, page0 == 0);
            if (!done && page0 == 0 && tid == 0)
                *parts.begun(kvh, wg) = {run.ends(pages, work.wgs), first, r0, rows};
            for (int e = tid; e < ROWS * HD / 4; e += 64 * FEW_W) {
                const int row = e / (HD / 4), d = e % (HD / 4) * 4;
                float top = sm[0][row], rest = slo[0][row], sum = 0.f;
#pragma unroll
                for (int w = 1; w < FEW_W; w++) {
                    const bool more = (sm[w][row] - top) + (slo[w][row] - rest) > 0.f;
                    top = more ? sm[w][row] : top, rest = more ? slo[w][row] : rest;
                }
                f32x4 x = {};
#pragma unroll
                for (int w = 0; w < FEW_W; w++) {
                    const float keep = __builtin_amdgcn_exp2f((sm[w][row] - top) + (slo[w][row] - rest));
                    sum += sl[w][row] * keep;
                    const f32x4 y = *(const f32x4 *)&so[w][row][d];
#pragma unroll
                    for (int v = 0; v < 4; v++) x[v] = fmaf(y[v], keep, x[v]);
                }
                if (!done) {
                    *(f32x4 *)(part + row * HD + d) = x;
                    if (d == 0) part[ROWS * HD + row] = sum, part[ROWS * (HD + 1) + row] = top, part[ROWS * (HD + 2) + row] = rest;
                } else if (r0 + row < rows) {
                    const float inv = sum == 0.f ? 0.f : 1.f / sum;
                    const int tok = (r0 + row) / G, head = kvh * G + (r0 + row) % G;
#pragma unroll
                    for (int v = 0; v < 4; v++) x[v] = x[v] * inv * BACK;
                    store4(o, a.type, (int64_t)(first + tok) * ldo + head * HD + d, x);
                }
            }
            __syncthreads();
            run.u += page1 - page0;
        } else {
            run.u += pages - page0;
        }
    } while (run.u < run.end && kv_next(c, s, work, run));
}

// Joins the parts of a divided tile in order, 4-7 us (many rows 13).  A workgroup takes RB rows of the tile
// that workgroup blockIdx.x of key head blockIdx.y began; SB groups of threads take
// every SB-th part each.
template <int HD, int SB>
__global__ __launch_bounds__(256) void k_kv_join(Fh3kAttn a, Fh3kKv c, void *__restrict__ o, int64_t ldo, KvWork work,
                                                 const float *__restrict__ ws) {
    constexpr int RB = 1024 / HD / SB;
    __shared__ __align__(16) float so[SB][RB * HD];
    __shared__ float sm[SB][RB], slo[SB][RB], sl[SB][RB];
    const int tid = threadIdx.x, wg = blockIdx.x, kvh = blockIdx.y, G = work.G, ROWS = 1 << work.shift;
    const Parts<HD> parts = {(float *)ws, ROWS, c.kv_heads, work.wgs};
    const Begun b = *parts.begun(kvh, wg);
    const int row0 = blockIdx.z * RB;
    if (b.last == 0 || b.r0 + row0 >= b.rows) return;
    const int grp = tid / (256 / SB), t = tid % (256 / SB), r = t / (HD / 4), d = t % (HD / 4) * 4, row = row0 + r;
    float top = M_NONE, rest = 0.f, sum = 0.f;
    f32x4 x = {};
#pragma unroll 4
    for (int w = wg + grp; w <= b.last; w += SB) {
        const float *p = parts.of(kvh, w, w == wg);
        const float pl = p[ROWS * HD + row], pm = p[ROWS * (HD + 1) + row], plo = p[ROWS * (HD + 2) + row];
        const f32x4 y = *(const f32x4 *)(p + row * HD + d);
        float keep, add;
        join_offsets(top, rest, pm, plo, keep, add);
        sum = sum * keep + pl * add;
#pragma unroll
        for (int v = 0; v < 4; v++) x[v] = x[v] * keep + y[v] * add;
    }
    if constexpr (SB > 1) {
        *(f32x4 *)&so[grp][r * HD + d] = x;
        if (d == 0) sm[grp][r] = top, slo[grp][r] = rest, sl[grp][r] = sum;
        __syncthreads();
        if (grp) return;
#pragma unroll
        for (int e = 1; e < SB; e++) {
            float keep, add;
            join_offsets(top, rest, sm[e][r], slo[e][r], keep, add);
            const f32x4 y = *(const f32x4 *)&so[e][r * HD + d];
            sum = sum * keep + sl[e][r] * add;
#pragma unroll
            for (int v = 0; v < 4; v++) x[v] = x[v] * keep + y[v] * add;
        }
    }
    if (b.r0 + row >= b.rows) return;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int tok = (b.r0 + row) / G, head = kvh * G + (b.r0 + row) % G;
#pragma unroll
    for (int v = 0; v < 4; v++) x[v] = x[v] * inv * BACK;
    store4(o, a.type, (int64_t)(b.first + tok) * ldo + head * HD + d, x);
}

// Many rows to a sequence: tiles of 128, 32 to a wavefront.  A page is turned
// into fp16 once for all of them, through double-buffered LDS: K as rows, V
// transposed with the keys of each 16 in the order of the first product's
// accumulator (0-3, 8-11, 4-7, 12-15).  Bound by the vector instructions of the softmax and
// the conversion (8 to a matrix instruction; each tile of rows converts its pages anew) beside
// the matrix ones: 1000 tokens of 64 heads behind 31000 in 550 us, 0.82 PFLOP/s, the matrix
// pipe busy 37 %.  fp32 (two terms of q and of the weights): 500 tokens behind 31500 in 505
// us, busy 46 %; at hd 128 46 registers spill.
constexpr int MANY_W = 4;
template <int HD, int NT>
__global__ __launch_bounds__(64 * MANY_W, 2) void k_kv_many(Fh3kAttn a, Fh3kKv c, const void *__restrict__ q,
                                                            int64_t ldq, void *__restrict__ o, int64_t ldo, Fh3kSeqs s,
                                                            KvWork work, float *__restrict__ ws) {
    typedef Rows<HD, _Float16, _Float16, NT> R;
    constexpr int ROWS = WAVE_R * MANY_W, NTH = 64 * MANY_W, KU = HD / 64, VROW = KV_PAGE + 8;
    constexpr int CH = KV_PAGE * HD / 16 / NTH;  // 16-byte pieces of K, and of V, to a thread
    __shared__ __align__(16) _Float16 sk[2][KV_PAGE][R::KROW];
    __shared__ __align__(16) _Float16 sv[2][HD][VROW];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, hf = lane >> 5;
    const int kvh = blockIdx.x % c.kv_heads, wg = blockIdx.x / c.kv_heads, G = work.G;
    const Score sc = score_of(a);
    const Parts<HD> parts = {ws, ROWS, c.kv_heads, work.wgs};
    KvRun run;
    const bool any = kv_run(c, s, work, wg, run);
    if (ws && tid == 0) parts.begun(kvh, wg)->last = 0;
    if (!any) return;
    do {
        const int page0 = run.page, pages = run.q.pages;
        const bool whole = pages <= WHOLE;
        if (!(whole && page0)) {
            const int page1 = whole || pages - page0 <= run.end - run.u ? pages : page0 + run.end - run.u;
            const int seq = run.seq, first = run.q.first, cnt = run.q.cnt, len = run.q.len, base = run.q.base;
            const int rows = cnt * G, r0 = run.tile * ROWS;
            auto limit = [&](int tok) { return a.causal && base + tok + 1 < len ? base + tok + 1 : len; };
            const int row = r0 + WAVE_R * wave + l32, rc = row < rows ? row : rows - 1;
            const int tok = rc / G, head = kvh * G + rc % G;
            R w;
            w.template load_q<true>(q, a.type, (int64_t)(first + tok) * ldq + head * HD, sc);
            w.clear();
            w.pos = base + tok;
            w.lim = limit(tok);
            w.slope2 = sc.bias ? a.slopes[head] * LOG2E : 0.f;
            const bool active = r0 + WAVE_R * wave < rows;
            const int lo = __builtin_amdgcn_readfirstlane(w.lim), hi = __builtin_amdgcn_readlane(w.lim, 31);
            const int seen = limit((r0 + ROWS < rows ? r0 + ROWS - 1 : rows - 1) / G);  // by the tile's last row
            const int page_n = seen <= page0 * KV_PAGE ? page0 : seen >= page1 * KV_PAGE ? page1 : (seen + KV_PAGE - 1) / KV_PAGE;
            float ref = 0.f;  // the sums are in units of this value scale

            int ids = -1;
            f32x2 scs = {};
            auto load_ids = [&](int n) {  // 64 pages at a time, one to a lane
                const int p = page0 + n + lane;
                ids = p < page_n ? kv_page(c, seq, p) : -1;
                scs = f32x2{};
                if (ids >= 0) scs = *(const f32x2 *)(c.scales + ((int64_t)ids * c.kv_heads + kvh) * 2);
            };
            u32x4 rk[CH], rv[CH];
            auto load = [&](int n) {
                const int id = __builtin_amdgcn_readlane(ids, n & 63);
                const u32x4 *b = (const u32x4 *)(c.pool + ((int64_t)(id < 0 ? 0 : id) * c.kv_heads + kvh) * 2 * KV_PAGE * HD) + tid;
#pragma unroll
                for (int i = 0; i < CH; i++) rk[i] = b[NTH * i], rv[i] = b[NTH * (CH + i)];
            };
            auto store = [&](int n) {
#pragma unroll
                for (int i = 0; i < CH; i++) {
                    const int p = tid + NTH * i, x = p & 15, g = (p >> 4) & 3, b = p >> 6;
                    _Float16 *kd = &sk[n & 1][16 * (b / KU) + x][64 * (b % KU) + 16 * g];
                    *(half8 *)kd = to_half(rk[i][0], rk[i][1]);
                    *(half8 *)(kd + 8) = to_half(rk[i][2], rk[i][3]);
                    _Float16 *vd = &sv[n & 1][16 * b + x][8 * (g & 1) + 4 * (g >> 1)];
                    const u32x4 lo4 = __builtin_bit_cast(u32x4, to_half(rv[i][0], rv[i][1]));
                    const u32x4 hi4 = __builtin_bit_cast(u32x4, to_half(rv[i][2], rv[i][3]));
                    *(u32x2 *)vd = u32x2{lo4[0], lo4[1]};
                    *(u32x2 *)(vd + 16) = u32x2{lo4[2], lo4[3]};
                    *(u32x2 *)(vd + 32) = u32x2{hi4[0], hi4[1]};
                    *(u32x2 *)(vd + 48) = u32x2{hi4[2], hi4[3]};
                }
            };
            const int n_pages = page_n - page0;
            float ks = 0.f, vs = 0.f;
            bool there = false;
            auto scales = [&](int n) {
                there = __builtin_amdgcn_readlane(ids, n & 63) >= 0;
                ks = lane_value(scs[0], n);
                vs = lane_value(scs[1], n);
            };
            __syncthreads();  // the last tile's readers are done
            if (n_pages > 0) {
                load_ids(0);
                load(0);
                scales(0);
                store(0);
            }
            __syncthreads();
            for (int n = 0; n < n_pages; n++) {
                const int j0 = (page0 + n) * KV_PAGE;
                const float ks_n = ks, vs_n = vs;
                const bool there_n = there;
                if (n + 1 < n_pages) {
                    if (((n + 1) & 63) == 0) load_ids(n + 1);
                    load(n + 1);
                    scales(n + 1);
                }
                if (active && there_n && j0 < hi) {
                    half8 pf[NT][4];
                    f32x16 x[2];
                    w.products(&sk[n & 1][0][0], x);
                    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);  // LDS reads, four ahead
#pragma unroll
                    for (int i = 0; i < 2 * R::KS; i++) {
                        __builtin_amdgcn_sched_group_barrier(0x008, NT, 0);
                        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                    }
                    float nm;
                    const float c = w.template scores<false>(x, sc, ks_n, nullptr, j0, j0 + KV_PAGE > lo, w.lim, nm);
                    w.weights(x, c, nm, pf);
                    // pages of the same scale add up in the product's accumulator
                    if (vs_n > ref) {
                        const float down = ref / vs_n;
                        ref = vs_n;
#pragma unroll
                        for (int i = 0; i < R::DB; i++) w.o[i] *= down;
                    }
                    if (vs_n == ref) {
#pragma unroll
                        for (int db = 0; db < R::DB; db++)
#pragma unroll
                            for (int tt = 0; tt < 4; tt++) {
                                const half8 x = *(const half8 *)&sv[n & 1][32 * db + l32][16 * tt + 8 * hf];
#pragma unroll
                                for (int e = NT - 1; e >= 0; e--) w.o[db] = mfma32(x, pf[e][tt], w.o[db]);
                            }
                        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
                        for (int i = 0; i < 4 * R::DB; i++) {
                            __builtin_amdgcn_sched_group_barrier(0x008, NT, 0);
                            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                        }
                    } else {
                        const float down = vs_n / ref;
#pragma unroll
                        for (int db = 0; db < R::DB; db++) {
                            f32x16 y = {};
#pragma unroll
                            for (int tt = 0; tt < 4; tt++) {
                                const half8 x = *(const half8 *)&sv[n & 1][32 * db + l32][16 * tt + 8 * hf];
#pragma unroll
                                for (int e = NT - 1; e >= 0; e--) y = mfma32(x, pf[e][tt], y);
                            }
#pragma unroll
                            for (int i = 0; i < 16; i++) w.o[db][i] = fmaf(y[i], down, w.o[db][i]);
                        }
                    }
                }
                if (n + 1 < n_pages) store(n + 1);
                __syncthreads();
            }

            const float l = sum32(w.l);
            const bool done = page0 == 0 && page1 == pages;
            if (!done && page0 == 0 && tid == 0)
                *parts.begun(kvh, wg) = {run.ends(pages, work.wgs), first, r0, rows};
            if (row < rows) {
                float *part = done ? nullptr : parts.of(kvh, wg, page0 == 0);
                const float inv = done ? (l == 0.f ? 0.f : 1.f / l) : 1.f, unit = done ? ref : ref * DOWN;
                const int64_t at_o = (int64_t)(first + tok) * ldo + head * HD;
                const int r = WAVE_R * wave + l32;
                if (!done && hf == 0) part[ROWS * HD + r] = l, part[ROWS * (HD + 1) + r] = w.m, part[ROWS * (HD + 2) + r] = w.lo;
#pragma unroll
                for (int db = 0; db < R::DB; db++)
#pragma unroll
                    for (int g = 0; g < 4; g++) {
                        const int d = 32 * db + 8 * g + 4 * hf;
                        f32x4 x;
#pragma unroll
                        for (int i = 0; i < 4; i++) x[i] = w.o[db][4 * g + i] * inv * unit;
                        if (done) store4(o, a.type, at_o + d, x);
                        else *(f32x4 *)(part + r * HD + d) = x;
                    }
            }
            run.u += page1 - page0;
        } else {
            run.u += pages - page0;
        }
    } while (run.u < run.end && kv_next(c, s, work, run));
}

}  // namespace

extern "C" hipError_t fh3k_kv_extend(int *len, Fh3kSeqs s, hipStream_t st) {
    hipLaunchKernelGGL(k_kv_extend, dim3((s.n_seq + ROW_T - 1) / ROW_T), dim3(ROW_T), 0, st, len, s);
    return hipGetLastError();
}

extern "C" hipError_t fh3k_kv_append(const Fh3kKv *c, int type, const void *k, int64_t ldk, const void *v, int64_t ldv,
                                     Fh3kSeqs s, hipStream_t st) {
    const dim3 grid((unsigned)touched_most(s), 2 * c->kv_heads);
    if (c->hd == 128)
        hipLaunchKernelGGL(k_kv_append<128>, grid, dim3(ROW_T), 0, st, *c, type, k, ldk, v, ldv, s);
    else
        hipLaunchKernelGGL(k_kv_append<64>, grid, dim3(ROW_T), 0, st, *c, type, k, ldk, v, ldv, s);
    return hipGetLastError();
}

extern "C" hipError_t fh3k_kv_read(const Fh3kKv *c, int type, void *k, int64_t ldk, void *v, int64_t ldv, Fh3kSeqs s,
                                   hipStream_t st) {
    const dim3 grid((unsigned)touched_most(s), 2 * c->kv_heads);
    if (c->hd == 128)
        hipLaunchKernelGGL(k_kv_read<128>, grid, dim3(ROW_T), 0, st, *c, type, k, ldk, v, ldv, s);
    else
        hipLaunchKernelGGL(k_kv_read<64>, grid, dim3(ROW_T), 0, st, *c, type, k, ldk, v, ldv, s);
    return hipGetLastError();
}

// How the rows of a call are tiled: by the average sequence, which is what the
// host knows (any tiling is right for any sequence).  8 key heads, us with tiles of 16 / 32 /
// 128 rows, one to some tokens of each sequence:
//                           fp16, hd 128      fp32, hd 128      fp16, hd 64       fp32, hd 64
//   16 x 4000,   8 rows   31.5/37.5/49.6    33.3/57.6/83.2    20.7/25.4/33.0    22.1/29.3/41.0
//                16       33.7/40.1/50.9    36.0/61.0/85.0    22.3/27.1/33.5    23.5/31.1/41.4
//                32       37.2/43.8/53.9    44.2/65.6/88.8    25.3/29.1/34.9    29.1/34.2/43.3
//                40       68.5/54.3/60.1    70.8/81.1/98.5    36.7/35.9/41.3    37.9/42.8/53.0
//    1 x 300,    32       14.1/12.3/16.7    16.0/16.8/22.3    10.6/ 9.0/11.3    11.7/10.3/13.6
//    4 x 300,    32       14.8/22.2/30.5    16.5/30.5/41.8    11.0/15.6/20.1    12.2/18.0/24.6
//    1 x 120000, 32       69.1/63.4/98.7    73.5/88.8/ 152    35.6/37.2/61.4    40.0/42.8/75.0
//   64 x 2000,   32       85.6/52.8/79.8    86.4/86.8/ 140    44.9/30.3/48.2    46.7/35.8/63.0
//  200 x 1000,   32        138/ 109/ 142     149/ 163/ 251    71.6/58.1/85.0    81.7/71.2/ 108
//   32 x 2000,   64       52.6/42.6/55.2    64.3/67.8/90.2    34.0/28.8/37.2    40.3/35.6/49.4
//               128        101/76.7/70.5     120/ 121/ 109    62.4/49.8/44.5    76.7/62.5/60.1
// fp32 at hd 128 has no 32-row form: its 53 spilled registers leave it behind 16 rows (the 46 of
// its 128-row form do not leave that behind where a sequence has that many).  Otherwise
// 32 rows win by more than they lose by from 17 to 32, as the number of tiles fits the card.
// One chunk in a call with single tokens (bf16, hd 128, all of 4000 tokens, 8 rows to a token):
// 512 tokens alone 114, 127 single tokens alone 188, together 350 (in 128-row tiles); 255
// single tokens alone 369, with the chunk 445 (in 32-row tiles).
struct KvForm {
    KvWork work;
    int64_t tiles;  // of all sequences at most
    bool few, join;
};
static KvForm kv_form(const Fh3kAttn &a, const Fh3kKv &c, const Fh3kSeqs &s) {
    KvForm f;
    const int64_t G = a.heads / a.kv_heads, rows = s.n_tok * G, avg = (rows + s.n_seq - 1) / s.n_seq;
    f.few = avg <= 32;
    static_assert(WAVE_R * MANY_W == 1 << 7, "");
    const int shift = avg <= (a.type == FH3K_F32 && a.hd == 128 ? 32 : 16) ? 4 : avg <= 32 ? 5 : 7;
    f.tiles = (rows >> shift) + (s.n_seq < s.n_tok ? s.n_seq : s.n_tok);
    const int64_t runs = (f.tiles * c.max_pages + WHOLE - 1) / WHOLE, most = (512 + a.kv_heads - 1) / a.kv_heads;
    f.work = {(int)G, shift, (int)(runs < most ? runs : most)};
    f.join = c.max_pages > WHOLE && f.work.wgs > 1;
    return f;
}

extern "C" int fh3k_kv_attn_fits(const Fh3kAttn *a, const Fh3kKv *c, Fh3kSeqs s) {
    return kv_form(*a, *c, s).tiles * c->max_pages <= 0x7FFFFFFF;
}

extern "C" size_t fh3k_kv_attn_ws_bytes(const Fh3kAttn *a, const Fh3kKv *c, Fh3kSeqs s) {
    const KvForm f = kv_form(*a, *c, s);
    return f.join ? (size_t)parts_bytes(a->hd, 1 << f.work.shift, a->kv_heads, f.work.wgs) : 0;
}

template <int HD>
static hipError_t kv_attn(const Fh3kAttn &a, const Fh3kKv &c, const void *q, int64_t ldq, void *o, int64_t ldo,
                          const Fh3kSeqs &s, float *ws, hipStream_t st) {
    const KvForm f = kv_form(a, c, s);
    const dim3 grid((unsigned)f.work.wgs * a.kv_heads);
    const bool two = a.type == FH3K_F32;
#define FH3K_KV(K, W) hipLaunchKernelGGL(K, grid, dim3(64 * W), 0, st, a, c, q, ldq, o, ldo, s, f.work, f.join ? ws : nullptr)
    if (f.work.shift == 4) {
        if (two) FH3K_KV((k_kv_few<HD, 1, 2>), FEW_W);
        else FH3K_KV((k_kv_few<HD, 1, 1>), FEW_W);
    } else if (f.few) {
        if constexpr (HD == 64) {
            if (two) FH3K_KV((k_kv_few<HD, 2, 2>), FEW_W);
        }
        if (!two) FH3K_KV((k_kv_few<HD, 2, 1>), FEW_W);
    } else {
        if (two) FH3K_KV((k_kv_many<HD, 2>), MANY_W);
        else FH3K_KV((k_kv_many<HD, 1>), MANY_W);
    }
#undef FH3K_KV
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !f.join) return e;
    // few rows: divided among up to 64 workgroups; many: between two or three
    const int rb = 1024 / HD / (f.few ? 4 : 1);
    const dim3 jg(f.work.wgs, a.kv_heads, (1 << f.work.shift) / rb);
    if (f.few) hipLaunchKernelGGL((k_kv_join<HD, 4>), jg, dim3(256), 0, st, a, c, o, ldo, f.work, ws);
    else hipLaunchKernelGGL((k_kv_join<HD, 1>), jg, dim3(256), 0, st, a, c, o, ldo, f.work, ws);
    return hipGetLastError();
}

extern "C" hipError_t fh3k_kv_attn(const Fh3kAttn *a, const Fh3kKv *c, const void *q, int64_t ldq, void *o,
                                   int64_t ldo, Fh3kSeqs s, void *ws, hipStream_t st) {
    return a->hd == 128 ? kv_attn<128>(*a, *c, q, ldq, o, ldo, s, (float *)ws, st)
                        : kv_attn<64>(*a, *c, q, ldq, o, ldo, s, (float *)ws, st);
}
