// fh3_kv.hip -- the 8-bit key/value cache: new rows written to it
// (fh3_hip_kv_append_dev), read back (fh3_hip_kv_read_dev), lengths moved on
// (fh3_hip_kv_extend_dev) and attention over it (fh3_hip_kv_attention_dev).
#include "fh3_seqs.h"

namespace {

// Pages that a sequence's cnt rows touch at most, and the touched pages of sequence i.
__host__ __device__ __forceinline__ int64_t most_pages(int64_t cnt) { return cnt > 0 ? (cnt + 62) / 64 + 1 : 0; }
__device__ __forceinline__ int64_t touched_pages(const Fh3kKv &c, const Fh3kSeqs &s, int i, int &p0) {
    int a, cnt, len, base;
    seq_rows(s, i, a, cnt);
    kv_len(c, i, cnt, len, base);
    p0 = base >> 6;  // base may be negative: rows that no page holds
    return cnt > 0 ? (int64_t)((base + cnt - 1) >> 6) - p0 + 1 : 0;
}
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
// x / s as a stored byte; the clamp takes infinities, a NaN becomes 0.
__device__ __forceinline__ uint32_t to_byte(float x, float inv) {
    const float y = x == x ? fminf(fmaxf(rintf(x * inv), -127.f), 127.f) : 0.f;
    return (uint32_t)((int)y + 128);
}
// A stored byte at a new scale: ratio = old / new <= 1, exactly a power of two.
__device__ __forceinline__ uint32_t again(uint32_t b, float ratio) {
    return (uint32_t)((int)fminf(fmaxf(rintf((float)((int)b - 128) * ratio), -127.f), 127.f) + 128);
}

constexpr int ROW_T = 256;  // threads of the kernels that move rows

// One workgroup to a page that new rows touch, a head, and K or V (blockIdx.y).
// The rows go through LDS as fp32: their largest finite value gives the scale,
// then each thread makes whole 16-byte pieces of the page.
template <int HD>
__global__ __launch_bounds__(ROW_T) void k_kv_append(Fh3kKv c, int type, const void *__restrict__ k, int64_t ldk,
                                                     const void *__restrict__ v, int64_t ldv, Fh3kSeqs s) {
    constexpr int LD = HD + 4;
    __shared__ __align__(16) float sx[KV_PAGE * LD];
    __shared__ float smax[ROW_T / 64];
    const int t = threadIdx.x, h = blockIdx.y >> 1, which = blockIdx.y & 1;
    int seq, a, cnt, len, base, p0;
    int64_t at;
    if (!find_unit(blockIdx.x, s.n_seq, [&](int i) { int p; return touched_pages(c, s, i, p); }, seq, at)) return;
    seq_rows(s, seq, a, cnt);
    kv_len(c, seq, cnt, len, base);
    touched_pages(c, s, seq, p0);
    const int p = p0 + (int)at, id = kv_page(c, seq, p);
    if (id < 0) return;
    const int64_t pos0 = (int64_t)p * KV_PAGE;
    const int lo = (int)(base > pos0 ? base - pos0 : 0);  // slots lo .. hi - 1 are new, those below lo held
    const int hi = (int)(base + cnt < pos0 + KV_PAGE ? base + cnt - pos0 : KV_PAGE);
    const void *x = which ? v : k;
    const int64_t ld = which ? ldv : ldk;
    float m = 0.f;
    for (int e = t; e < (hi - lo) * HD; e += ROW_T) {
        const int slot = lo + e / HD, d = e % HD;
        const float y = value_at(x, type, (a + (pos0 + slot - base)) * ld + h * HD + d);
        sx[slot * LD + d] = y;
        m = fmaxf(m, finite_abs(y));
    }
    float *scale = c.scales + ((int64_t)id * c.kv_heads + h) * 2 + which;
    const float before = *scale;
#pragma unroll
    for (int w = 1; w < 64; w <<= 1) m = fmaxf(m, __shfl_xor(m, w));
    if ((t & 63) == 0) smax[t >> 6] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < ROW_T / 64; w++) m = fmaxf(m, smax[w]);
    float now = page_scale(m);
    if (lo > 0) now = fmaxf(now, before);
    const float inv = 1.f / now, ratio = before * inv;
    const bool redo = lo > 0 && before != now;
    if (t == 0) *scale = now;
    u32x4 *page = (u32x4 *)(c.pool + (((int64_t)id * c.kv_heads + h) * 2 + which) * KV_PAGE * HD);
    for (int u = t; u < KV_PAGE * HD / 16; u += ROW_T) {
        // K: 16 channels of slot; V: slots 16 b + 4 g + r of a channel
        const int i = u & 15, g = (u >> 4) & 3, b = u >> 6;
        const int slot = which ? 4 * g : 16 * (b / (HD / 64)) + i;
        const int d = which ? 16 * b + i : 64 * (b % (HD / 64)) + 16 * g;
        uint32_t any = 0;  // bit e: byte e is written
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const int sl = which ? slot + 16 * (e >> 2) + (e & 3) : slot;
            any |= (uint32_t)((sl >= lo && sl < hi) || (redo && sl < lo)) << e;
        }
        if (!any) continue;
        u32x4 w = {};
        if (any != 0xFFFF || redo) w = page[u];
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const int sl = which ? slot + 16 * (e >> 2) + (e & 3) : slot;
            const uint32_t old = (w[e >> 2] >> (8 * (e & 3))) & 255;
            uint32_t y = old;
            if (sl >= lo && sl < hi) y = to_byte(sx[sl * LD + (which ? d : d + e)], inv);
            else if (redo && sl < lo) y = again(old, ratio);
            w[e >> 2] ^= (y ^ old) << (8 * (e & 3));
        }
        page[u] = w;
    }
}

// The same pages read back as rows; rows that no page holds become zeros.
template <int HD>
__global__ __launch_bounds__(ROW_T) void k_kv_read(Fh3kKv c, int type, void *__restrict__ k, int64_t ldk,
                                                   void *__restrict__ v, int64_t ldv, Fh3kSeqs s) {
    const int t = threadIdx.x, h = blockIdx.y >> 1, which = blockIdx.y & 1;
    void *x = which ? v : k;
    if (!x) return;
    int seq, a, cnt, len, base, p0;
    int64_t at;
    if (!find_unit(blockIdx.x, s.n_seq, [&](int i) { int p; return touched_pages(c, s, i, p); }, seq, at)) return;
    seq_rows(s, seq, a, cnt);
    kv_len(c, seq, cnt, len, base);
    touched_pages(c, s, seq, p0);
    const int p = p0 + (int)at, id = kv_page(c, seq, p);
    const int64_t pos0 = (int64_t)p * KV_PAGE, ld = which ? ldv : ldk;
    const int lo = (int)(base > pos0 ? base - pos0 : 0);
    const int hi = (int)(base + cnt < pos0 + KV_PAGE ? base + cnt - pos0 : KV_PAGE);
    const int64_t blk = ((int64_t)id * c.kv_heads + h) * 2 + which;
    const float scale = id >= 0 ? c.scales[blk] : 0.f;
    const uint8_t *page = c.pool + blk * KV_PAGE * HD;
    for (int e = t; e < (hi - lo) * HD; e += ROW_T) {
        const int slot = lo + e / HD, d = e % HD;
        const float y = id >= 0 ? (float)((int)page[which ? v_byte<HD>(slot, d) : k_byte<HD>(slot, d)] - 128) * scale
                                : 0.f;
        put_value(x, type, (a + (pos0 + slot - base)) * ld + h * HD + d, y);
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

// One wavefront to a row and query head: 64 keys at a time, a key to a lane, then
// HD / 64 channels to a lane.
template <int HD>
__global__ __launch_bounds__(64) void k_kv_rows(Fh3kAttn a, Fh3kKv c, const void *__restrict__ q, int64_t ldq,
                                                void *__restrict__ o, int64_t ldo, Fh3kSeqs s) {
    __shared__ float sq[HD], sp[64];
    const int lane = threadIdx.x, h = blockIdx.y, m = h / (a.heads / a.kv_heads);
    int seq, first, cnt, len, base;
    int64_t at;
    if (!find_unit(blockIdx.x, s.n_seq, [&](int i) { int b, n; seq_rows(s, i, b, n); return (int64_t)n; }, seq, at))
        return;
    seq_rows(s, seq, first, cnt);
    kv_len(c, seq, cnt, len, base);
    const int row = first + (int)at, pos = base + (int)at;
    for (int d = lane; d < HD; d += 64) sq[d] = value_at(q, a.type, row * ldq + h * HD + d);
    __syncthreads();
    const int end = a.causal && pos + 1 < len ? pos + 1 : len;
    bool some = false;  // the row sees a key
    float top = -INFINITY, sum = 0.f, acc[HD / 64] = {};
    for (int j0 = 0; j0 < end; j0 += 64) {
        const int j = j0 + lane, id = kv_page(c, seq, j0 >> 6);
        if (id < 0) continue;
        some = true;
        const int64_t blk = ((int64_t)id * c.kv_heads + m) * 2;
        const uint8_t *kp = c.pool + blk * KV_PAGE * HD, *vp = kp + KV_PAGE * HD;
        float x = -INFINITY;
        if (j < end) {
            x = 0.f;
            for (int d = 0; d < HD; d++) x = fmaf(sq[d], (float)((int)kp[k_byte<HD>(lane, d)] - 128), x);
            x *= c.scales[blk] * a.scale;
            if (a.softcap > 0.f) x = a.softcap * tanhf(x / a.softcap);
            if (a.slopes) x -= a.slopes[h] * fabsf((float)(pos - j));
        }
        float t = x;
        for (int w = 1; w < 64; w <<= 1) t = fmaxf(t, __shfl_xor(t, w));
        t = fmaxf(t, top);
        const float keep = top == -INFINITY ? 0.f : expf(top - t);
        const float p = j < end ? expf(x - t) : 0.f;
        top = t;
        sum = sum * keep + p;
        __syncthreads();
        sp[lane] = p * c.scales[blk + 1];
        __syncthreads();
        for (int e = 0; e < HD / 64; e++) {
            acc[e] *= keep;
            for (int l = 0; l < 64 && j0 + l < end; l++)
                acc[e] = fmaf(sp[l], (float)((int)vp[v_byte<HD>(l, 64 * e + lane)] - 128), acc[e]);
        }
    }
    for (int w = 1; w < 64; w <<= 1) sum += __shfl_xor(sum, w);
    for (int e = 0; e < HD / 64; e++)
        put_value(o, a.type, row * ldo + h * HD + 64 * e + lane, some ? acc[e] / sum : 0.f);
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

extern "C" size_t fh3k_kv_attn_ws_bytes(const Fh3kAttn *, const Fh3kKv *, Fh3kSeqs) { return 0; }

extern "C" hipError_t fh3k_kv_attn(const Fh3kAttn *a, const Fh3kKv *c, const void *q, int64_t ldq, void *o,
                                   int64_t ldo, Fh3kSeqs s, void *, hipStream_t st) {
    const dim3 grid(s.n_tok, a->heads);
    if (a->hd == 128)
        hipLaunchKernelGGL(k_kv_rows<128>, grid, dim3(64), 0, st, *a, *c, q, ldq, o, ldo, s);
    else
        hipLaunchKernelGGL(k_kv_rows<64>, grid, dim3(64), 0, st, *a, *c, q, ldq, o, ldo, s);
    return hipGetLastError();
}
