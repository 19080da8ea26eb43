// fh3_seqs.hip -- attention within packed sequences (fh3_hip_attention_seqs_dev).
#include "fh3_seqs.h"

namespace {

// One wavefront to a row and query head: 64 keys at a time, a key to a lane, then
// HD / 64 channels to a lane.
template <int HD>
__global__ __launch_bounds__(64) void k_attn_rows(Fh3kAttn a, const void *__restrict__ q, int64_t ldq,
                                                  const void *__restrict__ k, int64_t ldk,
                                                  const void *__restrict__ v, int64_t ldv, void *__restrict__ o,
                                                  int64_t ldo, Fh3kSeqs s, const int *__restrict__ prefix) {
    __shared__ float sq[HD], sp[64];
    const int lane = threadIdx.x, h = blockIdx.y, m = h / (a.heads / a.kv_heads);
    int seq, first, cnt;
    int64_t at;
    if (!find_unit(blockIdx.x, s.n_seq, [&](int i) { int b, n; seq_rows(s, i, b, n); return (int64_t)n; }, seq, at))
        return;
    seq_rows(s, seq, first, cnt);
    const int i = (int)at, pre = prefix ? prefix[seq] : 0;
    for (int d = lane; d < HD; d += 64) sq[d] = value_at(q, a.type, (first + i) * ldq + h * HD + d);
    __syncthreads();
    const int end = a.causal ? (pre > i + 1 ? (pre < cnt ? pre : cnt) : i + 1) : cnt;
    float top = -INFINITY, sum = 0.f, acc[HD / 64] = {};
    for (int j0 = 0; j0 < end; j0 += 64) {
        const int j = j0 + lane;
        float x = -INFINITY;
        if (j < end) {
            x = 0.f;
            for (int d = 0; d < HD; d++) x = fmaf(sq[d], value_at(k, a.type, (first + j) * ldk + m * HD + d), x);
            x *= a.scale;
            if (a.softcap > 0.f) x = a.softcap * tanhf(x / a.softcap);
            if (a.slopes) x -= a.slopes[h] * fabsf((float)(i - j));
        }
        float t = x;
        for (int w = 1; w < 64; w <<= 1) t = fmaxf(t, __shfl_xor(t, w));
        t = fmaxf(t, top);
        const float keep = top == -INFINITY ? 0.f : expf(top - t);
        const float p = j < end ? expf(x - t) : 0.f;
        top = t;
        sum = sum * keep + p;
        __syncthreads();
        sp[lane] = p;
        __syncthreads();
        for (int c = 0; c < HD / 64; c++) {
            acc[c] *= keep;
            for (int e = 0; e < 64 && j0 + e < end; e++)
                acc[c] = fmaf(sp[e], value_at(v, a.type, (first + j0 + e) * ldv + m * HD + 64 * c + lane), acc[c]);
        }
    }
    for (int w = 1; w < 64; w <<= 1) sum += __shfl_xor(sum, w);
    for (int c = 0; c < HD / 64; c++)
        put_value(o, a.type, (first + i) * ldo + h * HD + 64 * c + lane, end > 0 ? acc[c] / sum : 0.f);
}

}  // namespace

extern "C" hipError_t fh3k_attn_seqs(const Fh3kAttn *a, const void *q, int64_t ldq, const void *k, int64_t ldk,
                                     const void *v, int64_t ldv, void *o, int64_t ldo, Fh3kSeqs s, const int *prefix,
                                     hipStream_t st) {
    const dim3 grid(s.n_tok, a->heads);
    if (a->hd == 128)
        hipLaunchKernelGGL(k_attn_rows<128>, grid, dim3(64), 0, st, *a, q, ldq, k, ldk, v, ldv, o, ldo, s, prefix);
    else
        hipLaunchKernelGGL(k_attn_rows<64>, grid, dim3(64), 0, st, *a, q, ldq, k, ldk, v, ldv, o, ldo, s, prefix);
    return hipGetLastError();
}
