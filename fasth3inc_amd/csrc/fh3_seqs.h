// fh3_seqs.h -- device helpers of the kernels over packed sequences
// (fh3_seqs.hip, fh3_kv.hip): rows of the three value types, which rows are
// which sequence's, and the cache's byte order.
#ifndef FH3_SEQS_H
#define FH3_SEQS_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fh3_kernels.h"

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int KV_PAGE = 64;
constexpr float LOG2E = 1.4426950408889634f;

// value i of an array of F32, F16 or BF16
__device__ __forceinline__ float value_at(const void *p, int type, int64_t i) {
    if (type == FH3K_F32) return ((const float *)p)[i];
    if (type == FH3K_F16) return (float)((const _Float16 *)p)[i];
    return __builtin_bit_cast(float, (uint32_t)((const uint16_t *)p)[i] << 16);
}

// Rows a .. a + cnt - 1 of sequence s.  Whatever first holds, they lie within n_tok.
__device__ __forceinline__ void seq_rows(const Fh3kSeqs &s, int i, int &a, int &cnt) {
    if (s.first) {
        const int lo = s.first[i], hi = s.first[i + 1];
        a = lo < 0 ? 0 : lo > s.n_tok ? s.n_tok : lo;
        const int b = hi < 0 ? 0 : hi > s.n_tok ? s.n_tok : hi;
        cnt = b > a ? b - a : 0;
    } else {
        cnt = s.n_tok / s.n_seq;
        a = i * cnt;
    }
}

// Sums over the lanes below and this one.
__device__ __forceinline__ int wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);  // row_shr 1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // row_bcast 15, 31
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);
    return x;
}
// Work unit w when sequence i has units(i) of them (fewer than 2^31 in all): its
// sequence and its place there, or false past the last.  Every lane of a
// wavefront calls it with the same w; 64 sequences at a time.  What units() noted of
// its sequence is then in lane seq % 64 (of_lane), and need not be read again.
__device__ __forceinline__ int of_lane(int x, int seq) { return __builtin_amdgcn_readlane(x, seq & 63); }
template <class F> __device__ __forceinline__ bool find_unit(int w, int n_seq, F units, int &seq, int &at) {
    const int lane = threadIdx.x & 63;
    for (int s0 = 0; s0 < n_seq; s0 += 64) {
        const int u = s0 + lane < n_seq ? units(s0 + lane) : 0;
        const int end = wave_scan(u);
        const uint64_t past = __ballot(end > w);
        if (past) {
            const int l = __builtin_ctzll(past);
            seq = s0 + l;
            at = w - (__builtin_amdgcn_readlane(end, l) - __builtin_amdgcn_readlane(u, l));
            return true;
        }
        w -= __builtin_amdgcn_readlane(end, 63);
    }
    return false;
}

// The cache's byte order within the 64 x hd bytes of K or V of one page and head.
template <int HD> __device__ __forceinline__ int k_byte(int tok, int d) {
    return (((tok >> 4) * (HD / 64) + (d >> 6)) * 4 + ((d >> 4) & 3)) * 256 + (tok & 15) * 16 + (d & 15);
}
template <int HD> __device__ __forceinline__ int v_byte(int tok, int d) {
    return ((d >> 4) * 4 + ((tok >> 2) & 3)) * 256 + (d & 15) * 16 + (tok >> 4) * 4 + (tok & 3);
}

// Tokens that sequence i of a cache holds, and the position of its first new row.
__device__ __forceinline__ void kv_len(const Fh3kKv &c, int i, int cnt, int &len, int &base) {
    const int l = c.len[i] > 0 ? c.len[i] : 0, cap = c.max_pages * KV_PAGE;
    base = l - cnt;
    len = l < cap ? l : cap;
}
// The page that holds tokens 64 p .. of sequence i, or -1.
__device__ __forceinline__ int kv_page(const Fh3kKv &c, int i, int p) {
    if (p < 0 || p >= c.max_pages) return -1;
    const int id = c.table[(int64_t)i * c.max_pages + p];
    return id >= 0 && id < c.pages ? id : -1;
}

}  // namespace

#endif
