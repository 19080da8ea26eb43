// fh3_mx.hip -- microscaled (MX) operands: rows quantised to FP4 or FP8 codes
// with a power of two for each 32 of them (fh3_hip_mx_quantize_dev), read back
// (fh3_hip_mx_dequant_dev), made by the norm before a product
// (fh3_hip_mx_norm_dev), and their products on the block-scaled matrix
// instructions (fh3_hip_mx_matmul_dev, fh3_hip_mx_matmul_swiglu_dev).
#include "fh3_seqs.h"

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef short i16x2 __attribute__((ext_vector_type(2)));

constexpr int MX_BLOCK = 32;

// ---------------------------------------------------------------------------
// Values, eight to a lane: a block of 32 is the four lanes of a quad
// ---------------------------------------------------------------------------
template <int T> __device__ __forceinline__ void load8(const void *p, int64_t i, float (&v)[8]) {
    if constexpr (T == FH3K_F32) {
        const f32x4 a = *(const f32x4 *)((const float *)p + i), b = *(const f32x4 *)((const float *)p + i + 4);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            v[k] = a[k];
            v[4 + k] = b[k];
        }
    } else {
        const u32x4 a = *(const u32x4 *)((const uint16_t *)p + i);
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const uint32_t h = a[k >> 1] >> (16 * (k & 1)) & 0xFFFFu;
            if constexpr (T == FH3K_F16) v[k] = (float)__builtin_bit_cast(_Float16, (uint16_t)h);
            else v[k] = __builtin_bit_cast(float, h << 16);
        }
    }
}

template <int T> __device__ __forceinline__ uint16_t to_half(float v) {
    if constexpr (T == FH3K_F16) return __builtin_bit_cast(uint16_t, (_Float16)v);
    else return __builtin_bit_cast(uint16_t, (__bf16)v);
}

// Stores eight values, each rounded once to the type, and leaves them as they were stored.
template <int T> __device__ __forceinline__ void store8(void *p, int64_t i, float (&v)[8]) {
    if constexpr (T == FH3K_F32) {
        *(f32x4 *)((float *)p + i) = f32x4{v[0], v[1], v[2], v[3]};
        *(f32x4 *)((float *)p + i + 4) = f32x4{v[4], v[5], v[6], v[7]};
    } else {
        u32x4 a;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const uint32_t lo = to_half<T>(v[2 * k]), hi = to_half<T>(v[2 * k + 1]);
            a[k] = lo | hi << 16;
            if constexpr (T == FH3K_F16) {
                v[2 * k] = (float)__builtin_bit_cast(_Float16, (uint16_t)lo);
                v[2 * k + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)hi);
            } else {
                v[2 * k] = __builtin_bit_cast(float, lo << 16);
                v[2 * k + 1] = __builtin_bit_cast(float, hi << 16);
            }
        }
        *(u32x4 *)((uint16_t *)p + i) = a;
    }
}

__device__ __forceinline__ uint32_t quad_max(uint32_t a) {
    const uint32_t b = __builtin_amdgcn_update_dpp(0, a, 0xB1, 0xF, 0xF, true);  // lanes 1 0 3 2
    a = a > b ? a : b;
    const uint32_t c = __builtin_amdgcn_update_dpp(0, a, 0x4E, 0xF, 0xF, true);  // lanes 2 3 0 1
    return a > c ? a : c;
}

// The scale byte of a block whose largest magnitude has the bits u: the least s >= 0
// with amax <= top * 2^(s - 127).  448 = 1.75 * 2^8 and 6 = 1.5 * 2^2, so one more
// power of two is needed where the fraction is above .75 (.5): where the sum carries.
// NaN and infinity (whose bits are above all others) give 255.
template <bool F8> __device__ __forceinline__ uint32_t mx_scale(uint32_t u) {
    const int s = (int)((u + (F8 ? 0x1FFFFFu : 0x3FFFFFu)) >> 23) - (F8 ? 8 : 2);
    return u >= 0x7F800000u ? 255u : s > 0 ? (uint32_t)s : 0u;
}
// 2^(s - 127); the conversions take its exponent alone, so zero bits serve for s = 0
__device__ __forceinline__ float mx_unit(uint32_t s) { return __builtin_bit_cast(float, s << 23); }

// A quad's block to codes (eight of each lane: 4 or 8 bytes) and its scale byte.  The
// conversions divide by the scale and round to the nearest, ties to even, in one.
template <bool F8> __device__ __forceinline__ void mx_codes(const float (&in)[8], u32x2 &code, uint32_t &s) {
    float v[8];
    uint32_t u = 0;
#pragma unroll
    for (int k = 0; k < 8; k++) {
        const uint32_t b = __builtin_bit_cast(uint32_t, in[k]) & 0x7FFFFFFFu;
        u = u > b ? u : b;
    }
    s = mx_scale<F8>(quad_max(u));
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] = s == 255u ? 0.f : in[k];
    const float unit = mx_unit(s == 255u ? 127u : s);
    if constexpr (F8) {
        i16x2 a = {0, 0}, b = {0, 0};
        a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(a, v[0], v[1], unit, false);
        a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(a, v[2], v[3], unit, true);
        b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, v[4], v[5], unit, false);
        b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, v[6], v[7], unit, true);
        code = u32x2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
    } else {
        uint32_t a = 0;
        a = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(a, v[0], v[1], unit, 0);
        a = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(a, v[2], v[3], unit, 1);
        a = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(a, v[4], v[5], unit, 2);
        a = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(a, v[6], v[7], unit, 3);
        code = u32x2{a, 0};
    }
}
// Values col .. col + 7 of a row; every lane of the quad calls it.
template <bool F8> __device__ __forceinline__ void mx_store(const Fh3kMx &y, int64_t row, int col, const float (&v)[8]) {
    u32x2 code;
    uint32_t s;
    mx_codes<F8>(v, code, s);
    if constexpr (F8) *(u32x2 *)(y.codes + row * y.ld + col) = code;
    else *(uint32_t *)(y.codes + row * y.ld + col / 2) = code.x;
    if ((col & (MX_BLOCK - 1)) == 0) y.scales[row * y.lds + col / MX_BLOCK] = (uint8_t)s;
}

__device__ __forceinline__ float fp4_value(uint32_t c) {
    const uint32_t m = c & 7;
    const float a = m < 2 ? 0.5f * (float)m : __builtin_bit_cast(float, (126u + (m >> 1)) << 23 | (m & 1) << 22);
    return c & 8 ? -a : a;
}
__device__ __forceinline__ float fp8_value(uint32_t c) {
    const uint32_t e = c >> 3 & 15, f = c & 7;
    float a = e ? __builtin_bit_cast(float, (e + 120) << 23 | f << 20) : (float)f * 0x1p-9f;
    if ((c & 127) == 127) a = __builtin_bit_cast(float, 0x7FC00000u);
    return c & 128 ? -a : a;
}
// 2^(s - 127) as a factor: 2^-127 lies below fp32's normal numbers, 255 is NaN
__device__ __forceinline__ float mx_factor(uint32_t s) {
    return __builtin_bit_cast(float, s == 255u ? 0x7FC00000u : s ? s << 23 : 0x00400000u);
}

// Rows to codes.  rpw rows to a workgroup, eight values to a lane.  Bound by memory.
template <int T, bool F8> __global__ __launch_bounds__(256) void k_mx_quantize(const void *__restrict__ x, int64_t ldx,
                                                                               Fh3kMx y, int lanes) {
    const int64_t row = (int64_t)blockIdx.x * (256 / lanes) + threadIdx.x / lanes;
    const int col = 8 * (blockIdx.y * lanes + threadIdx.x % lanes);
    if (row >= y.rows || col >= y.in) return;  // whole quads: in is a multiple of 32
    float v[8];
    load8<T>(x, row * ldx + col, v);
    mx_store<F8>(y, row, col, v);
}

template <int T> __global__ __launch_bounds__(256) void k_mx_dequant(Fh3kMx x, void *__restrict__ y, int64_t ldy, int lanes) {
    const int64_t row = (int64_t)blockIdx.x * (256 / lanes) + threadIdx.x / lanes;
    const int col = 8 * (blockIdx.y * lanes + threadIdx.x % lanes);
    if (row >= x.rows || col >= x.in) return;
    const float f = mx_factor(x.scales[row * x.lds + col / MX_BLOCK]);
    float v[8];
    if (x.type == FH3K_MX_FP8) {
        const u32x2 c = *(const u32x2 *)(x.codes + row * x.ld + col);
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = fp8_value(c[k >> 2] >> (8 * (k & 3)) & 255) * f;
    } else {
        const uint32_t c = *(const uint32_t *)(x.codes + row * x.ld + col / 2);
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = fp4_value(c >> (4 * k) & 15) * f;
    }
    store8<T>(y, row * ldy + col, v);
}

// A 64-bit value cut to fp32, the last bit set where anything was cut off: rounding
// that to a code gives what rounding the value itself gives.
__device__ __forceinline__ float cut(double d) {
    const float f = (float)d;
    const double b = (double)f;
    uint32_t u = __builtin_bit_cast(uint32_t, f);
    if (b != d) u = (u - (fabs(b) > fabs(d) ? 1u : 0u)) | 1u;
    return __builtin_bit_cast(float, u);
}

// ---------------------------------------------------------------------------
// Norm: a workgroup to a row, which stays in registers between its two uses.
// Squares, their sum and the values up to their rounding are in 64 bits: rows of any
// finite size, and codes that are the formula's.  Bound by memory.
// ---------------------------------------------------------------------------
template <int T, bool F8, int C> __global__ __launch_bounds__(1024) void k_mx_norm(
    const void *__restrict__ x, int64_t ldx, const void *add, int64_t lda, void *sum, int64_t lds,
    const float *__restrict__ w, float eps, const float *__restrict__ shift, const float *__restrict__ scale, Fh3kMx y) {
    __shared__ double part[16];
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, nt = blockDim.x, n = (int)y.in;
    float v[C][8];
    double ss = 0;
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int col = 8 * (c * nt + tid);
        if (col < n) {
            load8<T>(x, row * ldx + col, v[c]);
            if (add) {
                float a[8];
                load8<T>(add, row * lda + col, a);
#pragma unroll
                for (int k = 0; k < 8; k++) v[c][k] += a[k];
            }
            if (sum) store8<T>(sum, row * lds + col, v[c]);
#pragma unroll
            for (int k = 0; k < 8; k++) ss += (double)v[c][k] * (double)v[c][k];
        }
    }
#pragma unroll
    for (int m = 32; m; m >>= 1) ss += __shfl_xor(ss, m);
    if ((tid & 63) == 0) part[tid >> 6] = ss;
    __syncthreads();
    ss = 0;
    for (int i = 0; i < nt >> 6; i++) ss += part[i];
    const double r = 1.0 / sqrt(ss / n + (double)eps);
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int col = 8 * (c * nt + tid);
        if (col < n) {
            double d[8];
            float u[8], p[8], q[8];
            load8<FH3K_F32>(w, col, p);
#pragma unroll
            for (int k = 0; k < 8; k++) d[k] = (double)v[c][k] * r * (double)p[k];
            if (shift) {
                load8<FH3K_F32>(scale, row * n + col, p);
                load8<FH3K_F32>(shift, row * n + col, q);
#pragma unroll
                for (int k = 0; k < 8; k++) d[k] = d[k] * (1.0 + (double)p[k]) + (double)q[k];
            }
#pragma unroll
            for (int k = 0; k < 8; k++) u[k] = cut(d[k]);
            mx_store<F8>(y, row, col, u);
        }
    }
}

// ---------------------------------------------------------------------------
// Product.  One wavefront: 16 weight rows (A) x 16 tokens (B), 128 values of a
// row at a step.  v_mfma_scale_f32_16x16x128: lane (r, g) holds of row r the FP4
// codes 32 g .. 32 g + 31, or the FP8 codes 16 g .. + 15 and 64 + 16 g .. + 15, and
// the scale of block g in either case.
// ---------------------------------------------------------------------------
__device__ __forceinline__ void set4(i32x8 &v, int at, const u32x4 &a) {
#pragma unroll
    for (int k = 0; k < 4; k++) v[at + k] = (int)a[k];
}
// e4m3 codes whose magnitude is 2 or more (bit 6 set); the others are c ^ that.  Within
// each part the products with e2m1 codes span no more than the 13 bits that the
// instruction keeps below the largest of eight, so both are summed exactly.
__device__ __forceinline__ uint32_t fp8_large(uint32_t c) {
    const uint32_t m = c & 0x40404040u, t = m << 1;
    return c & (t | (t - (m >> 6)));
}


template <bool F8> __global__ __launch_bounds__(256) void k_mx_simple(Fh3kMx w, Fh3kMx x, float *__restrict__ y) {
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int64_t n0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * 16, m0 = (int64_t)blockIdx.y * 16;
    if (n0 >= w.rows) return;
    const int64_t n = n0 + r < w.rows ? n0 + r : w.rows - 1, m = m0 + r < x.rows ? m0 + r : x.rows - 1;
    const uint8_t *wc = w.codes + n * w.ld, *xc = x.codes + m * x.ld, *ws = w.scales + n * w.lds, *xs = x.scales + m * x.lds;
    const int nb = (int)(w.in / MX_BLOCK);
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int b = 0; b < nb; b += 4) {
        i32x8 a = {}, c = {};
        int sa = 0, sb = 0;
        if (b + g < nb) {
            set4(a, 0, *(const u32x4 *)(wc + (b + g) * 16));
            sa = ws[b + g];
            sb = xs[b + g];
            if (!F8) set4(c, 0, *(const u32x4 *)(xc + (b + g) * 16));
        }
        if constexpr (F8) {
            if (b + (g >> 1) < nb) set4(c, 0, *(const u32x4 *)(xc + b * 32 + g * 16));
            if (b + 2 + (g >> 1) < nb) set4(c, 4, *(const u32x4 *)(xc + b * 32 + 64 + g * 16));
            i32x8 h;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                h[k] = (int)fp8_large((uint32_t)c[k]);
                c[k] ^= h[k];
            }
            acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, h, acc, 4, 0, 0, sa, 0, sb);
        }
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, c, acc, 4, F8 ? 0 : 4, 0, sa, 0, sb);
    }
    if (m0 + r < x.rows)
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (n0 + 4 * g + k < w.rows) y[(m0 + r) * w.rows + n0 + 4 * g + k] = acc[k];
}

// Sums to outputs, a value to a thread.
__device__ __forceinline__ float silu(float g) { return g / (1.f + __builtin_amdgcn_exp2f(-LOG2E * g)); }

template <int T> __global__ __launch_bounds__(256) void k_mx_finish(const float *__restrict__ p, int64_t rows, int64_t n, Fh3kMxOut o) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t t = i / n, c = i - t * n;
    if (t >= rows) return;
    float v = p[i];
    if (o.bias) v += o.bias[c];
    if (o.res) {
        const float h = value_at(o.res, T, t * o.ldres + c);
        v = o.gate ? __builtin_fmaf(o.gate[i], v, h) : h + v;
    }
    if constexpr (T == FH3K_F32) ((float *)o.out)[t * o.ldo + c] = v;
    else ((uint16_t *)o.out)[t * o.ldo + c] = to_half<T>(v);
}

template <bool F8> __global__ __launch_bounds__(256) void k_mx_swiglu(const float *__restrict__ p, const float *__restrict__ bias, Fh3kMx y) {
    const int64_t row = blockIdx.x, f = y.in;
    const int col = 8 * (blockIdx.y * 256 + threadIdx.x);
    if (col >= f) return;
    float v[8], g[8], a[8];
    load8<FH3K_F32>(p, row * 2 * f + col, v);
    load8<FH3K_F32>(p, row * 2 * f + f + col, g);
#pragma unroll
    for (int k = 0; k < 8; k++) {
        if (bias) {
            v[k] += bias[col + k];
            g[k] += bias[f + col + k];
        }
        a[k] = v[k] * silu(g[k]);
    }
    mx_store<F8>(y, row, col, a);
}

// lanes to a row: a power of two, eight values each
int row_lanes(int64_t in) {
    int n = 4;
    while (n < 256 && n * 8 < in) n *= 2;
    return n;
}

template <class F> hipError_t by_type(int type, F f) {
    switch (type) {
        case FH3K_F32: f(std::integral_constant<int, FH3K_F32>{}); break;
        case FH3K_F16: f(std::integral_constant<int, FH3K_F16>{}); break;
        default: f(std::integral_constant<int, FH3K_BF16>{}); break;
    }
    return hipGetLastError();
}

}  // namespace

extern "C" hipError_t fh3k_mx_quantize(int type, const void *x, int64_t ldx, const Fh3kMx *y, hipStream_t st) {
    const int lanes = row_lanes(y->in), rpw = 256 / lanes;
    const dim3 grid((unsigned)((y->rows + rpw - 1) / rpw), (unsigned)((y->in + 8 * lanes - 1) / (8 * lanes)));
    return by_type(type, [&](auto t) {
        if (y->type == FH3K_MX_FP8) k_mx_quantize<t(), true><<<grid, 256, 0, st>>>(x, ldx, *y, lanes);
        else k_mx_quantize<t(), false><<<grid, 256, 0, st>>>(x, ldx, *y, lanes);
    });
}

extern "C" hipError_t fh3k_mx_dequant(const Fh3kMx *x, int type, void *y, int64_t ldy, hipStream_t st) {
    const int lanes = row_lanes(x->in), rpw = 256 / lanes;
    const dim3 grid((unsigned)((x->rows + rpw - 1) / rpw), (unsigned)((x->in + 8 * lanes - 1) / (8 * lanes)));
    return by_type(type, [&](auto t) { k_mx_dequant<t()><<<grid, 256, 0, st>>>(*x, y, ldy, lanes); });
}

extern "C" hipError_t fh3k_mx_norm(int type, const void *x, int64_t ldx, const void *add, int64_t lda, void *sum, int64_t lds,
                                   const float *w, float eps, const float *shift, const float *scale, const Fh3kMx *y,
                                   hipStream_t st) {
    // chunks of eight values to a lane: as few as rows of up to 1024 lanes need
    int nt = 64;
    while (nt < 1024 && nt * 8 < y->in) nt += 64;
    const int c = (int)((y->in + 8 * nt - 1) / (8 * nt));
    return by_type(type, [&](auto t) {
        auto go = [&](auto f8, auto cc) {
            k_mx_norm<t(), f8(), cc()><<<(unsigned)y->rows, nt, 0, st>>>(x, ldx, add, lda, sum, lds, w, eps, shift, scale, *y);
        };
        auto pick = [&](auto f8) {
            if (c <= 1) go(f8, std::integral_constant<int, 1>{});
            else if (c <= 2) go(f8, std::integral_constant<int, 2>{});
            else go(f8, std::integral_constant<int, 4>{});
        };
        if (y->type == FH3K_MX_FP8) pick(std::true_type{});
        else pick(std::false_type{});
    });
}

extern "C" int fh3k_mx_matmul_fits(const Fh3kMx *w, const Fh3kMx *x) {
    return (w->rows + 63) / 64 < ((int64_t)1 << 31) && (x->rows + 15) / 16 < 65536 &&
           w->rows * x->rows <= ((int64_t)1 << 38);
}

extern "C" size_t fh3k_mx_matmul_ws_bytes(const Fh3kMx *w, const Fh3kMx *x, int) {
    return (size_t)w->rows * x->rows * sizeof(float);
}

extern "C" hipError_t fh3k_mx_matmul(const Fh3kMx *w, const Fh3kMx *x, const Fh3kMxOut *o, void *ws, hipStream_t st) {
    const dim3 grid((unsigned)((w->rows + 63) / 64), (unsigned)((x->rows + 15) / 16));
    float *p = (float *)ws;
    if (x->type == FH3K_MX_FP8) k_mx_simple<true><<<grid, 256, 0, st>>>(*w, *x, p);
    else k_mx_simple<false><<<grid, 256, 0, st>>>(*w, *x, p);
    if (o->y) {
        const dim3 g2((unsigned)x->rows, (unsigned)((o->y->in + 2047) / 2048));
        if (o->y->type == FH3K_MX_FP8) k_mx_swiglu<true><<<g2, 256, 0, st>>>(p, o->bias, *o->y);
        else k_mx_swiglu<false><<<g2, 256, 0, st>>>(p, o->bias, *o->y);
        return hipGetLastError();
    }
    return by_type(o->type, [&](auto t) {
        k_mx_finish<t()><<<(unsigned)((x->rows * w->rows + 255) / 256), 256, 0, st>>>(p, x->rows, w->rows, *o);
    });
}
