// fh3_mx.hip -- microscaled (MX) operands: rows quantised to FP4 or FP8 codes
// with a power of two for each 32 of them (fh3_hip_mx_quantize_dev), read back
// (fh3_hip_mx_dequant_dev), made by the norm before a product
// (fh3_hip_mx_norm_dev), and their products on the block-scaled matrix
// instructions (fh3_hip_mx_matmul_dev, fh3_hip_mx_matmul_swiglu_dev): k_mx_few and
// k_mx_stream for up to 64 rows, k_mx_gemm for more; plan_of picks.
#include "fh3_seqs.h"

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef short i16x2 __attribute__((ext_vector_type(2)));

constexpr int MX_BLOCK = 32;
constexpr float LOG2E_REST = 1.92596299e-08f;   // of log2(e) below LOG2E

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

// What is written once and not read here goes past L2's other lines: 13824 x 5120 fp32 to FP4 and back 99.6 -> 91.3 us,
// norm of 14430 x 5376 204 -> 198, 8192 x 5120 -> 15360 360 -> 328 (the tiles' operands stay in L2).
template <class V> __device__ __forceinline__ void put_past(const V &v, void *p) { __builtin_nontemporal_store(v, (V *)p); }

// Stores eight values, each rounded once to the type, and leaves them as they were stored.
template <int T> __device__ __forceinline__ void store8(void *p, int64_t i, float (&v)[8]) {
    if constexpr (T == FH3K_F32) {
        put_past(f32x4{v[0], v[1], v[2], v[3]}, (float *)p + i);
        put_past(f32x4{v[4], v[5], v[6], v[7]}, (float *)p + i + 4);
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
        put_past(a, (uint16_t *)p + i);
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

// Eight values to codes of a block with scale byte s: 4 or 8 bytes.  The conversions
// divide by the scale and round to the nearest, ties to even, in one.
template <bool F8> __device__ __forceinline__ u32x2 mx_encode(const float (&in)[8], uint32_t s) {
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] = s == 255u ? 0.f : in[k];
    const float unit = mx_unit(s == 255u ? 127u : s);
    if constexpr (F8) {
        i16x2 a = {0, 0}, b = {0, 0};
        a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(a, v[0], v[1], unit, false);
        a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(a, v[2], v[3], unit, true);
        b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, v[4], v[5], unit, false);
        b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, v[6], v[7], unit, true);
        return u32x2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
    } else {
        uint32_t a = 0;
        a = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(a, v[0], v[1], unit, 0);
        a = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(a, v[2], v[3], unit, 1);
        a = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(a, v[4], v[5], unit, 2);
        a = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(a, v[6], v[7], unit, 3);
        return u32x2{a, 0};
    }
}
// Values col .. col + 7 of a row; every lane of the quad calls it.
template <bool F8> __device__ __forceinline__ void mx_store(const Fh3kMx &y, int64_t row, int col, const float (&v)[8]) {
    uint32_t u = 0;
#pragma unroll
    for (int k = 0; k < 8; k++) {
        const uint32_t b = __builtin_bit_cast(uint32_t, v[k]) & 0x7FFFFFFFu;
        u = u > b ? u : b;
    }
    const uint32_t s = mx_scale<F8>(quad_max(u));
    const u32x2 code = mx_encode<F8>(v, s);
    if constexpr (F8) put_past(code, y.codes + row * y.ld + col);
    else put_past((uint32_t)code.x, y.codes + row * y.ld + col / 2);
    if ((col & (MX_BLOCK - 1)) == 0) y.scales[row * y.lds + col / MX_BLOCK] = (uint8_t)s;
}

// Eight codes' values under scale byte s; exact in fp32 (checked for every code and scale).
template <bool F8> __device__ __forceinline__ void mx_decode(const u32x2 &c, uint32_t s, float (&v)[8]) {
    const float unit = mx_unit(s);
#pragma unroll
    for (int k = 0; k < 4; k++) {
        f32x2 p;
        if constexpr (F8) {
            if (k & 1) p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c[k >> 1], unit, true);
            else p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c[k >> 1], unit, false);
        } else {
            if (k == 0) p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[0], unit, 0);
            else if (k == 1) p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[0], unit, 1);
            else if (k == 2) p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[0], unit, 2);
            else p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[0], unit, 3);
        }
        const float nan = __builtin_bit_cast(float, 0x7FC00000u);
        v[2 * k] = s == 255u ? nan : p[0];
        v[2 * k + 1] = s == 255u ? nan : p[1];
    }
}

// Rows to codes and back: a wavefront's lanes on neighbouring eights of values, MX_EACH
// of them to a lane a workgroup's width apart, loaded before the first is used.  Bound by memory:
// 13824 x 5120 fp32 to FP4 and back to bf16 in 91 us (500 MB, 5.5 TB/s; one eight to a lane 123).
constexpr int MX_EACH = 4;
// Workgroups by rows: a launch's x has fewer than 2^32 lanes, so 2^21 workgroups there, the rest by z.
constexpr int64_t MX_GRID = 1 << 21;
__device__ __forceinline__ int64_t first_row() { return blockIdx.x + MX_GRID * blockIdx.z; }
dim3 row_grid(int64_t groups, int64_t y) {
    return dim3((unsigned)(groups < MX_GRID ? groups : MX_GRID), (unsigned)y, (unsigned)((groups + MX_GRID - 1) / MX_GRID));
}
template <int T, bool F8> __global__ __launch_bounds__(256) void k_mx_quantize(const void *__restrict__ x, int64_t ldx,
                                                                               Fh3kMx y, int lanes) {
    const int64_t row = first_row() * (256 / lanes) + threadIdx.x / lanes;
    const int col = 8 * (blockIdx.y * lanes * MX_EACH + threadIdx.x % lanes);
    if (row >= y.rows) return;
    float v[MX_EACH][8];
#pragma unroll
    for (int i = 0; i < MX_EACH; i++)
        if (col + 8 * lanes * i < y.in) load8<T>(x, row * ldx + col + 8 * lanes * i, v[i]);
#pragma unroll
    for (int i = 0; i < MX_EACH; i++)   // whole quads: in is a multiple of 32
        if (col + 8 * lanes * i < y.in) mx_store<F8>(y, row, col + 8 * lanes * i, v[i]);
}

template <int T, bool F8> __global__ __launch_bounds__(256) void k_mx_dequant(Fh3kMx x, void *__restrict__ y, int64_t ldy, int lanes) {
    const int64_t row = first_row() * (256 / lanes) + threadIdx.x / lanes;
    const int col = 8 * (blockIdx.y * lanes * MX_EACH + threadIdx.x % lanes);
    if (row >= x.rows) return;
    u32x2 c[MX_EACH];
    uint32_t s[MX_EACH];
#pragma unroll
    for (int i = 0; i < MX_EACH; i++) {
        const int n = col + 8 * lanes * i;
        if (n >= x.in) continue;
        s[i] = x.scales[row * x.lds + n / MX_BLOCK];
        if constexpr (F8) c[i] = *(const u32x2 *)(x.codes + row * x.ld + n);
        else c[i].x = *(const uint32_t *)(x.codes + row * x.ld + n / 2);
    }
#pragma unroll
    for (int i = 0; i < MX_EACH; i++) {
        const int n = col + 8 * lanes * i;
        if (n >= x.in) continue;
        float v[8];
        mx_decode<F8>(c[i], s[i], v);
        store8<T>(y, row * ldy + n, v);
    }
}

// A 64-bit value cut to fp32, the last bit set where anything was cut off: rounding
// that to a code gives what rounding the value itself gives.  Past fp32's range: infinite.
__device__ __forceinline__ float cut(double d) {
    const float f = (float)d;
    const double b = (double)f;
    uint32_t u = __builtin_bit_cast(uint32_t, f);
    if (b != d && fabs(b) <= 3.4028234663852886e38) u = (u - (fabs(b) > fabs(d) ? 1u : 0u)) | 1u;
    return __builtin_bit_cast(float, u);
}

// ---------------------------------------------------------------------------
// Norm: a workgroup to a row, which stays in registers between its two uses.
// Squares, their sum and the values up to their rounding are in 64 bits: rows of any
// finite size, and codes that are the formula's.  Bound by memory: 14430 x 5376 bf16,
// modulated, 195 us (1.17 GB, 6.0 TB/s).
// ---------------------------------------------------------------------------
template <int T, bool F8, int C> __global__ __launch_bounds__(1024) void k_mx_norm(
    const void *x, int64_t ldx, const void *add, int64_t lda, void *sum, int64_t lds,
    const float *__restrict__ w, float eps, const float *__restrict__ shift, const float *__restrict__ scale, Fh3kMx y) {
    __shared__ double part[16];
    const int64_t row = first_row();
    if (row >= y.rows) return;
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
// Products
// ---------------------------------------------------------------------------
__device__ __forceinline__ void set4(i32x8 &v, int at, const u32x4 &a) {
#pragma unroll
    for (int k = 0; k < 4; k++) v[at + k] = (int)a[k];
}
// The instruction aligns eight products to 2^E, E the largest sum of two codes' exponents
// among them, and cuts off what lies below 2^(E - 13): up to seven times 2^-13 of the
// largest product, and where large ones cancel, all that is left (FP4 rows lose nothing:
// their products span 2^4 to 2^-2).  So FP8 rows come in two products, at half the rate:
// e4m3 codes whose magnitude is 2 or more (bit 6 set), and the others.  The first part's
// products have E of 10 at most (448 = 1.75 * 2^8, 6 = 1.5 * 2^2) and are multiples of
// 2^-3 (2.25 * 0.5), the second's E of 2 (1.875, 6) and multiples of 2^-10 (2^-9 * 0.5): 13 bits
// or less below 2^E, so eight of them are summed exactly.  In one product 600 x 5120 -> 17408
// bf16 took 56 us in place of 95, 32768 x 13824 -> 5120 1839 in place of 2980, and 16 x 25600 -> 5120
// 19.1 in place of 19.8, but differed from rounded fp32 sums by 2e-4 of their norm (in two: by 1e-6).
// The selector of a byte is its place, in the permutation's second word or (+ 4) its first.
__device__ __forceinline__ void fp8_split(uint32_t c, int &large, int &small) {
    const uint32_t sel = (c >> 4 & 0x04040404u) | 0x03020100u;
    large = (int)__builtin_amdgcn_perm(c, 0u, sel);
    small = (int)__builtin_amdgcn_perm(0u, c, sel);
}

// ---------------------------------------------------------------------------
// Many rows: tiles of BW weight rows x BX tokens, NW x NX wavefronts of TW x TX
// products of 32 x 32: 256 x 256 by eight or, where those are too few for the CUs, 128 x 128
// by four.  v_mfma_scale_f32_32x32x64: lane (r, g), g = 0 or 1, holds of
// row r the FP4 codes 32 g .. + 31, or the FP8 codes 16 g .. + 15 and 32 + 16 g .. + 15,
// and the scale of block g.  A stage is 256 values of a row (128 with FP8 rows), its
// blocks taken so that a lane's scales lie side by side: block g of step t is the
// stage's block g * T + t, and the instruction picks byte t.
// Rows come to LDS by DMA in 16-byte pieces (a line of 128 bytes to eight lanes), piece
// p of row r at place p ^ r / 2 % 8 (rows of 64 bytes: p ^ r / 4 % 4), so that the pieces
// p of sixteen rows lie in different banks.  Scales come for CH stages at a time (a
// request to L2 for each row's 8 or 4 bytes of a stage took as many requests as the
// codes) and are held in registers.
// 8192 x 5120 -> 15360 FP4 322 us (4.0 PFLOP/s: products alone 190, DMA alone 193, with the
// operands' reads 280); FP8 rows, in two products: 32768 x 13824 -> 5120 2980 (3.1 PFLOP/s of both),
// 3016 x 5376 -> 28672 SwiGLU 639 (2.9), 3016 x 7168 -> 5376 fp32 175, 600 x 5120 -> 17408 95.
// ---------------------------------------------------------------------------
typedef __attribute__((address_space(3))) void lds_void;

template <int TW_, int TX_, int NW_, int NX_, bool F8_, int KS_, int NBUF_> struct Gemm {
    static constexpr int TW = TW_, TX = TX_, NW = NW_, NX = NX_, WAVES = NW * NX;
    static constexpr bool F8 = F8_;
    static constexpr int KS = KS_, NB = KS / MX_BLOCK, T = NB / 2;
    static constexpr int WROW = KS / 2, XROW = F8 ? KS : KS / 2;   // bytes of a stage's row
    static constexpr int BW = NW * TW * 32, BX = NX * TX * 32;
    static constexpr int NBUF = NBUF_, CH = NBUF == 3 ? 3 : 4;     // stages in LDS, stages of a chunk of scales
    static constexpr int HALVES = F8 ? 1 : 2;                      // steps over which a stage's loads are spread
    static constexpr int SD = NB == 8 ? 8 : 4;                     // dwords of a row's chunk in LDS
    static constexpr int WI = BW * WROW / 1024 / WAVES, XI = BX * XROW / 1024 / WAVES, D = WI + XI;   // a wavefront's DMA instructions: a stage's codes
    static constexpr int WS = BW * SD / 64 / WAVES, XS = BX * SD / 64 / WAVES;                         // and a chunk's scales
    struct Buf {
        u32x4 x[BX * XROW / 16], w[BW * WROW / 16];
    };
    struct ScaleBuf {
        uint32_t x[BX * SD], w[BW * SD];
    };
};

// place of piece p of row r among its row's P pieces, or the piece at place p
template <int P> __device__ __forceinline__ int mx_place(int r, int p) { return p ^ (P == 8 ? (r >> 1) & 7 : (r >> 2) & 3); }

constexpr uint32_t MX_OUTSIDE = 0xC0000000u;   // past every buffer here: reads as zero

__device__ __forceinline__ u32x4 mx_rsrc(const void *p, uint32_t bytes) {
    const uint64_t a = (uint64_t)(uintptr_t)p;
    return u32x4{(uint32_t)a, (uint32_t)(a >> 32) & 0xFFFFu, bytes, 0x00020000u};
}
// DMA to LDS, 16 or 4 bytes of each lane to consecutive places.  As builtins they made
// the compiler wait for all of them (vmcnt(0)) before reads of other buffers here and
// there; as asm, which has no outputs, the waits are the kernel's own.  The nops stand
// between a scalar that the VALU may have written and the load that reads it.  m0 is
// used for nothing else here.
template <int BYTES> __device__ __forceinline__ void mx_dma(const u32x4 &r, void *to, uint32_t off, int at) {
    const uint32_t lds = (uint32_t)(uintptr_t)(lds_void *)to;
    at = __builtin_amdgcn_readfirstlane(at);   // uniform, which the compiler loses sight of where it runs short of scalars
    if constexpr (BYTES == 16)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" : : "s"(lds), "v"(off), "s"(r), "s"(at) : "memory");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dword %1, %2, %3 offen lds" : : "s"(lds), "v"(off), "s"(r), "s"(at) : "memory");
}
// All but the last VM loads have landed and all operands are read, in every wavefront.
template <int VM> __device__ __forceinline__ void mx_barrier() {
    static_assert(VM < 64, "the counter's range");
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(VM) : "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// What a wavefront loads of one operand: its share of the tile's rows.
template <class G, int ROW, int N, int NS> struct Rows {
    static constexpr int P = ROW / 16, RPI = 64 / P;   // pieces of a row, rows to an instruction
    u32x4 code, scale;
    uint32_t off[N], soff[NS];                         // of this lane, for each instruction
    int piece[2];                                      // of its row, in even and odd instructions

    // rows base .. of m; those past its end: its last row
    __device__ __forceinline__ void init(const Fh3kMx &m, int64_t base, int lane) {
        if (base >= m.rows) base = m.rows - 1;
        const int64_t left = m.rows - base;
        const int last = left < N * RPI ? (int)left - 1 : N * RPI - 1;
        code = mx_rsrc(m.codes + base * m.ld, (uint32_t)(last * m.ld + (m.type == FH3K_MX_FP8 ? m.in : m.in / 2)));
        scale = mx_rsrc(m.scales + base * m.lds, (uint32_t)(last * m.lds + (m.in / MX_BLOCK + 3) / 4 * 4));
#pragma unroll
        for (int j = 0; j < 2; j++) piece[j] = mx_place<P>(j * RPI + lane / P, lane % P);
#pragma unroll
        for (int j = 0; j < N; j++) {
            const int r = j * RPI + lane / P;
            off[j] = (uint32_t)((r < last ? r : last) * m.ld) + piece[j & 1] * 16;
        }
        // stages of eight blocks have two dwords of scales to a row, here in the order [g][stage]; those of four one
#pragma unroll
        for (int j = 0; j < NS; j++) {
            const int d = j * 64 + lane, r = d / G::SD, k = d % G::SD;
            soff[j] = (uint32_t)((r < last ? r : last) * m.lds) + 4 * (G::NB == 4 ? k : (k & 3) * 2 + (k >> 2));
            if (k >= (G::NB == 4 ? G::CH : 8)) soff[j] = MX_OUTSIDE;
        }
    }
    // instruction j of stage st, of whose row `pieces` pieces are there
    template <int j> __device__ __forceinline__ void dma(u32x4 *to, int wave, int st, int pieces) const {
        mx_dma<16>(code, to + (wave * N + j) * 64, piece[j & 1] < pieces ? off[j] : MX_OUTSIDE, st * ROW);
    }
    __device__ __forceinline__ void dma_scales(uint32_t *to, int wave, int st) const {
#pragma unroll
        for (int j = 0; j < NS; j++) mx_dma<4>(scale, to + (wave * NS + j) * 64, soff[j], st * G::NB);
    }
};
template <class G> struct Load {
    Rows<G, G::WROW, G::WI, G::WS> w;
    Rows<G, G::XROW, G::XI, G::XS> x;
    int wave, blocks, end;              // blocks of a row; stages past the end load nothing, with as many instructions

    template <int d, int to> __device__ __forceinline__ void codes(typename G::Buf &b, int st) const {
        if constexpr (d < to) {
            const int left = st < end ? blocks - st * G::NB : 0;
            const int at = st < end ? st : 0;   // no offset past the rows, whose range it is subtracted from
            if constexpr (d < G::WI) w.template dma<d>(b.w, wave, at, left);
            else x.template dma<d - G::WI>(b.x, wave, at, G::F8 ? 2 * left : left);
            codes<d + 1, to>(b, st);
        }
    }
    __device__ __forceinline__ void scales(typename G::ScaleBuf &b, int st) const {
        const int at = st < end ? st : 0;
        w.dma_scales(b.w, wave, at);
        x.dma_scales(b.x, wave, at);
    }
};

template <class G> struct Frags {
    u32x4 w[G::TW];
    typename std::conditional<G::F8, i32x8, u32x4>::type x[G::TX];
};
template <class G> struct Scales {       // of a chunk: a dword (of four blocks: both lanes' halves) for each stage
    u32x4 w[G::TW], x[G::TX];
};
template <class G> struct StageScales {
    int w[G::TW], x[G::TX];
};

// piece p of row r of a stage's rows
template <int ROW> __device__ __forceinline__ u32x4 mx_piece(const u32x4 *b, int r, int p) {
    return b[r * (ROW / 16) + mx_place<ROW / 16>(r, p)];
}

// Operand n (0 .. TW - 1: weights, then tokens) of step t.
template <class G, int t, int n> __device__ __forceinline__ void mx_read(Frags<G> &f, const typename G::Buf &b, int wr, int xr, int g) {
    if constexpr (n < G::TW) {
        f.w[n] = mx_piece<G::WROW>(b.w, wr + 32 * n, g * G::T + t);
    } else {
        constexpr int i = n - G::TW;
        if constexpr (G::F8) {
            set4(f.x[i], 0, mx_piece<G::XROW>(b.x, xr + 32 * i, 2 * t + g));
            set4(f.x[i], 4, mx_piece<G::XROW>(b.x, xr + 32 * i, 2 * (G::T + t) + g));
        } else {
            f.x[i] = mx_piece<G::XROW>(b.x, xr + 32 * i, g * G::T + t);
        }
    }
}
template <class G, int n> __device__ __forceinline__ void mx_read_scale(Scales<G> &s, const typename G::ScaleBuf &b, int wr, int xr, int g) {
    const uint32_t *p = n < G::TW ? b.w + (wr + 32 * n) * G::SD : b.x + (xr + 32 * (n - G::TW)) * G::SD;
    const u32x4 v = *(const u32x4 *)(p + (G::NB == 4 ? 0 : 4 * g));
    if constexpr (n < G::TW) s.w[n] = v;
    else s.x[n - G::TW] = v;
}
// The scales of the chunk's stage c; keep: zeros where the row has ended.
template <class G, int c> __device__ __forceinline__ void mx_stage_scales(StageScales<G> &o, const Scales<G> &s, int g, int keep) {
#pragma unroll
    for (int i = 0; i < G::TW; i++) o.w[i] = (int)(G::NB == 4 ? s.w[i][c] >> (16 * g) : s.w[i][c]) & keep;
#pragma unroll
    for (int i = 0; i < G::TX; i++) o.x[i] = (int)(G::NB == 4 ? s.x[i][c] >> (16 * g) : s.x[i][c]) & keep;
}

// The products of TW tiles of weights with one of tokens, sums in accumulation
// registers.  The nops stand between an operand made by the VALU (scales, split codes)
// and the matrix instruction that reads it, which the compiler does not see here.
#define MX_MFMA(C, W, S, FMT, SEL) "v_mfma_scale_f32_32x32x64_f8f6f4 " C ", " W ", %[x], " C ", " S ", %[xs] " SEL " cbsz:4" FMT "\n\t"
#define MX_MFMA4(FMT, SEL)                                                                                           \
    asm volatile("s_nop 1\n\t" MX_MFMA("%0", "%[w0]", "%[s0]", FMT, SEL) MX_MFMA("%1", "%[w1]", "%[s1]", FMT, SEL)   \
                     MX_MFMA("%2", "%[w2]", "%[s2]", FMT, SEL) MX_MFMA("%3", "%[w3]", "%[s3]", FMT, SEL)              \
                 : "+a"(acc[0]), "+a"(acc[1]), "+a"(acc[2]), "+a"(acc[3])                                            \
                 : [w0] "v"(w[0]), [w1] "v"(w[1]), [w2] "v"(w[2]), [w3] "v"(w[3]), [x] "v"(x), [s0] "v"(s[0]),        \
                   [s1] "v"(s[1]), [s2] "v"(s[2]), [s3] "v"(s[3]), [xs] "v"(xs))
#define MX_MFMA2(FMT, SEL)                                                                                           \
    asm volatile("s_nop 1\n\t" MX_MFMA("%0", "%[w0]", "%[s0]", FMT, SEL) MX_MFMA("%1", "%[w1]", "%[s1]", FMT, SEL)   \
                 : "+a"(acc[0]), "+a"(acc[1])                                                                        \
                 : [w0] "v"(w[0]), [w1] "v"(w[1]), [x] "v"(x), [s0] "v"(s[0]), [s1] "v"(s[1]), [xs] "v"(xs))
#define MX_SEL0 "op_sel:[0,0,0] op_sel_hi:[0,0,0]"
#define MX_SEL1 "op_sel:[1,1,0] op_sel_hi:[0,0,0]"
#define MX_SEL2 "op_sel:[0,0,0] op_sel_hi:[1,1,0]"
#define MX_SEL3 "op_sel:[1,1,0] op_sel_hi:[1,1,0]"
template <int t> __device__ __forceinline__ void mx_mfma(f32x16 (&acc)[4], const u32x4 (&w)[4], const int (&s)[4], const u32x4 &x, int xs) {
    if constexpr (t == 0) MX_MFMA4(" blgp:4", MX_SEL0);
    else if constexpr (t == 1) MX_MFMA4(" blgp:4", MX_SEL1);
    else if constexpr (t == 2) MX_MFMA4(" blgp:4", MX_SEL2);
    else MX_MFMA4(" blgp:4", MX_SEL3);
}
template <int t> __device__ __forceinline__ void mx_mfma(f32x16 (&acc)[4], const u32x4 (&w)[4], const int (&s)[4], const i32x8 &x, int xs) {
    if constexpr (t == 0) MX_MFMA4("", MX_SEL0);
    else MX_MFMA4("", MX_SEL1);
}
template <int t> __device__ __forceinline__ void mx_mfma(f32x16 (&acc)[2], const u32x4 (&w)[2], const int (&s)[2], const u32x4 &x, int xs) {
    if constexpr (t == 0) MX_MFMA2(" blgp:4", MX_SEL0);
    else if constexpr (t == 1) MX_MFMA2(" blgp:4", MX_SEL1);
    else if constexpr (t == 2) MX_MFMA2(" blgp:4", MX_SEL2);
    else MX_MFMA2(" blgp:4", MX_SEL3);
}
template <int t> __device__ __forceinline__ void mx_mfma(f32x16 (&acc)[2], const u32x4 (&w)[2], const int (&s)[2], const i32x8 &x, int xs) {
    if constexpr (t == 0) MX_MFMA2("", MX_SEL0);
    else MX_MFMA2("", MX_SEL1);
}

// Operands n .. end - 1 of step t, and (SC) the chunk of scales that goes with them.
template <class G, int t, bool SC, int n, int end> __device__ __forceinline__ void mx_reads(Frags<G> &f, Scales<G> &s, const typename G::Buf &b,
                                                                                           const typename G::ScaleBuf &sb, int wr, int xr, int g) {
    if constexpr (n < end) {
        mx_read<G, t, n>(f, b, wr, xr, g);
        if constexpr (SC) mx_read_scale<G, n>(s, sb, wr, xr, g);
        mx_reads<G, t, SC, n + 1, end>(f, s, b, sb, wr, xr, g);
    }
}

// One step's products; between them operand reads of step tn from nb (SC: and the
// next chunk's scales), and where Q is 0 or 1 that half of stage `to`'s loads into lb.
// Loads are issued a few at a time: all at once they kept the matrix instructions behind
// them waiting for the address unit.  Over one step or two: 8192 x 5120 -> 15360 FP4 362,
// 353 us; FP8, of half as many steps to a stage, 815-826, 842, and 32768 x 13824 -> 5120 2860, 2890.
template <class G, int t, int tn, bool SC, int Q, int j = 0> __device__ __forceinline__ void mx_step(
    f32x16 (&acc)[G::TX][G::TW], const Frags<G> &f, const StageScales<G> &s, Frags<G> &nf, Scales<G> &ns, const typename G::Buf &nb,
    const typename G::ScaleBuf &sb, const Load<G> &ld, typename G::Buf &lb, int to, int wr, int xr, int g) {
    if constexpr (j < G::TX) {
        constexpr int gap = Q * G::TX + j, gaps = G::HALVES * G::TX;
        auto between = [&]() {
            // (FP8 codes split in two leave registers for half of them)
            constexpr int N = G::TW + G::TX, n0 = G::F8 ? j * N / G::TX : j ? N : 0, n1 = G::F8 ? (j + 1) * N / G::TX : N;
            mx_reads<G, tn, SC, n0, n1>(nf, ns, nb, sb, wr, xr, g);
            if constexpr (Q >= 0 && Q < G::HALVES) ld.template codes<gap * G::D / gaps, (gap + 1) * G::D / gaps>(lb, to);
        };
        if constexpr (G::F8) {
            i32x8 h, l;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                int large, small;
                fp8_split((uint32_t)f.x[j][k], large, small);
                h[k] = large;
                l[k] = small;
            }
            mx_mfma<t>(acc[j], f.w, s.w, h, s.x[j]);
            between();
            __builtin_amdgcn_sched_barrier(0);
            mx_mfma<t>(acc[j], f.w, s.w, l, s.x[j]);
        } else {
            mx_mfma<t>(acc[j], f.w, s.w, f.x[j], s.x[j]);
            between();
        }
        __builtin_amdgcn_sched_barrier(0);
        mx_step<G, t, tn, SC, Q, j + 1>(acc, f, s, nf, ns, nb, sb, ld, lb, to, wr, xr, g);
    }
}

// Wait states between matrix instructions and others that touch their sums.
template <int TX, int TW> __device__ __forceinline__ void mx_settle(f32x16 (&acc)[TX][TW]) {
#pragma unroll
    for (int i = 0; i < TX; i++)
#pragma unroll
        for (int j = 0; j < TW; j++) asm volatile("" : "+a"(acc[i][j]));
    asm volatile("s_nop 15\n\ts_nop 15" : "+a"(acc[TX - 1][TW - 1]));
#pragma unroll
    for (int i = 0; i < TX; i++)
#pragma unroll
        for (int j = 0; j < TW; j++) asm volatile("" : "+a"(acc[i][j]));
}

// v * g / (1 + exp(-g)) to a few units in the last place: from e = exp(-|g|), which cannot overflow, with the rest of
// exp2's rounded argument (up to 1e-6 of e at |g| = 20) and the reciprocal's error taken out.  exp2's results below 2^-126 are
// zero, which with g from -87 on and large v would be seen (-88: -5e-37 v): where e is below 2^-100, it is kept 2^160 times as large, and
// that is taken from v and from the product in two halves, neither of which leaves fp32's range where a code is not zero anyway.
__device__ __forceinline__ float swiglu(float v, float g) {
    const float m = -fminf(fabsf(g), 230.f), a = m * LOG2E, rest = __builtin_fmaf(m, LOG2E, -a) + m * LOG2E_REST;
    const bool far = a < -100.f;
    float e = __builtin_amdgcn_exp2f(far ? a + 160.f : a);   // (exact: multiples of a's last place)
    e = __builtin_fmaf(e, rest * 0.69314718f, e);
    const float d = far ? 1.f : 1.f + e;
    float r = __builtin_amdgcn_rcpf(d);
    r = __builtin_fmaf(r, __builtin_fmaf(-d, r, 1.f), r);
    const float s = (g < 0.f ? g * e : g) * r;
    return far && g < 0.f ? v * 0x1p-80f * s * 0x1p-80f : v * s;
}

// Eight values of a row, or one, to where they go; Beside: what is read for them.
struct Beside {
    f32x4 gate[2], res[2];     // 16-bit residuals: as stored, in res[0]
};
template <int T, bool RES> __device__ __forceinline__ void mx_beside(Beside &b, const Fh3kMxOut &o, int64_t t, int n, int64_t cols) {
    if constexpr (RES) {
        const f32x4 *p = (const f32x4 *)((const uint8_t *)o.res + (t * o.ldres + n) * (T == FH3K_F32 ? 4 : 2));
        b.res[0] = p[0];
        if constexpr (T == FH3K_F32) b.res[1] = p[1];
        if (o.gate) {
            b.gate[0] = *(const f32x4 *)(o.gate + t * cols + n);
            b.gate[1] = *(const f32x4 *)(o.gate + t * cols + n + 4);
        }
    }
}
template <int T> __device__ __forceinline__ float half_value(uint32_t b) {
    return T == FH3K_F16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)b) : __builtin_bit_cast(float, b << 16);
}
template <int T, bool RES> __device__ __forceinline__ void mx_put(const Fh3kMxOut &o, int64_t t, int n, float (&v)[8], const Beside &b) {
    if (o.bias)
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] += o.bias[n + k];
    if constexpr (RES) {
#pragma unroll
        for (int k = 0; k < 8; k++) {
            float h;
            if constexpr (T == FH3K_F32) {
                h = b.res[k / 4][k % 4];
            } else {
                const float pair = b.res[0][k >> 1];
                h = half_value<T>(__builtin_bit_cast(uint32_t, pair) >> (16 * (k & 1)) & 0xFFFFu);
            }
            v[k] = o.gate ? __builtin_fmaf(b.gate[k / 4][k % 4], v[k], h) : v[k] + h;
        }
    }
    store8<T>(o.out, t * o.ldo + n, v);
}
template <int T> __device__ __forceinline__ void mx_put1(const Fh3kMxOut &o, int64_t t, int n, int64_t cols, float v) {
    if (o.bias) v += o.bias[n];
    if (o.res) {
        const float h = value_at(o.res, T, t * o.ldres + n);
        v = o.gate ? __builtin_fmaf(o.gate[t * cols + n], v, h) : h + v;
    }
    if constexpr (T == FH3K_F32) ((float *)o.out)[t * o.ldo + n] = v;
    else ((uint16_t *)o.out)[t * o.ldo + n] = to_half<T>(v);
}

// A tile's 32 columns of a token lie in lanes l and l + 32, four by four; after the
// exchange lane l has columns 0 .. 7 and 16 .. 23, l + 32 the others.
__device__ __forceinline__ void mx_columns(const f32x16 &a, float (&v)[2][8]) {
#pragma unroll
    for (int m = 0; m < 2; m++)
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float x = a[8 * m + k], y = a[8 * m + 4 + k];
            const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, y), false, false);
            const uint32_t p = r[0], q = r[1];
            v[m][k] = __builtin_bit_cast(float, p);
            v[m][4 + k] = __builtin_bit_cast(float, q);
        }
}

// acc[idx / TW][idx % TW], of a rolled loop: unrolled over the sums, the code of the stores ran once for each and was fetched each time.
template <int TX, int TW, int i = 0> __device__ __forceinline__ void mx_pick(f32x16 &v, const f32x16 (&acc)[TX][TW], int idx) {
    if constexpr (i < TX * TW) {
        if (idx == i) v = acc[i / TW][i % TW];
        else mx_pick<TX, TW, i + 1>(v, acc, idx);
    }
}

// A wavefront's sums to rows of the output through its own piece of LDS, 32 tokens at
// a time, [32][COLS / 4] pieces of four values with piece c of token t at c ^ t % 16:
// whole rows of COLS values to a store.  Straight from the registers a store covers 32
// bytes of 32 rows: 8192 x 5120 -> 15360 in FP4 398 against 387 us.
// What is read beside them and the pieces come for U stores at once: one by one, each
// waited for its own.
template <int T, bool RES, int TX, int TW> __device__ __forceinline__ void mx_rows_out(const Fh3kMxOut &o, const f32x16 (&acc)[TX][TW], f32x4 *stg,
                                                                                       int lane, int64_t t0, int64_t rows, int n0, int64_t cols,
                                                                                       bool vec) {
    constexpr int COLS = TW * 32, C = COLS / 4, L = COLS / 8, TPI = 64 / L, U = RES ? 2 : 4;   // eight values to a lane
    const int g = lane >> 5, l = lane & 31, e = lane % L, n = n0 + 8 * e;
    const bool whole = vec && n + 8 <= cols;
#pragma unroll
    for (int i = 0; i < TX; i++) {
        const int64_t ti = t0 + 32 * i;
#pragma unroll
        for (int j = 0; j < TW; j++)
#pragma unroll
            for (int q = 0; q < 4; q++)
                stg[l * C + ((8 * j + 2 * q + g) ^ (l & 15))] = f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
        for (int it = 0; it < 32; it += TPI * U) {
            const int tl = it + lane / L;
            if (whole) {
                Beside b[U];
                f32x4 a[U][2];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int t = tl + u * TPI;
                    mx_beside<T, RES>(b[u], o, ti + t < rows ? ti + t : rows - 1, n, cols);   // past the end: the last row's
#pragma unroll
                    for (int h = 0; h < 2; h++) a[u][h] = stg[t * C + ((2 * e + h) ^ (t & 15))];
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    float v[8] = {a[u][0][0], a[u][0][1], a[u][0][2], a[u][0][3], a[u][1][0], a[u][1][1], a[u][1][2], a[u][1][3]};
                    if (ti + tl + u * TPI < rows) mx_put<T, RES>(o, ti + tl + u * TPI, n, v, b[u]);
                }
            } else {
#pragma unroll 1
                for (int t = tl; t < tl + TPI * U; t += TPI)
#pragma unroll 1
                    for (int k = 0; k < 8; k++)
                        if (ti + t < rows && n + k < cols)
                            mx_put1<T>(o, ti + t, n + k, cols, ((const float *)(stg + t * C + ((2 * e + (k >> 2)) ^ (t & 15))))[k & 3]);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}
template <int T, int TX, int TW> __device__ __forceinline__ void mx_rows_out(const Fh3kMxOut &o, const f32x16 (&acc)[TX][TW], f32x4 *stg, int lane,
                                                                             int64_t t0, int64_t rows, int n0, int64_t cols, bool vec) {
    if (o.res) mx_rows_out<T, true>(o, acc, stg, lane, t0, rows, n0, cols, vec);
    else mx_rows_out<T, false>(o, acc, stg, lane, t0, rows, n0, cols, vec);
}
// The same where the wavefront's first tiles are values and the others their gates: SwiGLU to codes.  A block is a
// tile's 32 columns.  Codes and scales come together in the wavefront's piece of LDS, [32 TX][BYTES], and leave 16 bytes
// to a lane and a row's scales at once: from the registers a store covered 16 bytes of 32 rows (3016 x 5376 -> 28672, FP8 rows in one product, 402 -> 391 us).
template <bool F8, int TX, int TW> __device__ __forceinline__ void mx_swiglu_out(const Fh3kMxOut &o, const f32x16 (&acc)[TX][TW], uint8_t *stg, int lane,
                                                                                 int64_t t0, int64_t rows, int f0) {
    constexpr int J = TW / 2, BYTES = F8 ? 32 * J : 16 * J, LD = BYTES + 16, L = BYTES / 16, TOKENS = 32 * TX;   // + 16: other banks for each row
    static_assert(TOKENS == 64 && J <= 2, "scales: a token to a lane");
    const int64_t f = o.y.in;
    const int g = lane >> 5;
    if (f0 >= f) return;                      // f is a multiple of 64: all of the wavefront's columns or none
    uint8_t *sc = stg + TOKENS * LD;
#pragma unroll 1
    for (int idx = 0; idx < TX * J; idx++) {
        const int i = idx / J, j = idx % J, col = f0 + 32 * j, t = 32 * i + (lane & 31);
        f32x16 a, b;
        float v[2][8], q[2][8];
        mx_pick<TX, TW>(a, acc, i * TW + j);
        mx_pick<TX, TW>(b, acc, i * TW + j + J);
        mx_columns(a, v);
        mx_columns(b, q);
        uint32_t u = 0;
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int n = col + 16 * m + 8 * g + k;
                const float bv = o.bias ? o.bias[n] : 0.f, bg = o.bias ? o.bias[f + n] : 0.f;
                v[m][k] = swiglu(v[m][k] + bv, q[m][k] + bg);
                const uint32_t w = __builtin_bit_cast(uint32_t, v[m][k]) & 0x7FFFFFFFu;
                u = u > w ? u : w;
            }
        const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        const uint32_t r0 = r[0], r1 = r[1], s = mx_scale<F8>(r0 > r1 ? r0 : r1);
#pragma unroll
        for (int m = 0; m < 2; m++) {
            const u32x2 c = mx_encode<F8>(v[m], s);
            if constexpr (F8) *(u32x2 *)(stg + t * LD + 32 * j + 16 * m + 8 * g) = c;
            else *(uint32_t *)(stg + t * LD + 16 * j + 8 * m + 4 * g) = c.x;
        }
        if (!g) sc[t * J + j] = (uint8_t)s;
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int it = 0; it < TOKENS; it += 64 / L) {
        const int t = it + lane / L, p = 16 * (lane % L);
        const u32x4 c = *(const u32x4 *)(stg + t * LD + p);
        if (t0 + t < rows) put_past(c, o.y.codes + (t0 + t) * o.y.ld + (F8 ? f0 : f0 / 2) + p);
    }
    if (t0 + lane < rows) {
        uint8_t *p = o.y.scales + (t0 + lane) * o.y.lds + f0 / MX_BLOCK;
        if constexpr (J == 2) *(uint16_t *)p = *(const uint16_t *)(sc + lane * 2);
        else *p = sc[lane];
    }
}

template <class G> __global__ __launch_bounds__(64 * G::WAVES, 8 / G::WAVES) void k_mx_gemm(
    Fh3kMx w, Fh3kMx x, Fh3kMxOut o, float *part, int64_t ldp, int m_tiles, int n_tiles, int first, int per, bool vec) {
    constexpr int TW = G::TW, TX = G::TX;
    __shared__ typename G::Buf b0, b1;
    __shared__ typename std::conditional<G::NBUF == 3, typename G::Buf, int>::type b2;
    __shared__ typename G::ScaleBuf sb;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wn = wave % G::NW, wm = wave / G::NW, g = lane >> 5;
    // the tiles of a band of four token tiles, column by column, on one XCD
    constexpr int GB = 4;
    const int total = m_tiles * n_tiles, id = blockIdx.x, share = total >> 3;
    const int L = id < share * 8 ? (id & 7) * share + (id >> 3) : id;
    const int band = L / (GB * n_tiles), gs = min(GB, m_tiles - band * GB), in = L - band * GB * n_tiles;
    const int mt = band * GB + in % gs, nt = first + in / gs;   // columns of tiles from the first on
    const int64_t m0 = (int64_t)mt * G::BX;
    const bool swiglu = o.y.codes != nullptr && !part;

    Load<G> ld;
    const int64_t f = w.rows >> 1;
    // SwiGLU: each wavefront column's rows are the values' and then their gates'
    constexpr int RW = G::BW / G::WAVES, CW = G::BW / G::NW;
    const int wc = wave * RW / CW, wa = wave * RW % CW;
    ld.w.init(w, swiglu ? (wa >= CW / 2 ? f : 0) + (int64_t)nt * (G::BW / 2) + wc * (CW / 2) + wa % (CW / 2)
                        : (int64_t)nt * G::BW + wave * RW, lane);
    ld.x.init(x, m0 + wave * (G::BX / G::WAVES), lane);
    ld.wave = wave;
    ld.blocks = (int)(w.in / MX_BLOCK);
    const int s0 = blockIdx.y * per;
    ld.end = min(s0 + per, (ld.blocks + G::NB - 1) / G::NB);

    f32x16 acc[TX][TW];
#pragma unroll
    for (int i = 0; i < TX; i++)
#pragma unroll
        for (int j = 0; j < TW; j++) acc[i][j] = f32x16{};
    Frags<G> fr[2] = {};
    Scales<G> sc;
    StageScales<G> ss;
    const int wr = wn * CW + (lane & 31), xr = wm * (G::BX / G::NX) + (lane & 31);

    // the first stages (the last of them to half, where loads are spread: the other half is loaded in the first stage's first step)
    ld.scales(sb, s0);
    ld.template codes<0, G::D>(b0, s0);
    if constexpr (G::NBUF == 3) {
        ld.template codes<0, G::D>(b1, s0 + 1);
        ld.template codes<0, G::D / G::HALVES>(b2, s0 + 2);
    } else {
        ld.template codes<0, G::D / G::HALVES>(b1, s0 + 1);
    }
    mx_barrier<(G::NBUF - 2) * G::D + G::D / G::HALVES>();
    mx_reads<G, 0, true, 0, G::TW + G::TX>(fr[0], sc, b0, sb, wr, xr, g);

    // Stage s, the chunk's c-th.
    auto stage = [&](int s, auto ci, typename G::Buf &cur, const typename G::Buf &nxt, typename G::Buf &prev) {
        constexpr int c = ci();
        const int left = ld.blocks - s * G::NB - g * G::T;   // blocks of the row for this lane's scale bytes
        mx_stage_scales<G, c>(ss, sc, g, left >= G::T ? -1 : left <= 0 ? 0 : (int)((1u << (8 * left)) - 1));
        mx_step<G, 0, 1, false, 1>(acc, fr[0], ss, fr[1], sc, cur, sb, ld, prev, s + G::NBUF - 1, wr, xr, g);
        if constexpr (G::T == 4) {
            mx_step<G, 1, 2, false, -1>(acc, fr[1], ss, fr[0], sc, cur, sb, ld, prev, 0, wr, xr, g);
            mx_step<G, 2, 3, false, -1>(acc, fr[0], ss, fr[1], sc, cur, sb, ld, prev, 0, wr, xr, g);
        }
        // this stage's operands are all read, the next one's have landed
        mx_barrier<(G::NBUF - 2) * G::D>();
        if constexpr (c == 0) ld.scales(sb, s + G::CH);   // this chunk's are all in registers
        mx_step<G, G::T - 1, 0, c == G::CH - 1, 0>(acc, fr[1], ss, fr[0], sc, nxt, sb, ld, cur, s + G::NBUF, wr, xr, g);
    };
    mx_settle(acc);
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    using I3 = std::integral_constant<int, 3>;
    for (int s = s0;;) {
        if constexpr (G::NBUF == 3) {
            stage(s, I0{}, b0, b1, b2);
            if (++s >= ld.end) break;
            stage(s, I1{}, b1, b2, b0);
            if (++s >= ld.end) break;
            stage(s, I2{}, b2, b0, b1);
            if (++s >= ld.end) break;
        } else {
            stage(s, I0{}, b0, b1, b1);
            if (++s >= ld.end) break;
            stage(s, I1{}, b1, b0, b0);
            if (++s >= ld.end) break;
            stage(s, I2{}, b0, b1, b1);
            if (++s >= ld.end) break;
            stage(s, I3{}, b1, b0, b0);
            if (++s >= ld.end) break;
        }
    }
    mx_settle(acc);
    // nothing more comes to LDS, and nobody reads it
    mx_barrier<0>();
    constexpr int PIECE = TW * 32 * 32 / 4, PER = sizeof(typename G::Buf) / 16 / PIECE;   // 16-byte words of a wavefront, wavefronts to a buffer
    static_assert(G::NBUF * PER >= G::WAVES && PIECE * 16 >= 64 * (TW * 16 + 16 + 2), "the sums' room");
    f32x4 *stg = (f32x4 *)(wave < PER ? b0.x : wave < 2 * PER || G::NBUF == 2 ? b1.x : (u32x4 *)&b2) + wave % PER * PIECE;
    if (part) {
        o = Fh3kMxOut{};
        o.out = part + blockIdx.y * (x.rows * ldp);
        o.ldo = ldp;
    }
    const int64_t t0 = m0 + wm * (G::BX / G::NX);
    const int n0 = nt * G::BW + wn * CW;
    if (swiglu) {
        if (o.y.type == FH3K_MX_FP8) mx_swiglu_out<true>(o, acc, (uint8_t *)stg, lane, t0, x.rows, n0 / 2);
        else mx_swiglu_out<false>(o, acc, (uint8_t *)stg, lane, t0, x.rows, n0 / 2);
    } else if (o.type == FH3K_F32) mx_rows_out<FH3K_F32>(o, acc, stg, lane, t0, x.rows, n0, part ? ldp : w.rows, vec);
    else if (o.type == FH3K_F16) mx_rows_out<FH3K_F16>(o, acc, stg, lane, t0, x.rows, n0, w.rows, vec);
    else mx_rows_out<FH3K_BF16>(o, acc, stg, lane, t0, x.rows, n0, w.rows, vec);
}

// Eight sums' parts, n values apart, added in their order; four are loaded at once, since one by one each
// waited for its own.
__device__ __forceinline__ void mx_add_parts(const float *part, int S, int64_t n, int64_t at, float (&v)[8]) {
    for (int s = 0; s < S; s += 4) {
        float a[4][8];
#pragma unroll
        for (int i = 0; i < 4; i++) load8<FH3K_F32>(part, min(s + i, S - 1) * n + at, a[i]);
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] = s + i < S ? v[k] + a[i][k] : v[k];
    }
}
// The parts of a split product, added in their order, to rows of the output: eight values to a thread.
template <int T> __global__ __launch_bounds__(256) void k_mx_join(const float *__restrict__ part, int S, int64_t ldp, int64_t rows, int64_t cols,
                                                                  Fh3kMxOut o, bool vec) {
    const int64_t t = blockIdx.x;
    const int n = 8 * (blockIdx.y * 256 + threadIdx.x);
    if (n >= cols) return;
    float v[8] = {};
    mx_add_parts(part, S, rows * ldp, t * ldp + n, v);
    if (vec && n + 8 <= cols) {
        Beside b;
        if (o.res) {
            mx_beside<T, true>(b, o, t, n, cols);
            mx_put<T, true>(o, t, n, v, b);
        } else {
            mx_put<T, false>(o, t, n, v, b);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (n + k < cols) mx_put1<T>(o, t, n + k, cols, v[k]);
    }
}

template <bool F8> __global__ __launch_bounds__(256) void k_mx_join_swiglu(const float *__restrict__ part, int S, int64_t ldp, int64_t rows,
                                                                           Fh3kMxOut o) {
    const int64_t t = blockIdx.x, f = o.y.in;
    const int col = 8 * (blockIdx.y * 256 + threadIdx.x);
    if (col >= f) return;
    float v[8] = {}, q[8] = {}, a[8];
    mx_add_parts(part, S, rows * ldp, t * ldp + col, v);
    mx_add_parts(part, S, rows * ldp, t * ldp + f + col, q);
#pragma unroll
    for (int k = 0; k < 8; k++) a[k] = swiglu(v[k] + (o.bias ? o.bias[col + k] : 0.f), q[k] + (o.bias ? o.bias[f + col + k] : 0.f));
    mx_store<F8>(o.y, t, col, a);
}

// ---------------------------------------------------------------------------
// Few rows (up to 16 TT), not too many weights: bound by the weights' way from memory and,
// with x for each workgroup, from L2 (5120 -> 5120: 1 row 7.2 us, 32 rows 11.3).  A workgroup
// takes 16 R weight rows, its wavefronts a share each of the rows' windows of 128 S
// values, straight from memory into 16x16x128 products, and their sums meet in LDS.
// Lane (r, g), g = 0 .. 3, holds of row r the FP4 codes 32 g .. + 31 of a step's 128, or
// the FP8 codes 16 g .. + 15 and 64 + 16 g .. + 15, and the scale of block g.
// FP8 rows enter as two products (fp8_split).
// SwiGLU: half of the R tiles are values' rows, half their gates'.
// ---------------------------------------------------------------------------
constexpr int MX_WAVES = 12, MX_WAVES_AHEAD = 8;   // the most wavefronts to a workgroup

__device__ __forceinline__ u32x4 mx_load16(__amdgpu_buffer_rsrc_t r, uint32_t off) {
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 0, 0));
}
__device__ __forceinline__ u32x2 mx_load8(__amdgpu_buffer_rsrc_t r, uint32_t off) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, (int)off, 0, 0));
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t mx_buffer(const void *p, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), (short)0, (int)bytes, 0x00020000);
}

// Sixteen rows of an operand: those past the end are the last one.
struct Few {
    __amdgpu_buffer_rsrc_t code, scale;
    uint32_t off, soff;                  // of this lane's row
    __device__ __forceinline__ void init(const Fh3kMx &m, int64_t base, int r) {
        if (base >= m.rows) base = m.rows - 1;
        const int last = m.rows - base < 16 ? (int)(m.rows - base) - 1 : 15;
        code = mx_buffer(m.codes + base * m.ld, (uint32_t)(last * m.ld + (m.type == FH3K_MX_FP8 ? m.in : m.in / 2)));
        scale = mx_buffer(m.scales + base * m.lds, (uint32_t)(last * m.lds + (m.in / MX_BLOCK + 3) / 4 * 4));
        r = r < last ? r : last;
        off = (uint32_t)(r * m.ld);
        soff = (uint32_t)(r * m.lds);
    }
};

__device__ __forceinline__ f32x4 mx_mfma16(const u32x4 &w, const i32x8 &x, f32x4 acc, int ws, int xs, bool f8) {
    const i32x8 a = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
    if (f8) return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, x, acc, 4, 0, 0, ws, 0, xs);
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, x, acc, 4, 4, 0, ws, 0, xs);
}

template <bool F8, int TT, int R> struct Window {
    static constexpr int S = TT == 1 ? 4 : 2;                              // steps
    static constexpr int WB = 64 * S, XB = F8 ? 128 * S : 64 * S;          // bytes of a row
    typedef typename std::conditional<S == 4, u32x4, u32x2>::type Dwords;  // of scales, one for each step's four blocks
    u32x4 w[R][S];
    u32x4 x[TT][S][F8 ? 2 : 1];
    Dwords ws[R], xs[TT];

    __device__ __forceinline__ static void scales(Dwords &d, __amdgpu_buffer_rsrc_t r, uint32_t off) {
        if constexpr (S == 4) d = mx_load16(r, off);
        else d = mx_load8(r, off);
    }
    // window `at`, `left` blocks from its start to the rows' end
    __device__ __forceinline__ void load(const Few (&fw)[R], const Few (&fx)[TT], int at, int left, int g) {
#pragma unroll
        for (int i = 0; i < R; i++) scales(ws[i], fw[i].scale, fw[i].soff + at * (4 * S));
#pragma unroll
        for (int j = 0; j < TT; j++) scales(xs[j], fx[j].scale, fx[j].soff + at * (4 * S));
#pragma unroll
        for (int s = 0; s < S; s++) {
            const bool in = 4 * s + g < left;
#pragma unroll
            for (int i = 0; i < R; i++) w[i][s] = mx_load16(fw[i].code, in ? fw[i].off + at * WB + s * 64 + g * 16 : MX_OUTSIDE);
#pragma unroll
            for (int j = 0; j < TT; j++) {
                if constexpr (F8) {
                    const int b = 4 * s + (g >> 1);
                    const uint32_t off = fx[j].off + at * XB + s * 128 + g * 16;
                    x[j][s][0] = mx_load16(fx[j].code, b < left ? off : MX_OUTSIDE);
                    x[j][s][1] = mx_load16(fx[j].code, b + 2 < left ? off + 64 : MX_OUTSIDE);
                } else {
                    x[j][s][0] = mx_load16(fx[j].code, in ? fx[j].off + at * XB + s * 64 + g * 16 : MX_OUTSIDE);
                }
            }
        }
    }
    // the scale of step s's block g; past the row's end 0, whatever stands there
    __device__ __forceinline__ static int scale(uint32_t d, int s, int left, int g) { return 4 * s + g < left ? (int)(d >> (8 * g)) : 0; }

    __device__ __forceinline__ void products(f32x4 (&acc)[R][TT], int left, int g) const {
#pragma unroll
        for (int s = 0; s < S; s++) {
            int sw[R];
#pragma unroll
            for (int i = 0; i < R; i++) sw[i] = scale(ws[i][s], s, left, g);
#pragma unroll
            for (int j = 0; j < TT; j++) {
                const int sx = scale(xs[j][s], s, left, g);
                i32x8 v = {}, h;
                set4(v, 0, x[j][s][0]);
                if constexpr (F8) {
                    set4(v, 4, x[j][s][1]);
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        int large, small;
                        fp8_split((uint32_t)v[k], large, small);
                        h[k] = large;
                        v[k] = small;
                    }
#pragma unroll
                    for (int i = 0; i < R; i++) acc[i][j] = mx_mfma16(w[i][s], h, acc[i][j], sw[i], sx, true);
                }
#pragma unroll
                for (int i = 0; i < R; i++) acc[i][j] = mx_mfma16(w[i][s], v, acc[i][j], sw[i], sx, F8);
            }
        }
    }
};

// Both 16 x 16 tiles of a block of 32 outputs, values and gates: lane (t, g) has the block's outputs 4 g .. and 16 + 4 g .. of token t.
__device__ __forceinline__ void mx_swiglu16(const Fh3kMxOut &o, const f32x4 &v0, const f32x4 &q0, const f32x4 &v1, const f32x4 &q1, int64_t t,
                                            int64_t rows, int64_t n0, int g) {
    const int64_t f = o.y.in;
    float a[8];
    uint32_t u = 0;
#pragma unroll
    for (int k = 0; k < 8; k++) {
        const int64_t n = n0 + 16 * (k >> 2) + 4 * g + (k & 3);
        const float v = k < 4 ? v0[k & 3] : v1[k & 3], q = k < 4 ? q0[k & 3] : q1[k & 3];
        a[k] = swiglu(v + (o.bias ? o.bias[n] : 0.f), q + (o.bias ? o.bias[f + n] : 0.f));
        const float c = a[k];
        const uint32_t b = __builtin_bit_cast(uint32_t, c) & 0x7FFFFFFFu;
        u = u > b ? u : b;
    }
    u = max(u, (uint32_t)__shfl_xor((int)u, 16));
    u = max(u, (uint32_t)__shfl_xor((int)u, 32));
    const bool to8 = o.y.type == FH3K_MX_FP8;
    const uint32_t s = to8 ? mx_scale<true>(u) : mx_scale<false>(u);
    if (t >= rows) return;
    if (to8) {
        const u32x2 c = mx_encode<true>(a, s);
        uint8_t *p = o.y.codes + t * o.y.ld + n0 + 4 * g;
        *(uint32_t *)p = c.x;
        *(uint32_t *)(p + 16) = c.y;
    } else {
        const uint32_t c = mx_encode<false>(a, s).x;
        uint8_t *p = o.y.codes + t * o.y.ld + n0 / 2 + 2 * g;
        *(uint16_t *)p = (uint16_t)c;
        *(uint16_t *)(p + 8) = (uint16_t)(c >> 16);
    }
    if (g == 0) o.y.scales[t * o.y.lds + n0 / MX_BLOCK] = (uint8_t)s;
}
// Four outputs n .. n + 3 of token t, those of them that are there.
__device__ __forceinline__ void mx_put4(const Fh3kMxOut &o, int64_t t, int64_t n, int64_t cols, const f32x4 &v) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
        if (n + e >= cols) continue;
        if (o.type == FH3K_F32) mx_put1<FH3K_F32>(o, t, (int)n + e, cols, v[e]);
        else if (o.type == FH3K_F16) mx_put1<FH3K_F16>(o, t, (int)n + e, cols, v[e]);
        else mx_put1<FH3K_BF16>(o, t, (int)n + e, cols, v[e]);
    }
}

template <bool F8, int TT, int R, bool AHEAD> __global__ __launch_bounds__(64 * (AHEAD || TT == 4 || R * TT == 8 ? MX_WAVES_AHEAD : MX_WAVES)) void k_mx_few(Fh3kMx w, Fh3kMx x, Fh3kMxOut o) {
    extern __shared__ f32x4 parts[];         // [wavefront][R][TT][64]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int r = lane & 15, g = lane >> 4;
    const bool swiglu = o.y.codes != nullptr;
    const int64_t f = w.rows >> 1, n0 = (int64_t)blockIdx.x * (swiglu ? 8 * R : 16 * R);
    Few fw[R], fx[TT];
#pragma unroll
    for (int i = 0; i < R; i++) fw[i].init(w, swiglu ? (i < R / 2 ? 0 : f) + n0 + 16 * (i % (R / 2 > 0 ? R / 2 : 1)) : n0 + 16 * i, r);
#pragma unroll
    for (int j = 0; j < TT; j++) fx[j].init(x, 16 * j, r);
    typedef Window<F8, TT, R> Win;
    constexpr int WBL = 4 * Win::S;          // blocks of a window
    const int blocks = (int)(w.in / MX_BLOCK), windows = (blocks + WBL - 1) / WBL;
    f32x4 acc[R][TT] = {};
    // AHEAD: the next window's loads before this one's products
    Win v[AHEAD ? 2 : 1];
    if (AHEAD && wave < windows) v[0].load(fw, fx, wave, blocks - WBL * wave, g);
    for (int at = wave; at < windows; at += 2 * waves) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int a = at + h * waves, b = a + waves;
            if (a >= windows) break;
            if (!AHEAD) v[0].load(fw, fx, a, blocks - WBL * a, g);
            else if (b < windows) v[AHEAD ? 1 - h : 0].load(fw, fx, b, blocks - WBL * b, g);
            v[AHEAD ? h : 0].products(acc, blocks - WBL * a, g);
        }
    }
#pragma unroll
    for (int i = 0; i < R; i++)
#pragma unroll
        for (int j = 0; j < TT; j++) parts[((wave * R + i) * TT + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    // a wavefront to a tile of 16 x 16 (SwiGLU: to one of values and its gates)
    auto sum = [&](int i, int j) {
        f32x4 v = parts[(i * TT + j) * 64 + lane];
        for (int k = 1; k < waves; k++) {
            const f32x4 a = parts[((k * R + i) * TT + j) * 64 + lane];
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] += a[e];
        }
        return v;
    };
    if (swiglu) {
        if constexpr (R == 4) {
            for (int j = wave; j < TT; j += waves) mx_swiglu16(o, sum(0, j), sum(2, j), sum(1, j), sum(3, j), 16 * j + r, x.rows, n0, g);
        }
        return;
    }
    for (int tile = wave; tile < R * TT; tile += waves) {
        const int i = tile / TT, j = tile % TT;
        const int64_t t = 16 * j + r;
        const f32x4 v = sum(i, j);
        if (t < x.rows) mx_put4(o, t, n0 + 16 * i + 4 * g, w.rows, v);
    }
}

// ---------------------------------------------------------------------------
// Up to 64 rows (16 TT) against many weight rows: as k_mx_few, but a workgroup, one to a
// CU, keeps its part of the rows' length of x in registers (each wavefront NS steps of
// 128 values) and takes tile after tile of 16 weight rows, straight from memory, two of
// them while the next two are on their way; the wavefronts' sums meet in LDS four tiles at a time.
// k_mx_few reads all of x for each 16 R weight rows: 20 rows x 5120 -> 51200 SwiGLU, 139 MB
// of weights, take it 58 us, the tiles 65, this 39 (FP4 rows 48, 34, 30; one FP8 row 29): the splitting
// of FP8 codes is 32 VALU instructions to 32 codes (up to 16 rows the halves stay in registers: 31).
// Where x is longer than 40 steps (24), each part of it has its own workgroups, and the
// parts' sums are joined: 16 rows x 25600 -> 5120 30 us, tiles 39, this 21 with weights from memory.
// Two tiles to each splitting of FP8 codes: with one, that took longer than the loads.
// Nothing that is known before the loop is kept over it (the asm statements): the
// registers are full of loads, and a reload from scratch waits for all loads before it.
// ---------------------------------------------------------------------------
// byte xb of xs; a constant once unrolled
__device__ __forceinline__ f32x4 mx_mfma16(const u32x4 &w, const i32x8 &x, f32x4 acc, int ws, int xs, int xb, bool f8) {
    const i32x8 a = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
#define MX_M16(B) (f8 ? __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, x, acc, 4, 0, 0, ws, B, xs) : __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, x, acc, 4, 4, 0, ws, B, xs))
    switch (xb) {
        case 0: return MX_M16(0);
        case 1: return MX_M16(1);
        case 2: return MX_M16(2);
        default: return MX_M16(3);
    }
}
constexpr int MX_STREAM = 8;    // wavefronts of a workgroup
// NS steps' scales of a row, one dword each
template <int NS> __device__ __forceinline__ void mx_step_scales(uint32_t (&s)[NS], __amdgpu_buffer_rsrc_t r, uint32_t off) {
#pragma unroll
    for (int i = 0; i + 4 <= NS; i += 4) {
        const u32x4 v = mx_load16(r, off + 4 * i);
#pragma unroll
        for (int k = 0; k < 4; k++) s[i + k] = v[k];
    }
#pragma unroll
    for (int i = NS & ~3; i < NS; i++) s[i] = __builtin_amdgcn_raw_buffer_load_b32(r, (int)(off + 4 * i), 0, 0);
}
template <int NS> struct Streamed {
    u32x4 w[NS];
    uint32_t s[NS];
    // rows n0 .. of w (rows: how many are there), for this wavefront's steps from `first` on, n of them
    __device__ __forceinline__ void load(const Fh3kMx &m, int64_t n0, bool any, int r, int g, int first, int blocks) {
        if (n0 >= m.rows) n0 = m.rows - 1;
        const int last = m.rows - n0 < 16 ? (int)(m.rows - n0) - 1 : 15;
        const __amdgpu_buffer_rsrc_t code = mx_buffer(m.codes + n0 * m.ld, any ? (uint32_t)(last * m.ld + m.in / 2) : 0u);
        const __amdgpu_buffer_rsrc_t scale = mx_buffer(m.scales + n0 * m.lds, any ? (uint32_t)(last * m.lds + (m.in / MX_BLOCK + 3) / 4 * 4) : 0u);
        r = r < last ? r : last;
        const uint32_t off = (uint32_t)(r * m.ld) + first * 64 + g * 16;
        mx_step_scales<NS>(s, scale, (uint32_t)(r * m.lds) + first * 4);
#pragma unroll
        for (int i = 0; i < NS; i++) w[i] = mx_load16(code, 4 * i + g < blocks ? off + i * 64 : MX_OUTSIDE);
    }
};

template <bool F8, int TT, int NS> __global__ __launch_bounds__(64 * MX_STREAM, 2) void k_mx_stream(
    Fh3kMx w, Fh3kMx x, Fh3kMxOut o, float *part, int64_t ldp, int units, int per) {
    __shared__ f32x4 sums[4][TT][MX_STREAM][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, g = lane >> 4;
    const bool swiglu = o.y.codes != nullptr && !part;
    const int64_t f = w.rows >> 1;
    const int G = gridDim.x;
    // this wavefront's steps
    const int steps = (int)((w.in + 127) / 128), end = min((int)(blockIdx.y + 1) * per, steps);
    const int share = (per + MX_STREAM - 1) / MX_STREAM, first = blockIdx.y * per + wave * share;
    int blocks = min(min(first + share, end) * 4, (int)(w.in / MX_BLOCK)) - first * 4;   // of it, 0 or less: none
    const int count = swiglu ? (units - (int)blockIdx.x + G - 1) / G * 4 : (units - (int)blockIdx.x + G - 1) / G;
    auto row = [&](int k, int q) -> int64_t {
        if (swiglu) return ((q & 1) ? f : 0) + (int64_t)(blockIdx.x + (k >> 2) * G) * 32 + (q >> 1) * 16;
        return (int64_t)(blockIdx.x + (k + q) * G) * 16;
    };
    u32x4 xc[TT][NS][F8 ? 2 : 1];
    uint32_t xs[TT][(NS + 3) / 4] = {}, xd[TT][NS];
#pragma unroll
    for (int j = 0; j < TT; j++) {
        Few fx;
        fx.init(x, 16 * j, r);
        mx_step_scales<NS>(xd[j], fx.scale, fx.soff + first * 4);
#pragma unroll
        for (int i = 0; i < NS; i++) {
            if constexpr (F8) {
                const int b = 4 * i + (g >> 1);
                const uint32_t off = fx.off + (first + i) * 128 + g * 16;
                xc[j][i][0] = mx_load16(fx.code, b < blocks ? off : MX_OUTSIDE);
                xc[j][i][1] = mx_load16(fx.code, b + 2 < blocks ? off + 64 : MX_OUTSIDE);
            } else {
                xc[j][i][0] = mx_load16(fx.code, 4 * i + g < blocks ? fx.off + (first + i) * 64 + g * 16 : MX_OUTSIDE);
            }
        }
    }
    // two tiles at a time, the next two on their way
    Streamed<NS> v[2][2];
#pragma unroll
    for (int i = 0; i < 2; i++) v[0][i].load(w, row(0, i), i < count, r, g, first, blocks);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < TT; j++)
#pragma unroll
        for (int i = 0; i < NS; i++) xs[j][i >> 2] |= (4 * i + g < blocks ? xd[j][i] >> (8 * g) & 0xFFu : 0u) << (8 * (i & 3));
    for (int k = 0; k < count; k += 4) {
#pragma unroll
        for (int d = 0; d < 2; d++) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int a = 2 * d + 2 + i;
                v[1 - d][i].load(w, row(k + (a & ~3), a & 3), k + a < count, r, g, first, blocks);
            }
            __builtin_amdgcn_sched_barrier(0);
            f32x4 acc[2][TT] = {};
#pragma unroll
            for (int s = 0; s < NS; s++) {
                int sw[2];
#pragma unroll
                for (int i = 0; i < 2; i++) sw[i] = 4 * s + g < blocks ? (int)(v[d][i].s[s] >> (8 * g)) : 0;
#pragma unroll
                for (int j = 0; j < TT; j++) {
                    i32x8 c = {}, h;
                    // split here each time: kept, the halves take twice the registers (one tile of rows: there is room for them)
                    if constexpr (F8 && TT > 1) asm volatile("" : "+v"(xc[j][s][0]), "+v"(xc[j][s][1]));
                    set4(c, 0, xc[j][s][0]);
                    if constexpr (F8) {
                        set4(c, 4, xc[j][s][1]);
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            int large, small;
                            fp8_split((uint32_t)c[e], large, small);
                            h[e] = large;
                            c[e] = small;
                        }
#pragma unroll
                        for (int i = 0; i < 2; i++) acc[i][j] = mx_mfma16(v[d][i].w[s], h, acc[i][j], sw[i], (int)xs[j][s >> 2], s & 3, true);
                    }
#pragma unroll
                    for (int i = 0; i < 2; i++) acc[i][j] = mx_mfma16(v[d][i].w[s], c, acc[i][j], sw[i], (int)xs[j][s >> 2], s & 3, F8);
                }
            }
            // the sums of the last trip are read
            if (d == 0) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int j = 0; j < TT; j++) sums[2 * d + i][j][wave][lane] = acc[i][j];
            asm volatile("" : : : "memory");
            __builtin_amdgcn_sched_barrier(0);
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");
        int to = lane;
        asm volatile("" : "+v"(to));   // addresses made from it are not kept over the loads
        auto sum = [&](int d, int j) {
            f32x4 v = sums[d][j][0][to];
#pragma unroll
            for (int i = 1; i < MX_STREAM; i++) {
                const f32x4 a = sums[d][j][i][to];
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] += a[e];
                if (i & 1) asm volatile("" : "+v"(v) : : "memory");   // the registers are full of loads
            }
            return v;
        };
        if (swiglu) {
            if (wave < TT) {
                const f32x4 v0 = sum(0, wave), q0 = sum(1, wave), v1 = sum(2, wave), q1 = sum(3, wave);
                mx_swiglu16(o, v0, q0, v1, q1, 16 * wave + (to & 15), x.rows, row(k, 0), to >> 4);
            }
        } else {
#pragma unroll 1
            for (int i = wave; i < 4 * TT; i += MX_STREAM) {
                const int d = i / TT, j = i % TT;
                if (k + d >= count) break;
                const f32x4 v = sum(d, j);
                const int64_t t = 16 * j + (to & 15), n = row(k, d) + 4 * (to >> 4);
                if (t >= x.rows) continue;
                if (part) {
                    if (n < ldp) *(f32x4 *)(part + (blockIdx.y * x.rows + t) * ldp + n) = v;
                } else {
                    mx_put4(o, t, n, w.rows, v);
                }
            }
        }
    }
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
    const dim3 grid = row_grid((y->rows + rpw - 1) / rpw, (y->in + 8 * MX_EACH * lanes - 1) / (8 * MX_EACH * lanes));
    return by_type(type, [&](auto t) {
        if (y->type == FH3K_MX_FP8) k_mx_quantize<t(), true><<<grid, 256, 0, st>>>(x, ldx, *y, lanes);
        else k_mx_quantize<t(), false><<<grid, 256, 0, st>>>(x, ldx, *y, lanes);
    });
}

extern "C" hipError_t fh3k_mx_dequant(const Fh3kMx *x, int type, void *y, int64_t ldy, hipStream_t st) {
    const int lanes = row_lanes(x->in), rpw = 256 / lanes;
    const dim3 grid = row_grid((x->rows + rpw - 1) / rpw, (x->in + 8 * MX_EACH * lanes - 1) / (8 * MX_EACH * lanes));
    return by_type(type, [&](auto t) {
        if (x->type == FH3K_MX_FP8) k_mx_dequant<t(), true><<<grid, 256, 0, st>>>(*x, y, ldy, lanes);
        else k_mx_dequant<t(), false><<<grid, 256, 0, st>>>(*x, y, ldy, lanes);
    });
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
            k_mx_norm<t(), f8(), cc()><<<row_grid(y->rows, 1), nt, 0, st>>>(x, ldx, add, lda, sum, lds, w, eps, shift, scale, *y);
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

namespace {

// How a product is cut: tiles, and parts of the rows' length.
struct Plan {
    enum { FEW, STREAM, TILES } kernel;
    int bw, bx, parts, per;       // per: stages (STREAM: steps) of a part
    int64_t m_tiles, n_tiles, ldp;
    int64_t large;                // columns of larger tiles, where the others are left to smaller ones
};
// Tiles of 16 weight rows to a workgroup of k_mx_few: the most that leave 150
// workgroups, since each reads all rows of x.  SwiGLU: a block of 32 outputs.
int few_tiles(const Fh3kMx *w, const Fh3kMx *x, bool swiglu) {
    const int64_t n16 = (w->rows + 15) / 16;
    return swiglu || (n16 >= 600 && x->rows <= 16) ? 4 : n16 >= 300 ? 2 : 1;
}

// Each kernel's time in us by what was measured (weights from memory), of which the least is taken.
// FP8 rows to bf16, k_mx_few, k_mx_stream and the tiles:
//    5120 -> 5120           1 row 7.3, 8.5, 14.7     32 rows 11.3, 15.0, 15.9   64 rows 20.6, 18.7, 17.5
//    5120 -> 15360          1 row 13.3, 11.6, 24.6   17 rows 20.5, 16.7, 26.6   64 rows 43.5, 29.0, 28.4
//    25600 -> 5120          1 row 21.2, 19.5, 36.5   16 rows 30.3, 21.6, 38.7   64 rows 78.4, 39.0, 40.7
//    5120 -> 51200 SwiGLU   1 row 39.1, 29.1, 64.4   17 rows 56.5, 39.2, 65.5   64 rows 79.6, 68.6, 66.8
// and FP4 rows:
//    5120 -> 5120           1 row 6.2, 7.6, 10.8     32 rows 8.7, 9.8, 12.2     64 rows 12.3, 13.8, 13.7
//    5120 -> 15360          1 row 12.9, 10.9, 16.8   17 rows 15.0, 12.2, 17.5   64 rows 27.6, 18.3, 20.5
//    25600 -> 5120          1 row 19.1, 18.6, 24.4   16 rows 24.5, 20.1, 25.7   64 rows 50.6, 25.5, 28.5
double few_us(const Fh3kMx *w, const Fh3kMx *x, bool swiglu) {
    const int64_t rows = 16 * few_tiles(w, x, swiglu), groups = (w->rows + rows - 1) / rows;
    const double row = (double)w->in * (x->type == FH3K_MX_FP8 ? 1.0 : 0.5), each = (double)rows * w->in / 2 + x->rows * row;
    // a workgroup's bytes through one CU, or all weights from memory and the rows for each workgroup from L2
    const double one = each / (x->rows <= 16 ? 38e3 : x->rows <= 32 ? 36e3 : rows == 64 ? 20e3 : 32e3);
    const double all = (double)w->rows * w->in * 0.53 / (4.4e6 * (groups < 200 ? groups / 200.0 : 1.0)) + groups * x->rows * row / 12e6;
    const double more = x->type == FH3K_MX_FP4 || x->rows <= 16 ? 1 : x->rows <= 32 ? 1.35 : 1.8, a = 3.9 + one * more, b = (swiglu || x->rows > 32 ? 3.9 : 2.6) + all * more;
    return a > b ? a : b;
}
// Steps of 128 values that a wavefront of k_mx_stream holds of x: what fits its registers
int stream_steps(const Fh3kMx *x) {
    const int steps = (int)((x->in + 127) / 128);
    return x->rows <= 32 || (x->type == FH3K_MX_FP4 && steps <= 5 * MX_STREAM) ? 5 : 3;
}
double stream_us(const Fh3kMx *w, const Fh3kMx *x, bool swiglu, Plan &p) {
    const int steps = (int)((w->in + 127) / 128), most = MX_STREAM * stream_steps(x);
    p.kernel = Plan::STREAM;
    p.per = (steps + (steps + most - 1) / most - 1) / ((steps + most - 1) / most);
    p.parts = (steps + p.per - 1) / p.per;
    // a workgroup to a CU; tiles of 16 rows, or blocks of 32 outputs
    const bool blocks = swiglu && p.parts == 1;
    p.n_tiles = blocks ? w->rows / 64 : (w->rows + 15) / 16;
    p.m_tiles = p.parts < 256 ? 256 / p.parts : 1;
    if (p.m_tiles > p.n_tiles) p.m_tiles = p.n_tiles;
    p.ldp = (w->rows + 7) / 8 * 8;
    const int tt = x->rows <= 16 ? 1 : x->rows <= 32 ? 2 : 4;
    const double each = (double)((p.n_tiles + p.m_tiles - 1) / p.m_tiles) * (blocks ? 4 : 1) * p.per;
    const double held = (double)x->rows * p.per * (x->type == FH3K_MX_FP8 ? 128 : 64);
    double t = 5 + each * 0.038 + held / 45e3 + (tt == 4 ? 1.5 : 0);
    if (x->type == FH3K_MX_FP8 && tt > 1) t += tt * (1 + each * 0.008);
    if (p.parts > 1) t += 2.5 + (double)p.parts * x->rows * w->rows * 8 / 4e6;
    return t;
}
// Tiles: for a stage on a CU that has one workgroup of 128 x 128, two, or one of 256 x 256, and for a round's
// beginning and end; parts are written and read at 4 MB a us and joined by a launch of 3.5 us.  FP8 rows of 5120, weights
// in the caches, small and large tiles: 600 rows -> 5120 39, 52 us; 400 -> 17408 93, 91; 1000 -> 15360 129, 108;
// 13824 -> 5120: 600 rows 96, 91, 1000 rows 148, 122.  FP4 rows: 21, 31; 40, 32; 53, 41; 42, 46, 56, 65.
double tiles_us(const Fh3kMx *w, const Fh3kMx *x, Plan &p) {
    const bool f8 = x->type == FH3K_MX_FP8;
    const int ks = f8 ? 128 : 256, stages = (int)((w->in + ks - 1) / ks);
    const double one = f8 ? 0.765 : 0.88, few = f8 ? 1.17 : 0.95, two = f8 ? 1.425 : 1.15, big = f8 ? 1.8 : 1.6;
    double least = 0;
    p.kernel = Plan::TILES;
    // a last round of smaller tiles: one to a CU, two to a few or to all
    auto some = [&](int64_t n, int per) { return n <= 256 ? per * one + 3 : per * (few + (two - few) * (n - 256) / 256) + 4; };
    for (int b = 128; b <= 256; b += 128) {
        const int64_t m = (x->rows + b - 1) / b, n = (w->rows + b - 1) / b;
        for (int parts = 1; parts <= 32 && (parts == 1 || parts * 4 <= stages); parts++) {
            const int per = (stages + parts - 1) / parts;
            if (parts > 1 && (stages + per - 1) / per != parts) continue;
            const int64_t groups = m * n * parts, slots = b == 128 ? 512 : 256, rest = groups % slots;
            const double round = b == 256 ? per * big + 8 : per * two + 4, last = b == 256 ? round : some(rest, per);
            double t = (double)(groups / slots) * round + (rest ? last : 0);
            if (parts > 1) t += 3.5 + (double)parts * x->rows * w->rows * 8 / 4e6;
            // the last round, where it is not full, in smaller tiles: a launch of its own for the last columns
            // (4096 x 13824 -> 5120, 1.25 rounds, FP8 432 -> 380 us, FP4 170 -> 146; 3016 x 5376 -> 28672, 5.25 rounds, 678 -> 643)
            const int64_t large = b == 256 && parts == 1 ? groups / 256 * 256 / m : 0;
            bool mixed = false;
            if (large > 0 && large < n) {
                const int64_t small = (x->rows + 127) / 128 * ((w->rows + 127) / 128 - 2 * large), over = small % 512;
                const double both = (double)(groups / 256) * round + (double)(small / 512) * (per * two + 4) +
                                    (over ? some(over, per) : 0) + 3;
                mixed = both * 1.02 < t;
                if (mixed) t = both;
            }
            if (least == 0 || t < least) {
                least = t;
                p.large = mixed ? large : 0;
                p.bw = p.bx = b;
                p.parts = parts;
                p.per = per;
                p.m_tiles = m;
                p.n_tiles = n;
            }
        }
    }
    p.ldp = (w->rows + 7) / 8 * 8;
    return least;
}
Plan plan_of(const Fh3kMx *w, const Fh3kMx *x, bool swiglu) {
    Plan few = {}, tiles = {}, stream = {};
    few.kernel = Plan::FEW;
    few.parts = 1;
    if (x->rows > 64) {
        tiles_us(w, x, tiles);
        return tiles;
    }
    const double s = stream_us(w, x, swiglu, stream), f = few_us(w, x, swiglu), least = s < f ? s : f;
    // tiles: no less than the weights' way from memory (16 rows: never the least)
    if (x->rows > 16 && 8 + (double)w->rows * w->in * 0.53 / 3.2e6 < least && tiles_us(w, x, tiles) < least) return tiles;
    return f <= s ? few : stream;
}

// Columns first .. of tiles, all or those before `end`.
template <class G> void launch_gemm(const Fh3kMx *w, const Fh3kMx *x, const Fh3kMxOut *o, const Plan &p, int64_t first, int64_t end,
                                                float *part, bool vec, hipStream_t st) {
    const int64_t m = (x->rows + G::BX - 1) / G::BX, all = (w->rows + G::BW - 1) / G::BW, n = (end ? end : all) - first;
    const dim3 grid((unsigned)(m * n), (unsigned)p.parts);
    k_mx_gemm<G><<<grid, 64 * G::WAVES, 0, st>>>(*w, *x, *o, part, p.ldp, (int)m, (int)n, (int)first, p.per, vec || part);
}

template <bool F8, int TT, int R> void launch_few(const Fh3kMx *w, const Fh3kMx *x, const Fh3kMxOut *o, hipStream_t st) {
    const int64_t n = o->y.codes ? w->rows / 2 : w->rows, per = o->y.codes ? 8 * R : 16 * R;
    // as many wavefronts as share the windows evenly, and whose sums fit 64 KiB; where
    // that leaves each more than one, eight that load ahead
    constexpr int WIN = 128 * Window<F8, TT, R>::S;
    const int room = 64 / (R * TT), windows = (int)((w->in + WIN - 1) / WIN);
    auto go = [&](auto ahead, int most) {
        if (most > room) most = room;
        const int each = (windows + most - 1) / most, waves = (windows + each - 1) / each;
        k_mx_few<F8, TT, R, ahead()><<<(unsigned)((n + per - 1) / per), 64 * waves, waves * R * TT * 1024, st>>>(*w, *x, *o);
    };
    // (registers for two windows)
    if constexpr (Window<F8, TT, R>::S * (R + TT * (F8 ? 2 : 1)) <= 20) {
        if (windows > MX_WAVES) return go(std::true_type{}, MX_WAVES_AHEAD);
    }
    go(std::false_type{}, TT == 4 || R * TT == 8 ? MX_WAVES_AHEAD : MX_WAVES);
}

// Whether rows of an array, ld values apart, can be taken 16 bytes at a time.
bool sixteens(const void *p, int64_t ld, int size) { return !p || ((uintptr_t)p % 16 == 0 && ld * size % 16 == 0); }

}  // namespace

extern "C" int fh3k_mx_matmul_fits(const Fh3kMx *w, const Fh3kMx *x) {
    if ((x->rows + 127) / 128 * ((w->rows + 127) / 128) < ((int64_t)1 << 23) && (w->rows + 7) / 8 * 8 * x->rows <= ((int64_t)1 << 40)) return 1;
    const Plan p = plan_of(w, x, false);
    return (p.kernel != Plan::TILES || p.m_tiles * p.n_tiles < ((int64_t)1 << 23)) && p.ldp * x->rows <= ((int64_t)1 << 40);
}

extern "C" size_t fh3k_mx_matmul_ws_bytes(const Fh3kMx *w, const Fh3kMx *x, int swiglu) {
    const Plan p = plan_of(w, x, swiglu);
    return p.parts > 1 ? (size_t)p.parts * p.ldp * x->rows * sizeof(float) : 0;
}

extern "C" hipError_t fh3k_mx_matmul(const Fh3kMx *w, const Fh3kMx *x, const Fh3kMxOut *o, void *ws, hipStream_t st) {
    const bool f8 = x->type == FH3K_MX_FP8;
    const Plan p = plan_of(w, x, o->y.codes);
    float *part = p.parts > 1 ? (float *)ws : nullptr;
    const int size = o->type == FH3K_F32 ? 4 : 2;
    const bool vec = sixteens(o->out, o->ldo, size) && sixteens(o->res, o->ldres, size) && sixteens(o->gate, w->rows, 4);
    using N1 = std::integral_constant<int, 1>;
    using N2 = std::integral_constant<int, 2>;
    using N3 = std::integral_constant<int, 3>;
    using N4 = std::integral_constant<int, 4>;
    using N5 = std::integral_constant<int, 5>;
    using Big4 = Gemm<4, 2, 2, 4, false, 256, 2>;
    using Big8 = Gemm<4, 2, 2, 4, true, 128, 3>;
    using Small4 = Gemm<2, 2, 2, 2, false, 256, 2>;
    using Small8 = Gemm<2, 2, 2, 2, true, 128, 3>;
    auto few = [&](auto f) {
        const int r = few_tiles(w, x, o->y.codes);
        auto go = [&](auto tt) {
            if (r == 4) launch_few<f(), tt(), 4>(w, x, o, st);
            else if (r == 2) launch_few<f(), tt(), 2>(w, x, o, st);
            else launch_few<f(), tt(), 1>(w, x, o, st);
        };
        if (x->rows <= 16) go(N1{});
        else if (x->rows <= 32) go(N2{});
        else go(N4{});
    };
    auto stream = [&](auto f) {
        auto go = [&](auto tt, auto ns) {
            const dim3 grid((unsigned)p.m_tiles, (unsigned)p.parts);
            k_mx_stream<f(), tt(), ns()><<<grid, 64 * MX_STREAM, 0, st>>>(*w, *x, *o, part, p.ldp, (int)p.n_tiles, p.per);
        };
        if (x->rows <= 16) go(N1{}, N5{});
        else if (x->rows <= 32) go(N2{}, N5{});
        else if (stream_steps(x) == 3) go(N4{}, N3{});
        else if constexpr (!f()) go(N4{}, N5{});
    };
    auto tiles = [&](auto large, auto small) {
        if (p.bw == 256) launch_gemm<decltype(large)>(w, x, o, p, 0, p.large, part, vec, st);
        if (p.bw == 128 || p.large) launch_gemm<decltype(small)>(w, x, o, p, 2 * p.large, 0, part, vec, st);
    };
    auto by_rows = [&](auto go) {
        if (f8) go(std::true_type{});
        else go(std::false_type{});
    };
    if (p.kernel == Plan::FEW) by_rows(few);
    else if (p.kernel == Plan::STREAM) by_rows(stream);
    else if (f8) tiles(Big8{}, Small8{});
    else tiles(Big4{}, Small4{});
    if (!part) return hipGetLastError();
    if (o->y.codes) {
        const dim3 grid((unsigned)x->rows, (unsigned)((o->y.in + 2047) / 2048));
        if (o->y.type == FH3K_MX_FP8) k_mx_join_swiglu<true><<<grid, 256, 0, st>>>(part, p.parts, p.ldp, x->rows, *o);
        else k_mx_join_swiglu<false><<<grid, 256, 0, st>>>(part, p.parts, p.ldp, x->rows, *o);
        return hipGetLastError();
    }
    const dim3 grid((unsigned)x->rows, (unsigned)((w->rows + 2047) / 2048));
    return by_type(o->type, [&](auto t) { k_mx_join<t()><<<grid, 256, 0, st>>>(part, p.parts, p.ldp, x->rows, w->rows, *o, vec); });
}
