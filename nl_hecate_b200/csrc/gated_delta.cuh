// Gated delta rule in matrix form over chunks of 64 tokens: shared device code.
//
//   M_t = e^{g_t} M_{t-1} + u_t k_t^T,  u_t = theta_t e_t,  e_t = v_t - e^{g_t} M_{t-1} k_t,  y_t = scale M_t q_t
//
// M [dv, dk] fp32. Inside a chunk, with G_i = g_1 + ... + g_i and the state M_0 in front of it:
//   B_ij = e^{G_i - G_j} k_i.k_j (j < i),  T = (I + B diag(theta))^-1,  E = T (V - diag(e^G) K M_0^T),
//   Y = scale (diag(e^G) Q M_0^T + tril(e^{G_i - G_j} Q K^T) diag(theta) E),
//   M_L = e^{G_L} M_0 + (diag(theta e^{G_L - G}) E)^T K.
// theta scales the columns of B, not the rows, so that no gradient has to divide by a theta that may be 0.
//
// Products run on the tensor cores as tf32 (mma.sync m16n8k8). A fp32 operand is split into two tf32 numbers
// (22 significand bits) and the product takes three passes, low terms first; an operand that came in as bf16 is
// exact in one. A product whose result is rounded to bf16 takes one pass with operands rounded to tf32 (11 bits,
// 2^-12 of the value against the result's 2^-9). Why not tcgen05: the matrices are 64 x 64 x 64 and each depends
// on the one before it. One M64 N64 K16 tcgen05.mma takes 55 cycles (1190 multiply-adds a cycle), a bf16
// mma.sync 983, a tf32 one 486, and the results of mma.sync are in registers where the next product needs
// them; tcgen05 needs a commit, a wait and a trip through TMEM and shared memory for each.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace nlh {
namespace gd {

constexpr int C = 64;          // tokens per chunk
constexpr int LD = 68;         // floats between rows of a 64-column tile: = 4 (mod 32), see gemm16
constexpr float G_FLOOR = -200.f;      // e^-200 is 0 in fp32: a retention of 0 (g = -inf) without inf - inf
constexpr float THETA_TINY = 8.673617379884035e-19f;   // 2^-60, see gd_prep_kernel

struct Args {
    const void *k, *v, *q, *dy;
    const float *g, *theta, *m0;
    const int* starts;                 // [n_seqs + 1], NULL = dense batch
    long long kb, kt, kh, vb, vt, vh, qb, qt, qh, gb, gt, gh, yb, yt, yh;   // strides in elements: batch, token, head (y: d_y)
    int batch, seq, hk, hv, share, dk, dv, n_seqs, dkp, dvp;   // dkp, dvp: padded to 64 and 32
    float scale;
    int slots, nc;                     // chunk slots; chunks per sequence of a dense batch
    // private buffers, one tile per slot and value head
    float* tmat;                       // [slot, hv, 64, 64]
    float4* gates;                     // [slot, hv, 64] {G high, G low, e^G, e^(G_L - G)}
    float* theta_eff;                  // [slot, hv, 64]
    float* e;                          // [slot, hv, 64, dvp]
    float* m_chunk;                    // [slot, hv, dvp, dkp] state in front of the chunk
    int4* map;                         // [slot] {sequence, first token, length, -} of a ragged batch
    int *start, *off;                  // [n_seqs + 1] first token and first slot of each sequence
    void* y;
    float* m_final;
    // backward
    const float* d_m_final;
    float *f, *x, *d_chunk;            // like e, e, m_chunk
    float* dg_part;                    // [dkp / 64, slot, hv, 64] gradient of G, then [dkp / 64, slot, hv] of the chunk's last G
    float* dgl_part;
    float *dk_part, *dq_part;          // [batch * seq, hv, dk] when heads share keys
    void *d_k, *d_v, *d_q;
    float *d_g, *d_theta, *d_m0;
};

struct Chunk {
    int seq, b, t0, len;
    __device__ long long row0(const Args& A) const { return (long long)b * A.seq + t0; }   // row of [batch * seq]
};

__device__ __forceinline__ Chunk get_chunk(const Args& A, int slot)
{
    Chunk c;
    if (A.starts) {
        const int4 m = A.map[slot];
        c.seq = m.x; c.b = 0; c.t0 = m.y; c.len = m.z;
    } else {
        c.seq = c.b = slot / A.nc;
        c.t0 = (slot - c.seq * A.nc) * C;
        c.len = min(C, A.seq - c.t0);
    }
    return c;
}

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16(x); }

__device__ __forceinline__ void st2(float* p, float a, float b) { *reinterpret_cast<float2*>(p) = make_float2(a, b); }
__device__ __forceinline__ void st2(__nv_bfloat16* p, float a, float b)
{
    *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(a, b);
}

// Four consecutive elements as floats.
__device__ __forceinline__ float4 ld4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 ld4(const __nv_bfloat16* p)
{
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x));
    const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
    return make_float4(a.x, a.y, b.x, b.y);
}

// rows x COLS of a strided matrix -> shared memory, zero outside [0, rows) x [0, cols). `base` points at column 0 of
// row 0. Vector loads where every row start is aligned to four elements and cols is a multiple of 4.
template <typename T, int COLS, int THREADS>
__device__ __forceinline__ void load_tile(float* dst, int ld, const T* base, long long stride, int rows, int cols)
{
    constexpr int PER_ROW = COLS / 4;
    const bool vec = ((reinterpret_cast<uintptr_t>(base) | (uintptr_t)(stride * (long long)sizeof(T))) & (4 * sizeof(T) - 1)) == 0 &&
                     (cols & 3) == 0;
    if (vec) {
#pragma unroll
        for (int i = 0; i < C * PER_ROW / THREADS; i++) {
            const int at = threadIdx.x + i * THREADS, r = at / PER_ROW, c = (at - r * PER_ROW) * 4;
            const float4 v = r < rows && c < cols ? ld4(base + r * stride + c) : make_float4(0.f, 0.f, 0.f, 0.f);
            *reinterpret_cast<float4*>(dst + r * ld + c) = v;
        }
    } else {
#pragma unroll 4
        for (int i = 0; i < C * COLS / THREADS; i++) {
            const int at = threadIdx.x + i * THREADS, r = at / COLS, c = at - r * COLS;
            dst[r * ld + c] = r < rows && c < cols ? to_f(base[r * stride + c]) : 0.f;
        }
    }
}
// The same for the private, padded buffers: always aligned, ROWS x COLS whole.
template <int ROWS, int COLS, int THREADS>
__device__ __forceinline__ void load_own(float* dst, int ld, const float* base, int stride)
{
    constexpr int PER_ROW = COLS / 4;
#pragma unroll
    for (int i = 0; i < ROWS * PER_ROW / THREADS; i++) {
        const int at = threadIdx.x + i * THREADS, r = at / PER_ROW, c = (at - r * PER_ROW) * 4;
        *reinterpret_cast<float4*>(dst + r * ld + c) = *reinterpret_cast<const float4*>(base + (long long)r * stride + c);
    }
}

// ── tf32 products ──
enum Planes { EXACT = 0, ONE = 1, TWO = 2 };   // operand exact in tf32; rounded to tf32; split into two

// x = hi + lo, hi rounded to 11 bits by Dekker's splitting (the constant is 2^13 + 1). A NaN stays a NaN in hi, an infinity
// or a value above 4e34 becomes one; adding half a unit to the bits instead would turn the NaN 0x7fffffff into -0.
__device__ __forceinline__ float round_tf32(float x)
{
    const float c = __fmul_rn(x, 8193.f);
    return __fsub_rn(c, __fsub_rn(c, x));
}
template <int P>
__device__ __forceinline__ void split(float x, unsigned& hi, unsigned& lo)
{
    if (P == EXACT) { hi = __float_as_uint(x); return; }
    const float h = round_tf32(x);
    hi = __float_as_uint(h);
    if (P == TWO) lo = __float_as_uint(__fsub_rn(x, h));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1)
{
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// One warp: acc (16 x 8 NT) += A (16 x K) B (K x 8 NT) over k in [k0, k1), both multiples of 8.
// AK / BK: the operand is stored with k as its row index (A[k][m], B[k][n]) instead of A[m][k], B[n][k].
// Rows are LD = 4 (mod 32) floats apart. A row of the product's k-step may take any eight k as long as both operands
// agree: with k-rows in play lane t takes k + 2t and k + 2t + 1, which makes reads of k-rows free of bank conflicts
// (bank 8t + g) and reads of the other kind 8-byte loads; without them it takes k + t and k + t + 4 (bank 4g + t).
// The tensor core cuts its sums off instead of rounding them, and 24 of them on one accumulator add up to 1.4e-6; so
// a k-step starts from 0 and is added to the accumulator with rounding: 2.4e-6 -> 3.5e-7 against 64 bits over a
// training step of 512 tokens (a chunked form in fp32 FMA: 3.5e-7), for 12 % of the time.
template <int NT, bool AK, bool BK, int PA, int PB>
__device__ __forceinline__ void gemm16(float (&acc)[NT][4], const float* A, int lda, const float* B, int ldb, int k0, int k1)
{
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    constexpr bool PAIR = AK || BK;
#pragma unroll 2
    for (int k = k0; k < k1; k += 8) {
        float af[4];
        if (AK) {
            const float* p = A + (k + 2 * t) * lda + g;
            af[0] = p[0]; af[1] = p[8]; af[2] = p[lda]; af[3] = p[lda + 8];
        } else if (PAIR) {
            const float2 x = *reinterpret_cast<const float2*>(A + g * lda + k + 2 * t);
            const float2 y = *reinterpret_cast<const float2*>(A + (g + 8) * lda + k + 2 * t);
            af[0] = x.x; af[2] = x.y; af[1] = y.x; af[3] = y.y;
        } else {
            const float* p = A + g * lda + k + t;
            af[0] = p[0]; af[1] = p[8 * lda]; af[2] = p[4]; af[3] = p[8 * lda + 4];
        }
        unsigned ah[4], al[4];
#pragma unroll
        for (int i = 0; i < 4; i++) split<PA>(af[i], ah[i], al[i]);
#pragma unroll
        for (int n = 0; n < NT; n++) {
            float b0, b1;
            if (BK) {
                const float* p = B + (k + 2 * t) * ldb + n * 8 + g;
                b0 = p[0]; b1 = p[ldb];
            } else if (PAIR) {
                const float2 x = *reinterpret_cast<const float2*>(B + (n * 8 + g) * ldb + k + 2 * t);
                b0 = x.x; b1 = x.y;
            } else {
                const float* p = B + (n * 8 + g) * ldb + k + t;
                b0 = p[0]; b1 = p[4];
            }
            unsigned h0, h1, l0, l1;
            split<PB>(b0, h0, l0);
            split<PB>(b1, h1, l1);
            float s[4] = {0.f, 0.f, 0.f, 0.f};
            if (PA == TWO) mma_tf32(s, al, h0, h1);
            if (PB == TWO) mma_tf32(s, ah, l0, l1);
            mma_tf32(s, ah, h0, h1);
#pragma unroll
            for (int i = 0; i < 4; i++) acc[n][i] += s[i];
        }
    }
}
// The same with B split beforehand into pairs (hi, lo): a matrix that several warps read is split once, by who writes it.
// B[n][k] rows are 4 (mod 16) pairs apart, B[k][n] rows 2 (mod 8), for 8-byte reads without bank conflicts.
template <int NT, bool AK, bool BK, int PA>
__device__ __forceinline__ void gemm16s(float (&acc)[NT][4], const float* A, int lda, const float2* B, int ldb, int k0, int k1)
{
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    constexpr bool PAIR = AK || BK;
#pragma unroll 4
    for (int k = k0; k < k1; k += 8) {
        float af[4];
        if (AK) {
            const float* p = A + (k + 2 * t) * lda + g;
            af[0] = p[0]; af[1] = p[8]; af[2] = p[lda]; af[3] = p[lda + 8];
        } else if (PAIR) {
            const float2 x = *reinterpret_cast<const float2*>(A + g * lda + k + 2 * t);
            const float2 y = *reinterpret_cast<const float2*>(A + (g + 8) * lda + k + 2 * t);
            af[0] = x.x; af[2] = x.y; af[1] = y.x; af[3] = y.y;
        } else {
            const float* p = A + g * lda + k + t;
            af[0] = p[0]; af[1] = p[8 * lda]; af[2] = p[4]; af[3] = p[8 * lda + 4];
        }
        unsigned ah[4], al[4];
#pragma unroll
        for (int i = 0; i < 4; i++) split<PA>(af[i], ah[i], al[i]);
#pragma unroll
        for (int n = 0; n < NT; n++) {
            float2 b0, b1;
            if (BK) {
                const float2* p = B + (k + 2 * t) * ldb + n * 8 + g;
                b0 = p[0]; b1 = p[ldb];
            } else if (PAIR) {
                const float2* p = B + (n * 8 + g) * ldb + k + 2 * t;
                b0 = p[0]; b1 = p[1];
            } else {
                const float2* p = B + (n * 8 + g) * ldb + k + t;
                b0 = p[0]; b1 = p[4];
            }
            float s[4] = {0.f, 0.f, 0.f, 0.f};
            if (PA == TWO) mma_tf32(s, al, __float_as_uint(b0.x), __float_as_uint(b1.x));
            mma_tf32(s, ah, __float_as_uint(b0.y), __float_as_uint(b1.y));
            mma_tf32(s, ah, __float_as_uint(b0.x), __float_as_uint(b1.x));
#pragma unroll
            for (int i = 0; i < 4; i++) acc[n][i] += s[i];
        }
    }
}
__device__ __forceinline__ float2 split_pair(float x)
{
    const float h = round_tf32(x);
    return make_float2(h, __fsub_rn(x, h));
}

// A tile on its way from global to shared memory, in registers: loaded while the chunk before it is computed. Rows that do
// not allow vector loads are read when they are stored instead.
template <typename T> struct Raw { typedef float4 type; };
template <> struct Raw<__nv_bfloat16> { typedef uint2 type; };
__device__ __forceinline__ float4 widen(float4 v) { return v; }
__device__ __forceinline__ float4 widen(uint2 u)
{
    const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x));
    const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
    return make_float4(a.x, a.y, b.x, b.y);
}
// Loads that stay where they are written: left to itself the compiler moves them down to their first use.
__device__ __forceinline__ void ldg(float4& v, const float* p)
{
    asm volatile("ld.global.v4.f32 {%0, %1, %2, %3}, [%4];\n" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
}
__device__ __forceinline__ void ldg(uint2& v, const __nv_bfloat16* p)
{
    asm volatile("ld.global.v2.u32 {%0, %1}, [%2];\n" : "=r"(v.x), "=r"(v.y) : "l"(p));
}
__device__ __forceinline__ void ldg(float& v, const float* p) { asm volatile("ld.global.f32 %0, [%1];\n" : "=f"(v) : "l"(p)); }
__device__ __forceinline__ void ldg(float2& v, const float* p)
{
    asm volatile("ld.global.v2.f32 {%0, %1}, [%2];\n" : "=f"(v.x), "=f"(v.y) : "l"(p));
}
__device__ __forceinline__ void ldg(unsigned& v, const __nv_bfloat16* p) { asm volatile("ld.global.u32 %0, [%1];\n" : "=r"(v) : "l"(p)); }

// Two neighbouring columns of a strided matrix, as they came; `pair` says that one load may take both.
template <typename T> struct Pair;
template <> struct Pair<float> {
    float2 r;
    __device__ __forceinline__ void load(const float* p, bool a, bool b, bool pair)
    {
        r = make_float2(0.f, 0.f);
        if (pair) { if (a) ldg(r, p); }
        else { if (a) r.x = p[0]; if (b) r.y = p[1]; }
    }
    __device__ __forceinline__ float2 get() const { return r; }
};
template <> struct Pair<__nv_bfloat16> {
    unsigned r;
    __device__ __forceinline__ void load(const __nv_bfloat16* p, bool a, bool b, bool pair)
    {
        r = 0;
        if (pair) { if (a) ldg(r, p); }
        else {
            const unsigned short *u = reinterpret_cast<const unsigned short*>(p);
            r = (a ? (unsigned)u[0] : 0u) | (b ? (unsigned)u[1] << 16 : 0u);
        }
    }
    __device__ __forceinline__ float2 get() const { return make_float2(__uint_as_float(r << 16), __uint_as_float(r & 0xffff0000u)); }
};

template <typename T, int COLS, int THREADS> struct Prefetch {
    typedef typename Raw<T>::type R;
    static constexpr int PER_ROW = COLS / 4, N = C * PER_ROW / THREADS;
    R r[N];
    const T* base;
    long long stride;
    int rows, cols;
    bool vec;
    __device__ __forceinline__ void load(const T* b, long long st, int nr, int nc)
    {
        base = b; stride = st; rows = nr; cols = nc;
        vec = ((reinterpret_cast<uintptr_t>(b) | (uintptr_t)(st * (long long)sizeof(T))) & (4 * sizeof(T) - 1)) == 0 && (nc & 3) == 0;
        if (!vec) return;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int at = threadIdx.x + i * THREADS, row = at / PER_ROW, c = (at - row * PER_ROW) * 4;
            r[i] = R{};
            if (row < rows && c < cols) ldg(r[i], base + row * stride + c);
        }
    }
    __device__ __forceinline__ void store(float* dst, int ld) const
    {
        if (!vec) { load_tile<T, COLS, THREADS>(dst, ld, base, stride, rows, cols); return; }
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int at = threadIdx.x + i * THREADS, row = at / PER_ROW, c = (at - row * PER_ROW) * 4;
            *reinterpret_cast<float4*>(dst + row * ld + c) = widen(r[i]);
        }
    }
};

template <int NT> __device__ __forceinline__ void zero(float (&acc)[NT][4])
{
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[n][i] = 0.f;
}

// e^{G_i - G_j} from the pairs (high, low)
__device__ __forceinline__ float decay(float2 gi, float2 gj) { return expf((gi.x - gj.x) + (gi.y - gj.y)); }

// Planes of an operand that came in as T, of a fp32 one, and of operands of a product that is stored as T.
template <typename T> struct Pl { static constexpr int in = TWO, mid = TWO, out = TWO; };
template <> struct Pl<__nv_bfloat16> { static constexpr int in = EXACT, mid = TWO, out = ONE; };

}  // namespace gd
}  // namespace nlh
