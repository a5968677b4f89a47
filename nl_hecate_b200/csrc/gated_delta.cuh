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
// Products run on the tensor cores in bf16 (mma.sync m16n8k16) with fp32 sums. A fp32 operand is split into three bf16 planes
// (24 significand bits) when it is written to shared memory, and a product of two such takes six passes, smallest terms
// first; an operand that came in as bf16 is one plane, exact. So the bf16 form computes what the fp32 form computes from the same
// values, and rounds it once. (Two planes for the operands of a bf16 y, whose own rounding hides the difference, saved 1 to 4 % of a
// pass, but then a prompt's y and the recurrent step's, which works in fp32, were of different accuracy.) Two tf32 numbers for a fp32 one take the same time on the tensor cores, but their splitting,
// redone by every warp that reads them, and twice the instructions around each pass cost more: a training step of 64 sequences
// x 8 heads x 512 tokens took 1435 us that way against 1308 (4 x 16 x 4096 in bf16: 1336 against 1122).
// Why not tcgen05: in the kernels that walk the states the matrices are 64 x 64 x 64 and each depends on the one before it. One M64
// N64 K16 tcgen05.mma takes 55 cycles (1190 multiply-adds a cycle), mma.sync does 983, and its results are in registers where the
// next product needs them; tcgen05 needs a commit, a wait and a trip through TMEM and shared memory for each. That does not
// hold for the kernels that form the outputs of all chunks: there tiles could be stacked to 128 x 128, and no product waits for
// another chunk's. They run on mma.sync too, bound by the shared-memory path and latency; what stands against tcgen05 there is the sum of
// many k-steps in one accumulator, which the tensor core cuts off instead of rounding (see gemm), for fp32 streams.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace nlh {
namespace gd {

constexpr int C = 64;          // tokens per chunk
constexpr int LD = 68;         // floats between rows of a 64-column fp32 tile
constexpr int LP = 72;         // bf16 between rows of a 64-column plane: 16-byte pieces of eight rows hit all banks
constexpr int T_BYTES = 3 * C * LP * 2;    // the three planes of T, in global memory as they are in shared memory
constexpr float G_FLOOR = -200.f;      // e^-200 is 0 in fp32: a retention of 0 (g = -inf) without inf - inf
constexpr float THETA_TINY = 8.673617379884035e-19f;   // 2^-60, see gd_prep_kernel

struct Args {
    const void *k, *v, *q, *dy;
    const float *g, *theta, *m0;
    const int* starts;                 // [n_seqs + 1], NULL = dense batch
    long long kb, kt, kh, vb, vt, vh, qb, qt, qh, gb, gt, gh, yb, yt, yh;   // strides in elements: batch, token, head (y: d_y)
    int batch, seq, hk, hv, share, dk, dv, n_seqs, dkp, dvp;   // dkp, dvp: dk, dv padded to 64
    float scale;
    int slots, nc;                     // chunk slots; chunks per sequence of a dense batch
    // private buffers, one tile per slot and value head
    unsigned char* tmat;               // [slot, hv] three planes of T, T_BYTES each
    float4* gates;                     // [slot, hv, 64] {G high, G low, e^G, e^(G_L - G)}
    float* theta_eff;                  // [slot, hv, 64]
    float* e;                          // [slot, hv, 64, dvp]
    float* m_chunk;                    // [slot, hv, dkp, dvp] state in front of the chunk, transposed
    int4* map;                         // [slot] {sequence, first token, length, -} of a ragged batch
    int *start, *off;                  // [n_seqs + 1] first token and first slot of each sequence
    int *order;                        // [n_seqs] sequences in the order in which the state kernels begin them
    void* y;
    float* m_final;
    // backward
    const float* d_m_final;
    float *f, *x, *d_chunk;            // like e, e, m_chunk
    float* dg_part;                    // [dkp / 64, slot, hv, 64] parts of the gradient of log_retain, where there are two
    float *dk_part, *dq_part;          // [batch * seq, hv, dk] when heads share keys
    void *d_k, *d_v, *d_q;
    float *d_g, *d_theta, *d_m0;
    unsigned wait_cycles;              // of the state kernels' waits for T
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

// ── bf16 planes in shared memory ──
typedef __nv_bfloat16 bf;
template <typename T> struct Pl { static constexpr int in = 3; };      // planes of an input
template <> struct Pl<__nv_bfloat16> { static constexpr int in = 1; };

__device__ __forceinline__ unsigned pack2(float x, float y)
{
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const unsigned*>(&h);
}
__device__ __forceinline__ float lo_f(unsigned u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float hi_f(unsigned u) { return __uint_as_float(u & 0xffff0000u); }
// Two neighbouring values -> P planes, `ps` elements apart. What a plane leaves over is exact in fp32.
template <int P> __device__ __forceinline__ void put2(bf* p, int ps, float x, float y)
{
#pragma unroll
    for (int i = 0; i < P; i++) {
        const unsigned h = pack2(x, y);
        *reinterpret_cast<unsigned*>(p + i * ps) = h;
        if (i + 1 < P) { x -= lo_f(h); y -= hi_f(h); }
    }
}
template <int P> __device__ __forceinline__ float2 get2(const bf* p, int ps)
{
    float2 r = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = P - 1; i >= 0; i--) {
        const unsigned h = *reinterpret_cast<const unsigned*>(p + i * ps);
        r.x += lo_f(h);
        r.y += hi_f(h);
    }
    return r;
}
template <int P> __device__ __forceinline__ void put4(bf* p, int ps, float4 v)
{
#pragma unroll
    for (int i = 0; i < P; i++) {
        const unsigned a = pack2(v.x, v.y), b = pack2(v.z, v.w);
        *reinterpret_cast<uint2*>(p + i * ps) = make_uint2(a, b);
        if (i + 1 < P) { v.x -= lo_f(a); v.y -= hi_f(a); v.z -= lo_f(b); v.w -= hi_f(b); }
    }
}
// Four elements of an input as they came -> its planes.
__device__ __forceinline__ void put_raw(bf* p, int ps, float4 v) { put4<3>(p, ps, v); }
__device__ __forceinline__ void put_raw(bf* p, int ps, uint2 v) { *reinterpret_cast<uint2*>(p) = v; }
__device__ __forceinline__ void put_one(bf* p, int ps, float x)
{
#pragma unroll
    for (int i = 0; i < 3; i++) { p[i * ps] = __float2bfloat16(x); x -= __bfloat162float(p[i * ps]); }
}
__device__ __forceinline__ void put_one(bf* p, int ps, bf x) { *p = x; }

template <typename T> struct Raw { typedef float4 type; };
template <> struct Raw<bf> { typedef uint2 type; };
template <typename T> __device__ __forceinline__ bool vec_ok(const T* base, long long stride, int cols)
{
    return ((reinterpret_cast<uintptr_t>(base) | (uintptr_t)(stride * (long long)sizeof(T))) & (4 * sizeof(T) - 1)) == 0 && (cols & 3) == 0;
}

// 64 x COLS of a strided input -> its planes, zero outside [0, rows) x [0, cols). `base` points at column 0 of row 0. Vector loads
// where every row start is aligned to four elements and cols is a multiple of 4.
template <typename T, int COLS, int THREADS>
__device__ __forceinline__ void load_tile(bf* dst, int ld, int ps, const T* base, long long stride, int rows, int cols)
{
    constexpr int PER_ROW = COLS / 4;
    typedef typename Raw<T>::type R;
    if (vec_ok(base, stride, cols)) {
#pragma unroll
        for (int i = 0; i < C * PER_ROW / THREADS; i++) {
            const int at = threadIdx.x + i * THREADS, r = at / PER_ROW, c = (at - r * PER_ROW) * 4;
            R v = R{};
            if (r < rows && c < cols) v = *reinterpret_cast<const R*>(base + r * stride + c);
            put_raw(dst + r * ld + c, ps, v);
        }
    } else {
#pragma unroll 4
        for (int i = 0; i < C * COLS / THREADS; i++) {
            const int at = threadIdx.x + i * THREADS, r = at / COLS, c = at - r * COLS;
            put_one(dst + r * ld + c, ps, r < rows && c < cols ? base[r * stride + c] : from_f<T>(0.f));
        }
    }
}
// 64 x 64 of an input, each row times factor scale[row].z, in three planes.
template <typename T, int THREADS>
__device__ __forceinline__ void load_scaled(bf* dst, const T* base, long long stride, int rows, int cols, float factor, const float4* scale)
{
    if (vec_ok(base, stride, cols)) {
#pragma unroll
        for (int i = 0; i < C * 16 / THREADS; i++) {
            const int at = threadIdx.x + i * THREADS, r = at >> 4, c = (at & 15) * 4;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < rows && c < cols) v = ld4(base + r * stride + c);
            const float s = factor * scale[r].z;
            put4<3>(dst + r * LP + c, C * LP, make_float4(s * v.x, s * v.y, s * v.z, s * v.w));
        }
    } else {
#pragma unroll 4
        for (int i = 0; i < C * 64 / THREADS; i++) {
            const int at = threadIdx.x + i * THREADS, r = at >> 6, c = at & 63;
            put_one(dst + r * LP + c, C * LP, r < rows && c < cols ? factor * scale[r].z * to_f(base[r * stride + c]) : 0.f);
        }
    }
}
__device__ __forceinline__ bool odd(float x) { return !(fabsf(x) <= 3.402823466e38f); }      // an infinity or a NaN
// A lower triangle's 0 times a later token's infinity or NaN is a NaN. Where a chunk holds such a value the two triangular
// products of the forward are formed again token by token: row `row` of lower (planes) times the rows j <= row of x's column.
template <int P> __device__ __noinline__ float triangle_at(const bf* lower, int psl, const bf* x, int ldx, int psx, int row)
{
    float s = 0.f;
    for (int j = 0; j <= row; j++) {
        float a = 0.f, b = 0.f;
        for (int q = P - 1; q >= 0; q--) {
            a += __bfloat162float(lower[q * psl + row * LP + j]);
            b += __bfloat162float(x[q * psx + j * ldx]);
        }
        s = fmaf(a, b, s);
    }
    return s;
}
template <int P, int NT>
__device__ __forceinline__ void triangle_by_token(float (&acc)[NT][4], const bf* lower, int psl, const bf* x, int ldx, int psx, int r0, int c0)
{
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[n][i] += triangle_at<P>(lower, psl, x + c0 + 8 * n + 2 * t + (i & 1), ldx, psx, r0 + g + 8 * (i >> 1));
}

// 64 x 64 of a private, padded buffer, each row times scale[row] where a scale is given; whether the thread's part is odd.
template <int P, int THREADS>
__device__ __forceinline__ bool load_own(bf* dst, const float* base, int stride, const float* scale = nullptr)
{
    bool any = false;
#pragma unroll
    for (int i = 0; i < C * 16 / THREADS; i++) {
        const int at = threadIdx.x + i * THREADS, r = at >> 4, c = (at & 15) * 4;
        float4 v = *reinterpret_cast<const float4*>(base + (long long)r * stride + c);
        if (scale) { const float s = scale[r]; v.x *= s; v.y *= s; v.z *= s; v.w *= s; }
        any |= odd(v.x) | odd(v.y) | odd(v.z) | odd(v.w);
        put4<P>(dst + r * LP + c, C * LP, v);
    }
    return any;
}

// ── products ──
__device__ __forceinline__ unsigned smem_addr(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
template <bool TRANS> __device__ __forceinline__ void ldsm4(unsigned (&r)[4], unsigned a)
{
    if (TRANS) asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
    else asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
template <bool TRANS> __device__ __forceinline__ void ldsm2(unsigned& r0, unsigned& r1, unsigned a)
{
    if (TRANS) asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2];\n" : "=r"(r0), "=r"(r1) : "r"(a) : "memory");
    else asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0,%1}, [%2];\n" : "=r"(r0), "=r"(r1) : "r"(a) : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// One warp: acc (16 x 8 NT) += A (16 x K) B (K x 8 NT) over k in [k0, k1), multiples of 16.
// AK / BK: the operand is stored with k as its row index (A[k][m], B[k][n]) instead of A[m][k], B[n][k]. PA, PB planes,
// psa, psb elements apart. Terms of planes i and j with i + j below the larger count are taken.
// The tensor core cuts its sums off instead of rounding them, and 24 of them on one accumulator add up to 1.4e-6; so a
// k-step starts from 0 and is added to the accumulator with rounding.
template <int NT, bool AK, bool BK, int PA, int PB>
__device__ __forceinline__ void gemm(float (&acc)[NT][4], const bf* A, int lda, int psa, const bf* B, int ldb, int psb, int k0, int k1)
{
    constexpr int TOP = (PA > PB ? PA : PB) - 1;
    const int l = threadIdx.x & 31, l8 = l & 7, q = l >> 3;
    const unsigned a0 = smem_addr(AK ? A + ((q >> 1) * 8 + l8) * lda + (q & 1) * 8 : A + ((q & 1) * 8 + l8) * lda + (q >> 1) * 8);
    const unsigned b0 = smem_addr(BK ? B + ((q & 1) * 8 + l8) * ldb + (q >> 1) * 8 : B + ((q >> 1) * 8 + l8) * ldb + (q & 1) * 8);
#pragma unroll 2
    for (int k = k0; k < k1; k += 16) {
        unsigned a[PA][4];
#pragma unroll
        for (int i = 0; i < PA; i++) ldsm4<AK>(a[i], a0 + 2 * (i * psa + (AK ? k * lda : k)));
#pragma unroll
        for (int n = 0; n < NT; n += 2) {
            unsigned b[PB][4];
#pragma unroll
            for (int j = 0; j < PB; j++) {
                const unsigned at = b0 + 2 * (j * psb + (BK ? k * ldb + n * 8 : k + n * 8 * ldb));
                if (n + 1 < NT) ldsm4<BK>(b[j], at);
                else ldsm2<BK>(b[j][0], b[j][1], at);
            }
#pragma unroll
            for (int e = 0; e < 2; e++) {
                if (n + e < NT) {
                    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int o = TOP; o >= 0; o--)
#pragma unroll
                        for (int i = 0; i < PA; i++)
                            if (o - i >= 0 && o - i < PB) mma_bf16(s, a[i], b[o - i][2 * e], b[o - i][2 * e + 1]);
#pragma unroll
                    for (int x = 0; x < 4; x++) acc[n + e][x] += s[x];
                }
            }
        }
    }
}
// The same for 32 rows: every B fragment serves two A fragments.
template <int NT, bool AK, bool BK, int PA, int PB>
__device__ __forceinline__ void gemm_2(float (&acc)[2][NT][4], const bf* A, int lda, int psa, const bf* B, int ldb, int psb, int k0, int k1)
{
    constexpr int TOP = (PA > PB ? PA : PB) - 1;
    const int l = threadIdx.x & 31, l8 = l & 7, q = l >> 3;
    const unsigned a0 = smem_addr(AK ? A + ((q >> 1) * 8 + l8) * lda + (q & 1) * 8 : A + ((q & 1) * 8 + l8) * lda + (q >> 1) * 8);
    const unsigned b0 = smem_addr(BK ? B + ((q & 1) * 8 + l8) * ldb + (q >> 1) * 8 : B + ((q >> 1) * 8 + l8) * ldb + (q & 1) * 8);
#pragma unroll 1
    for (int k = k0; k < k1; k += 16) {
        unsigned a[2][PA][4];
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
            for (int i = 0; i < PA; i++) ldsm4<AK>(a[m][i], a0 + 2 * (i * psa + (AK ? k * lda + 16 * m : k + 16 * m * lda)));
#pragma unroll
        for (int n = 0; n < NT; n += 2) {
            unsigned b[PB][4];
#pragma unroll
            for (int j = 0; j < PB; j++) ldsm4<BK>(b[j], b0 + 2 * (j * psb + (BK ? k * ldb + n * 8 : k + n * 8 * ldb)));
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int o = TOP; o >= 0; o--)
#pragma unroll
                        for (int i = 0; i < PA; i++)
                            if (o - i >= 0 && o - i < PB) mma_bf16(s, a[m][i], b[o - i][2 * e], b[o - i][2 * e + 1]);
#pragma unroll
                    for (int x = 0; x < 4; x++) acc[m][n + e][x] += s[x];
                }
        }
    }
}
template <int NT> __device__ __forceinline__ void zero(float (&acc)[NT][4])
{
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[n][i] = 0.f;
}

// e^{G_i - G_j} from the pairs (high, low)
__device__ __forceinline__ float decay(float2 gi, float2 gj) { return expf((gi.x - gj.x) + (gi.y - gj.y)); }

// ── loads that stay where they are written: left to itself the compiler moves them down to their first use ──
__device__ __forceinline__ void ldg(float4& v, const float* p)
{
    asm volatile("ld.global.v4.f32 {%0, %1, %2, %3}, [%4];\n" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
}
__device__ __forceinline__ void ldg(uint4& v, const void* p)
{
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
}
__device__ __forceinline__ void ldg(uint2& v, const bf* p)
{
    asm volatile("ld.global.v2.u32 {%0, %1}, [%2];\n" : "=r"(v.x), "=r"(v.y) : "l"(p));
}
__device__ __forceinline__ void ldg(float& v, const float* p) { asm volatile("ld.global.f32 %0, [%1];\n" : "=f"(v) : "l"(p)); }
__device__ __forceinline__ void ldg(float2& v, const float* p)
{
    asm volatile("ld.global.v2.f32 {%0, %1}, [%2];\n" : "=f"(v.x), "=f"(v.y) : "l"(p));
}
__device__ __forceinline__ void ldg(unsigned& v, const bf* p) { asm volatile("ld.global.u32 %0, [%1];\n" : "=r"(v) : "l"(p)); }

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
template <> struct Pair<bf> {
    unsigned r;
    __device__ __forceinline__ void load(const bf* p, bool a, bool b, bool pair)
    {
        r = 0;
        if (pair) { if (a) ldg(r, p); }
        else {
            const unsigned short* u = reinterpret_cast<const unsigned short*>(p);
            r = (a ? (unsigned)u[0] : 0u) | (b ? (unsigned)u[1] << 16 : 0u);
        }
    }
    __device__ __forceinline__ float2 get() const { return make_float2(lo_f(r), hi_f(r)); }
};

// A tile of an input on its way from global to shared memory, in registers: loaded while the chunk before it is computed. Rows
// that do not allow vector loads are read when they are stored instead. Addresses are a thread's own, made once: with 64-bit products and
// divisions in the loop they were a quarter of a chunk's time, since few warps share a scheduler.
template <typename T, int COLS, int THREADS> struct Prefetch {
    typedef typename Raw<T>::type R;
    static constexpr int PER_ROW = COLS / 4, ROWS = THREADS / PER_ROW, N = C / ROWS;
    R r[N];
    const T *base, *mine;                // chunk 0; this thread's part of it
    long long stride;
    int cols, chunk, rows;
    bool vec, has;
    __device__ __forceinline__ void init(const T* b, long long st, int nc)
    {
        base = b; stride = st; cols = nc;
        vec = vec_ok(b, st, nc);
        const int c = (threadIdx.x % PER_ROW) * 4;
        has = vec && c < nc;
        mine = b + threadIdx.x / PER_ROW * st + c;
    }
    __device__ __forceinline__ void load(int c, int nr)
    {
        chunk = c; rows = nr;
        const T* p = mine + c * (C * stride);
#pragma unroll
        for (int i = 0; i < N; i++) {
            r[i] = R{};
            if (has && threadIdx.x / PER_ROW + i * ROWS < nr) ldg(r[i], p);
            p += ROWS * stride;
        }
    }
    __device__ __forceinline__ void store(bf* dst, int ld, int ps) const
    {
        if (!vec) { load_tile<T, COLS, THREADS>(dst, ld, ps, base + chunk * (C * stride), stride, rows, cols); return; }
#pragma unroll
        for (int i = 0; i < N; i++) put_raw(dst + (threadIdx.x / PER_ROW + i * ROWS) * ld + (threadIdx.x % PER_ROW) * 4, ps, r[i]);
    }
};
// The planes of T, copied as they are, straight into shared memory: one bulk copy by one thread, issued when the chunk before has no
// more use for its T, waited for when the next one needs it, half a chunk later. (As 16-byte cp.async by all threads the
// issue alone held the warps up for some 900 cycles of a chunk's 4000.) The wait is bounded by the clock: a second or so, where
// a copy takes a microsecond. Where it runs out, in any thread, the CTA gives the copy in flight as long again, issues no
// more, sets g_gd_timeout, and takes NaN for the product with T: so is its share of the state from there on, and all that follows.
__device__ int g_gd_timeout = 0;
constexpr unsigned T_WAIT_CYCLES = 2000000000u;
__device__ __forceinline__ void init_t(unsigned long long* bar)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;\n" ::"r"(smem_addr(bar)) : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
}
__device__ __forceinline__ void copy_t(bf* dst, const unsigned char* src, unsigned long long* bar)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(smem_addr(bar)), "r"(T_BYTES) : "memory");
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n"
                 ::"r"(smem_addr(dst)), "l"(src), "r"(T_BYTES), "r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ bool test_t(unsigned long long* bar, unsigned parity)
{
    unsigned ok;
    asm volatile("{\n\t.reg .pred P;\n\tmbarrier.try_wait.parity.shared::cta.b64 P, [%1], %2;\n\tselp.u32 %0, 1, 0, P;\n\t}\n"
                 : "=r"(ok) : "r"(smem_addr(bar)), "r"(parity) : "memory");
    return ok != 0;
}
// Whether the copy has arrived before `cycles` have passed.
__device__ __forceinline__ bool wait_t(unsigned long long* bar, unsigned parity, unsigned cycles)
{
    if (cycles > 0 && test_t(bar, parity)) return true;
    for (const unsigned t0 = (unsigned)clock(); (unsigned)clock() - t0 < cycles;)
        if (test_t(bar, parity)) return true;
    return false;
}
template <int NT> __device__ __forceinline__ void fill_nan(float (&acc)[NT][4])
{
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[n][i] = __int_as_float(0x7fffffff);
}
// The wait of a chunk: whether its copy, or one before it, has not come. The answers of a CTA's threads meet in the barrier behind it.
__device__ __forceinline__ bool not_arrived(int* dead, unsigned long long* bar, unsigned parity, unsigned cycles)
{
    if (cycles > 0 && test_t(bar, parity)) return false;
    if (*dead == 0 && wait_t(bar, parity, cycles)) return false;
    if (*dead == 0) *dead = 1;
    return true;
}
// Behind that barrier, where a thread answered so: whether a copy is lost (the same for all threads, and from now on).
__device__ __forceinline__ bool lost_t(int* dead, unsigned long long* bar, unsigned parity)
{
    const int d = *dead;                          // 1: not reported yet
    if (threadIdx.x == 0 && d == 1) {
        wait_t(bar, parity, T_WAIT_CYCLES);
        atomicExch(&g_gd_timeout, 1);
        *dead = 2;
    }
    return d != 0;
}

}  // namespace gd
}  // namespace nlh
