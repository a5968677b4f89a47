// Distillation from a teacher's top logits: loss and gradient.
//
// A row of student logits z [vocab] comes with k teacher entries (id, logit t) and, optionally, a target id:
//   p = softmax(t / tau) over the row's valid entries,
//   loss = hard_weight mean(lse(z) - z_target) + soft_weight tau^2 mean(sum_k p_k (log p_k - z_k / tau + lse(z / tau))),
//   dz_j = hard_weight / n_hard (softmax(z)_j - [j = target]) + soft_weight tau / n_soft (softmax(z / tau)_j - p_j),
// each mean over the rows that have a target / a teacher entry. Both sums come out of one pass over the row with a
// running maximum, and the gradient out of one more: z is read twice and dz written once, which bounds the pair by HBM.
// The exponentials are next (two an element; 16 a cycle and SM): at tau = 2 the one of z is the square of the one of z / tau.
// Every exponential is of z - max, a subtraction that is exact near the maximum, and a row keeps {max, sum, sum}, not a log-sum-exp:
// rounded to one number that would carry an error of 2^-24 of the logits' own size into every probability (4e-5 at logits of 1000).
// Sums over rows and over entries of one id have one order; no atomics.
#include <cuda_bf16.h>
#include <math_constants.h>

#include "nlh_common.cuh"
#include "../../include/nlh_ffi.h"

namespace nlh {
namespace distill {

constexpr int MAX_K = 1024, MAX_N = 1 << 30;          // MAX_N: rows, and vocabulary; strided loops stay in 32 bits
constexpr float LOG2E = 1.4426950408889634f;

struct Args {
    const void* z;
    long long z_row, d_row;              // elements between rows of logits and of d_logits
    const int *targets, *ids;
    const void* t;
    void* d;
    const float* grad;
    int n, vocab, k, t_bf16, splits, per_split;
    float tau, inv_tau, hard_w, soft_w;
    bool hard, soft;                     // which terms exist
    // saved
    float4* stat;                        // [n] {max, sum e^(z - max), sum e^((z - max) / tau), -}
    float2* row;                         // [n] cross-entropy, divergence; -infinity (which neither can be) where a row has none
    float* stats;                        // {-, hard_weight / n_hard, soft_weight tau / n_soft, -}
    float* loss;
    float4* part;                        // [n, splits] {max, sum e^(z - max), sum e^((z - max) / tau), -}
};

__device__ __forceinline__ float ld(const float* p) { return *p; }
__device__ __forceinline__ float ld(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two fp32 operations in one instruction: the kernels are bound by instruction issue next to the exponentials.
typedef unsigned long long f2;
__device__ __forceinline__ f2 pair(float a, float b)
{
    f2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 both(f2 v)
{
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c)
{
    f2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b)
{
    f2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b)
{
    f2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f2 ex2_2(f2 v)
{
    const float2 x = both(v);
    return pair(ex2(x.x), ex2(x.y));
}

// Which exponentials a row needs. ONE: e^((z - max) c) alone (a single term, or tau = 1); SQUARE: tau = 2; BOTH: any other tau.
enum Mode { ONE = 0, SQUARE = 1, BOTH = 2 };

template <typename T> struct Vec { static constexpr int N = 16 / sizeof(T); };
template <typename T> __device__ __forceinline__ void unpack(const uint4& u, float* f);
template <> __device__ __forceinline__ void unpack<float>(const uint4& u, float* f)
{
    f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
}
template <> __device__ __forceinline__ void unpack<__nv_bfloat16>(const uint4& u, float* f)
{
    const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
template <typename T> __device__ __forceinline__ uint4 pack(const float* f);
template <> __device__ __forceinline__ uint4 pack<float>(const float* f)
{
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}
template <> __device__ __forceinline__ uint4 pack<__nv_bfloat16>(const float* f)
{
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const unsigned*>(&b);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

struct Stat { float m, h, s; };          // maximum, sum e^(z - m), sum e^((z - m) / tau)

template <int MODE>
__device__ __forceinline__ void add_one(float x, float m, float cs, float ch, float& h, float& s)
{
    const float e = ex2((x - m) * cs);
    s += e;
    if (MODE == SQUARE) h = fmaf(e, e, h);
    if (MODE == BOTH) h += ex2((x - m) * ch);
}
template <int MODE> __device__ __forceinline__ void raise(Stat& a, float m, float cs, float ch)
{
    if (m > a.m) {
        a.s *= ex2((a.m - m) * cs);
        if (MODE != ONE) a.h *= ex2((a.m - m) * ch);
        a.m = m;
    }
}
template <int MODE> __device__ __forceinline__ void add_scalar(Stat& a, float x, float cs, float ch)
{
    const float m = fmaxf(a.m, x);
    if (m == -CUDART_INF_F) {
        if (x != x) a.h = a.s = x;                // nothing but -infinity so far; a NaN, which fmaxf passes over, must not be lost
        return;
    }
    raise<MODE>(a, m, cs, ch);
    add_one<MODE>(x, m, cs, ch, a.h, a.s);
}
__device__ __forceinline__ float max_of(const uint4& u, const float*)
{
    return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
}
__device__ __forceinline__ float max_of(const uint4& u, const __nv_bfloat16*)
{
    const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(&u);
    const __nv_bfloat162 m = __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
    return fmaxf(__low2float(m), __high2float(m));
}
// V 16-byte vectors at once: one step of the running maximum, in the elements' own type, then their exponentials.
template <typename T, int MODE, int V>
__device__ __forceinline__ void add_vectors(Stat& a, const uint4* u, float cs, float ch)
{
    constexpr int N = Vec<T>::N;
    float m = a.m;
#pragma unroll
    for (int v = 0; v < V; v++) m = fmaxf(m, max_of(u[v], (const T*)nullptr));
    if (m == -CUDART_INF_F) {
#pragma unroll
        for (int v = 0; v < V; v++) {
            float f[N];
            unpack<T>(u[v], f);
            for (int i = 0; i < N; i++) add_scalar<MODE>(a, f[i], cs, ch);
        }
        return;
    }
    raise<MODE>(a, m, cs, ch);
    const f2 c2 = pair(cs, cs), m2 = pair(-m, -m), ch2 = pair(ch, ch);
    f2 h = pair(0.f, 0.f), s = pair(0.f, 0.f);
#pragma unroll
    for (int v = 0; v < V; v++) {
        float f[N];
        unpack<T>(u[v], f);
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const f2 x = add2(pair(f[i], f[i + 1]), m2), e = ex2_2(mul2(x, c2));
            s = add2(s, e);
            if (MODE == SQUARE) h = fma2(e, e, h);
            if (MODE == BOTH) h = add2(h, ex2_2(mul2(x, ch2)));
        }
    }
    a.h += both(h).x + both(h).y;
    a.s += both(s).x + both(s).y;
}
template <int MODE>
__device__ __forceinline__ Stat merge(const Stat& a, const Stat& b, float cs, float ch)
{
    Stat o;
    o.m = fmaxf(a.m, b.m);
    if (o.m == -CUDART_INF_F) { o.h = a.h + b.h; o.s = a.s + b.s; return o; }
    o.s = a.s * ex2((a.m - o.m) * cs) + b.s * ex2((b.m - o.m) * cs);
    o.h = MODE == ONE ? o.s : a.h * ex2((a.m - o.m) * ch) + b.h * ex2((b.m - o.m) * ch);
    return o;
}

__device__ __forceinline__ float warp_max(float v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// Statistics of columns [j0, j1) of a row by TH threads: aligned 16-byte loads, four in flight, scalars at the ragged ends.
// The calling warp's share.
template <typename T, int MODE, int TH>
__device__ __forceinline__ Stat row_stat(const T* row, int j0, int j1, float cs, float ch, int tid)
{
    constexpr int N = Vec<T>::N;
    Stat a = {-CUDART_INF_F, 0.f, 0.f};
    const int lead = min(j1 - j0, (int)(((16 - ((uintptr_t)(row + j0) & 15)) & 15) / sizeof(T)));
    const int nvec = (j1 - j0 - lead) / N, tail = j0 + lead + nvec * N;
    const uint4* r4 = reinterpret_cast<const uint4*>(row + j0 + lead);
    for (int i = tid; i < nvec; i += 4 * TH) {
        uint4 u[4];
#pragma unroll
        for (int q = 0; q < 4; q++) if (i + q * TH < nvec) u[q] = __ldg(r4 + i + q * TH);
        if (i + 3 * TH < nvec) add_vectors<T, MODE, 4>(a, u, cs, ch);
        else {
#pragma unroll
            for (int q = 0; q < 3; q++) if (i + q * TH < nvec) add_vectors<T, MODE, 1>(a, u + q, cs, ch);
        }
    }
    if (tid < lead) add_scalar<MODE>(a, ld(row + j0 + tid), cs, ch);
    if (tid < j1 - tail) add_scalar<MODE>(a, ld(row + tail + tid), cs, ch);
    const float m = warp_max(a.m);
    if (m != -CUDART_INF_F) raise<MODE>(a, m, cs, ch);
    a.s = warp_sum(a.s);
    if (MODE != ONE) a.h = warp_sum(a.h);
    return a;
}

__device__ __forceinline__ float teacher(const Args& A, long long at)
{
    return A.t_bf16 ? ld((const __nv_bfloat16*)A.t + at) : ((const float*)A.t)[at];
}
// Entry i of a row: its id if it counts, -1 if not (an id outside the vocabulary, a logit of -infinity).
__device__ __forceinline__ int entry(const Args& A, long long row, int i, float& t)
{
    const int id = A.ids[row * A.k + i];
    t = teacher(A, row * A.k + i);
    return id >= 0 && id < A.vocab && t != -CUDART_INF_F ? id : -1;
}
__device__ __forceinline__ bool has_target(const Args& A, int row)
{
    return A.hard && A.targets[row] >= 0 && A.targets[row] < A.vocab;
}
// One warp: {sum_k p_k (log p_k - (z_k - ref) / tau), ref} of a row, ref the largest of the entries' logits; {-infinity, -} where it
// has no entry.
template <typename T> __device__ float2 teacher_cross(const Args& A, int row, const T* z)
{
    const int lane = threadIdx.x & 31;
    float top = -CUDART_INF_F, ref = -CUDART_INF_F;
    bool mine = false;
    for (int i = lane; i < A.k; i += 32) {
        float t;
        const int id = entry(A, row, i, t);
        if (id >= 0) { top = t != t ? t : fmaxf(top, t); ref = fmaxf(ref, ld(z + id)); mine = true; }
    }
    if (!__any_sync(0xffffffffu, mine)) return make_float2(-CUDART_INF_F, 0.f);
    top = warp_max(top);
    ref = warp_max(ref);
    if (ref == -CUDART_INF_F) ref = 0.f;          // no mass of the student's on any entry: infinite, not NaN
    float sum = 0.f, cross = 0.f;                 // t' = (t - top) / tau: sum e^t'; sum e^t' (t' - (z - ref) / tau)
    for (int i = lane; i < A.k; i += 32) {
        float t;
        const int id = entry(A, row, i, t);
        if (id < 0) continue;
        t = (t - top) * A.inv_tau;
        const float e = expf(t);
        sum += e;
        if (e != 0.f) cross += e * (t - (ld(z + id) - ref) * A.inv_tau);
    }
    sum = warp_sum(sum);
    cross = warp_sum(cross);
    return make_float2(cross / sum - logf(sum), ref);
}
// One thread: the row's values from its statistics; zt is the target's logit.
__device__ __forceinline__ void finish_row(const Args& A, int row, const Stat& a, bool target, float zt, float2 cross)
{
    const float h = A.hard && A.soft && A.tau != 1.f ? a.h : a.s;
    A.stat[row] = make_float4(a.m, h, a.s, 0.f);
    A.row[row] = make_float2(target ? logf(h) + (a.m - zt) : -CUDART_INF_F,
                             cross.x != -CUDART_INF_F ? cross.x + ((a.m - cross.y) * A.inv_tau + logf(a.s)) : -CUDART_INF_F);
}

// TH threads read the row; one more warp reads the teacher's entries meanwhile.
template <typename T, int MODE, int TH>
__global__ void __launch_bounds__(TH + 32, TH == 128 ? 8 : 6) fwd_kernel(Args A, float cs, float ch)
{
    __shared__ Stat s_stat[TH / 32];
    __shared__ float2 s_cross;
    __shared__ float s_target;
    const int row = blockIdx.x / A.splits, sp = blockIdx.x - row * A.splits;
    const bool target = has_target(A, row);
    if (!A.soft && !target) {                     // no term: the row is not read
        if (sp == 0 && threadIdx.x == 0) A.row[row] = make_float2(-CUDART_INF_F, -CUDART_INF_F);
        return;
    }
    const T* z = (const T*)A.z + (long long)row * A.z_row;
    if (threadIdx.x < TH) {
        const int j0 = sp * A.per_split, j1 = min(A.vocab, j0 + A.per_split);
        const Stat a = row_stat<T, MODE, TH>(z, j0, j1, cs, ch, threadIdx.x);
        if ((threadIdx.x & 31) == 0) s_stat[threadIdx.x >> 5] = a;
    } else {
        if (threadIdx.x == TH) s_target = target && A.splits == 1 ? ld(z + A.targets[row]) : 0.f;
        const float2 x = A.soft && A.splits == 1 ? teacher_cross<T>(A, row, z) : make_float2(-CUDART_INF_F, 0.f);
        if (threadIdx.x == TH) s_cross = x;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        Stat a = s_stat[0];
        for (int w = 1; w < TH / 32; w++) a = merge<MODE>(a, s_stat[w], cs, ch);
        if (A.splits > 1) A.part[(long long)row * A.splits + sp] = make_float4(a.m, a.h, a.s, 0.f);
        else finish_row(A, row, a, target, s_target, s_cross);
    }
}
// A warp per row, four rows a CTA.
template <typename T, int MODE>
__global__ void __launch_bounds__(128, 12) fwd_warp_kernel(Args A, float cs, float ch)
{
    const int row = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (row >= A.n) return;
    const bool target = has_target(A, row);
    if (!A.soft && !target) {
        if (lane == 0) A.row[row] = make_float2(-CUDART_INF_F, -CUDART_INF_F);
        return;
    }
    const T* z = (const T*)A.z + (long long)row * A.z_row;
    const float zt = target ? ld(z + A.targets[row]) : 0.f;
    const float2 cross = A.soft ? teacher_cross<T>(A, row, z) : make_float2(-CUDART_INF_F, 0.f);
    const Stat a = row_stat<T, MODE, 32>(z, 0, A.vocab, cs, ch, lane);
    if (lane == 0) finish_row(A, row, a, target, zt, cross);
}
template <typename T, int MODE>
__global__ void __launch_bounds__(32) join_kernel(Args A, float cs, float ch)
{
    const int row = blockIdx.x;
    const bool target = has_target(A, row);
    if (!A.soft && !target) return;
    const T* z = (const T*)A.z + (long long)row * A.z_row;
    const float zt = target ? ld(z + A.targets[row]) : 0.f;
    const float2 cross = A.soft ? teacher_cross<T>(A, row, z) : make_float2(-CUDART_INF_F, 0.f);
    if (threadIdx.x != 0) return;
    Stat a = {-CUDART_INF_F, 0.f, 0.f};
#pragma unroll 8
    for (int i = 0; i < A.splits; i++) {
        const float4 p = A.part[(long long)row * A.splits + i];
        a = merge<MODE>(a, Stat{p.x, p.y, p.z}, cs, ch);
    }
    finish_row(A, row, a, target, zt, cross);
}

// Means over the rows. One CTA, one order: thread i adds rows i, i + 1024, ... in 64 bits.
__global__ void __launch_bounds__(1024) mean_kernel(Args A)
{
    __shared__ double s_d[2][32];
    __shared__ int s_i[2][32];
    double ce = 0., kl = 0.;
    int nh = 0, ns = 0;
#pragma unroll 16
    for (int i = threadIdx.x; i < A.n; i += 1024) {
        const float2 x = A.row[i];
        if (x.x != -CUDART_INF_F) { ce += x.x; nh++; }
        if (x.y != -CUDART_INF_F) { kl += x.y; ns++; }
    }
    for (int o = 16; o > 0; o >>= 1) {
        ce += __shfl_xor_sync(0xffffffffu, ce, o);
        kl += __shfl_xor_sync(0xffffffffu, kl, o);
        nh += __shfl_xor_sync(0xffffffffu, nh, o);
        ns += __shfl_xor_sync(0xffffffffu, ns, o);
    }
    const int w = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) { s_d[0][w] = ce; s_d[1][w] = kl; s_i[0][w] = nh; s_i[1][w] = ns; }
    __syncthreads();
    if (threadIdx.x == 0) {
        ce = kl = 0.;
        nh = ns = 0;
        for (int i = 0; i < 32; i++) { ce += s_d[0][i]; kl += s_d[1][i]; nh += s_i[0][i]; ns += s_i[1][i]; }
        const double h = A.hard ? (double)A.hard_w / max(nh, 1) : 0., s = A.soft ? (double)A.soft_w / max(ns, 1) : 0.;
        *A.loss = (float)((A.hard ? h * ce : 0.) + (A.soft ? s * A.tau * A.tau * kl : 0.));
        A.stats[1] = (float)h;
        A.stats[2] = (float)(s * A.tau);
    }
}

// What a row's gradient is made of. m: its maximum. ONE: a single softmax, e^((z - m) c) gs. SQUARE: e^(z - m) = (e^((z - m) / 2))^2.
// gs, gh: the terms' weights over their sums.
struct RowGrad {
    bool hard, soft;
    float wh, ws;                        // what the target / an entry's p takes off
    float m, gs, gh;
};
template <int MODE> __device__ __forceinline__ RowGrad row_grad(const Args& A, int row)
{
    RowGrad r;
    const float2 rv = A.row[row];
    const float4 st = A.stat[row];       // all on their way at once; of no meaning where the row has no term
    const float g = A.grad ? *A.grad : 1.f, sh = A.stats[1], ss = A.stats[2];
    r.hard = rv.x != -CUDART_INF_F;
    r.soft = rv.y != -CUDART_INF_F;
    r.wh = r.hard ? g * sh : 0.f;
    r.ws = r.soft ? g * ss : 0.f;
    r.m = st.x;
    r.gh = 0.f;
    if (MODE == ONE) r.gs = (r.ws + r.wh) / st.z;        // of the only term, or of both at tau = 1
    else { r.gs = r.ws / st.z; r.gh = r.wh / st.y; }
    return r;
}
template <int MODE> __device__ __forceinline__ float grad_of(float x, const RowGrad& r, float cs, float ch)
{
    const float e = ex2((x - r.m) * cs);
    if (MODE == ONE) return r.gs * e;
    if (MODE == SQUARE) return e * fmaf(r.gh, e, r.gs);
    return fmaf(r.gs, e, r.gh * ex2((x - r.m) * ch));
}
// Two elements at once.
template <int MODE> __device__ __forceinline__ float2 grad_of2(float x, float y, const RowGrad& r, float cs, float ch)
{
    const f2 d = add2(pair(x, y), pair(-r.m, -r.m)), e = ex2_2(mul2(d, pair(cs, cs))), gs = pair(r.gs, r.gs), gh = pair(r.gh, r.gh);
    if (MODE == ONE) return both(mul2(gs, e));
    if (MODE == SQUARE) return both(mul2(e, fma2(gh, e, gs)));
    return both(fma2(gs, e, mul2(gh, ex2_2(mul2(d, pair(ch, ch))))));
}

// Columns [j0, j1) of a row by TH threads.
template <typename T> struct Span {
    int j0, j1, lead, nvec, body, tail;
    __device__ __forceinline__ Span(const T* z, const T* d, int a, int b) : j0(a), j1(b)
    {
        lead = min(j1 - j0, (int)(((16 - ((uintptr_t)(z + j0) & 15)) & 15) / sizeof(T)));
        nvec = (((uintptr_t)z ^ (uintptr_t)d) & 15) ? 0 : (j1 - j0 - lead) / Vec<T>::N;    // 16-byte stores where both rows align
        body = j0 + lead;
        tail = body + nvec * Vec<T>::N;
    }
};
template <typename T, int TH> __device__ __forceinline__ void load_first(uint4 (&u)[4], const T* z, const Span<T>& s, int tid)
{
    const uint4* r4 = reinterpret_cast<const uint4*>(z + s.body);
#pragma unroll
    for (int q = 0; q < 4; q++) if (tid + q * TH < s.nvec) u[q] = r4[tid + q * TH];
}
template <typename T, int MODE, int TH>
__device__ __forceinline__ void write_row(const T* z, T* d, const Span<T>& s, uint4 (&u)[4], const RowGrad& r, float cs, float ch, int tid)
{
    constexpr int N = Vec<T>::N;
    const uint4* r4 = reinterpret_cast<const uint4*>(z + s.body);
    uint4* d4 = reinterpret_cast<uint4*>(d + s.body);
    for (int i = tid; i < s.nvec; i += 4 * TH) {
        if (i != tid) {
#pragma unroll
            for (int q = 0; q < 4; q++) if (i + q * TH < s.nvec) u[q] = r4[i + q * TH];
        }
#pragma unroll
        for (int q = 0; q < 4; q++) {
            if (i + q * TH < s.nvec) {
                float f[N];
                unpack<T>(u[q], f);
#pragma unroll
                for (int e = 0; e < N; e += 2) {
                    const float2 o = grad_of2<MODE>(f[e], f[e + 1], r, cs, ch);
                    f[e] = o.x;
                    f[e + 1] = o.y;
                }
                d4[i + q * TH] = pack<T>(f);
            }
        }
    }
    if (tid < s.lead) d[s.j0 + tid] = T(grad_of<MODE>(ld(z + s.j0 + tid), r, cs, ch));
    for (int j = s.tail + tid; j < s.j1; j += TH) d[j] = T(grad_of<MODE>(ld(z + j), r, cs, ch));
}
template <typename T, int TH> __device__ __forceinline__ void zero_row(T* d, const Span<T>& s, int tid)
{
    for (int i = tid; i < s.nvec; i += TH) reinterpret_cast<uint4*>(d + s.body)[i] = make_uint4(0, 0, 0, 0);
    if (tid < s.lead) d[s.j0 + tid] = T(0.f);
    for (int j = s.tail + tid; j < s.j1; j += TH) d[j] = T(0.f);
}

// The row's entries in shared memory by one warp: ids inside [j0, j1), logits z there, and (in weigh) p times its weight; the
// target is one more entry.
struct Entries { int* id; float *w, *z; };
template <typename T> __device__ __forceinline__ float read_entries(const Args& A, const Entries& E, int row, const T* z, int j0, int j1, int k,
                                                                    const RowGrad& r)
{
    const int lane = threadIdx.x & 31;
    float top = -CUDART_INF_F;
    for (int i = lane; i < k; i += 32) {
        float t;
        const int id = entry(A, row, i, t);
        const bool here = id >= j0 && id < j1;
        E.id[i] = here ? id : -1;
        E.z[i] = here ? ld(z + id) : 0.f;
        E.w[i] = id >= 0 ? t : -CUDART_INF_F;
        if (id >= 0) top = t != t ? t : fmaxf(top, t);
    }
    if (lane == 0) {
        const int id = r.hard ? A.targets[row] : -1;
        const bool here = id >= j0 && id < j1;
        E.id[k] = here ? id : -1;
        for (int i = k + 1; i & 3; i++) E.id[i] = -1;
        E.w[k] = r.wh;
        E.z[k] = here ? ld(z + id) : 0.f;
    }
    return top;
}
__device__ __forceinline__ void weigh(const Entries& E, int k, float top, float inv_tau, float ws)
{
    const int lane = threadIdx.x & 31;
    float sum = 0.f;
    top = warp_max(top);
    for (int i = lane; i < k; i += 32) {
        const float e = expf((E.w[i] - top) * inv_tau);       // 0 for an entry that does not count
        E.w[i] = e;
        sum += e;
    }
    const float wn = ws / warp_sum(sum);
    for (int i = lane; i < k; i += 32) E.w[i] *= wn;
}
// An id that several entries name is written by the first of them, with all their p in the entries' order.
template <typename T, int MODE, int TH>
__device__ __forceinline__ void write_entries(const Entries& E, int k, T* d, const RowGrad& r, float cs, float ch, int tid)
{
    for (int i = tid; i <= k; i += TH) {
        const int id = E.id[i];
        if (id < 0) continue;
        float w = E.w[i];
        bool first = true;
        int same = 0;
        for (int j = 0; j <= k; j += 4) {
            const int4 o = *reinterpret_cast<const int4*>(E.id + j);
            same += (o.x == id) + (o.y == id) + (o.z == id) + (o.w == id);
        }
        if (same > 1) {
            w = 0.f;
            for (int j = 0; j <= k; j++)
                if (E.id[j] == id) { first &= j >= i; w += E.w[j]; }
        }
        if (first) d[id] = T(grad_of<MODE>(E.z[i], r, cs, ch) - w);
    }
}

// Barrier that the two kinds of warps reach at different places, where the gradient goes over the logits: the entries' elements
// have been read.
template <int TH> __device__ __forceinline__ void entries_read() { asm volatile("bar.sync 1, %0;\n" ::"n"(TH + 32) : "memory"); }

// TH threads write the row; one more warp has the entries. d_logits may be logits: a thread reads its elements before it writes
// them, and the elements of the entries, which are written once more at the end with their p taken off, are read before
// anything is written. 32768 rows of 8192 bf16 at tau 2: 198 us with nine CTAs an SM (twelve spill registers: 211, ten: 208).
template <typename T, int MODE, int TH>
__global__ void __launch_bounds__(TH + 32, TH == 128 ? 9 : 5) bwd_kernel(Args A, float cs, float ch)
{
    __shared__ __align__(16) int s_id[MAX_K + 4];
    __shared__ float s_w[MAX_K + 1], s_z[MAX_K + 1];
    const Entries E = {s_id, s_w, s_z};
    const int row = blockIdx.x / A.splits, sp = blockIdx.x - row * A.splits;
    const int j0 = sp * A.per_split, j1 = min(A.vocab, j0 + A.per_split);
    const T* z = (const T*)A.z + (long long)row * A.z_row;
    T* d = (T*)A.d + (long long)row * A.d_row;
    const Span<T> s(z, d, j0, j1);
    uint4 u[4];                                   // on their way while the row's statistics come in
    if (threadIdx.x < TH) load_first<T, TH>(u, z, s, threadIdx.x);
    const RowGrad r = row_grad<MODE>(A, row);
    if (!r.hard && !r.soft) { zero_row<T, TH + 32>(d, s, threadIdx.x); return; }
    const int k = r.soft ? A.k : 0;
    const bool in_place = A.d == A.z;             // else nothing that is written is still to be read
    if (threadIdx.x < TH) {
        if (in_place) entries_read<TH>();
        write_row<T, MODE, TH>(z, d, s, u, r, cs, ch, threadIdx.x);
    } else {
        const float top = read_entries<T>(A, E, row, z, j0, j1, k, r);
        if (in_place) entries_read<TH>();
        else __syncwarp();
        weigh(E, k, top, A.inv_tau, r.ws);
    }
    __syncthreads();
    write_entries<T, MODE, TH + 32>(E, k, d, r, cs, ch, threadIdx.x);
}
// ── host ──
static int64_t place(Args& A, char* base)
{
    int64_t at = 0;
    auto take = [&](int64_t bytes) { char* p = base + at; at += (bytes + 255) & ~(int64_t)255; return (void*)p; };
    A.stat = (float4*)take((int64_t)A.n * 16);
    A.row = (float2*)take((int64_t)A.n * 8);
    A.stats = (float*)take(16);
    A.part = A.splits > 1 ? (float4*)take((int64_t)A.n * A.splits * 16) : nullptr;
    return at;
}
// Few rows: each is divided over CTAs until every SM has two, in pieces of 4096 columns at least.
static void divide(Args& A)
{
    const int most = (A.vocab + 4095) / 4096, want = A.n > 0 ? (2 * 148 + A.n - 1) / A.n : 1;
    A.splits = A.n >= 148 ? 1 : (want < most ? want : most);
    if (A.splits < 1) A.splits = 1;
    A.per_split = ((A.vocab + A.splits - 1) / A.splits + 7) & ~7;
    A.splits = (A.vocab + A.per_split - 1) / A.per_split;
}
static bool fill(const char* where, Args& A, const void* logits, int64_t row_stride, const int32_t* targets, const int32_t* teacher_ids,
                 const void* teacher_logits, int32_t teacher_is_bf16, int32_t n, int32_t vocab, int32_t k, float temperature,
                 float hard_weight, float soft_weight)
{
    A = Args{};
    const char* bad = nullptr;
    A.hard = targets != nullptr && hard_weight != 0.f;
    A.soft = teacher_ids != nullptr && soft_weight != 0.f;
    if (n < 0 || n > MAX_N || vocab <= 0 || vocab > MAX_N || k < 0 || k > MAX_K || row_stride < vocab)
        bad = "bad dimensions (k is at most 1024, n and vocab 2^30)";
    else if (!(temperature > 0.f) || temperature > 1e6f || temperature < 1e-6f) bad = "the temperature must be in [1e-6, 1e6]";
    else if (n > 0 && (!logits || (A.soft && k > 0 && !teacher_logits))) bad = "NULL pointer";
    if (bad) { record_status(NLH_ERR_INVALID_ARG, where, bad); return false; }
    A.z = logits; A.z_row = row_stride; A.targets = targets; A.ids = teacher_ids; A.t = teacher_logits; A.t_bf16 = teacher_is_bf16;
    A.n = n; A.vocab = vocab; A.k = A.soft ? k : 0; A.tau = temperature; A.inv_tau = 1.f / temperature; A.hard_w = hard_weight; A.soft_w = soft_weight;
    divide(A);
    return true;
}
// Whether the gradient's rows share an element with the logits', other than as the same elements in the same places: exact for rows
// of one stride, else whether the address ranges meet.
static bool overlaps(const Args& A, int64_t size)
{
    const int64_t n = A.n, width = A.vocab, apart = ((intptr_t)A.d - (intptr_t)A.z) / size, row = n > 1 ? A.z_row : 0;
    if (n > 1 && A.d_row != row) return apart > -((n - 1) * A.d_row + width) && apart < (n - 1) * row + width;
    int64_t k = 0;                       // rows of logits that a row of the gradient can meet: this far ahead, and the next
    if (row) { k = apart / row; if (k * row > apart) k--; }
    for (int i = 0; i < 2; i++, k++) {
        const int64_t off = apart - k * row;
        if (apart != 0 && k < n && -k < n && off < width && -off < width) return true;
    }
    return false;
}
static int mode_of(const Args& A) { return !(A.hard && A.soft) || A.tau == 1.f ? ONE : A.tau == 2.f ? SQUARE : BOTH; }

// Who reads a row in the forward: with many short rows a warp, which waits at no barrier (32768 x 8192 bf16 at tau 2: 110 us
// against 132), else a CTA (8192 x 16000: 63 us against 65). The backward writes as well, and is faster with a CTA at every size
// (32768 x 8192 when both were measured: 196 us against 216).
static bool warp_rows(const Args& A) { return A.vocab <= 12288 && A.n >= 4096; }

template <typename T, int MODE, int TH> static bool forward(const Args& A, float cs, const char* where)
{
    cudaStream_t st = current_stream();
    fwd_kernel<T, MODE, TH><<<(unsigned)((long long)A.n * A.splits), TH + 32, 0, st>>>(A, cs, LOG2E);
    if (!check_launch(where)) return false;
    if (A.splits > 1) {
        join_kernel<T, MODE><<<A.n, 32, 0, st>>>(A, cs, LOG2E);
        if (!check_launch(where)) return false;
    }
    return true;
}
template <typename T, int MODE, int TH> static bool backward(const Args& A, float cs, const char* where)
{
    bwd_kernel<T, MODE, TH><<<(unsigned)((long long)A.n * A.splits), TH + 32, 0, current_stream()>>>(A, cs, LOG2E);
    return check_launch(where);
}
template <typename T, int MODE> static bool launch_mode(const Args& A, bool bwd, const char* where)
{
    const float cs = LOG2E / (A.soft ? A.tau : 1.f);
    if (!bwd && warp_rows(A)) {
        fwd_warp_kernel<T, MODE><<<(unsigned)(((long long)A.n + 3) / 4), 128, 0, current_stream()>>>(A, cs, LOG2E);
        return check_launch(where);
    }
    if (A.vocab <= 16384) return bwd ? backward<T, MODE, 128>(A, cs, where) : forward<T, MODE, 128>(A, cs, where);
    return bwd ? backward<T, MODE, 256>(A, cs, where) : forward<T, MODE, 256>(A, cs, where);
}
template <typename T> static bool launch(const Args& A, bool bwd, const char* where)
{
    switch (mode_of(A)) {
    case ONE: return launch_mode<T, ONE>(A, bwd, where);
    case SQUARE: return launch_mode<T, SQUARE>(A, bwd, where);
    default: return launch_mode<T, BOTH>(A, bwd, where);
    }
}

}  // namespace distill
}  // namespace nlh

using namespace nlh;

extern "C" {

int64_t nlh_distill_saved_bytes(int32_t n, int32_t vocab)
{
    if (n < 0 || n > distill::MAX_N || vocab <= 0 || vocab > distill::MAX_N) return -1;
    distill::Args A{};
    A.n = n; A.vocab = vocab;
    distill::divide(A);
    return distill::place(A, nullptr);
}

int32_t nlh_distill_forward(const void* logits, int32_t logits_is_bf16, int64_t row_stride, const int32_t* target_ids,
    const int32_t* teacher_ids, const void* teacher_logits, int32_t teacher_is_bf16, float* loss, void* saved, int64_t saved_bytes,
    int32_t n, int32_t vocab, int32_t k, float temperature, float hard_weight, float soft_weight)
{
    const char* where = "nlh_distill_forward";
    distill::Args A;
    if (!distill::fill(where, A, logits, row_stride, target_ids, teacher_ids, teacher_logits, teacher_is_bf16, n, vocab, k, temperature,
                       hard_weight, soft_weight)) return NLH_ERR_INVALID_ARG;
    if (!loss || !saved || !aligned16(saved) || saved_bytes < distill::place(A, (char*)saved)) {
        record_status(NLH_ERR_INVALID_ARG, where, "NULL output, or a saved buffer that is too small or not 16-byte aligned");
        return NLH_ERR_INVALID_ARG;
    }
    A.loss = loss;
    if (n > 0 && !(logits_is_bf16 ? distill::launch<__nv_bfloat16>(A, false, where) : distill::launch<float>(A, false, where)))
        return NLH_ERR_CUDA;
    distill::mean_kernel<<<1, 1024, 0, current_stream()>>>(A);
    if (!check_launch(where)) return NLH_ERR_CUDA;
    return NLH_OK;
}

int32_t nlh_distill_backward(const void* logits, int32_t logits_is_bf16, int64_t row_stride, const int32_t* target_ids,
    const int32_t* teacher_ids, const void* teacher_logits, int32_t teacher_is_bf16, const void* saved, int64_t saved_bytes,
    const float* grad_scale, void* d_logits, int64_t d_row_stride, int32_t n, int32_t vocab, int32_t k, float temperature,
    float hard_weight, float soft_weight)
{
    const char* where = "nlh_distill_backward";
    distill::Args A;
    if (!distill::fill(where, A, logits, row_stride, target_ids, teacher_ids, teacher_logits, teacher_is_bf16, n, vocab, k, temperature,
                       hard_weight, soft_weight)) return NLH_ERR_INVALID_ARG;
    if (!saved || !aligned16(saved) || saved_bytes < distill::place(A, (char*)saved) || d_row_stride < vocab || (n > 0 && !d_logits)) {
        record_status(NLH_ERR_INVALID_ARG, where, "NULL pointer, a bad stride, or a saved buffer that is too small or not 16-byte aligned");
        return NLH_ERR_INVALID_ARG;
    }
    if (n == 0) return NLH_OK;
    A.d = d_logits; A.d_row = d_row_stride; A.grad = grad_scale;
    if (distill::overlaps(A, logits_is_bf16 ? 2 : 4)) {
        record_status(NLH_ERR_INVALID_ARG, where, "d_logits overlaps logits without being logits");
        return NLH_ERR_INVALID_ARG;
    }
    return (logits_is_bf16 ? distill::launch<__nv_bfloat16>(A, true, where) : distill::launch<float>(A, true, where)) ? NLH_OK : NLH_ERR_CUDA;
}

}  // extern "C"
