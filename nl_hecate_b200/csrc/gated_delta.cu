// Gated delta rule: chunked forward and backward, recurrent step. Mathematics and products: gated_delta.cuh.
//
// Only the state in front of each chunk is a recurrence; the rest of a chunk is known once that state is.
// So a pass has three parts: what needs no state, for all chunks at once (prep); the states, one after the
// other, divided over the columns of V, which never meet (state); what needs them, for all chunks at once
// (out). The backward has the same three parts. Every sum has one order: no atomics.
#include <atomic>

#include "gated_delta.cuh"
#include "nlh_common.cuh"
#include "../../include/nlh_ffi.h"

namespace nlh {
namespace gd {

// ── ragged batches: sequence, first token and length of every chunk slot ──
// Starts are taken at their running maximum inside [0, seq], so that no value of them can lead out of the buffers:
// the lengths are not negative and add up to seq at most, which bounds the chunks by seq / 64 + n_seqs.
__device__ __forceinline__ int block_scan(int v, bool take_max, int* s_warp)
{
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v = take_max ? max(v, y) : v + y;
    }
    if (lane == 31) s_warp[w] = v;
    __syncthreads();
    for (int j = 0; j < w; j++) v = take_max ? max(v, s_warp[j]) : v + s_warp[j];
    return v;
}
constexpr int RANKED = 256;
__global__ void __launch_bounds__(1024) gd_map_kernel(Args A)
{
    __shared__ int s_warp[32], s_last;
    for (int pass = 0; pass < 2; pass++) {          // running maximum of the starts, then the sum of the chunks before each
        int carry = 0;
        for (int base = 0; base <= A.n_seqs; base += 1024) {
            const int i = base + threadIdx.x;
            int v = 0, n = 0;
            if (pass == 0) v = i <= A.n_seqs ? min(max(A.starts[i], 0), A.seq) : 0;
            else v = n = i < A.n_seqs ? (A.start[i + 1] - A.start[i] + C - 1) / C : 0;
            v = block_scan(v, pass == 0, s_warp);
            v = pass == 0 ? max(v, carry) : v + carry;
            if (i <= A.n_seqs) (pass == 0 ? A.start : A.off)[i] = v - n;
            if (threadIdx.x == 1023) s_last = v;
            __syncthreads();
            carry = s_last;
            __syncthreads();
        }
    }
    // The state kernels begin long sequences first: their chains are what a pass waits for. (13 prompts x 8 heads, the longest the last in
    // the batch: 72 + 80 us against 84 + 94 in the batch's order; 40 prompts: 94 + 114 against 122 + 145.) Many sequences even out by themselves.
    __shared__ int s_len[RANKED];
    const bool ranked = A.n_seqs <= RANKED;
    if (ranked && threadIdx.x < A.n_seqs) s_len[threadIdx.x] = A.off[threadIdx.x + 1] - A.off[threadIdx.x];
    __syncthreads();
    for (int i = threadIdx.x; i < A.n_seqs; i += 1024) {
        int rank = i;
        if (ranked) {
            rank = 0;
            for (int j = 0; j < A.n_seqs; j++) rank += s_len[j] > s_len[i] || (s_len[j] == s_len[i] && j < i);
        }
        A.order[rank] = i;
    }
    for (int slot = threadIdx.x; slot < A.slots; slot += 1024) {
        int lo = 0, hi = A.n_seqs;                  // off[lo] <= slot; the last such lo
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (A.off[mid] <= slot) lo = mid; else hi = mid - 1;
        }
        int4 m = make_int4(0, 0, 0, 0);
        if (lo < A.n_seqs) {
            const int t0 = A.start[lo] + (slot - A.off[lo]) * C;
            m = make_int4(lo, t0, min(C, A.start[lo + 1] - t0), 0);
        }
        A.map[slot] = m;
    }
}

__device__ __forceinline__ int first_slot(const Args& A, int seq) { return A.starts ? A.off[seq] : seq * A.nc; }
__device__ __forceinline__ int chunk_count(const Args& A, int seq) { return A.starts ? A.off[seq + 1] - A.off[seq] : A.nc; }

// ── prep: gates and T = (I + B diag(theta))^-1 of a chunk ──
// One CTA of eight warps per chunk and value head. T is built from the inverses of its 16 x 16 diagonal blocks (forward substitution,
// a thread per column) by [[P, 0], [R, S]]^-1 = [[P', 0], [-S' R P', S']]: to 32 x 32 in fp32 FMA, to 64 x 64 on the tensor
// cores, in the planes that leave for global memory. (All of it in FMA: 138 us for 4096 tiles of fp32 keys, against 99.)
// A theta of 0 is taken as 2^-60: then u is 2^-60 e, which no sum of fp32 sees, and the gradient e.x / theta of
// theta needs no case of its own (x, the gradient of v, carries the factor theta).
template <typename T>
__global__ void __launch_bounds__(256, 3) gd_prep_kernel(Args A)
{
    constexpr int IN = Pl<T>::in, PS = C * LP;
    extern __shared__ float4 smem4[];
    bf* Tp = reinterpret_cast<bf*>(smem4);        // K's planes, then T's
    float* Am = reinterpret_cast<float*>(Tp + 3 * PS);
    float* Tm = Am + C * LD;
    float* Z = Am + C / 2;                        // [32][LD] inside Am's upper right quarter, which no one reads
    __shared__ float2 s_g[C];
    __shared__ float s_theta[C];
    const int slot = blockIdx.x / A.hv, h = blockIdx.x - slot * A.hv;
    const Chunk ch = get_chunk(A, slot);
    if (ch.len <= 0) return;
    const long long tile = (long long)slot * A.hv + h;
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, rb = w & 3, hf = w >> 2, g = lane >> 2, t = lane & 3;

    if (w == 4) {                                 // all of its part of K K^T is above the diagonal
        const long long at = ch.b * A.gb + ch.t0 * A.gt + h * A.gh;
        double x[2], th[2];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int i = 2 * lane + j;
            float gv = 0.f, tv = 0.f;
            if (i < ch.len) { gv = A.g[at + i * A.gt]; tv = A.theta[at + i * A.gt]; }
            x[j] = gv < G_FLOOR ? G_FLOOR : gv;
            th[j] = fabsf(tv) < THETA_TINY ? THETA_TINY : tv;
        }
        double s = x[0] + x[1];
        for (int o = 1; o < 32; o <<= 1) { const double y = __shfl_up_sync(0xffffffffu, s, o); if (lane >= o) s += y; }
        const double last = __shfl_sync(0xffffffffu, s, 31);
        double before = __shfl_up_sync(0xffffffffu, s, 1);       // not s - x[1]: a NaN there would reach the token before it
        if (lane == 0) before = 0.;
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int i = 2 * lane + j;
            const double G = j == 1 ? s : before + x[0];
            const float hi = (float)G;
            const float4 o = make_float4(hi, (float)(G - hi), expf(hi), expf((float)(last - G)));
            A.gates[tile * C + i] = o;
            A.theta_eff[tile * C + i] = (float)th[j];
            s_g[i] = make_float2(o.x, o.y);
            s_theta[i] = (float)th[j];
        }
    }
    float kk[4][4];
    zero(kk);
    const bool need = 32 * hf <= 16 * rb + 15;
    const T* kp = (const T*)A.k + ch.b * A.kb + ch.t0 * A.kt + (h / A.share) * A.kh;
    for (int c0 = 0; c0 < A.dk; c0 += 64) {
        __syncthreads();
        load_tile<T, 64, 256>(Tp, LP, PS, kp + c0, A.kt, ch.len, A.dk - c0);
        __syncthreads();
        if (need) gemm<4, false, false, IN, IN>(kk, Tp + 16 * rb * LP, LP, PS, Tp + 32 * hf * LP, LP, PS, 0, 64);
    }
    bool any = false;
    if (need) {
#pragma unroll
        for (int n = 0; n < 4; n++) {
            if (32 * hf + 8 * n > 16 * rb + 15) continue;
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const int i = 16 * rb + g + 8 * r, j = 32 * hf + 8 * n + 2 * t;
                const float2 gi = s_g[i];
                float a[2];
#pragma unroll
                for (int e = 0; e < 2; e++) a[e] = j + e < i ? decay(gi, s_g[j + e]) * kk[n][2 * r + e] * s_theta[j + e] : 0.f;
                any |= odd(a[0]) | odd(a[1]);
                st2(Am + i * LD + j, a[0], a[1]);
            }
        }
    }
    uint4* out = reinterpret_cast<uint4*>(A.tmat + tile * T_BYTES);
    if (__syncthreads_or(any)) {                  // a value that is not finite: rows from the ones before them alone, see triangle_by_token
        if (tid < 64)
            for (int i = 0; i < C; i++) {
                float s = i == tid ? 1.f : 0.f;
                for (int l = tid; l < i; l++) s = fmaf(-Am[i * LD + l], Tm[l * LD + tid], s);
                Tm[i * LD + tid] = s;
            }
        __syncthreads();
        for (int i = tid; i < C * 16; i += 256)
            put4<3>(Tp + (i >> 4) * LP + (i & 15) * 4, PS, *reinterpret_cast<const float4*>(Tm + (i >> 4) * LD + (i & 15) * 4));
        __syncthreads();
        for (int i = tid; i < T_BYTES / 16; i += 256) out[i] = reinterpret_cast<const uint4*>(Tp)[i];
        return;
    }
    if (tid < 64) {
        const int b = tid & ~15, j = tid & 15;
        float col[16];
#pragma unroll
        for (int i = 0; i < 16; i++) {
            float s = i == j ? 1.f : 0.f;
            const float* row = Am + (b + i) * LD + b;
#pragma unroll
            for (int l = 0; l < i; l++) s = fmaf(-row[l], col[l], s);       // col[l] is 0 above the diagonal
            col[i] = s;
            Tm[(b + i) * LD + b + j] = s;
        }
    } else {
        // meanwhile the planes' blocks that need no inverse: zeros, and B diag(theta) where T's lower left quarter will be
        for (int i = tid - 64; i < C * 16; i += 192) {
            const int r = i >> 4, c = (i & 15) * 4;
            if (r < 32 && c >= 32) put4<3>(Tp + r * LP + c, PS, make_float4(0.f, 0.f, 0.f, 0.f));
            if (r >= 32 && c < 32) put4<3>(Tp + r * LP + c, PS, *reinterpret_cast<const float4*>(Am + r * LD + c));
        }
    }
    __syncthreads();
    {   // 16 -> 32, both pairs of blocks at once, two columns a thread
        const int p = tid >> 7, r = (tid >> 3) & 15, c = (tid & 7) * 2, r0 = 32 * p + 16, c0 = 32 * p;
        float2 z = make_float2(0.f, 0.f);
#pragma unroll
        for (int l = 0; l < 16; l++) {
            const float a = Am[(r0 + r) * LD + c0 + l];
            const float2 b = *reinterpret_cast<const float2*>(Tm + (c0 + l) * LD + c0 + c);
            z.x = fmaf(a, b.x, z.x);
            z.y = fmaf(a, b.y, z.y);
        }
        *reinterpret_cast<float2*>(Z + (16 * p + r) * LD + c) = z;
        __syncthreads();
        float2 o = make_float2(0.f, 0.f);
#pragma unroll
        for (int l = 0; l < 16; l++) {
            const float a = -Tm[(r0 + r) * LD + r0 + l];
            const float2 b = *reinterpret_cast<const float2*>(Z + (16 * p + l) * LD + c);
            o.x = fmaf(a, b.x, o.x);
            o.y = fmaf(a, b.y, o.y);
        }
        *reinterpret_cast<float2*>(Tm + (r0 + r) * LD + c0 + c) = o;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; i++) {                 // the 32 x 32 inverses into the planes
        const int at = tid + i * 256, q = at >> 8, r = (at >> 3) & 31, c = (at & 7) * 4;
        float4 v = *reinterpret_cast<const float4*>(Tm + (32 * q + r) * LD + 32 * q + c);
        if (r < 16 && c >= 16) v = make_float4(0.f, 0.f, 0.f, 0.f);         // never written in Tm
        put4<3>(Tp + (32 * q + r) * LP + 32 * q + c, PS, v);
    }
    __syncthreads();
    {   // 32 -> 64: warp = 16 x 8 of the lower left quarter
        const int r0 = 32 + 16 * (w & 1), c0 = 8 * (w >> 1);
        float z[1][4];
        zero(z);
        gemm<1, false, true, 3, 3>(z, Tp + r0 * LP, LP, PS, Tp + c0, LP, PS, 0, 32);
        __syncthreads();
        put2<3>(Tp + (r0 + g) * LP + c0 + 2 * t, PS, z[0][0], z[0][1]);
        put2<3>(Tp + (r0 + g + 8) * LP + c0 + 2 * t, PS, z[0][2], z[0][3]);
        __syncthreads();
        zero(z);
        gemm<1, false, true, 3, 3>(z, Tp + r0 * LP + 32, LP, PS, Tp + 32 * LP + c0, LP, PS, 0, 32);
        __syncthreads();
        put2<3>(Tp + (r0 + g) * LP + c0 + 2 * t, PS, -z[0][0], -z[0][1]);
        put2<3>(Tp + (r0 + g + 8) * LP + c0 + 2 * t, PS, -z[0][2], -z[0][3]);
    }
    __syncthreads();
    for (int i = tid; i < T_BYTES / 16; i += 256) out[i] = reinterpret_cast<const uint4*>(Tp)[i];
}

// ── forward states: the recurrence over chunks for NS columns of V ──
// Eight warps: warp = 16 rows (tokens; state rows of each 64 of dk in the update) x half of the columns. The state (transposed, S
// [dk, dv]) stays in the update's accumulators from chunk to chunk. While a chunk is computed the next one's K, V and gates are
// on their way in registers, and its T in a bulk copy. Bound by the chain of three products of 64 x NS x 64 a chunk: NS = 32 shares the loads of K and T
// among more columns, NS = 16 gives twice the CTAs where heads are few. A bf16 K has two buffers, so that only the
// products' own barriers are left; three planes of a fp32 one have one buffer, which lets two CTAs share an SM.
template <typename T, int DKP, int NS> struct StateSmem {
    static constexpr int LK = DKP + 8, LS = NS + 8, KB = Pl<T>::in == 1 ? 2 : 1;       // bf16 between rows of K, of [..][NS] matrices
    static constexpr int PK = C * LK, PM = DKP * LS, PR = C * LS;                      // bf16 of one plane
    static constexpr int BYTES = T_BYTES + 2 * (KB * Pl<T>::in * PK + 3 * PM + 6 * PR);
};
struct GateRow { float4 g; float theta; };
// A sequence: its first token in its batch, its length.
struct Seq { int b, t0, len; };
__device__ __forceinline__ Seq get_seq(const Args& A, int seq)
{
    if (!A.starts) return Seq{seq, 0, A.seq};
    const int t0 = A.start[seq];
    return Seq{0, t0, A.start[seq + 1] - t0};
}

template <typename T, int DKP, int NS>
__global__ void __launch_bounds__(256, DKP == 64 ? 2 : 1) gd_state_fwd_kernel(Args A)
{
    typedef StateSmem<T, DKP, NS> L;
    constexpr int LK = L::LK, LS = L::LS, MT = DKP / 64, NT = NS / 16, H = NS / 2, IN = Pl<T>::in;
    extern __shared__ float4 smem4[];
    bf* Ts = reinterpret_cast<bf*>(smem4);              // [64][LP], three planes
    bf* Kb = Ts + T_BYTES / 2;                          // [KB] [64][LK]
    bf* Ms = Kb + L::KB * IN * L::PK;                   // [DKP][LS]
    bf *Rs = Ms + 3 * L::PM, *Us = Rs + 3 * L::PR;      // [64][LS]
    __shared__ float4 s_gate[2][C];
    __shared__ float s_w[2][C];
    __shared__ __align__(8) unsigned long long s_bar;
    __shared__ int s_dead;
    const int nsl = A.dvp / NS, sl = blockIdx.x % nsl, p = blockIdx.x / nsl, h = p % A.hv, seq = A.starts ? A.order[p / A.hv] : p / A.hv;
    const int n0 = sl * NS, tid = threadIdx.x, lane = tid & 31, w = tid >> 5, rb = w & 3, hf = w >> 2, g = lane >> 2, t = lane & 3;
    const int slot0 = first_slot(A, seq), count = chunk_count(A, seq);

    float S[MT][NT][4];
    const float* m0 = A.m0 ? A.m0 + ((long long)seq * A.hv + h) * A.dv * A.dk : nullptr;
    auto put_state = [&](int m) {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int r = 0; r < 2; r++)
                put2<3>(Ms + (64 * m + 16 * rb + g + 8 * r) * LS + H * hf + 8 * n + 2 * t, L::PM, S[m][n][2 * r], S[m][n][2 * r + 1]);
    };
#pragma unroll
    for (int m = 0; m < MT; m++) {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int row = 64 * m + 16 * rb + g + 8 * (i >> 1), col = n0 + H * hf + 8 * n + 2 * t + (i & 1);   // dk, dv
                S[m][n][i] = m0 && row < A.dk && col < A.dv ? m0[(long long)col * A.dk + row] : 0.f;
            }
        put_state(m);
    }
    Prefetch<T, DKP, 256> pk;
    GateRow pg;
    Pair<T> pv[NT][2];
    const bool vpair = ((reinterpret_cast<uintptr_t>((const T*)A.v + n0) | (uintptr_t)((A.vb | A.vt | A.vh) * (long long)sizeof(T))) &
                        (2 * sizeof(T) - 1)) == 0 && (A.dv & 1) == 0;
    const Seq sq = get_seq(A, seq);
    const long long tile0 = (long long)slot0 * A.hv + h, tok0 = sq.b * A.vb + sq.t0 * A.vt;
    const int row0 = 16 * rb + g, col0 = H * hf + 2 * t;
    const T* vp0 = (const T*)A.v + tok0 + h * A.vh + n0 + row0 * A.vt + col0;
    const float4* gp0 = A.gates + tile0 * C + tid;
    const float* tp0 = A.theta_eff + tile0 * C + tid;
    float* mc = A.m_chunk + (tile0 * DKP + row0) * A.dvp + n0 + col0;
    float* ep = A.e + (tile0 * C + row0) * A.dvp + n0 + col0;
    const long long v_step = C * A.vt, g_step = (long long)A.hv * C, m_step = (long long)A.hv * DKP * A.dvp, e_step = g_step * A.dvp;
    pk.init((const T*)A.k + sq.b * A.kb + sq.t0 * A.kt + (h / A.share) * A.kh, A.kt, A.dk);
    auto fetch = [&](int c) {
        const int len = min(C, sq.len - c * C);
        pk.load(c, len);
        if (tid < C) { ldg(pg.g, reinterpret_cast<const float*>(gp0 + c * g_step)); ldg(pg.theta, tp0 + c * g_step); }
        const T* vp = vp0 + c * v_step;
#pragma unroll
        for (int r = 0; r < 2; r++) {
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const int col = n0 + col0 + 8 * n;
                pv[n][r].load(vp + 8 * n, row0 + 8 * r < len && col < A.dv, row0 + 8 * r < len && col + 1 < A.dv, vpair);
            }
            vp += 8 * A.vt;
        }
    };
    auto commit = [&](int buf) {
        if (L::KB == 1) __syncthreads();              // the one buffer of K has been read
        pk.store(Kb + (L::KB == 1 ? 0 : buf) * IN * L::PK, LK, L::PK);
        if (tid < C) { s_gate[buf][tid] = pg.g; s_w[buf][tid] = pg.g.w * pg.theta; }
    };
    if (tid == 0) {
        s_dead = 0;
        init_t(&s_bar);
        if (count > 0) copy_t(Ts, A.tmat + tile0 * T_BYTES, &s_bar);
    }
    if (count > 0) { fetch(0); commit(0); }
    __syncthreads();
    for (int c = 0; c < count; c++) {
        const int buf = c & 1;
        const bf* Ks = Kb + (L::KB == 1 ? 0 : buf) * IN * L::PK;
        Pair<T> v[NT][2];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int r = 0; r < 2; r++) {
                v[n][r] = pv[n][r];
#pragma unroll
                for (int m = 0; m < MT; m++) st2(mc + (64 * m + 8 * r) * A.dvp + 8 * n, S[m][n][2 * r], S[m][n][2 * r + 1]);
            }
        mc += m_step;
        if (c + 1 < count) fetch(c + 1);
        float acc[NT][4];
        zero(acc);
        gemm<NT, false, true, IN, 3>(acc, Ks + 16 * rb * LK, LK, L::PK, Ms + H * hf, LS, L::PM, 0, DKP);
        bool any = false;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const int row = 16 * rb + g + 8 * r;
                float2 x = v[n][r].get();
                x.x -= s_gate[buf][row].z * acc[n][2 * r];
                x.y -= s_gate[buf][row].z * acc[n][2 * r + 1];
                any |= odd(x.x) | odd(x.y);
                put2<3>(Rs + row * LS + H * hf + 8 * n + 2 * t, L::PR, x.x, x.y);
            }
        any |= not_arrived(&s_dead, &s_bar, buf, A.wait_cycles);
        any = __syncthreads_or(any);
        zero(acc);
        if (any) {
            if (lost_t(&s_dead, &s_bar, buf)) fill_nan(acc);
            else triangle_by_token<3, NT>(acc, Ts, C * LP, Rs, LS, L::PR, 16 * rb, H * hf);
        }
        else gemm<NT, false, true, 3, 3>(acc, Ts + 16 * rb * LP, LP, C * LP, Rs + H * hf, LS, L::PR, 0, 16 * (rb + 1));
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const int row = row0 + 8 * r, col = col0 + 8 * n;
                const float a = acc[n][2 * r], b = acc[n][2 * r + 1], wt = s_w[buf][row];
                st2(ep + 8 * r * A.dvp + 8 * n, a, b);
                put2<3>(Us + row * LS + col, L::PR, wt * a, wt * b);
            }
        __syncthreads();
        ep += e_step;
        if (tid == 0 && c + 1 < count && s_dead == 0) copy_t(Ts, A.tmat + (tile0 + (long long)(c + 1) * A.hv) * T_BYTES, &s_bar);
        const float gl = s_gate[buf][C - 1].z;
#pragma unroll
        for (int m = 0; m < MT; m++) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int i = 0; i < 4; i++) S[m][n][i] *= gl;
            gemm<NT, true, true, IN, 3>(S[m], Ks + 64 * m + 16 * rb, LK, L::PK, Us + H * hf, LS, L::PR, 0, C);
            put_state(m);
        }
        if (c + 1 < count) commit(buf ^ 1);
        __syncthreads();
    }
    float* mf = A.m_final + ((long long)seq * A.hv + h) * A.dv * A.dk;
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int row = 64 * m + 16 * rb + g + 8 * (i >> 1), col = n0 + H * hf + 8 * n + 2 * t + (i & 1);
                if (row < A.dk && col < A.dv) mf[(long long)col * A.dk + row] = S[m][n][i];
            }
}

// Row-major store of a 16 x 32 accumulator block into a contiguous [row, heads, d] output.
template <typename T>
__device__ __forceinline__ void store_rows(T* out, const float (&acc)[4][4], int r0, int rows, int c0, int d, long long row_stride)
{
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const bool pair = ((d | (int)(row_stride & 1)) & 1) == 0 && (reinterpret_cast<uintptr_t>(out) & (2 * sizeof(T) - 1)) == 0;
#pragma unroll
    for (int n = 0; n < 4; n++)
#pragma unroll
        for (int r = 0; r < 2; r++) {
            const int i = r0 + g + 8 * r, col = c0 + 8 * n + 2 * t;
            if (i >= rows) continue;
            T* p = out + i * row_stride + col;
            if (pair) {
                if (col < d) st2(p, acc[n][2 * r], acc[n][2 * r + 1]);
            } else {
                if (col < d) p[0] = from_f<T>(acc[n][2 * r]);
                if (col + 1 < d) p[1] = from_f<T>(acc[n][2 * r + 1]);
            }
        }
}

// ── forward outputs ──
// Four warps: warp = 32 tokens x 32 of the tile's 64 columns. Two places in shared memory, Q then P, and K, then S, then U: four
// CTAs share an SM and cover each other's loads. 4096 tiles fp32: 143 us; eight warps of 16 x 32, which read a third more from shared memory, 152; those with three places and two
// CTAs 166, with three CTAs and the next tile on its way in registers 174.
constexpr int OUT_FWD_BYTES = 2 * 3 * C * LP * 2;
template <typename T>
__global__ void __launch_bounds__(128, 4) gd_out_fwd_kernel(Args A)
{
    constexpr int PS = C * LP, IN = Pl<T>::in;
    extern __shared__ float4 smem4[];
    bf* Qs = reinterpret_cast<bf*>(smem4);
    bf* Ks = Qs + 3 * PS;
    __shared__ float4 s_gate[C];
    __shared__ float s_theta[C];
    const int slot = blockIdx.x / A.hv, h = blockIdx.x - slot * A.hv, n0 = blockIdx.y * 64;
    const Chunk ch = get_chunk(A, slot);
    if (ch.len <= 0) return;
    const long long tile = (long long)slot * A.hv + h;
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, rb = w & 1, hf = w >> 1, g = lane >> 2, t = lane & 3;
    if (tid < C) { s_gate[tid] = A.gates[tile * C + tid]; s_theta[tid] = A.theta_eff[tile * C + tid]; }
    const T* kp = (const T*)A.k + ch.b * A.kb + ch.t0 * A.kt + (h / A.share) * A.kh;
    const T* qp = (const T*)A.q + ch.b * A.qb + ch.t0 * A.qt + (h / A.share) * A.qh;
    float att[2][4][4], y[2][4][4];
    zero(att[0]); zero(att[1]);
    zero(y[0]); zero(y[1]);
    const bool need = hf <= rb;
    for (int c0 = 0; c0 < A.dk; c0 += 64) {
        if (c0) __syncthreads();
        load_tile<T, 64, 128>(Qs, LP, PS, qp + c0, A.qt, ch.len, A.dk - c0);
        load_tile<T, 64, 128>(Ks, LP, PS, kp + c0, A.kt, ch.len, A.dk - c0);
        __syncthreads();
        if (need) gemm_2<4, false, false, IN, IN>(att, Qs + 32 * rb * LP, LP, PS, Ks + 32 * hf * LP, LP, PS, 0, 64);
        __syncthreads();
        load_own<3, 128>(Ks, A.m_chunk + (tile * A.dkp + c0) * A.dvp + n0, A.dvp);
        __syncthreads();
        gemm_2<4, false, true, IN, 3>(y, Qs + 32 * rb * LP, LP, PS, Ks + 32 * hf, LP, PS, 0, 64);
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < 4; n++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int i = 32 * rb + g + 8 * r, j = 32 * hf + 8 * n + 2 * t, m = r >> 1, o = 2 * (r & 1);
            const float4 gi = s_gate[i];
            float x[2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float4 gj = s_gate[j + e];
                x[e] = j + e <= i ? decay(make_float2(gi.x, gi.y), make_float2(gj.x, gj.y)) * A.scale * att[m][n][o + e] : 0.f;
                y[m][n][o + e] *= A.scale * gi.z;
            }
            put2<3>(Qs + i * LP + j, PS, x[0], x[1]);
        }
    const bool any = load_own<3, 128>(Ks, A.e + tile * C * A.dvp + n0, A.dvp, s_theta);
    if (__syncthreads_or(any)) {
        triangle_by_token<3, 4>(y[0], Qs, PS, Ks, LP, PS, 32 * rb, 32 * hf);
        triangle_by_token<3, 4>(y[1], Qs, PS, Ks, LP, PS, 32 * rb + 16, 32 * hf);
    } else gemm_2<4, false, true, 3, 3>(y, Qs + 32 * rb * LP, LP, PS, Ks + 32 * hf, LP, PS, 0, 32 * (rb + 1));
    T* out = (T*)A.y + (ch.row0(A) * A.hv + h) * A.dv;
    store_rows<T>(out, y[0], 32 * rb, ch.len, n0 + 32 * hf, A.dv, (long long)A.hv * A.dv);
    store_rows<T>(out, y[1], 32 * rb + 16, ch.len, n0 + 32 * hf, A.dv, (long long)A.hv * A.dv);
}

// ── backward, what needs no state gradient: F = P^T dY, and N = scale (e^G Q)^T dY into the place of D ──
// Two places in shared memory, Q then P^T, and K, then scale e^G dY, then dY: four CTAs share an SM.
constexpr int PRE_BWD_BYTES = 2 * 3 * C * LP * 2;
template <typename T>
__global__ void __launch_bounds__(256, 4) gd_pre_bwd_kernel(Args A)
{
    constexpr int PS = C * LP, IN = Pl<T>::in;
    extern __shared__ float4 smem4[];
    bf* Qs = reinterpret_cast<bf*>(smem4);
    bf* Ks = Qs + 3 * PS;
    __shared__ float4 s_gate[C];
    const int slot = blockIdx.x / A.hv, h = blockIdx.x - slot * A.hv, n0 = blockIdx.y * 64;
    const Chunk ch = get_chunk(A, slot);
    if (ch.len <= 0) return;
    const long long tile = (long long)slot * A.hv + h;
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, rb = w & 3, hf = w >> 2, g = lane >> 2, t = lane & 3;
    if (tid < C) s_gate[tid] = A.gates[tile * C + tid];
    const T* kp = (const T*)A.k + ch.b * A.kb + ch.t0 * A.kt + (h / A.share) * A.kh;
    const T* qp = (const T*)A.q + ch.b * A.qb + ch.t0 * A.qt + (h / A.share) * A.qh;
    const T* yp = (const T*)A.dy + ch.b * A.yb + ch.t0 * A.yt + h * A.yh + n0;
    float att[4][4];                              // rows: j, columns: i >= j
    zero(att);
    const bool need = 32 * hf + 31 >= 16 * rb;
    for (int c0 = 0; c0 < A.dk; c0 += 64) {
        if (c0) __syncthreads();
        load_tile<T, 64, 256>(Qs, LP, PS, qp + c0, A.qt, ch.len, A.dk - c0);
        load_tile<T, 64, 256>(Ks, LP, PS, kp + c0, A.kt, ch.len, A.dk - c0);
        __syncthreads();
        if (need) gemm<4, false, false, IN, IN>(att, Ks + 16 * rb * LP, LP, PS, Qs + 32 * hf * LP, LP, PS, 0, 64);
        __syncthreads();
        load_scaled<T, 256>(Ks, yp, A.yt, ch.len, A.dv - n0, A.scale, s_gate);
        __syncthreads();
        float nn[4][4];                           // rows: dk, columns: dv
        zero(nn);
        gemm<4, true, true, IN, 3>(nn, Qs + 16 * rb, LP, PS, Ks + 32 * hf, LP, PS, 0, C);
        float* np = A.d_chunk + (tile * A.dkp + c0) * A.dvp + n0 + 32 * hf;
#pragma unroll
        for (int n = 0; n < 4; n++)
#pragma unroll
            for (int r = 0; r < 2; r++)
                st2(np + (16 * rb + g + 8 * r) * A.dvp + 8 * n + 2 * t, nn[n][2 * r], nn[n][2 * r + 1]);
    }
    __syncthreads();
    load_tile<T, 64, 256>(Ks, LP, PS, yp, A.yt, ch.len, A.dv - n0);
    bf* Pt = Qs;                                  // [j][i]
#pragma unroll
    for (int n = 0; n < 4; n++)
#pragma unroll
        for (int r = 0; r < 2; r++) {
            const int j = 16 * rb + g + 8 * r, i = 32 * hf + 8 * n + 2 * t;
            const float4 gj = s_gate[j];
            float x[2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float4 gi = s_gate[i + e];
                x[e] = j <= i + e ? decay(make_float2(gi.x, gi.y), make_float2(gj.x, gj.y)) * A.scale * att[n][2 * r + e] : 0.f;
            }
            put2<3>(Pt + j * LP + i, PS, x[0], x[1]);
        }
    __syncthreads();
    float f[4][4];
    zero(f);
    gemm<4, false, true, 3, IN>(f, Pt + 16 * rb * LP, LP, PS, Ks + 32 * hf, LP, PS, 16 * rb, C);
    float* fp = A.f + tile * C * A.dvp + n0 + 32 * hf;
#pragma unroll
    for (int n = 0; n < 4; n++)
#pragma unroll
        for (int r = 0; r < 2; r++)
            st2(fp + (long long)(16 * rb + g + 8 * r) * A.dvp + 8 * n + 2 * t, f[n][2 * r], f[n][2 * r + 1]);
}

// ── backward states: the gradient D of the state behind each chunk, last chunk first ──
//   F = P^T dY + e^{G_L - G} K D,  X = T^T (theta F),  D <- e^{G_L} D + N - (e^G K)^T X,  N = scale (e^G Q)^T dY.
// The forward kernel's structure. N is in D's place in d_chunk when a chunk is reached, and is read a chunk ahead.
template <typename T, int DKP, int NS>
__global__ void __launch_bounds__(256, DKP == 64 ? 2 : 1) gd_state_bwd_kernel(Args A)
{
    typedef StateSmem<T, DKP, NS> L;
    constexpr int LK = L::LK, LS = L::LS, MT = DKP / 64, NT = NS / 16, H = NS / 2, IN = Pl<T>::in;
    extern __shared__ float4 smem4[];
    bf* Ts = reinterpret_cast<bf*>(smem4);
    bf* Kb = Ts + T_BYTES / 2;
    bf* Ds = Kb + L::KB * IN * L::PK;
    bf *Rs = Ds + 3 * L::PM, *Us = Rs + 3 * L::PR;
    __shared__ float4 s_gate[2][C];
    __shared__ float s_theta[2][C];
    __shared__ __align__(8) unsigned long long s_bar;
    __shared__ int s_dead;
    const int nsl = A.dvp / NS, sl = blockIdx.x % nsl, p = blockIdx.x / nsl, h = p % A.hv, seq = A.starts ? A.order[p / A.hv] : p / A.hv;
    const int n0 = sl * NS, tid = threadIdx.x, lane = tid & 31, w = tid >> 5, rb = w & 3, hf = w >> 2, g = lane >> 2, t = lane & 3;
    const int slot0 = first_slot(A, seq), count = chunk_count(A, seq);

    float S[MT][NT][4];
    const float* dm = A.d_m_final ? A.d_m_final + ((long long)seq * A.hv + h) * A.dv * A.dk : nullptr;
    auto put_state = [&](int m) {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int r = 0; r < 2; r++)
                put2<3>(Ds + (64 * m + 16 * rb + g + 8 * r) * LS + H * hf + 8 * n + 2 * t, L::PM, S[m][n][2 * r], S[m][n][2 * r + 1]);
    };
#pragma unroll
    for (int m = 0; m < MT; m++) {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int row = 64 * m + 16 * rb + g + 8 * (i >> 1), col = n0 + H * hf + 8 * n + 2 * t + (i & 1);
                S[m][n][i] = dm && row < A.dk && col < A.dv ? dm[(long long)col * A.dk + row] : 0.f;
            }
        put_state(m);
    }
    Prefetch<T, DKP, 256> pk;
    GateRow pg;
    float2 pf[NT][2], pn[MT][NT][2];
    const Seq sq = get_seq(A, seq);
    const int row0 = 16 * rb + g, col0 = H * hf + 2 * t;
    const long long dv_row = (long long)A.hv * A.dv, g_step = (long long)A.hv * C, m_step = (long long)A.hv * DKP * A.dvp, e_step = g_step * A.dvp;
    long long tile = (long long)(slot0 + count - 1) * A.hv + h, g_at = tile * C + tid;     // of the chunk that is computed
    long long m_at = (tile * DKP + row0) * A.dvp + n0 + col0, e_at = (tile * C + row0) * A.dvp + n0 + col0;
    T* dv = (T*)A.d_v + ((long long)sq.b * A.seq + sq.t0 + (long long)(count - 1) * C + row0) * dv_row + h * A.dv + n0 + col0;
    pk.init((const T*)A.k + sq.b * A.kb + sq.t0 * A.kt + (h / A.share) * A.kh, A.kt, A.dk);
    auto fetch = [&](int c, long long ga, long long ea, long long ma) {
        pk.load(c, min(C, sq.len - c * C));
        if (tid < C) { ldg(pg.g, reinterpret_cast<const float*>(A.gates + ga)); ldg(pg.theta, A.theta_eff + ga); }
        const float *fp = A.f + ea, *np = A.d_chunk + ma;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int r = 0; r < 2; r++) {
                ldg(pf[n][r], fp + 8 * r * A.dvp + 8 * n);
#pragma unroll
                for (int m = 0; m < MT; m++) ldg(pn[m][n][r], np + (64 * m + 8 * r) * A.dvp + 8 * n);
            }
    };
    auto commit = [&](int buf) {
        if (L::KB == 1) __syncthreads();
        pk.store(Kb + (L::KB == 1 ? 0 : buf) * IN * L::PK, LK, L::PK);
        if (tid < C) { s_gate[buf][tid] = pg.g; s_theta[buf][tid] = pg.theta; }
    };
    if (tid == 0) {
        s_dead = 0;
        init_t(&s_bar);
        if (count > 0) copy_t(Ts, A.tmat + tile * T_BYTES, &s_bar);
    }
    if (count > 0) { fetch(count - 1, g_at, e_at, m_at); commit(0); }
    __syncthreads();
    for (int c = count - 1; c >= 0; c--) {
        const int buf = (count - 1 - c) & 1, len = min(C, sq.len - c * C);
        const bf* Ks = Kb + (L::KB == 1 ? 0 : buf) * IN * L::PK;
        float2 f[NT][2], nn[MT][NT][2];
        float* dc = A.d_chunk + m_at;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int r = 0; r < 2; r++) {
                f[n][r] = pf[n][r];
#pragma unroll
                for (int m = 0; m < MT; m++) {
                    nn[m][n][r] = pn[m][n][r];
                    st2(dc + (64 * m + 8 * r) * A.dvp + 8 * n, S[m][n][2 * r], S[m][n][2 * r + 1]);
                }
            }
        if (c > 0) fetch(c - 1, g_at - g_step, e_at - e_step, m_at - m_step);
        float acc[NT][4];
        zero(acc);
        gemm<NT, false, true, IN, 3>(acc, Ks + 16 * rb * LK, LK, L::PK, Ds + H * hf, LS, L::PM, 0, DKP);
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const int row = 16 * rb + g + 8 * r;
                const float wi = s_gate[buf][row].w, th = s_theta[buf][row];
                put2<3>(Rs + row * LS + H * hf + 8 * n + 2 * t, L::PR, th * (f[n][r].x + wi * acc[n][2 * r]), th * (f[n][r].y + wi * acc[n][2 * r + 1]));
            }
        const bool lost = __syncthreads_or(not_arrived(&s_dead, &s_bar, buf, A.wait_cycles));
        zero(acc);
        if (lost) { lost_t(&s_dead, &s_bar, buf); fill_nan(acc); }
        else gemm<NT, true, true, 3, 3>(acc, Ts + 16 * rb, LP, C * LP, Rs + H * hf, LS, L::PR, 16 * rb, C);
        float* xp = A.x + e_at;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const int row = row0 + 8 * r, col = col0 + 8 * n;
                const float a = acc[n][2 * r], b = acc[n][2 * r + 1], eg = -s_gate[buf][row].z;
                st2(xp + 8 * r * A.dvp + 8 * n, a, b);
                put2<3>(Us + row * LS + col, L::PR, eg * a, eg * b);
                if (row < len) {
                    const bool none = fabsf(s_theta[buf][row]) <= THETA_TINY;     // theta was 0: so is the gradient of v
                    T* o = dv + 8 * r * dv_row + 8 * n;
                    if (n0 + col < A.dv) o[0] = from_f<T>(none ? 0.f : a);
                    if (n0 + col + 1 < A.dv) o[1] = from_f<T>(none ? 0.f : b);
                }
            }
        __syncthreads();
        tile -= A.hv;
        g_at -= g_step;
        e_at -= e_step;
        m_at -= m_step;
        dv -= C * dv_row;
        if (tid == 0 && c > 0 && s_dead == 0) copy_t(Ts, A.tmat + tile * T_BYTES, &s_bar);
        const float gl = s_gate[buf][C - 1].z;
#pragma unroll
        for (int m = 0; m < MT; m++) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    S[m][n][2 * r] = fmaf(gl, S[m][n][2 * r], nn[m][n][r].x);
                    S[m][n][2 * r + 1] = fmaf(gl, S[m][n][2 * r + 1], nn[m][n][r].y);
                }
            gemm<NT, true, true, IN, 3>(S[m], Ks + 64 * m + 16 * rb, LK, L::PK, Us + H * hf, LS, L::PR, 0, C);
            put_state(m);
        }
        if (c > 0) commit(buf ^ 1);
        __syncthreads();
    }
    if (A.d_m0) {
        float* o = A.d_m0 + ((long long)seq * A.hv + h) * A.dv * A.dk;
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int row = 64 * m + 16 * rb + g + 8 * (i >> 1), col = n0 + H * hf + 8 * n + 2 * t + (i & 1);
                    if (row < A.dk && col < A.dv) o[(long long)col * A.dk + row] = S[m][n][i];
                }
    }
}

// One warp: the gradient of log_retain of a chunk's tokens 2 lane, 2 lane + 1. Token t's retention is a factor of just those terms in which
// something from before t meets something from t on: pairs of tokens (r: their sums), the state in front of the chunk with the queries
// from t on (a), keys before t with the state behind the chunk (b), and the two states (through). Every sum is of such terms
// alone. (Sums of the gradient of G over the tokens from t on are the same number, but between terms of full size that
// cancel: at a retention of 1e-4 they left the gradient of the retention 2e-3 off, at 1e-6 by a fifth. A step of
// 64 x 8 x 512 tokens in fp32 took 1136 us with them, against 1195.)
__device__ __forceinline__ float2 gate_gradient(float2 r, float2 a, float2 b, float through)
{
    const int lane = threadIdx.x & 31;
    float sa = a.x + a.y, sb = b.x + b.y;
    for (int o = 1; o < 32; o <<= 1) {
        const float x = __shfl_down_sync(0xffffffffu, sa, o), y = __shfl_up_sync(0xffffffffu, sb, o);
        if (lane + o < 32) sa += x;
        if (lane >= o) sb += y;
    }
    float behind = __shfl_down_sync(0xffffffffu, sa, 1), before = __shfl_up_sync(0xffffffffu, sb, 1);
    if (lane == 31) behind = 0.f;
    if (lane == 0) before = 0.f;
    behind += a.y;
    return make_float2(r.x + (behind + a.x) + before + through, r.y + behind + (before + b.x) + through);
}
__device__ __forceinline__ void store_gate(const Args& A, const Chunk& ch, int h, float2 v)
{
    const int i = 2 * (threadIdx.x & 31);
    float* out = A.d_g + (ch.row0(A) + i) * A.hv + h;
    if (i < ch.len) out[0] = v.x;
    if (i + 1 < ch.len) out[A.hv] = v.y;
}

// ── backward outputs: d_q, d_k, d_theta and the gradient of G, for 64 columns of dk ──
//   Mq_ij = scale e^{G_i - G_j} (dy_i.e_j) theta_j (j <= i),  Mb_ij = -e^{G_i - G_j} (x_i.e_j) theta_j (j < i)
//   d_q = scale e^G dY M_0 + Mq K;  k as a query: -e^G X M_0 + Mb K;  k as a key: theta e^{G_L - G} E D + Mq^T Q + Mb^T K
//   log_retain_t: sum over i >= t > j of W_ij = Mq_ij q_i.k_j + Mb_ij k_i.k_j, and the parts with the states: see gate_gradient.
// Four tiles at a time in shared memory: dY, X, E with M_0, then with D; Mq, Mb, Q, K take their places. Two CTAs per SM.
template <typename T> struct OutBwdSmem {
    static constexpr int PS = C * LP, IN = Pl<T>::in, BYTES = 2 * PS * (IN + 9);
};
template <typename T>
__global__ void __launch_bounds__(256, 2) gd_out_bwd_kernel(Args A)
{
    typedef OutBwdSmem<T> L;
    constexpr int PS = L::PS, IN = L::IN;
    extern __shared__ float4 smem4[];
    bf* Ys = reinterpret_cast<bf*>(smem4);
    bf *Xs = Ys + IN * PS, *Es = Xs + 3 * PS, *Ms = Es + 3 * PS;
    __shared__ float4 s_gate[C];
    __shared__ float s_theta[C], s_a[2][C], s_b[2][C], s_r[8][C], s_red[8];
    const int slot = blockIdx.x / A.hv, h = blockIdx.x - slot * A.hv, kt = blockIdx.y, k0 = kt * 64;
    const Chunk ch = get_chunk(A, slot);
    if (ch.len <= 0) return;
    const long long tile = (long long)slot * A.hv + h;
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, rb = w & 3, hf = w >> 2, g = lane >> 2, t = lane & 3;
    if (tid < C) { s_gate[tid] = A.gates[tile * C + tid]; s_theta[tid] = A.theta_eff[tile * C + tid]; }
    const T* yp = (const T*)A.dy + ch.b * A.yb + ch.t0 * A.yt + h * A.yh;
    const bool need = 32 * hf <= 16 * rb + 15;
    float dp[4][4], xe[4][4], dq[4][4], kq[4][4], ks[4][4], xdot = 0.f, gsum = 0.f;
    zero(dp);
    zero(xe);
    zero(dq);
    zero(kq);
    zero(ks);
    for (int n = 0; n < A.dvp; n += 64) {
        if (n) __syncthreads();
        load_tile<T, 64, 256>(Ys, LP, PS, yp + n, A.yt, ch.len, A.dv - n);
        const long long at = (tile * A.dkp + k0) * A.dvp + n;
        load_own<3, 256>(Ms, A.m_chunk + at, A.dvp);
        const float *xg = A.x + tile * C * A.dvp + n, *eg = A.e + tile * C * A.dvp + n;
#pragma unroll
        for (int i = 0; i < 4; i++) {             // X and E; the gradient of theta is x.e / theta
            const int r = (tid + i * 256) >> 4, c = (tid & 15) * 4;
            const float4 x = *reinterpret_cast<const float4*>(xg + (long long)r * A.dvp + c);
            const float4 e = *reinterpret_cast<const float4*>(eg + (long long)r * A.dvp + c);
            put4<3>(Xs + r * LP + c, PS, x);
            put4<3>(Es + r * LP + c, PS, e);
            float s = x.x * e.x + x.y * e.y + x.z * e.z + x.w * e.w;      // 16 lanes hold a row
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            if ((tid & 15) == i) xdot += s;       // lane i keeps row (tid + 256 i) / 16
        }
        __syncthreads();
        if (need) {
            gemm<4, false, false, IN, 3>(dp, Ys + 16 * rb * LP, LP, PS, Es + 32 * hf * LP, LP, PS, 0, 64);
            gemm<4, false, false, 3, 3>(xe, Xs + 16 * rb * LP, LP, PS, Es + 32 * hf * LP, LP, PS, 0, 64);
        }
        gemm<4, false, false, IN, 3>(dq, Ys + 16 * rb * LP, LP, PS, Ms + 32 * hf * LP, LP, PS, 0, 64);
        gemm<4, false, false, 3, 3>(kq, Xs + 16 * rb * LP, LP, PS, Ms + 32 * hf * LP, LP, PS, 0, 64);
        __syncthreads();
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = (tid + i * 256) >> 4, c = (tid & 15) * 4;
            const long long o = at + (long long)r * A.dvp + c;
            const float4 v = *reinterpret_cast<const float4*>(A.d_chunk + o), m = *reinterpret_cast<const float4*>(A.m_chunk + o);
            s += v.x * m.x + v.y * m.y + v.z * m.z + v.w * m.w;
            put4<3>(Ms + r * LP + c, PS, v);
        }
        gsum = fmaf(s_gate[C - 1].z, s, gsum);
        __syncthreads();
        gemm<4, false, false, 3, 3>(ks, Es + 16 * rb * LP, LP, PS, Ms + 32 * hf * LP, LP, PS, 0, 64);
    }
    if (kt == 0 && (tid & 15) < 4) {
        const int r = (tid + (tid & 15) * 256) >> 4;
        if (r < ch.len) A.d_theta[(ch.row0(A) + r) * A.hv + h] = xdot / s_theta[r];
    }
    __syncthreads();
    bf *Mq = Xs, *Mb = Es, *Qs = Ys, *Ks = Ms;
    load_tile<T, 64, 256>(Qs, LP, PS, (const T*)A.q + ch.b * A.qb + ch.t0 * A.qt + (h / A.share) * A.qh + k0, A.qt, ch.len, A.dk - k0);
    load_tile<T, 64, 256>(Ks, LP, PS, (const T*)A.k + ch.b * A.kb + ch.t0 * A.kt + (h / A.share) * A.kh + k0, A.kt, ch.len, A.dk - k0);
#pragma unroll
    for (int n = 0; n < 4; n++)
#pragma unroll
        for (int r = 0; r < 2; r++) {
            const int i = 16 * rb + g + 8 * r, j = 32 * hf + 8 * n + 2 * t;
            const float4 gi = s_gate[i];
            float a[2], b[2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float4 gj = s_gate[j + e];
                const float d = j + e <= i ? decay(make_float2(gi.x, gi.y), make_float2(gj.x, gj.y)) * s_theta[j + e] : 0.f;
                a[e] = j + e <= i ? A.scale * d * dp[n][2 * r + e] : 0.f;
                b[e] = j + e < i ? -d * xe[n][2 * r + e] : 0.f;
            }
            put2<3>(Mq + i * LP + j, PS, a[0], a[1]);
            put2<3>(Mb + i * LP + j, PS, b[0], b[1]);
        }
    __syncthreads();
    float ra[2] = {0.f, 0.f}, rk[2] = {0.f, 0.f};
#pragma unroll
    for (int n = 0; n < 4; n++)
#pragma unroll
        for (int r = 0; r < 2; r++) {
            const int i = 16 * rb + g + 8 * r, col = 32 * hf + 8 * n + 2 * t;
            const float2 q2 = get2<IN>(Qs + i * LP + col, PS), k2 = get2<IN>(Ks + i * LP + col, PS);
            const float eg = s_gate[i].z, wt = s_theta[i] * s_gate[i].w;
#pragma unroll
            for (int e = 0; e < 2; e++) {
                dq[n][2 * r + e] *= A.scale * eg;
                kq[n][2 * r + e] *= -eg;
                ks[n][2 * r + e] *= wt;
            }
            ra[r] += q2.x * dq[n][2 * r] + q2.y * dq[n][2 * r + 1] + k2.x * kq[n][2 * r] + k2.y * kq[n][2 * r + 1];
            rk[r] += k2.x * ks[n][2 * r] + k2.y * ks[n][2 * r + 1];
        }
#pragma unroll
    for (int r = 0; r < 2; r++) {
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            ra[r] += __shfl_xor_sync(0xffffffffu, ra[r], o);
            rk[r] += __shfl_xor_sync(0xffffffffu, rk[r], o);
        }
        if (t == 0) { s_a[hf][16 * rb + g + 8 * r] = ra[r]; s_b[hf][16 * rb + g + 8 * r] = rk[r]; }
    }
    gemm<4, false, true, 3, IN>(dq, Mq + 16 * rb * LP, LP, PS, Ks + 32 * hf, LP, PS, 0, 16 * (rb + 1));
    gemm<4, false, true, 3, IN>(kq, Mb + 16 * rb * LP, LP, PS, Ks + 32 * hf, LP, PS, 0, 16 * (rb + 1));
    gemm<4, true, true, 3, IN>(ks, Mq + 16 * rb, LP, PS, Qs + 32 * hf, LP, PS, 16 * rb, C);
    gemm<4, true, true, 3, IN>(ks, Mb + 16 * rb, LP, PS, Ks + 32 * hf, LP, PS, 16 * rb, C);
#pragma unroll
    for (int n = 0; n < 4; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) kq[n][i] += ks[n][i];
    if (A.share == 1) {
        const long long at = (ch.row0(A) * A.hk + h) * A.dk, st = (long long)A.hk * A.dk;
        store_rows<T>((T*)A.d_q + at, dq, 16 * rb, ch.len, k0 + 32 * hf, A.dk, st);
        store_rows<T>((T*)A.d_k + at, kq, 16 * rb, ch.len, k0 + 32 * hf, A.dk, st);
    } else {
        const long long at = (ch.row0(A) * A.hv + h) * A.dk, st = (long long)A.hv * A.dk;
        store_rows<float>(A.dq_part + at, dq, 16 * rb, ch.len, k0 + 32 * hf, A.dk, st);
        store_rows<float>(A.dk_part + at, kq, 16 * rb, ch.len, k0 + 32 * hf, A.dk, st);
    }
    // W, strictly lower
    zero(dp);
    zero(xe);
    if (need) {
        gemm<4, false, false, IN, IN>(dp, Qs + 16 * rb * LP, LP, PS, Ks + 32 * hf * LP, LP, PS, 0, 64);
        gemm<4, false, false, IN, IN>(xe, Ks + 16 * rb * LP, LP, PS, Ks + 32 * hf * LP, LP, PS, 0, 64);
    }
#pragma unroll
    for (int n = 0; n < 4; n++)
#pragma unroll
        for (int r = 0; r < 2; r++) {
            const int i = 16 * rb + g + 8 * r, j = 32 * hf + 8 * n + 2 * t;
            const float2 a = get2<3>(Mq + i * LP + j, PS), b = get2<3>(Mb + i * LP + j, PS);
            dp[n][2 * r] = j < i ? a.x * dp[n][2 * r] + b.x * xe[n][2 * r] : 0.f;
            dp[n][2 * r + 1] = j + 1 < i ? a.y * dp[n][2 * r + 1] + b.y * xe[n][2 * r + 1] : 0.f;
        }
    gsum = warp_sum(gsum);
    if (lane == 0) s_red[w] = gsum;
    __syncthreads();
    constexpr int LW = C + 1;
    float* W = reinterpret_cast<float*>(Mq);      // takes the place of Mq
#pragma unroll
    for (int n = 0; n < 4; n++)
#pragma unroll
        for (int r = 0; r < 2; r++) {
            float* p = W + (16 * rb + g + 8 * r) * LW + 32 * hf + 8 * n + 2 * t;
            p[0] = dp[n][2 * r];
            p[1] = dp[n][2 * r + 1];
        }
    __syncthreads();
    float r0 = 0.f, r1 = 0.f;                     // warp = eight of W's columns: sums from each row down, where the row is below the diagonal
#pragma unroll
    for (int c = 0; c < 8; c++) {
        const int j = 8 * w + c;
        const float a = W[2 * lane * LW + j], b = W[(2 * lane + 1) * LW + j];
        float s = a + b;
        for (int o = 1; o < 32; o <<= 1) { const float y = __shfl_down_sync(0xffffffffu, s, o); if (lane + o < 32) s += y; }
        s = __shfl_down_sync(0xffffffffu, s, 1);
        s = lane == 31 ? b : b + s;
        if (j < 2 * lane) r0 += a + s;
        if (j < 2 * lane + 1) r1 += s;
    }
    s_r[w][2 * lane] = r0;
    s_r[w][2 * lane + 1] = r1;
    __syncthreads();
    if (w != 0) return;
    float through = 0.f;
    r0 = r1 = 0.f;
    for (int i = 0; i < 8; i++) { through += s_red[i]; r0 += s_r[i][2 * lane]; r1 += s_r[i][2 * lane + 1]; }
    const float2 v = gate_gradient(make_float2(r0, r1), make_float2(s_a[0][2 * lane] + s_a[1][2 * lane], s_a[0][2 * lane + 1] + s_a[1][2 * lane + 1]),
                                   make_float2(s_b[0][2 * lane] + s_b[1][2 * lane], s_b[0][2 * lane + 1] + s_b[1][2 * lane + 1]), through);
    if (gridDim.y == 1) store_gate(A, ch, h, v);
    else *reinterpret_cast<float2*>(A.dg_part + ((long long)kt * A.slots * A.hv + tile) * C + 2 * lane) = v;
}

// Where dk takes two CTAs of the kernel above: the sum of their parts of the gradient of log_retain. One warp per chunk and head.
__global__ void __launch_bounds__(128) gd_gate_bwd_kernel(Args A)
{
    const long long tile = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (tile >= (long long)A.slots * A.hv) return;
    const int slot = (int)(tile / A.hv), h = (int)(tile - (long long)slot * A.hv), lane = threadIdx.x & 31;
    const Chunk ch = get_chunk(A, slot);
    if (ch.len <= 0) return;
    float2 v = make_float2(0.f, 0.f);
    for (int kt = 0; kt < A.dkp / 64; kt++) {
        const float2 x = *reinterpret_cast<const float2*>(A.dg_part + ((long long)kt * A.slots * A.hv + tile) * C + 2 * lane);
        v.x += x.x;
        v.y += x.y;
    }
    store_gate(A, ch, h, v);
}

// Gradients of shared keys and queries: the value heads of a group, added in their order. Rows outside the sequences of a packed
// batch have no sums and are left as they are.
template <typename T>
__global__ void __launch_bounds__(256) gd_group_kernel(Args A, long long n)
{
    const long long per_row = (long long)A.hk * A.dk;
    const long long i0 = A.starts ? A.start[0] * per_row : 0, i1 = A.starts ? A.start[A.n_seqs] * per_row : n;
    for (long long i = i0 + (long long)blockIdx.x * 256 + threadIdx.x; i < i1; i += (long long)gridDim.x * 256) {
        const long long rh = i / A.dk;                    // row * hk + key head
        const int c = (int)(i - rh * A.dk);
        const long long at = rh * A.share * A.dk + c;
        float q = 0.f, k = 0.f;
        for (int s = 0; s < A.share; s++) { q += A.dq_part[at + (long long)s * A.dk]; k += A.dk_part[at + (long long)s * A.dk]; }
        ((T*)A.d_q)[i] = from_f<T>(q);
        ((T*)A.d_k)[i] = from_f<T>(k);
    }
}

// ── recurrent step ──
// Bound by the state: read once, written once. Eight lanes hold a row of M (dk / 8 numbers each, in groups of four so
// that a row's 128-byte pieces are whole), a thread RP rows at a time; a CTA holds `rows` rows of one head. Small CTAs, so that
// some of an SM's load while others store: 256 x 16 states of 128 x 128 take 99 us (5.4 TB/s) with 64 rows a CTA and three
// CTAs per SM, 128 us with two, 180 us with 128 rows and two.
// Sequences that name the same slot are stepped one after the other, in their order, by the CTA of the first: a slot behaves
// as if they came in as further tokens.
template <typename T, int NV, bool VEC>
__global__ void __launch_bounds__(256, 3) gd_step_kernel(Args A, float* M, const int* slots, int pool, int rows)
{
    constexpr int RP = 8 / NV;
    const int per = (A.dv + rows - 1) / rows;
    const int part = blockIdx.x % per, p = blockIdx.x / per, h = p % A.hv, first = p / A.hv;
    const int lane8 = threadIdx.x & 7, grp = threadIdx.x >> 3, end = min(A.dv, (part + 1) * rows);
    const int slot = slots ? slots[first] : first;
    if (slot < 0 || slot >= pool) {                       // no sequence in this place
        for (long long i = threadIdx.x; i < (long long)A.seq * rows; i += 256) {
            const long long tok = i / rows;
            const int row = part * rows + (int)(i - tok * rows);
            if (row < A.dv) ((T*)A.y)[(((long long)first * A.seq + tok) * A.hv + h) * A.dv + row] = from_f<T>(0.f);
        }
        return;
    }
    int last = first + 1;                                 // sequences first .. last - 1 may be of this slot
    bool looked = slots == nullptr;
    for (int r0 = part * rows; r0 < end; r0 += 32 * RP) {
        float4 m[RP][NV];
        float* base = M + ((long long)slot * A.hv + h) * A.dv * A.dk;
#pragma unroll
        for (int r = 0; r < RP; r++) {
            const int row = r0 + grp + 32 * r;
#pragma unroll
            for (int v = 0; v < NV; v++) {
                const int c = 4 * lane8 + 32 * v;
                float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
                if (row < end) {
                    const float* s = base + (long long)row * A.dk + c;
                    if (VEC) { if (c < A.dk) ldg(x, s); }
                    else {
                        if (c < A.dk) x.x = s[0];
                        if (c + 1 < A.dk) x.y = s[1];
                        if (c + 2 < A.dk) x.z = s[2];
                        if (c + 3 < A.dk) x.w = s[3];
                    }
                }
                m[r][v] = x;
            }
        }
        if (!looked) {                                    // while the rows are on their way: who else names this slot?
            looked = true;
            bool seen = false, again = false;
            for (int i = threadIdx.x; i < A.batch; i += 256) {
                const bool same = slots[i] == slot;
                seen |= same && i < first;
                again |= same && i > first;
            }
            if (__syncthreads_or(seen)) return;
            if (__syncthreads_or(again)) last = A.batch;
        }
        for (int b = first; b < last; b++) {
            if (b != first && slots[b] != slot) continue;
            for (int tok = 0; tok < A.seq; tok++) {
                const T* kp = (const T*)A.k + b * A.kb + tok * A.kt + (h / A.share) * A.kh;
                const T* qp = (const T*)A.q + b * A.qb + tok * A.qt + (h / A.share) * A.qh;
                const T* vp = (const T*)A.v + b * A.vb + tok * A.vt + h * A.vh;
                const long long ga = b * A.gb + tok * A.gt + h * A.gh;
                const float rt = expf(A.g[ga]), th = A.theta[ga];
                float kf[NV][4], qf[NV][4];
#pragma unroll
                for (int v = 0; v < NV; v++) {
                    const int c = 4 * lane8 + 32 * v;
                    if (VEC) {
                        float4 a = make_float4(0.f, 0.f, 0.f, 0.f), o = a;
                        if (c < A.dk) { a = ld4(kp + c); o = ld4(qp + c); }
                        kf[v][0] = a.x; kf[v][1] = a.y; kf[v][2] = a.z; kf[v][3] = a.w;
                        qf[v][0] = o.x; qf[v][1] = o.y; qf[v][2] = o.z; qf[v][3] = o.w;
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            kf[v][i] = c + i < A.dk ? to_f(kp[c + i]) : 0.f;
                            qf[v][i] = c + i < A.dk ? to_f(qp[c + i]) : 0.f;
                        }
                    }
                }
#pragma unroll
                for (int r = 0; r < RP; r++) {
                    const int row = r0 + grp + 32 * r;
                    const float val = row < end ? to_f(vp[row]) : 0.f;
                    float s = 0.f;
#pragma unroll
                    for (int v = 0; v < NV; v++) {
                        m[r][v].x *= rt; m[r][v].y *= rt; m[r][v].z *= rt; m[r][v].w *= rt;
                        s = fmaf(m[r][v].x, kf[v][0], s); s = fmaf(m[r][v].y, kf[v][1], s);
                        s = fmaf(m[r][v].z, kf[v][2], s); s = fmaf(m[r][v].w, kf[v][3], s);
                    }
                    s += __shfl_xor_sync(0xffffffffu, s, 1);
                    s += __shfl_xor_sync(0xffffffffu, s, 2);
                    s += __shfl_xor_sync(0xffffffffu, s, 4);
                    const float u = th * (val - s);
                    float y = 0.f;
#pragma unroll
                    for (int v = 0; v < NV; v++) {
                        m[r][v].x = fmaf(u, kf[v][0], m[r][v].x); m[r][v].y = fmaf(u, kf[v][1], m[r][v].y);
                        m[r][v].z = fmaf(u, kf[v][2], m[r][v].z); m[r][v].w = fmaf(u, kf[v][3], m[r][v].w);
                        y = fmaf(m[r][v].x, qf[v][0], y); y = fmaf(m[r][v].y, qf[v][1], y);
                        y = fmaf(m[r][v].z, qf[v][2], y); y = fmaf(m[r][v].w, qf[v][3], y);
                    }
                    y += __shfl_xor_sync(0xffffffffu, y, 1);
                    y += __shfl_xor_sync(0xffffffffu, y, 2);
                    y += __shfl_xor_sync(0xffffffffu, y, 4);
                    if (row < end && lane8 == 0)
                        ((T*)A.y)[(((long long)b * A.seq + tok) * A.hv + h) * A.dv + row] = from_f<T>(A.scale * y);
                }
            }
        }
#pragma unroll
        for (int r = 0; r < RP; r++) {
            const int row = r0 + grp + 32 * r;
            if (row >= end) continue;
#pragma unroll
            for (int v = 0; v < NV; v++) {
                const int c = 4 * lane8 + 32 * v;
                float* s = base + (long long)row * A.dk + c;
                if (VEC) { if (c < A.dk) *reinterpret_cast<float4*>(s) = m[r][v]; }
                else {
                    if (c < A.dk) s[0] = m[r][v].x;
                    if (c + 1 < A.dk) s[1] = m[r][v].y;
                    if (c + 2 < A.dk) s[2] = m[r][v].z;
                    if (c + 3 < A.dk) s[3] = m[r][v].w;
                }
            }
        }
    }
}

// ── host ──
constexpr int MAX_N = 1 << 30;       // tokens, and chunks of all heads: strided loops stay in 32 bits
static bool fill(const char* where, const nlh_gated_delta_desc* d, Args& A)
{
    A = Args{};
    const char* bad = nullptr;
    if (!d) bad = "NULL descriptor";
    else if (d->batch < 0 || d->seq < 0 || d->heads_k <= 0 || d->heads_v <= 0 || d->n_seqs < 0) bad = "bad dimensions";
    else if (d->heads_v % d->heads_k != 0) bad = "heads_v is no multiple of heads_k";
    else if (d->dk < 1 || d->dk > 128 || d->dv < 1 || d->dv > 128) bad = "dk and dv must be in 1..128";
    else if (d->n_seqs > 0 && d->batch != 1) bad = "a packed batch has batch = 1";
    else if ((long long)d->batch * d->seq > MAX_N || d->n_seqs > MAX_N) bad = "batch * seq and n_seqs are 2^30 at most";
    if (bad) { record_status(NLH_ERR_INVALID_ARG, where, bad); return false; }
    A.batch = d->batch; A.seq = d->seq; A.hk = d->heads_k; A.hv = d->heads_v; A.share = d->heads_v / d->heads_k;
    A.dk = d->dk; A.dv = d->dv; A.n_seqs = d->n_seqs;
    A.dkp = (d->dk + 63) / 64 * 64; A.dvp = (d->dv + 63) / 64 * 64;
    A.kb = d->k_batch; A.kt = d->k_token; A.kh = d->k_head;
    A.vb = d->v_batch; A.vt = d->v_token; A.vh = d->v_head;
    A.qb = d->q_batch; A.qt = d->q_token; A.qh = d->q_head;
    A.gb = d->gate_batch; A.gt = d->gate_token; A.gh = d->gate_head;
    A.yb = d->dy_batch; A.yt = d->dy_token; A.yh = d->dy_head;
    A.scale = d->scale;
    A.wait_cycles = option_value(NLH_OPT_GATED_DELTA_WAIT) ? T_WAIT_CYCLES : 0u;
    A.nc = (d->seq + C - 1) / C;
    const long long slots = d->n_seqs > 0 ? (long long)d->seq / C + d->n_seqs : (long long)d->batch * A.nc;
    if (slots * d->heads_v > MAX_N) { record_status(NLH_ERR_INVALID_ARG, where, "too many chunks"); return false; }
    A.slots = (int)slots;
    return true;
}

// Places the private buffers that forward hands on to backward behind `base`; returns their bytes.
static int64_t place_saved(Args& A, char* base)
{
    const int64_t tiles = (int64_t)A.slots * A.hv;
    int64_t at = 0;
    auto take = [&](int64_t bytes) { char* p = base + at; at += (bytes + 255) & ~(int64_t)255; return (void*)p; };
    A.tmat = (unsigned char*)take(tiles * T_BYTES);
    A.gates = (float4*)take(tiles * C * 16);
    A.theta_eff = (float*)take(tiles * C * 4);
    A.e = (float*)take(tiles * C * A.dvp * 4);
    A.m_chunk = (float*)take(tiles * A.dvp * A.dkp * 4);
    if (A.n_seqs > 0) {
        A.map = (int4*)take((int64_t)A.slots * 16);
        A.start = (int*)take((int64_t)(A.n_seqs + 1) * 4);
        A.off = (int*)take((int64_t)(A.n_seqs + 1) * 4);
        A.order = (int*)take((int64_t)A.n_seqs * 4);
    }
    return at;
}
static int64_t place_bwd(Args& A, char* base)
{
    const int64_t tiles = (int64_t)A.slots * A.hv, nk = A.dkp / 64;
    int64_t at = 0;
    auto take = [&](int64_t bytes) { char* p = base + at; at += (bytes + 255) & ~(int64_t)255; return (void*)p; };
    A.f = (float*)take(tiles * C * A.dvp * 4);
    A.x = (float*)take(tiles * C * A.dvp * 4);
    A.d_chunk = (float*)take(tiles * A.dvp * A.dkp * 4);
    A.dg_part = (float*)take(nk * tiles * C * 4);
    if (A.share > 1) {
        A.dk_part = (float*)take((int64_t)A.batch * A.seq * A.hv * A.dk * 4);
        A.dq_part = (float*)take((int64_t)A.batch * A.seq * A.hv * A.dk * 4);
    }
    return at;
}

// Opts a kernel in to its dynamic shared memory, once per device (the attribute belongs to the device that is current).
template <auto KERNEL, int BYTES> static bool allow_smem(const char* where)
{
    static std::atomic<uint64_t> done[2];        // devices 0 .. 127
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev > 127) dev = -1;
    if (dev >= 0 && (done[dev >> 6].load(std::memory_order_relaxed) >> (dev & 63) & 1)) return true;
    const cudaError_t e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, BYTES);
    if (e != cudaSuccess) { record_status(NLH_ERR_CUDA, where, cudaGetErrorString(e)); return false; }
    if (dev >= 0) done[dev >> 6].fetch_or(1ull << (dev & 63), std::memory_order_relaxed);
    return true;
}

template <typename T, int DKP, int NS>
static bool launch_states_ns(const Args& A, long long heads, bool backward, cudaStream_t st, const char* where)
{
    const long long grid = heads * (A.dvp / NS);
    if (grid >= (1LL << 31)) { record_status(NLH_ERR_INVALID_ARG, where, "too many sequences"); return false; }
    constexpr int bytes = StateSmem<T, DKP, NS>::BYTES;
    if (backward) {
        if (!allow_smem<gd_state_bwd_kernel<T, DKP, NS>, bytes>(where)) return false;
        gd_state_bwd_kernel<T, DKP, NS><<<(unsigned)grid, 256, bytes, st>>>(A);
    } else {
        if (!allow_smem<gd_state_fwd_kernel<T, DKP, NS>, bytes>(where)) return false;
        gd_state_fwd_kernel<T, DKP, NS><<<(unsigned)grid, 256, bytes, st>>>(A);
    }
    return check_launch(where);
}
template <typename T, int DKP> static bool launch_states(const Args& A, bool backward, cudaStream_t st, const char* where)
{
    const long long heads = (long long)(A.n_seqs > 0 ? A.n_seqs : A.batch) * A.hv;
    if (heads == 0) return true;
    // 16 columns a CTA while each of those CTAs finds an SM of its own (forward + backward, 2 x 8 heads of 128 x 128: 39 + 43 us against
    // 60 + 69 with 32 columns; 3 x 16 of 64 x 64, which does not: 83 + 99 against 80 + 93). For packed batches longer, since their few
    // longest sequences run alone in the end: up to three CTAs of 32 columns an SM where two fit one, up to two where one does. Whole pass,
    // 16 | 32 columns, bf16, lengths drawn from x^3 (CTAs of 32 columns): dk 64: 495 | 539 us (208), 420 | 476 (416), 167 | 155 (600),
    // 440 | 414 (640); dk 128: 322 | 420 (104), 280 | 336 (208), 291 | 274 (320), 855 | 793 (416). Equal lengths: 0 to 8 % the other way.
    const bool narrow = A.n_seqs > 0 ? heads * (A.dvp / 32) < (DKP == 64 ? 3 : 2) * 148 : heads * (A.dvp / 16) <= 148;
    if (narrow) return launch_states_ns<T, DKP, 16>(A, heads, backward, st, where);
    return launch_states_ns<T, DKP, 32>(A, heads, backward, st, where);
}

template <typename T> static bool run_forward(Args& A, cudaStream_t st, const char* where)
{
    if (A.n_seqs > 0) {
        gd_map_kernel<<<1, 1024, 0, st>>>(A);
        if (!check_launch(where)) return false;
    }
    const unsigned tiles = (unsigned)((long long)A.slots * A.hv);
    if (tiles) {
        constexpr int bytes = T_BYTES + 2 * C * LD * 4;
        if (!allow_smem<gd_prep_kernel<T>, bytes>(where)) return false;
        gd_prep_kernel<T><<<tiles, 256, bytes, st>>>(A);
        if (!check_launch(where)) return false;
    }
    if (!(A.dkp == 64 ? launch_states<T, 64>(A, false, st, where) : launch_states<T, 128>(A, false, st, where))) return false;
    if (tiles) {
        if (!allow_smem<gd_out_fwd_kernel<T>, OUT_FWD_BYTES>(where)) return false;
        gd_out_fwd_kernel<T><<<dim3(tiles, A.dvp / 64), 128, OUT_FWD_BYTES, st>>>(A);
        if (!check_launch(where)) return false;
    }
    return true;
}

template <typename T> static bool run_backward(Args& A, cudaStream_t st, const char* where)
{
    const unsigned tiles = (unsigned)((long long)A.slots * A.hv);
    if (tiles) {
        if (!allow_smem<gd_pre_bwd_kernel<T>, PRE_BWD_BYTES>(where)) return false;
        gd_pre_bwd_kernel<T><<<dim3(tiles, A.dvp / 64), 256, PRE_BWD_BYTES, st>>>(A);
        if (!check_launch(where)) return false;
    }
    if (!(A.dkp == 64 ? launch_states<T, 64>(A, true, st, where) : launch_states<T, 128>(A, true, st, where))) return false;
    if (!tiles) return true;
    constexpr int bytes = OutBwdSmem<T>::BYTES;
    if (!allow_smem<gd_out_bwd_kernel<T>, bytes>(where)) return false;
    gd_out_bwd_kernel<T><<<dim3(tiles, A.dkp / 64), 256, bytes, st>>>(A);
    if (!check_launch(where)) return false;
    if (A.dkp > 64) {
        gd_gate_bwd_kernel<<<(tiles + 3) / 4, 128, 0, st>>>(A);
        if (!check_launch(where)) return false;
    }
    const long long n = (long long)A.batch * A.seq * A.hk * A.dk;
    if (A.share > 1 && n > 0) {                   // a packed batch without a token has chunk slots, but no rows
        const long long need = (n + 255) / 256;
        gd_group_kernel<T><<<(unsigned)(need < 148 * 16 ? need : 148 * 16), 256, 0, st>>>(A, n);
        if (!check_launch(where)) return false;
    }
    return true;
}

}  // namespace gd
}  // namespace nlh

using namespace nlh;
using namespace nlh::gd;

extern "C" {

int64_t nlh_gated_delta_saved_bytes(const nlh_gated_delta_desc* desc)
{
    Args A;
    if (!fill("nlh_gated_delta_saved_bytes", desc, A)) return -1;
    return place_saved(A, nullptr);
}

int64_t nlh_gated_delta_backward_bytes(const nlh_gated_delta_desc* desc)
{
    Args A;
    if (!fill("nlh_gated_delta_backward_bytes", desc, A)) return -1;
    return place_bwd(A, nullptr);
}

static bool gd_inputs(const char* where, Args& A, const nlh_gated_delta_desc* desc, const void* k, const void* v, const void* q,
                      const float* log_retain, const float* theta, const int32_t* seq_starts)
{
    if (!fill(where, desc, A)) return false;
    const bool tokens = (long long)A.batch * A.seq > 0;
    if ((tokens && (!k || !v || !q || !log_retain || !theta)) || (A.n_seqs > 0) != (seq_starts != nullptr)) {
        record_status(NLH_ERR_INVALID_ARG, where, "NULL pointer, or seq_starts without n_seqs");
        return false;
    }
    A.k = k; A.v = v; A.q = q; A.g = log_retain; A.theta = theta; A.starts = seq_starts;
    return true;
}

int32_t nlh_gated_delta_forward(const nlh_gated_delta_desc* desc, const void* k, const void* v, const void* q,
    const float* log_retain, const float* theta, const float* m_initial, const int32_t* seq_starts, void* y, float* m_final,
    void* saved, int64_t saved_bytes)
{
    const char* where = "nlh_gated_delta_forward";
    Args A;
    if (!gd_inputs(where, A, desc, k, v, q, log_retain, theta, seq_starts)) return NLH_ERR_INVALID_ARG;
    const bool tokens = (long long)A.batch * A.seq > 0;
    const int64_t need = place_saved(A, (char*)saved);       // a packed batch has chunk slots without a token too
    if ((tokens && !y) || (!m_final && (A.n_seqs > 0 || A.batch > 0)) || ((uintptr_t)saved & 15) || saved_bytes < need || (need > 0 && !saved)) {
        record_status(NLH_ERR_INVALID_ARG, where, "NULL output, or a saved buffer that is too small or not 16-byte aligned");
        return NLH_ERR_INVALID_ARG;
    }
    A.m0 = m_initial; A.y = y; A.m_final = m_final;
    const bool ok = desc->is_bf16 ? run_forward<__nv_bfloat16>(A, current_stream(), where) : run_forward<float>(A, current_stream(), where);
    return ok ? NLH_OK : NLH_ERR_CUDA;
}

int32_t nlh_gated_delta_backward(const nlh_gated_delta_desc* desc, const void* k, const void* v, const void* q,
    const float* log_retain, const float* theta, const int32_t* seq_starts, const void* saved, int64_t saved_bytes,
    const void* d_y, const float* d_m_final, void* d_k, void* d_v, void* d_q, float* d_log_retain, float* d_theta,
    float* d_m_initial, void* workspace, int64_t workspace_bytes)
{
    const char* where = "nlh_gated_delta_backward";
    Args A;
    if (!gd_inputs(where, A, desc, k, v, q, log_retain, theta, seq_starts)) return NLH_ERR_INVALID_ARG;
    const bool tokens = (long long)A.batch * A.seq > 0;
    const int64_t need_saved = place_saved(A, (char*)saved), need_work = place_bwd(A, (char*)workspace);
    if ((tokens && (!d_y || !d_k || !d_v || !d_q || !d_log_retain || !d_theta)) || (need_saved > 0 && !saved) || (need_work > 0 && !workspace) ||
        (((uintptr_t)saved | (uintptr_t)workspace) & 15) || saved_bytes < need_saved || workspace_bytes < need_work) {
        record_status(NLH_ERR_INVALID_ARG, where, "NULL pointer, or a buffer that is too small or not 16-byte aligned");
        return NLH_ERR_INVALID_ARG;
    }
    A.dy = d_y; A.d_m_final = d_m_final; A.d_k = d_k; A.d_v = d_v; A.d_q = d_q;
    A.d_g = d_log_retain; A.d_theta = d_theta; A.d_m0 = d_m_initial;
    const bool ok = desc->is_bf16 ? run_backward<__nv_bfloat16>(A, current_stream(), where) : run_backward<float>(A, current_stream(), where);
    return ok ? NLH_OK : NLH_ERR_CUDA;
}

int32_t nlh_gated_delta_timeout_flag(void)
{
    int v = 0;
    if (cudaStreamSynchronize(current_stream()) != cudaSuccess || cudaMemcpyFromSymbol(&v, g_gd_timeout, sizeof(int)) != cudaSuccess) return -1;
    return v;
}

int32_t nlh_gated_delta_timeout_clear(void)
{
    const int v = 0;
    if (cudaStreamSynchronize(current_stream()) != cudaSuccess || cudaMemcpyToSymbol(g_gd_timeout, &v, sizeof(int)) != cudaSuccess) {
        record_status(NLH_ERR_CUDA, "nlh_gated_delta_timeout_clear", cudaGetErrorString(cudaGetLastError()));
        return NLH_ERR_CUDA;
    }
    return NLH_OK;
}

int32_t nlh_gated_delta_step(const nlh_gated_delta_desc* desc, const void* k, const void* v, const void* q,
    const float* log_retain, const float* theta, float* m, const int32_t* slots, int32_t n_slots, void* y)
{
    const char* where = "nlh_gated_delta_step";
    Args A;
    if (!gd_inputs(where, A, desc, k, v, q, log_retain, theta, nullptr)) return NLH_ERR_INVALID_ARG;
    if ((long long)A.batch * A.seq == 0) return NLH_OK;
    if (!m || !y || n_slots < (slots ? 0 : A.batch)) {
        record_status(NLH_ERR_INVALID_ARG, where, "NULL pointer, or fewer states than sequences");
        return NLH_ERR_INVALID_ARG;
    }
    A.y = y;
    // one round of a CTA's threads (64 rows of dk > 64, 128 shorter ones) while that gives every SM two CTAs, else 32 rows
    const long long heads = (long long)A.batch * A.hv;
    const int full = A.dk > 64 ? 64 : 128, rows = heads * ((A.dv + full - 1) / full) >= 2 * 148 ? full : 32;
    const long long grid = heads * ((A.dv + rows - 1) / rows);
    if (grid >= (1LL << 31)) { record_status(NLH_ERR_INVALID_ARG, where, "too many sequences"); return NLH_ERR_INVALID_ARG; }
    cudaStream_t st = current_stream();
    const int es = desc->is_bf16 ? 2 : 4;
    const bool vec = (A.dk & 3) == 0 && aligned16(m) && (((uintptr_t)k | (uintptr_t)q) & (4 * es - 1)) == 0 &&
                     ((A.kb | A.kt | A.kh | A.qb | A.qt | A.qh) & 3) == 0;
#define NLH_GD_STEP(T, NV) (vec ? gd_step_kernel<T, NV, true><<<(unsigned)grid, 256, 0, st>>>(A, m, slots, n_slots, rows) \
                                : gd_step_kernel<T, NV, false><<<(unsigned)grid, 256, 0, st>>>(A, m, slots, n_slots, rows))
    if (desc->is_bf16) { if (A.dk <= 64) NLH_GD_STEP(__nv_bfloat16, 2); else NLH_GD_STEP(__nv_bfloat16, 4); }
    else { if (A.dk <= 64) NLH_GD_STEP(float, 2); else NLH_GD_STEP(float, 4); }
#undef NLH_GD_STEP
    return check_launch(where) ? NLH_OK : NLH_ERR_CUDA;
}

}  // extern "C"
