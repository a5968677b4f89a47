// Embedding lookup with scaling, and its gradient by sorted tokens.
//
//   out_t = scale w[id_t],   d_w[r] (+)= scale sum over {t : id_t = r} of d_out_t, in ascending t, in fp32.
//
// The gradient's rows meet wherever an id repeats, and in text a few ids are much of it. Instead of atomics (whose
// order, and so whose sum, changes from run to run, and which queue up on the hot rows) the tokens are sorted by id with a
// stable radix sort, every sum then has one order, and every row of d_w is touched once, by one writer:
//   sort    : least significant digit first, 9 bits a pass at most: one cluster of CTAs, or for long lists a histogram per 2048 tokens and
//             ranks from it
//   reduce  : a run of sorted tokens per group of lanes; an id that lies inside the run is written at once, the pieces of one
//             that crosses runs go to a buffer
//   join    : those pieces, added in order by the run in which the id begins
// A few tokens take one launch (one_launch): a CTA per token looks for its id in the whole list, and the first token of an id
// adds up its rows.
// Bound by HBM: d_out is read once, the touched rows of d_w once and written once.
#include <atomic>
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include "nlh_common.cuh"
#include "../../include/nlh_ffi.h"

namespace nlh {
namespace emb {

constexpr int BITS = 9, BINS = 1 << BITS;
constexpr int SORT_THREADS = 256, SORT_ITEMS = 8, SORT_TILE = SORT_THREADS * SORT_ITEMS;
constexpr int SMALL = 2048;
constexpr int THREADS = 128;
constexpr int MAX_N = 1 << 30, MAX_D = 1 << 20;       // tokens, width: strided loops and grids stay in their ranges

template <typename T> struct Vec { static constexpr int N = 16 / sizeof(T); };
// N elements as they came, and as floats
template <typename T, int N> struct Raw { uint4 r; };
template <> struct Raw<float, 1> { float r; };
template <> struct Raw<__nv_bfloat16, 1> { __nv_bfloat16 r; };
template <typename T, int N> __device__ __forceinline__ void load(const T* p, float* f);
template <> __device__ __forceinline__ void load<float, 4>(const float* p, float* f)
{
    const float4 v = *reinterpret_cast<const float4*>(p);
    f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
}
template <> __device__ __forceinline__ void load<__nv_bfloat16, 8>(const __nv_bfloat16* p, float* f)
{
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
template <> __device__ __forceinline__ void load<float, 1>(const float* p, float* f) { f[0] = *p; }
template <> __device__ __forceinline__ void load<__nv_bfloat16, 1>(const __nv_bfloat16* p, float* f) { f[0] = __bfloat162float(*p); }
// N floats to / from fp32 memory
template <int N> __device__ __forceinline__ void store_f32(float* p, const float* f)
{
    if constexpr (N == 1) p[0] = f[0];
    else {
#pragma unroll
        for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
    }
}
template <int N> __device__ __forceinline__ void load_f32(const float* p, float* f)
{
    if constexpr (N == 1) f[0] = p[0];
    else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 v = *reinterpret_cast<const float4*>(p + i);
            f[i] = v.x; f[i + 1] = v.y; f[i + 2] = v.z; f[i + 3] = v.w;
        }
    }
}
// One writer per row of d_w: a reduction without an answer, which no load waits for, has no other to race with.
template <int N, bool ADD> __device__ __forceinline__ void add_row(float* p, const float* acc, float scale)
{
    if (!ADD) {
        float o[N];
#pragma unroll
        for (int i = 0; i < N; i++) o[i] = scale * acc[i];
        store_f32<N>(p, o);
    } else if (N == 1) {
        atomicAdd(p, scale * acc[0]);
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4)
            atomicAdd(reinterpret_cast<float4*>(p + i), make_float4(scale * acc[i], scale * acc[(i + 1) % N], scale * acc[(i + 2) % N],
                                                                  scale * acc[(i + 3) % N]));
    }
}
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16(x); }

// ── lookup ──
// `lanes` lanes share a row (a power of two, 32 at most), N elements each and step.
template <typename T, int N>
__global__ void __launch_bounds__(256) lookup_kernel(const T* __restrict__ w, const int* __restrict__ ids, T* __restrict__ out, int n,
                                                     int vocab, int d, int lanes, float scale)
{
    const int per = 256 / lanes, lane = threadIdx.x & (lanes - 1);
    for (long long t = (long long)blockIdx.x * per + threadIdx.x / lanes; t < n; t += (long long)gridDim.x * per) {
        const int id = ids[t];
        const bool ok = id >= 0 && id < vocab;
        const T* src = w + (long long)(ok ? id : 0) * d;
        T* dst = out + t * d;
#pragma unroll 4
        for (int c = lane * N; c < d; c += lanes * N) {
            float f[N];
            if (ok) load<T, N>(src + c, f);
#pragma unroll
            for (int i = 0; i < N; i++) f[i] = ok ? f[i] * scale : 0.f;
            if (N == 1) put(dst + c, f[0]);
            else if (sizeof(T) == 4) store_f32<N>((float*)(dst + c), f);
            else {
                unsigned u[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const __nv_bfloat162 b = __floats2bfloat162_rn(f[(2 * i) % N], f[(2 * i + 1) % N]);
                    u[i] = *reinterpret_cast<const unsigned*>(&b);
                }
                *reinterpret_cast<uint4*>(dst + c) = make_uint4(u[0], u[1], u[2], u[3]);
            }
        }
    }
}

// ── sort ──
// Key of a token: its id, or vocab (behind all others) where the id is none.
__device__ __forceinline__ int key_of(const int* ids, const int2* in, int i, int vocab, int& pos)
{
    if (in) { const int2 x = in[i]; pos = x.y; return x.x; }
    pos = i;
    const int id = ids[i];
    return id >= 0 && id < vocab ? id : vocab;
}
// hist [BINS, blocks]: tokens of each digit in each tile
__global__ void __launch_bounds__(SORT_THREADS) hist_kernel(const int* ids, const int2* in, int* hist, int n, int vocab, int shift, int blocks)
{
    __shared__ int s[BINS];
    for (int i = threadIdx.x; i < BINS; i += SORT_THREADS) s[i] = 0;
    __syncthreads();
    for (int j = 0; j < SORT_ITEMS; j++) {
        const int i = blockIdx.x * SORT_TILE + j * SORT_THREADS + threadIdx.x;
        int pos;
        if (i < n) atomicAdd(&s[(key_of(ids, in, i, vocab, pos) >> shift) & (BINS - 1)], 1);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < BINS; i += SORT_THREADS) hist[(long long)i * blocks + blockIdx.x] = s[i];
}
// One warp per digit: counts -> sums over the tiles before; the digit's total behind them in `total`.
__global__ void __launch_bounds__(256) scan_kernel(int* hist, int* total, int blocks)
{
    const int digit = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    int* h = hist + (long long)digit * blocks;
    int carry = 0;
    for (int b = 0; b < blocks; b += 32) {
        const int c = b + lane < blocks ? h[b + lane] : 0;
        int s = c;
        for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, s, o); if (lane >= o) s += y; }
        if (b + lane < blocks) h[b + lane] = carry + s - c;
        carry += __shfl_sync(0xffffffffu, s, 31);
    }
    if (lane == 0) total[digit] = carry;
}
// Every token to its place: tokens of smaller digits, of this digit in the tiles before, in the warps before, in this warp before.
__global__ void __launch_bounds__(SORT_THREADS) scatter_kernel(const int* ids, const int2* in, int2* out, const int* hist, const int* total,
                                                               int n, int vocab, int shift, int blocks)
{
    constexpr int WARPS = SORT_THREADS / 32, SEG = SORT_TILE / WARPS;
    __shared__ int s_cnt[WARPS][BINS], s_scan[WARPS];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    for (int i = threadIdx.x; i < WARPS * BINS; i += SORT_THREADS) (&s_cnt[0][0])[i] = 0;
    __syncthreads();
    int key[SORT_ITEMS], pos[SORT_ITEMS], rank[SORT_ITEMS];
#pragma unroll
    for (int j = 0; j < SORT_ITEMS; j++) {
        const int i = blockIdx.x * SORT_TILE + w * SEG + j * 32 + lane;
        key[j] = -1;
        if (i < n) key[j] = key_of(ids, in, i, vocab, pos[j]);
    }
#pragma unroll
    for (int j = 0; j < SORT_ITEMS; j++) {
        const int digit = key[j] < 0 ? -1 : (key[j] >> shift) & (BINS - 1);
        const unsigned same = __match_any_sync(0xffffffffu, digit);
        int before = 0;
        if (digit >= 0) before = s_cnt[w][digit];
        __syncwarp();
        if (digit >= 0) {
            rank[j] = before + __popc(same & ((1u << lane) - 1));
            if (lane == __ffs(same) - 1) s_cnt[w][digit] = before + __popc(same);
        }
        __syncwarp();
    }
    __syncthreads();
    // digits 2 threadIdx.x, 2 threadIdx.x + 1: where this tile's first token of the digit goes, then each warp's
    int tot[2], first[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
        const int digit = 2 * threadIdx.x + e;
        tot[e] = total[digit];
        first[e] = hist[(long long)digit * blocks + blockIdx.x];
    }
    int s = tot[0] + tot[1];
    for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, s, o); if (lane >= o) s += y; }
    if (lane == 31) s_scan[w] = s;
    __syncthreads();
    for (int j = 0; j < w; j++) s += s_scan[j];
#pragma unroll
    for (int e = 0; e < 2; e++) {
        const int digit = 2 * threadIdx.x + e;
        int at = s - tot[0] - tot[1] + (e ? tot[0] : 0) + first[e];
        for (int j = 0; j < WARPS; j++) { const int c = s_cnt[j][digit]; s_cnt[j][digit] = at; at += c; }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < SORT_ITEMS; j++)
        if (key[j] >= 0) out[s_cnt[w][(key[j] >> shift) & (BINS - 1)] + rank[j]] = make_int2(key[j], pos[j]);
}

// The whole sort in one launch up to 131072 tokens: a cluster of sixteen CTAs, a thread ITEMS tokens, the digits' totals exchanged
// through distributed shared memory, digits only as wide as the passes need. A device (or a part of one) that cannot hold such a
// cluster takes the launches above. 32768 tokens of a vocabulary of 8192 take 12 us (the launches above: 27 and the gaps between
// them), 65521 of 50001 take 19 (37). Tokens of one digit in a warp are found by a ballot per bit, which beat a match instruction.
constexpr int CL = 16, CL_THREADS = 1024, CL_WARPS = CL_THREADS / 32, CL_MOST = CL * CL_THREADS * 8;
template <int ITEMS>
__global__ void __launch_bounds__(CL_THREADS, 1) sort_cluster_kernel(const int* ids, int2* bufa, int2* bufb, int n,
                                                                                               int vocab, int passes, int bits)
{
    extern __shared__ int s_dyn[];
    int* s_cnt = s_dyn;                          // [CL_WARPS][BINS]
    int* s_tot = s_dyn + CL_WARPS * BINS;        // [BINS] this CTA's tokens of each digit
    int* s_first = s_tot + BINS;                 // [BINS] where they go
    const int bins = 1 << bits;
    __shared__ int s_scan[BINS / 32];
    namespace cg = cooperative_groups;
    cg::cluster_group cl = cg::this_cluster();
    const int rank = (int)cl.block_rank(), tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
    const int base = (rank * CL_WARPS + w) * ITEMS * 32 + lane;    // warps hold stretches of the list, in order
    const int2* in = nullptr;
    int2* out = bufa;
    for (int p = 0; p < passes; p++) {
        const int shift = p * bits;
        for (int i = tid; i < CL_WARPS * bins; i += CL_THREADS) s_cnt[i] = 0;
        int key[ITEMS], pos[ITEMS], rnk[ITEMS];
#pragma unroll
        for (int j = 0; j < ITEMS; j++) {
            const int i = base + j * 32;
            key[j] = -1;
            if (i < n) key[j] = key_of(ids, in, i, vocab, pos[j]);
        }
        __syncthreads();
        int* mine = s_cnt + w * bins;
#pragma unroll
        for (int j = 0; j < ITEMS; j++) {
            const int digit = key[j] < 0 ? -1 : (key[j] >> shift) & (bins - 1);
            unsigned same = __ballot_sync(0xffffffffu, digit >= 0);
            if (digit < 0) same = ~same;
            for (int x = 0; x < bits; x++) {
                const bool one = (digit >> x) & 1;
                const unsigned m = __ballot_sync(0xffffffffu, one);
                same &= one ? m : ~m;
            }
            int before = 0;
            if (digit >= 0) before = mine[digit];
            __syncwarp();
            if (digit >= 0) {
                rnk[j] = before + __popc(same & ((1u << lane) - 1));
                if (lane == __ffs(same) - 1) mine[digit] = before + __popc(same);
            }
            __syncwarp();
        }
        __syncthreads();
        if (tid < bins) {                        // tokens of the digit in the warps before
            int at = 0;
#pragma unroll 8
            for (int j = 0; j < CL_WARPS; j++) { const int c = s_cnt[j * bins + tid]; s_cnt[j * bins + tid] = at; at += c; }
            s_tot[tid] = at;
        }
        cl.sync();
        int total = 0, first = 0;                // in all CTAs, in the CTAs before
        if (tid < bins) {
#pragma unroll
            for (int r = 0; r < CL; r++) {
                const int c = *cl.map_shared_rank(s_tot + tid, r);
                total += c;
                first += r < rank ? c : 0;
            }
            int s = total;
            for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, s, o); if (lane >= o) s += y; }
            if (lane == 31) s_scan[w] = s;
            first += s - total;
        }
        __syncthreads();
        if (tid < bins) {
            for (int j = 0; j < w; j++) first += s_scan[j];
            s_first[tid] = first;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < ITEMS; j++)
            if (key[j] >= 0) {
                const int digit = (key[j] >> shift) & (bins - 1);
                out[s_first[digit] + mine[digit] + rnk[j]] = make_int2(key[j], pos[j]);
            }
        cl.sync();                               // the list is whole for the next pass, and every s_tot has been read
        in = out;
        out = out == bufa ? bufb : bufa;
    }
}

// ── reduce ──
// A group of `lanes` lanes takes `run` sorted tokens (and columns blockIdx.y * lanes * N ..). part [runs, 2, d]: the piece of an id
// that began before the run, and of one that goes on behind it.
template <typename T, int N, bool ADD>
__global__ void __launch_bounds__(THREADS) reduce_kernel(const T* __restrict__ dy, const int2* __restrict__ sorted, float* __restrict__ dw,
                                                         float* __restrict__ part, int n, int vocab, int d, int lanes, int run, float scale)
{
    const int per = THREADS / lanes, lane = threadIdx.x & (lanes - 1), grp = threadIdx.x / lanes;
    const int r = blockIdx.x * per + grp, c = (blockIdx.y * lanes + lane) * N;
    extern __shared__ int2 s_all[];               // [per][run + 2]: the tokens of each run, the one before and the one behind
    for (int i = threadIdx.x; i < per * (run + 2); i += THREADS) {
        const int q = i / (run + 2);
        const long long at = ((long long)blockIdx.x * per + q) * run + (i - q * (run + 2)) - 1;
        s_all[i] = at >= 0 && at < n ? sorted[at] : make_int2(-1, 0);
    }
    __syncthreads();
    const int2* mine = s_all + grp * (run + 2) + 1;
    const long long b = (long long)r * run;
    if (b >= n || c >= d) return;
    const int e = (int)min((long long)run, n - b);
    const int prev = mine[-1].x, next = mine[e].x;
    float acc[N];
#pragma unroll
    for (int i = 0; i < N; i++) acc[i] = 0.f;
    int cur = mine[0].x;
    bool head = cur == prev;
    auto flush = [&](bool tail) {
        if (cur >= vocab) return;
        if (head || tail) {
            store_f32<N>(part + ((long long)r * 2 + (head ? 0 : 1)) * d + c, acc);
        } else {
            add_row<N, ADD>(dw + (long long)cur * d + c, acc, scale);
        }
    };
    constexpr int U = 8;
    for (int i = 0; i < e; i += U) {
        Raw<T, N> raw[U];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (i + u < e && mine[i + u].x < vocab) raw[u] = *reinterpret_cast<const Raw<T, N>*>(dy + (long long)mine[i + u].y * d + c);
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (i + u >= e) break;
            if (mine[i + u].x != cur) {
                flush(false);
                cur = mine[i + u].x;
                head = false;
#pragma unroll
                for (int x = 0; x < N; x++) acc[x] = 0.f;
            }
            if (cur < vocab) {
                float f[N];
                load<T, N>(reinterpret_cast<const T*>(&raw[u]), f);
#pragma unroll
                for (int x = 0; x < N; x++) acc[x] += f[x];
            }
        }
    }
    flush(cur == next);
}
// Ids that cross runs: the run in which one begins adds its pieces up, in their order. A warp per run and 32 N columns; most have
// nothing to do. A warp looks 32 runs ahead at once for the last one that begins with the id. Up to LONG pieces it adds by itself;
// for more the CTA's eight warps take a stretch each and join their sums (one warp walking the pieces of the most frequent id
// of a text of 32768 tokens took 51 us).
constexpr int LONG = 16;
template <int N>
__device__ __forceinline__ void add_pieces(float (&acc)[N], const float* part, long long r, long long i0, long long i1, int d, int c)
{
#pragma unroll
    for (int i = 0; i < N; i++) acc[i] = 0.f;
    if (c >= d) return;
#pragma unroll 8
    for (long long i = i0; i < i1; i++) {
        float f[N];
        load_f32<N>(part + ((r + i) * 2 + (i == 0)) * d + c, f);       // piece 0 is what run r left over, the others began before their runs
#pragma unroll
        for (int x = 0; x < N; x++) acc[x] += f[x];
    }
}
template <int N, bool ADD>
__global__ void __launch_bounds__(256) join_kernel(const int2* __restrict__ sorted, float* __restrict__ dw, const float* __restrict__ part,
                                                   int n, int vocab, int d, int run, float scale)
{
    __shared__ float s_acc[8][32 * N];
    __shared__ long long s_pieces[8];
    __shared__ int s_key[8];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = (blockIdx.y * 32 + lane) * N;
    const long long r = (long long)blockIdx.x * 8 + w, b = r * run, e = b + run;
    long long pieces = 0;                                              // runs behind r that begin with the id, if it begins in r
    int key = -1;
    if (e < n) {
        key = sorted[e - 1].x;
        if (key < vocab && sorted[e].x == key && !(b > 0 && sorted[b].x == key && sorted[b - 1].x == key)) {
            for (;;) {
                const long long q = r + 1 + pieces + lane;
                const int more = __popc(__ballot_sync(0xffffffffu, q * run < n && sorted[q * run].x == key));    // sorted: the first ones
                pieces += more;
                if (more < 32) break;
            }
        }
    }
    float acc[N];
    if (pieces > 0 && pieces <= LONG) {
        add_pieces<N>(acc, part, r, 0, pieces + 1, d, c);
        if (c < d) add_row<N, ADD>(dw + (long long)key * d + c, acc, scale);
    }
    if (lane == 0) { s_pieces[w] = pieces > LONG ? pieces : 0; s_key[w] = key; }
    __syncthreads();
    for (int o = 0; o < 8; o++) {
        const long long many = s_pieces[o];
        if (many == 0) continue;
        const long long each = (many + 8) / 8, i0 = w * each, i1 = min(many + 1, i0 + each);
        add_pieces<N>(acc, part, (long long)blockIdx.x * 8 + o, i0, i1, d, c);
#pragma unroll
        for (int i = 0; i < N; i++) s_acc[w][i * 32 + lane] = acc[i];
        __syncthreads();
        if (w == 0 && c < d) {
            for (int j = 1; j < 8; j++)
#pragma unroll
                for (int i = 0; i < N; i++) acc[i] += s_acc[j][i * 32 + lane];
            add_row<N, ADD>(dw + (long long)s_key[o] * d + c, acc, scale);
        }
        __syncthreads();
    }
}

// ── few tokens ──
// A CTA per token. Groups of `lanes` lanes take stretches of the id's tokens, joined in order.
template <typename T, int N, bool ADD>
__global__ void __launch_bounds__(THREADS) small_kernel(const T* __restrict__ dy, const int* __restrict__ ids, float* __restrict__ dw, int n,
                                                        int vocab, int d, int lanes, float scale)
{
    __shared__ int s_list[SMALL], s_warp[THREADS / 32];
    __shared__ float s_acc[THREADS * N];
    const int t = blockIdx.x, id = ids[t], w = threadIdx.x >> 5, wl = threadIdx.x & 31;
    if (id < 0 || id >= vocab) return;
    bool seen = false;
    for (int i = threadIdx.x; i < t; i += THREADS) seen |= ids[i] == id;
    if (__syncthreads_or(seen)) return;
    int count = 0;
    for (int base = t; base < n; base += THREADS) {
        const bool hit = base + threadIdx.x < n && ids[base + threadIdx.x] == id;
        const unsigned m = __ballot_sync(0xffffffffu, hit);
        if (wl == 0) s_warp[w] = __popc(m);
        __syncthreads();
        int at = count;
        for (int j = 0; j < w; j++) at += s_warp[j];
        if (hit) s_list[at + __popc(m & ((1u << wl) - 1))] = base + threadIdx.x;
        for (int j = 0; j < THREADS / 32; j++) count += s_warp[j];
        __syncthreads();
    }
    const int per = THREADS / lanes, lane = threadIdx.x & (lanes - 1), grp = threadIdx.x / lanes;
    const int stretch = (count + per - 1) / per, i0 = grp * stretch, i1 = min(count, i0 + stretch);
    for (int c0 = 0; c0 < d; c0 += lanes * N) {
        const int c = c0 + lane * N;
        float acc[N];
#pragma unroll
        for (int i = 0; i < N; i++) acc[i] = 0.f;
        if (c < d) {
#pragma unroll 8
            for (int i = i0; i < i1; i++) {
                float f[N];
                load<T, N>(dy + (long long)s_list[i] * d + c, f);
#pragma unroll
                for (int x = 0; x < N; x++) acc[x] += f[x];
            }
        }
        if (per > 1) {
#pragma unroll
            for (int i = 0; i < N; i++) s_acc[i * THREADS + threadIdx.x] = acc[i];
            __syncthreads();
            if (grp == 0) {
                for (int j = 1; j < per; j++)
#pragma unroll
                    for (int i = 0; i < N; i++) acc[i] += s_acc[i * THREADS + j * lanes + lane];
            }
            __syncthreads();
        }
        if (grp == 0 && c < d) add_row<N, ADD>(dw + (long long)id * d + c, acc, scale);
    }
}

// ── host ──
struct Plan {
    int passes, bits, blocks, run, runs;              // bits: of a digit in the one-launch sort
    int2 *a, *b;
    int *hist, *total;
    float* part;
};
// The single launch adds the rows of one id by one CTA, so its time goes by the most frequent id; the sorted path takes 15 to 23 us
// whatever the ids. us, one launch | sorted, fp32, for ids drawn as 1 / rank^1.1 of 256, and for a list of one id (padding, at worst):
//   tokens x width  512 x 64      1024 x 64     256 x 512     1024 x 128    256 x 1024    2048 x 512
//   drawn           5.2 | 16.9    7.7 | 17.0    8.1 | 15.7    9.7 | 16.7    12.9 | 15.6   43.1 | 18.6
//   one id          8.8 | 15.4    15.6 | 15.8   24.8 | 14.7   26.2 | 15.6   47.6 | 14.9   184 | 17.1
// (bf16 within a tenth of these.) Up to 2^17 elements it gains more on drawn ids than it loses on one.
static bool one_launch(int n, int d) { return n <= SMALL && (int64_t)n * d <= (1 << 17); }

static int64_t place(Plan& P, char* base, int n, int vocab, int d)
{
    P = Plan{};
    if (one_launch(n, d)) return 0;
    int bits = 1;
    while (bits < 31 && (vocab >> bits) != 0) bits++;          // keys 0 .. vocab
    P.passes = (bits + BITS - 1) / BITS;
    P.bits = (bits + P.passes - 1) / P.passes;
    if (P.bits < 5) P.bits = 5;                                // whole warps of digits
    P.blocks = (int)(((int64_t)n + SORT_TILE - 1) / SORT_TILE);
    // runs of 32 sorted tokens give every SM work from a few thousand tokens on; longer ones shorten the join of a hot id where there are plenty
    P.run = n <= (1 << 18) ? 32 : 128;
    P.runs = (int)(((int64_t)n + P.run - 1) / P.run);
    int64_t at = 0;
    auto take = [&](int64_t bytes) { char* p = base + at; at += (bytes + 255) & ~(int64_t)255; return (void*)p; };
    P.a = (int2*)take((int64_t)n * 8);
    P.b = (int2*)take((int64_t)n * 8);
    P.hist = (int*)take((int64_t)BINS * P.blocks * 4);
    P.total = (int*)take(BINS * 4);
    P.part = (float*)take((int64_t)P.runs * 2 * d * 4);
    return at;
}
static int lanes_for(int d, int per, int most)
{
    int l = 1;
    while (l < most && l * per < d) l <<= 1;
    return l;
}

template <int ITEMS> static cudaError_t sort_cluster(const int* ids, const Plan& P, int n, int vocab, bool* fits)
{
    constexpr int bytes = (CL_WARPS + 2) * BINS * 4;
    const auto kernel = sort_cluster_kernel<ITEMS>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = CL;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3(CL);
    c.blockDim = dim3(CL_THREADS);
    c.dynamicSmemBytes = bytes;
    c.stream = current_stream();
    c.attrs = &at;
    c.numAttrs = 1;
    if (fits) {
        int clusters = 0;
        *fits = cudaOccupancyMaxActiveClusters(&clusters, kernel, &c) == cudaSuccess && clusters > 0;
        cudaGetLastError();                      // a size that the device does not take is an answer, not an error
        return cudaSuccess;
    }
    return cudaLaunchKernelEx(&c, kernel, ids, P.a, P.b, n, vocab, P.passes, P.bits);
}
static bool sort_in_one(const int* ids, const Plan& P, int n, int vocab, const char* where)
{
    const int items = (n + CL * CL_THREADS - 1) / (CL * CL_THREADS);
    const cudaError_t e = items <= 2 ? sort_cluster<2>(ids, P, n, vocab, nullptr)
                          : items <= 4 ? sort_cluster<4>(ids, P, n, vocab, nullptr) : sort_cluster<8>(ids, P, n, vocab, nullptr);
    if (e != cudaSuccess) record_status(NLH_ERR_CUDA, where, cudaGetErrorString(e));
    return e == cudaSuccess;
}
// Whether the current device holds a cluster of sixteen of these CTAs; asked once per device.
static bool wide_clusters(const Plan& P)
{
    static std::atomic<int> known[64];           // 0: not asked, 1: no, 2: yes
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
    int k = known[dev].load(std::memory_order_relaxed);
    if (k == 0) {
        bool fits = false;
        if (sort_cluster<8>(nullptr, P, 0, 1, &fits) != cudaSuccess) { cudaGetLastError(); fits = false; }
        k = fits ? 2 : 1;
        known[dev].store(k, std::memory_order_relaxed);
    }
    return k == 2;
}

template <typename T, int N, bool ADD>
static bool backward(const T* dy, const int* ids, float* dw, int n, int vocab, int d, float scale, char* ws, const char* where)
{
    cudaStream_t st = current_stream();
    Plan P;
    place(P, ws, n, vocab, d);
    const int lanes = max(4, lanes_for(d, N, THREADS));         // four at least: the tokens of all runs of a CTA fit 48 KB
    if (one_launch(n, d)) {
        small_kernel<T, N, ADD><<<n, THREADS, 0, st>>>(dy, ids, dw, n, vocab, d, lanes, scale);
        return check_launch(where);
    }
    const int2* in = nullptr;
    if (n <= CL_MOST && wide_clusters(P)) {
        if (!sort_in_one(ids, P, n, vocab, where)) return false;
        in = P.passes & 1 ? P.a : P.b;
    } else {
        int2* out = P.a;
        for (int p = 0; p < P.passes; p++) {
            hist_kernel<<<P.blocks, SORT_THREADS, 0, st>>>(ids, in, P.hist, n, vocab, p * BITS, P.blocks);
            if (!check_launch(where)) return false;
            scan_kernel<<<BINS / 8, 256, 0, st>>>(P.hist, P.total, P.blocks);
            if (!check_launch(where)) return false;
            scatter_kernel<<<P.blocks, SORT_THREADS, 0, st>>>(ids, in, out, P.hist, P.total, n, vocab, p * BITS, P.blocks);
            if (!check_launch(where)) return false;
            in = out;
            out = out == P.a ? P.b : P.a;
        }
    }
    const int per = THREADS / lanes;
    const dim3 grid((P.runs + per - 1) / per, (d + lanes * N - 1) / (lanes * N));
    reduce_kernel<T, N, ADD><<<grid, THREADS, per * (P.run + 2) * sizeof(int2), st>>>(dy, in, dw, P.part, n, vocab, d, lanes, P.run, scale);
    if (!check_launch(where)) return false;
    join_kernel<N, ADD><<<dim3((P.runs + 7) / 8, (d + 32 * N - 1) / (32 * N)), 256, 0, st>>>(in, dw, P.part, n, vocab, d, P.run, scale);
    return check_launch(where);
}

template <typename T, int N> static bool lookup(const T* w, const int* ids, T* out, int n, int vocab, int d, float scale, const char* where)
{
    const int lanes = lanes_for(d, N, 32), per = 256 / lanes;
    const long long need = ((long long)n + per - 1) / per;
    lookup_kernel<T, N><<<(unsigned)(need < 148 * 32 ? need : 148 * 32), 256, 0, current_stream()>>>(w, ids, out, n, vocab, d, lanes, scale);
    return check_launch(where);
}

}  // namespace emb
}  // namespace nlh

using namespace nlh;

extern "C" {

int32_t nlh_embedding_forward(const void* w, int32_t w_is_bf16, const int32_t* ids, void* out, int32_t n, int32_t vocab, int32_t d,
    float scale)
{
    const char* where = "nlh_embedding_forward";
    if (n < 0 || vocab <= 0 || d <= 0 || d > emb::MAX_D || (n > 0 && (!w || !ids || !out))) {
        record_status(NLH_ERR_INVALID_ARG, where, "bad dimensions or NULL pointer");
        return NLH_ERR_INVALID_ARG;
    }
    if (n == 0) return NLH_OK;
    const bool vec = aligned16(w) && aligned16(out);
    bool ok;
    if (w_is_bf16) {
        typedef __nv_bfloat16 T;
        ok = vec && d % 8 == 0 ? emb::lookup<T, 8>((const T*)w, ids, (T*)out, n, vocab, d, scale, where)
                               : emb::lookup<T, 1>((const T*)w, ids, (T*)out, n, vocab, d, scale, where);
    } else {
        ok = vec && d % 4 == 0 ? emb::lookup<float, 4>((const float*)w, ids, (float*)out, n, vocab, d, scale, where)
                               : emb::lookup<float, 1>((const float*)w, ids, (float*)out, n, vocab, d, scale, where);
    }
    return ok ? NLH_OK : NLH_ERR_CUDA;
}

int64_t nlh_embedding_backward_bytes(int32_t n, int32_t vocab, int32_t d)
{
    if (n < 0 || n > emb::MAX_N || vocab <= 0 || d <= 0 || d > emb::MAX_D) return -1;
    emb::Plan P;
    return emb::place(P, nullptr, n, vocab, d);
}

int32_t nlh_embedding_backward(const void* d_out, int32_t d_out_is_bf16, const int32_t* ids, float* d_w, int32_t n, int32_t vocab,
    int32_t d, float scale, int32_t accumulate, void* workspace, int64_t workspace_bytes)
{
    const char* where = "nlh_embedding_backward";
    const int64_t need = nlh_embedding_backward_bytes(n, vocab, d);
    if (need < 0 || !d_w || (n > 0 && (!d_out || !ids)) || (need > 0 && (!workspace || !aligned16(workspace))) || workspace_bytes < need) {
        record_status(NLH_ERR_INVALID_ARG, where, "bad dimensions, NULL pointer, or a workspace that is too small or not 16-byte aligned");
        return NLH_ERR_INVALID_ARG;
    }
    if (!accumulate) {      // rows without a token
        const cudaError_t e = cudaMemsetAsync(d_w, 0, (size_t)vocab * d * 4, current_stream());
        if (e != cudaSuccess) { record_status(NLH_ERR_CUDA, where, cudaGetErrorString(e)); return NLH_ERR_CUDA; }
    }
    if (n == 0) return NLH_OK;
    const bool vec = aligned16(d_out) && aligned16(d_w);
    char* ws = (char*)workspace;
    bool ok;
#define NLH_EMB(T, N) (accumulate ? emb::backward<T, N, true>((const T*)d_out, ids, d_w, n, vocab, d, scale, ws, where) \
                                  : emb::backward<T, N, false>((const T*)d_out, ids, d_w, n, vocab, d, scale, ws, where))
    if (d_out_is_bf16) ok = vec && d % 8 == 0 ? NLH_EMB(__nv_bfloat16, 8) : NLH_EMB(__nv_bfloat16, 1);
    else ok = vec && d % 4 == 0 ? NLH_EMB(float, 4) : NLH_EMB(float, 1);
#undef NLH_EMB
    return ok ? NLH_OK : NLH_ERR_CUDA;
}

}  // extern "C"
