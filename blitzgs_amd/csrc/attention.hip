// Scaled dot-product attention, forward and backward.
//
//   forward    S = scale q k^T, P = softmax over the keys a row sees, o = P v
//   backward   delta = sum(do o),  dP = do v^T,  dS = P (dP - delta)
//              dv = P^T do,  dq = scale dS k,  dk = scale dS^T q
// Query i of batch b sees key j when j < key_lengths[b] and, when causal,
// j <= i + query_start[b].  A row that sees no key has o = 0 and no gradient.
//
// Nothing of size Tq x Tk is stored.  The forward walks the keys once with the
// running maximum and sum of the softmax and keeps one number per row, the
// logarithm (to base 2) of its sum of exponentials; the backward recomputes
// P = exp2(S scale log2(e) - lse) from it.
//
// Layout.  Every product keeps one side in a wave's registers as the columns
// of 16x16 matrix-core tiles and streams the other side through LDS as rows:
//   forward, dq: columns = queries.  S^T = k q^T leaves a query's scores in the
//     four lanes of its column, so the softmax is lane arithmetic with two
//     exchanges per 64 keys, and P^T is at once the right operand of
//     o^T = v^T P^T (dq^T = k^T dS^T), without a lane exchange.
//   dk, dv: columns = keys.  S = q k^T, then dv^T = do^T P and dk^T = q^T dS.
// The backward is two kernels that recompute S and dP each: seven products in
// place of five, but no gradient is summed by atomics, so the same inputs give
// the same bits, and no fp32 copy of dq goes through memory.
//
// The query heads that share a key head are rows of one matrix: their keys are
// read once for all of them, and dk and dv are summed over them in registers.
//
// Precision.  Scores, softmax statistics and all sums are fp32.  P and dS are
// rounded to the tensors' type as operands of the second product, which is the
// matrix core's operand type.  That adds to the rounding of the results themselves:
// o and the gradients are off by 0.0024 in bfloat16 and 0.00030 in float16, relative
// to their size, where rounding alone leaves 0.0017 and 0.00021 (float32: 4.4e-7).
// delta is subtracted from numbers of its own size, where a row looks at few keys,
// so a 16-bit forward also keeps what the rounding of o left, and delta is formed
// from both parts: in bfloat16 as many bits again, in float16 down to 2^-25, which
// for v of 2^-14 and more is below what the rounding of P has left in o.
//
// Bound and figures (bfloat16; a large library product reaches 1240 TFLOP/s on the
// card; after 200 passes, the first of which are up to 15 % slower).  Of a SIMD's
// cycles with work on its CU, the share with vector instructions issued and the share
// with the matrix core busy:
//   2 x 16 heads, 4096 x 4096, D 64
//     forward 183 us (752 TFLOP/s)                        64 %, 32 %
//     dq 197 us (1046 with its recomputation)             60 %, 50 %
//     dk, dv 276 us (997)                                 46 %, 42 %
//   16 heads on 4, 8192 causal, D 128
//     forward 308 us (891)                                53 %, 42 %
//     dq 380 us (1084)                                    46 %, 54 %
//     dk, dv 657 us (836), 22 to add                      32 %, 36 %, and LDS 41 %
// Neither is full: a wave's products, its exponentials and its second product follow
// one another, and two or three waves per SIMD do not cover all of that.  dk, dv want
// registers besides: 16 keys a wave at D = 128.  float16 takes the same but for fit().
//   8 x 32 heads on 8, one query, up to 32768 keys, D 128
//     104 us and 6 to join the splits (537 MB, 4.9 TB/s; a large copy: 5.15)
//   float32, 2 x 16 heads, 4096 x 4096, D 64
//     1098, 1535 and 2187 us (125, 134 and 126 TFLOP/s; a large library product: 153)
#include <algorithm>
#include <type_traits>

#include "gs_host.h"
#include "gs_matrix.h"
#include "../../include/blitzgs_amd.h"

namespace {

using gs::f4;
using gs::Frag;
using gs::Fill;
using gs::Stage;
using gs::Tile;

constexpr int BK = 64;   // rows of a streamed tile
constexpr float NEG_INF = -__builtin_inff();
constexpr float SLACK = 8.0f;   // of the softmax's running base, in powers of two
constexpr float LOG2E = 1.4426950408889634f;

// Workgroups per CU that the registers are shared out for; the tiles of wide fp32
// heads leave room for one in LDS.
template <typename T, int DP>
constexpr int PER_CU = sizeof(T) == 4 && DP > 64 ? 1 : 2;

struct Strides {
    int64_t b, h, t;
};

struct AttnArgs {
    const void *q, *k, *v, *o, *dout;
    void *out0, *out1;          // forward: o; dq: dq; dkv: dk, dv
    void* rest;                 // what rounding o to its type left, or null
    float* lse;                 // [B][Hq][Tq], base 2
    float* delta;               // [B][Hq][Tq]
    float* part;                // partial results of a split, or null
    float* part_ml;             // forward: (maximum, sum) of a split's row
    const int* key_lengths;
    const int* query_start;
    Strides qs, ks, vs, os, dos, s0, s1;
    int B, Hkv, G, Tq, Tk, D;
    int causal, splits, tiles;  // tiles: column tiles per (batch, key head)
    float scale, c;             // c = scale log2(e)
};

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// The sum and maximum over the four lanes of a column.
__device__ __forceinline__ float column_max(float v)
{
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float column_sum(float v)
{
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

__device__ __forceinline__ int length_of(const AttnArgs& A, int b)
{
    return A.key_lengths == nullptr ? A.Tk : max(0, min(A.Tk, A.key_lengths[b]));
}
__device__ __forceinline__ int64_t start_of(const AttnArgs& A, int b)
{
    return A.query_start == nullptr ? (int64_t)A.Tk - A.Tq : A.query_start[b];
}
// How many keys query i sees of `len`.
__device__ __forceinline__ int seen_of(const AttnArgs& A, int len, int64_t start, int i)
{
    if (!A.causal) return len;
    const int64_t n = start + i + 1;
    return n < 0 ? 0 : n < len ? (int)n : len;
}

// A workgroup's share: a column tile of one (batch, key head), and a split of
// its walk.  Where all tiles cost the same, each XCD gets a run of neighbours,
// which stream the same rows through its L2.  With a causal limit that holds for
// runs of whole heads only, else one XCD gets the costly half of a head; with
// key lengths it holds for none.  There the costliest tiles of all heads go
// first, dealt out in turn.  dk, dv of 4 key heads of 8192 keys, causal: 695 us,
// in runs 1181; 8 batches of up to 32768 keys, one query: 112 us, in runs 145.
struct Share {
    int bh, tile, split;
};

__device__ __forceinline__ Share share_of(const AttnArgs& A, int cost_heads)
{
    const uint32_t heads = (uint32_t)(A.B * A.Hkv), tiles = (uint32_t)A.tiles, splits = (uint32_t)A.splits;
    if (A.key_lengths == nullptr && (!A.causal || cost_heads % 8 == 0)) {
        const uint32_t item = gs::xcd_item(blockIdx.x, gridDim.x), rest = item / splits;
        return {(int)(rest / tiles), (int)(rest % tiles), (int)(item % splits)};
    }
    const uint32_t rest = blockIdx.x / splits;
    return {(int)(rest % heads), (int)(rest / heads), (int)(blockIdx.x % splits)};
}

// One column tile of the kernels whose columns are queries.
struct QueryTile {
    int b, hk, tile, split, bh;
    int len, seen_max, seen_min;   // keys that some / every row of the tile sees
    int t0, t1;                    // key tiles of this split
    int64_t start;
};

template <int COLS>
__device__ __forceinline__ QueryTile query_tile(const AttnArgs& A)
{
    QueryTile w;
    const Share share = share_of(A, A.B * A.Hkv * A.G);
    w.split = share.split;
    w.tile = A.tiles - 1 - share.tile;   // causal: the last tiles see the most keys
    w.bh = share.bh;
    w.b = w.bh / A.Hkv;
    w.hk = w.bh % A.Hkv;
    w.len = length_of(A, w.b);
    w.start = start_of(A, w.b);
    const int R = A.G * A.Tq, r0 = w.tile * COLS, r1 = min(R, r0 + COLS) - 1;
    const bool one_head = r0 / A.Tq == r1 / A.Tq;
    w.seen_max = seen_of(A, w.len, w.start, one_head ? r1 % A.Tq : A.Tq - 1);
    w.seen_min = seen_of(A, w.len, w.start, one_head ? r0 % A.Tq : 0);
    const int tiles = (w.seen_max + BK - 1) / BK, per = (tiles + A.splits - 1) / A.splits;
    w.t0 = min(tiles, w.split * per);
    w.t1 = min(tiles, w.t0 + per);
    return w;
}

// A query column of this lane: its head, position and the keys it sees.
struct Column {
    int r, h, i, seen;
    bool valid;
};

__device__ __forceinline__ Column column(const AttnArgs& A, const QueryTile& w, int r)
{
    Column c;
    const int R = A.G * A.Tq;
    c.r = r;
    c.valid = r < R;
    const int rr = c.valid ? r : 0;
    c.h = w.hk * A.G + rr / A.Tq;
    c.i = rr % A.Tq;
    c.seen = c.valid ? seen_of(A, w.len, w.start, c.i) : w.seen_max;
    return c;
}

// The first n of four neighbours; unless ODD, all of them or none.
template <bool ODD, typename T>
__device__ __forceinline__ void store4(T* p, f4 v, int n)
{
    if constexpr (!ODD) {
        if (n <= 0) return;
        T t[4];
#pragma unroll
        for (int r = 0; r < 4; r++) t[r] = (T)v[r];
        __builtin_memcpy(p, t, 4 * sizeof(T));
    } else {
#pragma unroll
        for (int r = 0; r < 4; r++)
            if (r < n) p[r] = (T)v[r];
    }
}

// o is a mean of values of v.  The rounding of P can leave it above the largest of them by
// 2^-11, which takes it from float16's largest numbers to infinity.
template <typename T>
__device__ __forceinline__ float mean_of(float x)
{
    if constexpr (__is_same(T, gs::f16))
        return fabsf(x) < -NEG_INF ? fminf(fmaxf(x, -65504.0f), 65504.0f) : x;
    return x;
}

// Four neighbours of o, and what their rounding leaves.
template <bool ODD, typename T>
__device__ __forceinline__ void store_o(T* p, T* rest, f4 v, int n)
{
#pragma unroll
    for (int r = 0; r < 4; r++) v[r] = mean_of<T>(v[r]);
    store4<ODD>(p, v, n);
    if (rest == nullptr) return;
    f4 left;
#pragma unroll
    for (int r = 0; r < 4; r++) left[r] = v[r] - (float)(T)v[r];
    store4<ODD>(rest, left, n);
}

// A weight of zero does not keep a NaN or an infinity of a tile's row from the
// columns that do not see the row.  So in the tiles that a mask cuts, put() makes
// such elements zero, and the columns that do see them get them after the walk,
// from memory.  With that work beside the product instead, under a branch that is
// never taken, its registers spilled; with a barrier of its own at the beginning of
// a step the 577 x 1025 forward took 34 us in place of 31.

// Adds to x those of the first n of four neighbours that are not finite.
template <typename T>
__device__ __forceinline__ void add_rest(f4& x, const T* p, int n)
{
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const float v = r < n ? (float)p[r] : 0.0f;
        if (!(fabsf(v) < -NEG_INF)) x[r] += v;
    }
}

// dS as an operand in float16.  It is as large as the gradients of o over the number of
// keys, and as the products of those with v, so both ends of float16's range are within
// reach: gradients of 1e-3 over 4096 keys left dq and dk with an error of 5.3e-3, of 1e4
// over 64 made them infinite.  So a column's dS is multiplied by a power of two, `up`,
// and its sum divided by it at the end.  As with the softmax's base, `up` falls when the
// column's largest dS so far asks for it: that keeps the largest between 2^7 and 2^15,
// and all of float16's bits in what is at least 2^-21 of it.  The error above becomes
// 6.9e-4, of which dq's own rounding is 6.6e-4; float16's dq, dk and dv take longer by it:
// 204 -> 225 and 285 -> 309 us at 2 x 16 heads of 4096 x 4096, D 64; 399 -> 416 and
// 681 -> 709 at 16 heads on 4 of 8192, causal, D 128.
template <typename T>
constexpr bool FITS = __is_same(T, gs::f16);
constexpr float UP = 0x1p60f;      // of columns that have met no dS yet
constexpr float UP_MOST = 0x1p15f; // of dS up

template <int U, int N, int DT>
__device__ __forceinline__ void fit(f4 (&ds)[U][N], f4 (&acc)[DT][N], float (&up)[N])
{
#pragma unroll
    for (int n = 0; n < N; n++) {
        float top = 0.0f;
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int r = 0; r < 4; r++) top = fmaxf(top, fabsf(ds[u][n][r]));
        if (__any(top * up[n] >= UP_MOST)) {
            top = column_max(top);
            // in powers of two: top up comes to between 2^7 and 2^8
            int to = 8 - __builtin_amdgcn_frexp_expf(top);
            const int from = __builtin_amdgcn_frexp_expf(up[n]) - 1;
            to = top * up[n] >= UP_MOST ? min(to, from) : from;
            up[n] = __builtin_ldexpf(1.0f, to);
            const float shrink = __builtin_ldexpf(1.0f, to - from);
#pragma unroll
            for (int d = 0; d < DT; d++) acc[d][n] *= shrink;
        }
#pragma unroll
        for (int u = 0; u < U; u++) ds[u][n] *= up[n];
    }
}

// P as an operand of dv in float16: about 1 over the number of keys, and float16 has fewer
// bits below 2^-14 (a probability of 2^-20 was off by up to 3 %).  The lse that dk, dv
// takes is smaller by P_UP: its P comes to at most 2^10, with all bits from 2^-24 on.
constexpr float P_UP = 10.0f, P_BACK = 0x1p-10f;

// The tile that is read and the one that is being loaded come to a step as two
// restricted pointers: only so does the compiler know that the loads need not
// have arrived before the reads.

// ------------------------------------------------------------------- forward

template <typename T, int DP, int NQ, Fill F>
__global__ __launch_bounds__(256, (PER_CU<T, DP>)) void attn_fwd_kernel(AttnArgs A)
{
    using L = Tile<T, DP>;
    constexpr int KC = DP / 32, DT = DP / 16, COLS = 64 * NQ, WORDS = BK * L::CHUNKS;
    extern __shared__ uint4 lds[];   // [2][k tile, v tile]
    __shared__ int found;            // whether put() made anything zero
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
    const L tile_of;
    const QueryTile w = query_tile<COLS>(A);
    const T* kb = (const T*)A.k + w.b * A.ks.b + w.hk * A.ks.h;
    const T* vb = (const T*)A.v + w.b * A.vs.b + w.hk * A.vs.h;

    Column col[NQ];
    Frag<T> q[NQ][KC];
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        col[n] = column(A, w, w.tile * COLS + (wave * NQ + n) * 16 + i);
        const T* p = (const T*)A.q + w.b * A.qs.b + col[n].h * A.qs.h + col[n].i * A.qs.t;
#pragma unroll
        for (int c = 0; c < KC; c++)
            q[n][c] = gs::frag_global<T, F == gs::ODD>(p + 32 * c + 8 * g, col[n].valid ? A.D - 32 * c - 8 * g : 0);
    }
    f4 o[DT][NQ];
    float m[NQ], l[NQ];
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        m[n] = NEG_INF;
        l[n] = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; d++) o[d][n] = f4{0, 0, 0, 0};
    }

    if (threadIdx.x == 0) found = 0;
    bool met = false;   // by this thread
    Stage<T, DP, BK, F> sk, sv;
    auto fetch = [&](int t, uint4* to) __attribute__((always_inline)) {
        sk.fetch(to, kb + (int64_t)t * BK * A.ks.t, A.ks.t, w.seen_max - t * BK, A.D);
        sv.fetch(to + WORDS, vb + (int64_t)t * BK * A.vs.t, A.vs.t, w.seen_max - t * BK, A.D);
    };
    auto put = [&](int t, uint4* to, bool cuts) __attribute__((always_inline)) {
        sk.put(to);
        met |= sv.put(to + WORDS, cuts && (t + 1) * BK > w.seen_min);
    };
    if (w.t0 < w.t1) {
#pragma unroll
        for (int k = 0; k < 4; k++) sk.clear(lds + k * WORDS, A.D);
        fetch(w.t0, lds);
        put(w.t0, lds, true);
    }
    __syncthreads();
    auto step = [&](auto cuts, int t, const uint4* __restrict__ kt, uint4* __restrict__ next)
                    __attribute__((always_inline)) {
        constexpr bool CUTS = decltype(cuts)::value;
        const uint4* vt = kt + WORDS;
        const int k0 = t * BK;
        if (t + 1 < w.t1) fetch(t + 1, next);
        f4 s[4][NQ];
#pragma unroll
        for (int u = 0; u < 4; u++) {
#pragma unroll
            for (int n = 0; n < NQ; n++) s[u][n] = f4{0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < KC; c++) {
                const Frag<T> a = tile_of.rows(kt, 16 * u, 32 * c);
#pragma unroll
                for (int n = 0; n < NQ; n++) s[u][n] = gs::mma(a, q[n][c], s[u][n]);
            }
        }
        // the parts stay apart, as the mask's branch keeps them (577 x 1025: 33 -> 31 us)
        if constexpr (!CUTS) __builtin_amdgcn_sched_barrier(0);
        if (CUTS && k0 + BK > w.seen_min) {
#pragma unroll
            for (int n = 0; n < NQ; n++)
#pragma unroll
                for (int u = 0; u < 4; u++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        if (k0 + 16 * u + 4 * g + r >= col[n].seen) s[u][n][r] = NEG_INF;
        }
#pragma unroll
        for (int n = 0; n < NQ; n++) {
            float top = s[0][n][0];
#pragma unroll
            for (int u = 0; u < 4; u++)
#pragma unroll
                for (int r = 0; r < 4; r++) top = fmaxf(top, s[u][n][r]);
            top = column_max(top) * A.c;
            // the base follows the maximum once that is 2^8 above it: sums and
            // products in between are larger by that much, which costs nothing
            if (__any(top > m[n] + SLACK)) {
                const float next = fmaxf(m[n], top);
                const float shrink = next == NEG_INF ? 1.0f : exp2_fast(m[n] - next);
                m[n] = next;
                l[n] *= shrink;
#pragma unroll
                for (int d = 0; d < DT; d++) o[d][n] *= shrink;
            }
            const float base = m[n] == NEG_INF ? 0.0f : m[n];
            float sum = 0.0f;
#pragma unroll
            for (int u = 0; u < 4; u++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    s[u][n][r] = exp2_fast(__builtin_fmaf(s[u][n][r], A.c, -base));
                    sum += s[u][n][r];
                }
            l[n] += sum;
        }
#pragma unroll
        for (int kk = 0; kk < 2; kk++) {
            Frag<T> p[NQ];
#pragma unroll
            for (int n = 0; n < NQ; n++) p[n] = gs::frag_of_tiles<T>(s[2 * kk][n], s[2 * kk + 1][n]);
#pragma unroll
            for (int d = 0; d < DT; d++) {
                const Frag<T> a = tile_of.cols(vt, 32 * kk, 16 * d);
#pragma unroll
                for (int n = 0; n < NQ; n++) o[d][n] = gs::mma(a, p[n], o[d][n]);
            }
        }
        if (t + 1 < w.t1) put(t + 1, next, CUTS);
        __syncthreads();
    };
    // tiles that no mask cuts, and whose next is none that one cuts, take a loop of
    // their own; at D <= 64 one loop schedules better (4096 keys of 64: 217 us, 226
    // in two; 8192 causal of 128: 330 and 326)
    int t = w.t0;
    if constexpr (DP > 64)
        for (const int whole = min(w.t1, w.seen_min / BK) - 1; t < whole; t++)
            step(std::false_type{}, t, lds + ((t - w.t0) & 1) * 2 * WORDS, lds + ((t + 1 - w.t0) & 1) * 2 * WORDS);
    for (; t < w.t1; t++)
        step(std::true_type{}, t, lds + ((t - w.t0) & 1) * 2 * WORDS, lds + ((t + 1 - w.t0) & 1) * 2 * WORDS);
    if (met) found = 1;
    __syncthreads();
    if (found) {
        // keys of the cut tiles
        const int from = max(w.t0 * BK, w.seen_min / BK * BK);
#pragma unroll
        for (int n = 0; n < NQ; n++)
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma nounroll
                for (int k = from; k < min(w.t1 * BK, col[n].seen); k++)
                    add_rest(o[d][n], vb + (int64_t)k * A.vs.t + 16 * d + 4 * g, A.D - 16 * d - 4 * g);
    }
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        const float sum = column_sum(l[n]);
        if (!col[n].valid) continue;
        const int64_t row = (int64_t)w.bh * A.G * A.Tq + col[n].r;   // = (b Hq + h) Tq + i
        if (A.part != nullptr) {
            const int64_t at = (int64_t)w.split * A.B * A.Hkv * A.G * A.Tq + row;
            float* p = A.part + at * A.D;
#pragma unroll
            for (int d = 0; d < DT; d++) store4<F == gs::ODD>(p + 16 * d + 4 * g, o[d][n], A.D - 16 * d - 4 * g);
            if (g == 0) {
                A.part_ml[2 * at] = m[n];
                A.part_ml[2 * at + 1] = sum;
            }
            continue;
        }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        const int64_t out = w.b * A.s0.b + col[n].h * A.s0.h + col[n].i * A.s0.t;
        T* rest = A.rest == nullptr ? nullptr : (T*)A.rest + out;
#pragma unroll
        for (int d = 0; d < DT; d++) {
            const int at = 16 * d + 4 * g;
            store_o<F == gs::ODD>((T*)A.out0 + out + at, rest == nullptr ? nullptr : rest + at, o[d][n] * inv,
                                  A.D - at);
        }
        if (g == 0 && A.lse != nullptr) A.lse[row] = sum == 0.0f ? -NEG_INF : m[n] + __builtin_log2f(sum);
    }
}

// Joins the splits of a row, W waves a row: wave w takes splits w, w + W, ...
// One wave where the rows alone fill the chip, 16 where few rows leave them the
// latency of many splits (8 rows of 128 splits: 14 us with four waves), else four.
template <typename T, int W>
__global__ __launch_bounds__(W > 4 ? 64 * W : 256) void attn_join_kernel(AttnArgs A)
{
    __shared__ float sums[W][130];
    const int64_t rows = (int64_t)A.B * A.Hkv * A.G * A.Tq;
    const int lane = threadIdx.x & 63, wave = W == 1 ? 0 : threadIdx.x >> 6;
    const int64_t row = W == 1 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
    if (row >= rows) return;
    const float* ml = A.part_ml + 2 * row;   // a split's maximum and sum, 2 rows apart
    float m = NEG_INF;
    for (int s = lane; s < A.splits; s += 64) m = fmaxf(m, ml[2 * s * rows]);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
    const float base = m == NEG_INF ? 0.0f : m;
    // of 64 of the wave's splits lane k keeps the k-th's factor
    float sum = 0.0f, o0 = 0.0f, o1 = 0.0f;
    for (int s0 = wave; s0 < A.splits; s0 += 64 * W) {
        const int s = s0 + W * lane, n = min(64, (A.splits - s0 + W - 1) / W);
        const float f = lane < n ? exp2_fast(ml[2 * s * rows] - base) : 0.0f;
        sum = __builtin_fmaf(lane < n ? ml[2 * s * rows + 1] : 0.0f, f, sum);
        const float* p = A.part + (s0 * rows + row) * A.D;
#pragma unroll 8
        for (int k = 0; k < n; k++) {
            const float fk = __shfl(f, k, 64);
            if (lane < A.D) o0 = __builtin_fmaf(p[lane], fk, o0);
            if (lane + 64 < A.D) o1 = __builtin_fmaf(p[lane + 64], fk, o1);
            p += W * rows * A.D;
        }
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d, 64);
    if constexpr (W > 1) {
        sums[wave][lane] = o0;
        sums[wave][64 + lane] = o1;
        if (lane == 0) sums[wave][128] = sum;
        __syncthreads();
        if (wave != 0) return;
        o0 = o1 = sum = 0.0f;
#pragma unroll
        for (int w = 0; w < W; w++) {
            o0 += sums[w][lane];
            o1 += sums[w][64 + lane];
            sum += sums[w][128];
        }
    }
    const uint32_t r = (uint32_t)row, i = r % (uint32_t)A.Tq, bh = r / (uint32_t)A.Tq, Hq = A.Hkv * A.G;
    const int64_t out = bh / Hq * A.s0.b + bh % Hq * A.s0.h + i * A.s0.t;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum, x0 = mean_of<T>(o0 * inv), x1 = mean_of<T>(o1 * inv);
    T *o = (T*)A.out0 + out, *rest = (T*)A.rest + out;
    if (lane < A.D) {
        o[lane] = (T)x0;
        if (A.rest != nullptr) rest[lane] = (T)(x0 - (float)(T)x0);
    }
    if (lane + 64 < A.D) {
        o[lane + 64] = (T)x1;
        if (A.rest != nullptr) rest[lane + 64] = (T)(x1 - (float)(T)x1);
    }
    if (lane == 0 && A.lse != nullptr) A.lse[row] = sum == 0.0f ? -NEG_INF : m + __builtin_log2f(sum);
}

// ------------------------------------------------------------------ backward

// dq, and delta for the other kernel.
template <typename T, int DP, int NQ, Fill F>
__global__ __launch_bounds__(256, (PER_CU<T, DP>)) void attn_dq_kernel(AttnArgs A)
{
    using L = Tile<T, DP>;
    constexpr int KC = DP / 32, DT = DP / 16, COLS = 64 * NQ, WORDS = BK * L::CHUNKS;
    extern __shared__ uint4 lds[];
    __shared__ int found;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
    const L tile_of;
    const QueryTile w = query_tile<COLS>(A);
    const T* kb = (const T*)A.k + w.b * A.ks.b + w.hk * A.ks.h;
    const T* vb = (const T*)A.v + w.b * A.vs.b + w.hk * A.vs.h;

    Column col[NQ];
    Frag<T> q[NQ][KC], go[NQ][KC];
    float lse[NQ], delta[NQ], up[NQ];
    f4 acc[DT][NQ];
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        up[n] = FITS<T> ? UP : 1.0f;
        col[n] = column(A, w, w.tile * COLS + (wave * NQ + n) * 16 + i);
        const T* p = (const T*)A.q + w.b * A.qs.b + col[n].h * A.qs.h + col[n].i * A.qs.t;
        const T* pg = (const T*)A.dout + w.b * A.dos.b + col[n].h * A.dos.h + col[n].i * A.dos.t;
        const int64_t oat = w.b * A.os.b + col[n].h * A.os.h + col[n].i * A.os.t;
        const T* po = (const T*)A.o + oat;
        const T* pr = (const T*)A.rest + oat;
        float d = 0.0f;
#pragma unroll
        for (int c = 0; c < KC; c++) {
            const int at = 32 * c + 8 * g, left = col[n].valid ? A.D - at : 0;
            q[n][c] = gs::frag_global<T, F == gs::ODD>(p + at, left);
            go[n][c] = gs::frag_global<T, F == gs::ODD>(pg + at, left);
            const Frag<T> fo = gs::frag_global<T, F == gs::ODD>(po + at, left);
            const Frag<T> fr = gs::frag_global<T, F == gs::ODD>(pr + at, A.rest == nullptr ? 0 : left);
            T a[8], b[8], e[8];
            __builtin_memcpy(a, &go[n][c], 8 * sizeof(T));
            __builtin_memcpy(b, &fo, 8 * sizeof(T));
            __builtin_memcpy(e, &fr, 8 * sizeof(T));
#pragma unroll
            for (int j = 0; j < 8; j++) d = __builtin_fmaf((float)a[j], (float)b[j] + (float)e[j], d);
        }
        delta[n] = column_sum(d);
        const int64_t row = (int64_t)w.bh * A.G * A.Tq + col[n].r;
        lse[n] = col[n].valid ? A.lse[row] : -NEG_INF;
        if (col[n].valid && g == 0 && w.split == 0) A.delta[row] = delta[n];
#pragma unroll
        for (int d2 = 0; d2 < DT; d2++) acc[d2][n] = f4{0, 0, 0, 0};
    }

    if (threadIdx.x == 0) found = 0;
    bool met = false;   // by this thread
    Stage<T, DP, BK, F> sk, sv;
    auto fetch = [&](int t, uint4* to) __attribute__((always_inline)) {
        sk.fetch(to, kb + (int64_t)t * BK * A.ks.t, A.ks.t, w.seen_max - t * BK, A.D);
        sv.fetch(to + WORDS, vb + (int64_t)t * BK * A.vs.t, A.vs.t, w.seen_max - t * BK, A.D);
    };
    auto put = [&](int t, uint4* to, bool cuts) __attribute__((always_inline)) {
        met |= sk.put(to, cuts && (t + 1) * BK > w.seen_min);
        sv.put(to + WORDS);
    };
    if (w.t0 < w.t1) {
#pragma unroll
        for (int k = 0; k < 4; k++) sk.clear(lds + k * WORDS, A.D);
        fetch(w.t0, lds);
        put(w.t0, lds, true);
    }
    __syncthreads();
    auto step = [&](auto cuts, int t, const uint4* __restrict__ kt, uint4* __restrict__ next)
                    __attribute__((always_inline)) {
        constexpr bool CUTS = decltype(cuts)::value;
        const uint4* vt = kt + WORDS;
        const int k0 = t * BK;
        if (!CUTS || t + 1 < w.t1) fetch(t + 1, next);
        const bool cut = CUTS && k0 + BK > w.seen_min;
#pragma unroll
        for (int kk = 0; kk < 2; kk++) {
            f4 s[2][NQ], dp[2][NQ];
#pragma unroll
            for (int u = 0; u < 2; u++) {
#pragma unroll
                for (int n = 0; n < NQ; n++) {
                    s[u][n] = f4{0, 0, 0, 0};
                    dp[u][n] = f4{-delta[n], -delta[n], -delta[n], -delta[n]};   // the sums start at -delta
                }
#pragma unroll
                for (int c = 0; c < KC; c++) {
                    const Frag<T> a = tile_of.rows(kt, 32 * kk + 16 * u, 32 * c);
                    const Frag<T> b = tile_of.rows(vt, 32 * kk + 16 * u, 32 * c);
#pragma unroll
                    for (int n = 0; n < NQ; n++) {
                        s[u][n] = gs::mma(a, q[n][c], s[u][n]);
                        dp[u][n] = gs::mma(b, go[n][c], dp[u][n]);
                    }
                }
            }
            if (cut) {
#pragma unroll
                for (int n = 0; n < NQ; n++)
#pragma unroll
                    for (int u = 0; u < 2; u++)
#pragma unroll
                        for (int r = 0; r < 4; r++)
                            if (k0 + 32 * kk + 16 * u + 4 * g + r >= col[n].seen) {
                                s[u][n][r] = NEG_INF;
                                dp[u][n][r] = 0.0f;
                            }
            }
            Frag<T> ds[NQ];
#pragma unroll
            for (int n = 0; n < NQ; n++)
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const float p = exp2_fast(__builtin_fmaf(s[u][n][r], A.c, -lse[n]));
                        s[u][n][r] = p * dp[u][n][r];
                    }
            if constexpr (FITS<T>) fit(s, acc, up);
#pragma unroll
            for (int n = 0; n < NQ; n++) ds[n] = gs::frag_of_tiles<T>(s[0][n], s[1][n]);
#pragma unroll
            for (int d = 0; d < DT; d++) {
                const Frag<T> a = tile_of.cols(kt, 32 * kk, 16 * d);
#pragma unroll
                for (int n = 0; n < NQ; n++) acc[d][n] = gs::mma(a, ds[n], acc[d][n]);
            }
        }
        if (!CUTS || t + 1 < w.t1) put(t + 1, next, CUTS);
        __syncthreads();
    };
    // as in the forward, at every D (4096 keys of 64: 219 us, in one loop 230)
    int t = w.t0;
    for (const int whole = min(w.t1, w.seen_min / BK) - 1; t < whole; t++)
        step(std::false_type{}, t, lds + ((t - w.t0) & 1) * 2 * WORDS, lds + ((t + 1 - w.t0) & 1) * 2 * WORDS);
    for (; t < w.t1; t++)
        step(std::true_type{}, t, lds + ((t - w.t0) & 1) * 2 * WORDS, lds + ((t + 1 - w.t0) & 1) * 2 * WORDS);
    if (met) found = 1;
    __syncthreads();
    if (found) {
        // a query that sees a key that is not finite has no gradient that is
        const int from = max(w.t0 * BK, w.seen_min / BK * BK);
#pragma unroll
        for (int n = 0; n < NQ; n++) {
            float x = 0.0f;
#pragma nounroll
            for (int k = from; k < min(w.t1 * BK, col[n].seen); k++)
#pragma nounroll
                for (int d = 0; d < A.D; d++) x += 0.0f * (float)kb[(int64_t)k * A.ks.t + d];
#pragma unroll
            for (int d = 0; d < DT; d++) acc[d][n] += x;
        }
    }
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        if (!col[n].valid) continue;
        const float scale = A.scale / up[n];
        if (A.part != nullptr) {
            const int64_t rows = (int64_t)A.B * A.Hkv * A.G * A.Tq;
            float* p = A.part + (w.split * rows + (int64_t)w.bh * A.G * A.Tq + col[n].r) * A.D;
#pragma unroll
            for (int d = 0; d < DT; d++)
                store4<F == gs::ODD>(p + 16 * d + 4 * g, acc[d][n] * scale, A.D - 16 * d - 4 * g);
        } else {
            T* p = (T*)A.out0 + w.b * A.s0.b + col[n].h * A.s0.h + col[n].i * A.s0.t;
#pragma unroll
            for (int d = 0; d < DT; d++)
                store4<F == gs::ODD>(p + 16 * d + 4 * g, acc[d][n] * scale, A.D - 16 * d - 4 * g);
        }
    }
}

// dk and dv.  A wave holds 16 NK keys; the block streams the queries of every
// head that shares them, QT rows at a time.
template <typename T, int DP, int NK, int QT, Fill F>
__global__ __launch_bounds__(256, (PER_CU<T, DP>)) void attn_dkv_kernel(AttnArgs A)
{
    using L = Tile<T, DP>;
    constexpr float p_up = FITS<T> ? P_UP : 0.0f, p_back = FITS<T> ? P_BACK : 1.0f;
    constexpr int KC = DP / 32, DT = DP / 16, COLS = 64 * NK, WORDS = QT * L::CHUNKS, BUF = 2 * WORDS + QT / 2;
    extern __shared__ uint4 lds[];   // [2][q tile, do tile, lse[QT], -delta[QT]]
    __shared__ int found;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
    const L tile_of;
    const Share share = share_of(A, A.B * A.Hkv);
    const int split = share.split, tile = share.tile, bh = share.bh;   // causal: the first keys are seen most
    const int b = bh / A.Hkv, hk = bh % A.Hkv, key0 = tile * COLS;
    const int64_t start = start_of(A, b);
    const int len = seen_of(A, length_of(A, b), start, A.Tq - 1);   // keys that the last query sees

    Frag<T> k[NK][KC], v[NK][KC];
    f4 dk[DT][NK], dv[DT][NK];
    float up[NK];
    int key[NK];
#pragma unroll
    for (int n = 0; n < NK; n++) {
        up[n] = FITS<T> ? UP : 1.0f;
        key[n] = key0 + (wave * NK + n) * 16 + i;
        const bool held = key[n] < len;
        const T* pk = (const T*)A.k + b * A.ks.b + hk * A.ks.h + (int64_t)(held ? key[n] : 0) * A.ks.t;
        const T* pv = (const T*)A.v + b * A.vs.b + hk * A.vs.h + (int64_t)(held ? key[n] : 0) * A.vs.t;
#pragma unroll
        for (int c = 0; c < KC; c++) {
            const int at = 32 * c + 8 * g, left = held ? A.D - at : 0;
            k[n][c] = gs::frag_global<T, F == gs::ODD>(pk + at, left);
            v[n][c] = gs::frag_global<T, F == gs::ODD>(pv + at, left);
        }
#pragma unroll
        for (int d = 0; d < DT; d++) dk[d][n] = dv[d][n] = f4{0, 0, 0, 0};
    }

    // the first query tile that sees the block's first key
    const int64_t first = A.causal ? (int64_t)key0 - start : 0;
    const int tiles = (A.Tq + QT - 1) / QT;
    const int from = key0 >= len ? tiles : first <= 0 ? 0 : first >= A.Tq ? tiles : (int)first / QT;
    const int per_head = tiles - from, total = per_head * A.G, per = (total + A.splits - 1) / A.splits;
    const int e0 = min(total, split * per), e1 = min(total, e0 + per);

    if (threadIdx.x == 0) found = 0;
    bool met = false;   // by this thread
    Stage<T, DP, QT, F> sq, sg;
    // threads 0 .. QT - 1: lse, QT .. 2 QT - 1: delta, as loaded; put() finishes them,
    // so that nothing waits for them, and the tiles' loads before them, until then
    float stat = 0.0f;
    bool real = false;
    const bool is_lse = threadIdx.x < QT;
    auto fetch = [&](int e, uint4* to) __attribute__((always_inline)) {
        const int h = hk * A.G + e / per_head, q0 = (from + e % per_head) * QT, n = A.Tq - q0;
        sq.fetch(to, (const T*)A.q + b * A.qs.b + h * A.qs.h + (int64_t)q0 * A.qs.t, A.qs.t, n, A.D);
        sg.fetch(to + WORDS, (const T*)A.dout + b * A.dos.b + h * A.dos.h + (int64_t)q0 * A.dos.t, A.dos.t, n, A.D);
        if (threadIdx.x < 2 * QT) {
            const int r = threadIdx.x % QT;
            const int64_t row = ((int64_t)b * A.Hkv * A.G + h) * A.Tq + q0 + min(r, n - 1);
            real = r < n;
            stat = *((is_lse ? A.lse : A.delta) + row);
        }
    };
    auto put = [&](int e, uint4* to) __attribute__((always_inline)) {
        const bool part = A.causal && start + (from + e % per_head) * QT < (int64_t)key0 + COLS - 1;
        met |= sq.put(to, part);
        met |= sg.put(to + WORDS, part);
        if (threadIdx.x < 2 * QT)
            ((float*)(to + 2 * WORDS))[threadIdx.x] = is_lse ? (real ? stat - p_up : -NEG_INF) : real ? -stat : 0.0f;
    };
    if (e0 < e1) {
#pragma unroll
        for (int k = 0; k < 4; k++) sq.clear(lds + k / 2 * BUF + k % 2 * WORDS, A.D);
        fetch(e0, lds);
        put(e0, lds);
    }
    __syncthreads();
    auto step = [&](int e, const uint4* __restrict__ qt, uint4* __restrict__ next) __attribute__((always_inline)) {
        const uint4* gt = qt + WORDS;
        const float* st = (const float*)(gt + WORDS);
        const int q0 = (from + e % per_head) * QT;
        if (e + 1 < e1) fetch(e + 1, next);
        // row r of the tile sees key `key` when r >= sees + key - key0
        const bool part = A.causal && start + q0 < (int64_t)key0 + COLS - 1;
        const int sees = part ? (int)(key0 - start - q0) : 0;   // between -COLS and QT
#pragma unroll
        for (int kk = 0; kk < QT / 32; kk++) {
            f4 s[2][NK], dp[2][NK];
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const f4 delta = *(const f4*)(st + QT + 32 * kk + 16 * u + 4 * g);
#pragma unroll
                for (int n = 0; n < NK; n++) {
                    s[u][n] = f4{0, 0, 0, 0};
                    dp[u][n] = delta;   // the sums start at -delta
                }
#pragma unroll
                for (int c = 0; c < KC; c++) {
                    const Frag<T> a = tile_of.rows(qt, 32 * kk + 16 * u, 32 * c);
                    const Frag<T> d = tile_of.rows(gt, 32 * kk + 16 * u, 32 * c);
#pragma unroll
                    for (int n = 0; n < NK; n++) {
                        s[u][n] = gs::mma(a, k[n][c], s[u][n]);
                        dp[u][n] = gs::mma(d, v[n][c], dp[u][n]);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int r0 = 32 * kk + 16 * u + 4 * g;
                const f4 lse = *(const f4*)(st + r0);
#pragma unroll
                for (int n = 0; n < NK; n++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const float p = exp2_fast(__builtin_fmaf(s[u][n][r], A.c, -lse[r]));
                        s[u][n][r] = p;
                        dp[u][n][r] = p * dp[u][n][r];
                    }
            }
            if (part) {
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int n = 0; n < NK; n++)
#pragma unroll
                        for (int r = 0; r < 4; r++)
                            if (32 * kk + 16 * u + 4 * g + r < sees + key[n] - key0) s[u][n][r] = dp[u][n][r] = 0.0f;
            }
            if constexpr (FITS<T>) fit(dp, dk, up);
            Frag<T> fp[NK], fs[NK];
#pragma unroll
            for (int n = 0; n < NK; n++) {
                fp[n] = gs::frag_of_tiles<T>(s[0][n], s[1][n]);
                fs[n] = gs::frag_of_tiles<T>(dp[0][n], dp[1][n]);
            }
#pragma unroll
            for (int d = 0; d < DT; d++) {
                const Frag<T> a = tile_of.cols(gt, 32 * kk, 16 * d), c = tile_of.cols(qt, 32 * kk, 16 * d);
#pragma unroll
                for (int n = 0; n < NK; n++) {
                    dv[d][n] = gs::mma(a, fp[n], dv[d][n]);
                    dk[d][n] = gs::mma(c, fs[n], dk[d][n]);
                }
            }
        }
        if (e + 1 < e1) put(e + 1, next);
        __syncthreads();
    };
    for (int e = e0; e < e1; e++) step(e, lds + ((e - e0) & 1) * BUF, lds + ((e + 1 - e0) & 1) * BUF);
    if (met) found = 1;
    __syncthreads();
    if (found) {
        // dv; to dk such a query's delta or lse has brought it already
#pragma unroll
        for (int n = 0; n < NK; n++)
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma nounroll
                for (int e = e0; e < e1; e++) {
                    const int h = hk * A.G + e / per_head, q0 = (from + e % per_head) * QT;
                    if (start + q0 >= (int64_t)key0 + COLS - 1) continue;   // not cut
                    const int64_t first_row = (int64_t)key[n] - start;
#pragma nounroll
                    for (int r = (int)max((int64_t)q0, first_row); r < min(A.Tq, q0 + QT); r++)
                        add_rest(dv[d][n], (const T*)A.dout + b * A.dos.b + h * A.dos.h + (int64_t)r * A.dos.t + 16 * d +
                                               4 * g, A.D - 16 * d - 4 * g);
                }
    }
#pragma unroll
    for (int n = 0; n < NK; n++) {
        if (key[n] >= A.Tk) continue;
        const bool held = key[n] < len;
        const float scale = A.scale / up[n] * p_back;
#pragma unroll
        for (int d = 0; d < DT; d++) {
            const int at = 16 * d + 4 * g, left = A.D - at;
            const f4 xk = held ? dk[d][n] * scale : f4{0, 0, 0, 0}, xv = held ? dv[d][n] * p_back : f4{0, 0, 0, 0};
            if (A.part != nullptr) {
                const int64_t rows = (int64_t)A.B * A.Hkv * A.Tk, row = (int64_t)bh * A.Tk + key[n];
                store4<F == gs::ODD>(A.part + (2 * split * rows + row) * A.D + at, xk, left);
                store4<F == gs::ODD>(A.part + ((2 * split + 1) * rows + row) * A.D + at, xv, left);
            } else {
                store4<F == gs::ODD>((T*)A.out0 + b * A.s0.b + hk * A.s0.h + (int64_t)key[n] * A.s0.t + at, xk, left);
                store4<F == gs::ODD>((T*)A.out1 + b * A.s1.b + hk * A.s1.h + (int64_t)key[n] * A.s1.t + at, xv, left);
            }
        }
    }
}

// Adds the splits' partial gradients: [splits][per][rows = B H Tn][D] to each of
// `per` tensors; a wave per row, its splits in order.
template <typename T>
__global__ __launch_bounds__(256) void attn_add_kernel(const float* __restrict__ part, int splits, int per,
                                                       int64_t rows, int H, int Tn, int D, T* out0, T* out1,
                                                       Strides s0, Strides s1)
{
    const int lane = threadIdx.x & 63, which = blockIdx.y;
    const Strides st = which == 0 ? s0 : s1;
    T* out = which == 0 ? out0 : out1;
    for (int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); row < rows; row += (int64_t)gridDim.x * 4) {
        float x0 = 0.0f, x1 = 0.0f;
        const float* p = part + (which * rows + row) * D;
#pragma unroll 8
        for (int k = 0; k < splits; k++, p += per * rows * D) {
            if (lane < D) x0 += p[lane];
            if (lane + 64 < D) x1 += p[lane + 64];
        }
        const uint32_t r = (uint32_t)row, t = r % (uint32_t)Tn, bh = r / (uint32_t)Tn, h = bh % H, b = bh / H;
        T* to = out + b * st.b + h * st.h + t * st.t;
        if (lane < D) to[lane] = (T)x0;
        if (lane + 64 < D) to[lane + 64] = (T)x1;
    }
}

// ------------------------------------------------------------------ launching

// Workgroups that keep the chip's 256 CUs busy at two per CU, with a second
// round to even out their ends.
constexpr int ENOUGH = 1024;

int padded(int D) { return (D + 31) / 32 * 32; }

// Splits of a walk of `steps` tiles when there are `blocks` column tiles: up to
// `enough` workgroups.  A split's partial results cost as much as `least` steps,
// which is as short as one gets.  With a tile per CU already, only long walks of
// unequal cost are split, none shorter than 32 (256 tiles of 32 steps: 37 us in
// two splits and 41 us to join them; whole, in 512 half as wide tiles, 41 us).
int splits_of(int64_t blocks, int steps, int least, int64_t enough, bool unequal)
{
    if (blocks >= ENOUGH / 4) {
        if (!unequal || blocks >= ENOUGH) return 1;
        least = 32;
    }
    if (steps < 2 * least) return 1;
    const int64_t want = (enough + blocks - 1) / blocks;
    return (int)std::max<int64_t>(1, std::min<int64_t>(want, steps / least));
}

enum Walk { FORWARD, DQ, DKV };

// Whether a wave's registers hold 32 columns, which halve the LDS reads per
// product, or 16.
constexpr bool two_columns(Walk w, bool f32, int DP) { return w == DKV ? DP <= (f32 ? 32 : 64) : !(f32 && DP > 64); }

// How the three walks of one problem are cut.
struct Plan {
    int nq, nk, splits_f, splits_q, splits_k, qt;
    size_t fwd_bytes, bwd_bytes;
};

Plan plan_of(int type, int B, int Hkv, int G, int Tq, int Tk, int D, bool unequal)
{
    Plan p{};
    const int DP = padded(D);
    const int64_t heads = (int64_t)B * Hkv, rows = (int64_t)G * Tq;
    // 16 columns also where 32 would leave less than two workgroups per CU, and for
    // head dimensions that end inside 16 bytes
    const bool whole = D % (16 / gs::dtype_bytes(type)) == 0, f32 = type == GS_F32;
    p.nq = whole && two_columns(DQ, f32, DP) && heads * ((rows + 127) / 128) >= ENOUGH / 2 ? 2 : 1;
    p.nk = whole && two_columns(DKV, f32, DP) && heads * (((int64_t)Tk + 127) / 128) >= ENOUGH / 2 ? 2 : 1;
    p.qt = 64;
    const int64_t tiles_q = (rows + 64 * p.nq - 1) / (64 * p.nq), tiles_k = ((int64_t)Tk + 64 * p.nk - 1) / (64 * p.nk);
    p.splits_f = p.splits_q = splits_of(heads * tiles_q, (Tk + BK - 1) / BK, 4, unequal ? 2 * ENOUGH : ENOUGH, unequal);
    const int64_t steps_k = (int64_t)G * ((Tq + p.qt - 1) / p.qt);
    p.splits_k = splits_of(heads * tiles_k, (int)std::min<int64_t>(steps_k, 1 << 20), 8, ENOUGH, unequal);
    const size_t all = (size_t)heads * (size_t)rows;
    p.fwd_bytes = p.splits_f > 1 ? (size_t)p.splits_f * all * (size_t)(D + 2) * 4 : 0;
    const size_t dq = p.splits_q > 1 ? (size_t)p.splits_q * all * (size_t)D * 4 : 0;
    const size_t dkv = p.splits_k > 1 ? (size_t)p.splits_k * 2 * (size_t)heads * (size_t)Tk * (size_t)D * 4 : 0;
    p.bwd_bytes = (all * 4 + 255) / 256 * 256 + std::max(dq, dkv);   // delta, then one walk's partial results
    return p;
}

template <typename K>
int launch(const char* name, K kernel, int64_t blocks, size_t lds, const AttnArgs& A, hipStream_t stream)
{
    GS_REQUIRE(blocks < (1 << 24), "attention: too many workgroups for one launch");
    if (lds > 65536)
        GS_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    GS_TIMED(name, stream, hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), lds, stream, A));
    GS_LAUNCH_CHECK(name);
    return GS_OK;
}

template <typename T, int DP, int NQ, Fill F>
int forward_one(const AttnArgs& A, hipStream_t stream)
{
    const size_t lds = (size_t)4 * BK * Tile<T, DP>::CHUNKS * 16;
    return launch("attn_fwd_kernel", attn_fwd_kernel<T, DP, NQ, F>, (int64_t)A.B * A.Hkv * A.tiles * A.splits, lds, A,
                  stream);
}

template <typename T, int DP, int NQ, Fill F>
int dq_one(const AttnArgs& A, hipStream_t stream)
{
    const size_t lds = (size_t)4 * BK * Tile<T, DP>::CHUNKS * 16;
    return launch("attn_dq_kernel", attn_dq_kernel<T, DP, NQ, F>, (int64_t)A.B * A.Hkv * A.tiles * A.splits, lds, A,
                  stream);
}

template <typename T, int DP, int NK, Fill F>
int dkv_one(const AttnArgs& A, hipStream_t stream)
{
    constexpr int QT = 64;
    const size_t lds = (size_t)2 * (2 * QT * Tile<T, DP>::CHUNKS + QT / 2) * 16;
    return launch("attn_dkv_kernel", attn_dkv_kernel<T, DP, NK, QT, F>, (int64_t)A.B * A.Hkv * A.tiles * A.splits,
                  lds, A, stream);
}

template <Walk W, typename T, int DP, int N, Fill F>
int run_one(AttnArgs A, hipStream_t stream)
{
    const int64_t columns = W == DKV ? A.Tk : (int64_t)A.G * A.Tq;
    A.tiles = (int)((columns + 64 * N - 1) / (64 * N));
    if constexpr (W == FORWARD) return forward_one<T, DP, N, F>(A, stream);
    else if constexpr (W == DQ) return dq_one<T, DP, N, F>(A, stream);
    else return dkv_one<T, DP, N, F>(A, stream);
}

// Whether a walk's streamed rows may be loaded straight to LDS: all but views at
// odd addresses, for which 16 columns per wave are enough.
bool direct(const void* p, const Strides& s, int elem)
{
    const int64_t v = 16 / elem;
    return ((uintptr_t)p & 15) == 0 && s.b % v == 0 && s.h % v == 0 && s.t % v == 0 && s.t >= 0 &&
           s.t * elem * BK < (1ll << 31);
}

template <Walk W, typename T, int DP>
int run_width(const AttnArgs& A, int wide, hipStream_t stream)
{
    if (A.D % gs::Vec<T>::N != 0) return run_one<W, T, DP, 1, gs::ODD>(A, stream);
    const bool aligned = W == DKV ? direct(A.q, A.qs, sizeof(T)) && direct(A.dout, A.dos, sizeof(T))
                                  : direct(A.k, A.ks, sizeof(T)) && direct(A.v, A.vs, sizeof(T));
    if (!aligned) return run_one<W, T, DP, 1, gs::WHOLE>(A, stream);
    if constexpr (two_columns(W, sizeof(T) == 4, DP))
        if (wide == 2) return run_one<W, T, DP, 2, gs::DIRECT>(A, stream);
    return run_one<W, T, DP, 1, gs::DIRECT>(A, stream);
}

template <Walk W, typename T>
int run_type(const AttnArgs& A, int wide, hipStream_t stream)
{
    switch (padded(A.D)) {
        case 32: return run_width<W, T, 32>(A, wide, stream);
        case 64: return run_width<W, T, 64>(A, wide, stream);
        case 96: return run_width<W, T, 96>(A, wide, stream);
        default: return run_width<W, T, 128>(A, wide, stream);
    }
}

template <Walk W>
int run(int type, const AttnArgs& A, int wide, hipStream_t stream)
{
    if (type == GS_F32) return run_type<W, float>(A, wide, stream);
    if (type == GS_BF16) return run_type<W, gs::bf16>(A, wide, stream);
    return run_type<W, gs::f16>(A, wide, stream);
}

template <typename T>
void join(const AttnArgs& A, hipStream_t stream)
{
    const int64_t rows = (int64_t)A.B * A.Hkv * A.G * A.Tq;
    if (rows >= 4096)
        GS_TIMED("attn_join_kernel", stream,
                 hipLaunchKernelGGL((attn_join_kernel<T, 1>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream,
                                    A));
    else if (rows < 512 && A.splits > 16)
        GS_TIMED("attn_join_kernel", stream,
                 hipLaunchKernelGGL((attn_join_kernel<T, 16>), dim3((unsigned)rows), dim3(1024), 0, stream, A));
    else
        GS_TIMED("attn_join_kernel", stream,
                 hipLaunchKernelGGL((attn_join_kernel<T, 4>), dim3((unsigned)rows), dim3(256), 0, stream, A));
}

template <typename T>
void add(const AttnArgs& A, int per, int H, int Tn, hipStream_t stream)
{
    const int64_t rows = (int64_t)A.B * H * Tn, blocks = std::min<int64_t>((rows + 3) / 4, 1 << 20);
    GS_TIMED("attn_add_kernel", stream,
             hipLaunchKernelGGL(attn_add_kernel<T>, dim3((unsigned)blocks, (unsigned)per), dim3(256), 0, stream, A.part,
                                A.splits, per, rows, H, Tn, A.D, (T*)A.out0, (T*)A.out1, A.s0, A.s1));
}

Strides strides_of(const int64_t* s) { return {s[0], s[1], s[2]}; }

int check(int type, int B, int Hq, int Hkv, int Tq, int Tk, int D, float scale)
{
    GS_REQUIRE(gs::dtype_known(type), "attention: unknown element type %d", type);
    GS_REQUIRE(B >= 0 && Tq >= 0 && Tk >= 0, "attention: sizes must not be negative");
    GS_REQUIRE(Hkv >= 1 && Hq >= Hkv && Hq % Hkv == 0,
               "attention: the number of query heads (%d) must be a multiple of the number of key heads (%d)", Hq, Hkv);
    GS_REQUIRE(D >= 1 && D <= 128, "attention: the head dimension must be in [1, 128], got %d", D);
    GS_REQUIRE(scale > 0.0f && scale * LOG2E < -NEG_INF, "attention: scale must be a positive number below 2.3e38");
    GS_REQUIRE((int64_t)(Hq / Hkv) * Tq < 0x7fffff00ll && Tk < 0x7fffff00,
               "attention: too many queries or keys for one head");
    GS_REQUIRE((int64_t)B * Hq * Tq < (1ll << 32) && (int64_t)B * Hkv * Tk < (1ll << 32),
               "attention: too many rows");
    return GS_OK;
}

AttnArgs args_of(int B, int Hq, int Hkv, int Tq, int Tk, int D, float scale, int causal, const int* key_lengths,
                 const int* query_start)
{
    AttnArgs A{};
    A.B = B;
    A.Hkv = Hkv;
    A.G = Hq / Hkv;
    A.Tq = Tq;
    A.Tk = Tk;
    A.D = D;
    A.scale = scale;
    A.c = scale * LOG2E;
    A.causal = causal != 0;
    A.key_lengths = key_lengths;
    A.query_start = query_start;
    return A;
}

}  // namespace

extern "C" size_t gs_attention_workspace_bytes(int type, int B, int Hq, int Hkv, int Tq, int Tk, int D, int unequal,
                                               int backward)
{
    if (check(type, B, Hq, Hkv, Tq, Tk, D, 1.0f) != GS_OK) return 0;
    const Plan p = plan_of(type, B, Hkv, Hq / Hkv, Tq, Tk, D, unequal != 0);
    return backward ? p.bwd_bytes : p.fwd_bytes;
}

extern "C" int gs_attention_forward(int type, int B, int Hq, int Hkv, int Tq, int Tk, int D, const void* q,
                                    const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v,
                                    const int64_t* v_strides, float scale, int causal, const int* key_lengths,
                                    const int* query_start, void* o, const int64_t* o_strides, void* o_rest,
                                    float* lse, void* workspace, hipStream_t stream)
{
    gs::clear_error();
    if (int rc = check(type, B, Hq, Hkv, Tq, Tk, D, scale)) return rc;
    if (B == 0 || Tq == 0) return GS_OK;
    GS_REQUIRE(q && o && q_strides && k_strides && v_strides && o_strides,
               "attention: q, o and all strides must be given");
    GS_REQUIRE(Tk == 0 || (k && v), "attention: k and v must be non-null");
    const Plan p = plan_of(type, B, Hkv, Hq / Hkv, Tq, Tk, D, causal || key_lengths);
    GS_REQUIRE(p.splits_f == 1 || workspace != nullptr, "attention: this size needs the workspace");
    AttnArgs A = args_of(B, Hq, Hkv, Tq, Tk, D, scale, causal, key_lengths, query_start);
    A.q = q;
    A.k = k;
    A.v = v;
    A.out0 = o;
    A.rest = o_rest;
    A.lse = lse;
    A.qs = strides_of(q_strides);
    A.ks = strides_of(k_strides);
    A.vs = strides_of(v_strides);
    A.s0 = strides_of(o_strides);
    A.splits = p.splits_f;
    if (A.splits > 1) {
        A.part = (float*)workspace;
        A.part_ml = A.part + (size_t)A.splits * B * Hq * (size_t)Tq * D;
    }
    if (int rc = run<FORWARD>(type, A, p.nq, stream)) return rc;
    if (A.splits > 1) {
        if (type == GS_F32) join<float>(A, stream);
        else if (type == GS_BF16) join<gs::bf16>(A, stream);
        else join<gs::f16>(A, stream);
        GS_LAUNCH_CHECK("attn_join_kernel");
    }
    return GS_OK;
}

extern "C" int gs_attention_backward(int type, int B, int Hq, int Hkv, int Tq, int Tk, int D, const void* q,
                                     const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v,
                                     const int64_t* v_strides, float scale, int causal, const int* key_lengths,
                                     const int* query_start, const void* o, const int64_t* o_strides,
                                     const void* o_rest, const float* lse, const void* dout,
                                     const int64_t* dout_strides, void* dq, const int64_t* dq_strides, void* dk,
                                     const int64_t* dk_strides, void* dv, const int64_t* dv_strides,
                                     void* workspace, hipStream_t stream)
{
    gs::clear_error();
    if (int rc = check(type, B, Hq, Hkv, Tq, Tk, D, scale)) return rc;
    if (B == 0 || (Tq == 0 && Tk == 0)) return GS_OK;
    GS_REQUIRE(q_strides && k_strides && v_strides && o_strides && dout_strides && dq_strides && dk_strides &&
                   dv_strides,
               "attention: all strides must be given");
    GS_REQUIRE(Tq == 0 || (q && o && lse && dout && dq), "attention: q, o, lse, dout and dq must be non-null");
    GS_REQUIRE(Tk == 0 || (k && v), "attention: k and v must be non-null");
    GS_REQUIRE((dk == nullptr) == (dv == nullptr), "attention: dk and dv come together");
    const Plan p = plan_of(type, B, Hkv, Hq / Hkv, Tq, Tk, D, causal || key_lengths);
    GS_REQUIRE(p.bwd_bytes == 0 || workspace != nullptr, "attention: the backward needs the workspace");
    AttnArgs A = args_of(B, Hq, Hkv, Tq, Tk, D, scale, causal, key_lengths, query_start);
    A.q = q;
    A.k = k;
    A.v = v;
    A.o = o;
    A.rest = const_cast<void*>(o_rest);
    A.dout = dout;
    A.lse = const_cast<float*>(lse);
    A.delta = (float*)workspace;
    A.qs = strides_of(q_strides);
    A.ks = strides_of(k_strides);
    A.vs = strides_of(v_strides);
    A.os = strides_of(o_strides);
    A.dos = strides_of(dout_strides);
    float* part = (float*)((char*)workspace + ((size_t)B * Hq * (size_t)Tq * 4 + 255) / 256 * 256);
    auto add_all = [&](int per, int H, int Tn) {
        if (type == GS_F32) add<float>(A, per, H, Tn, stream);
        else if (type == GS_BF16) add<gs::bf16>(A, per, H, Tn, stream);
        else add<gs::f16>(A, per, H, Tn, stream);
    };
    if (Tq > 0) {
        A.out0 = dq;
        A.s0 = strides_of(dq_strides);
        A.splits = p.splits_q;
        A.part = A.splits > 1 ? part : nullptr;
        if (int rc = run<DQ>(type, A, p.nq, stream)) return rc;
        if (A.splits > 1) {
            add_all(1, Hq, Tq);
            GS_LAUNCH_CHECK("attn_add_kernel");
        }
    }
    if (Tk > 0 && dk != nullptr) {
        A.out0 = dk;
        A.out1 = dv;
        A.s0 = strides_of(dk_strides);
        A.s1 = strides_of(dv_strides);
        A.splits = p.splits_k;
        A.part = A.splits > 1 ? part : nullptr;
        if (int rc = run<DKV>(type, A, p.nk, stream)) return rc;
        if (A.splits > 1) {
            add_all(2, Hkv, Tk);
            GS_LAUNCH_CHECK("attn_add_kernel");
        }
    }
    return GS_OK;
}
