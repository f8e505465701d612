// The orthogonalised update of weight matrices: G = U S V^T is replaced by a
// matrix near U V^T, by five (`steps`) steps of a quintic Newton-Schulz
// iteration on the shorter side's rows.
//
//   X = G / (|G|_F + 1e-7)                      (G transposed where it is tall)
//   repeat   A = X X^T,  B = a I + b A + c A A,  X = B X
//   a, b, c = 3.4445, -4.7750, 2.0315
// The polynomial takes every singular value in (0, 1] towards 1 and keeps it
// below 1.21, so no value here grows: |X| <= 1.21, |A| <= 1.47, |B| <= 3.5.
//
// Three products per step carry all the work, and a small singular value's
// error is multiplied by up to 3.4 in each step, so the products keep fp32's
// accuracy.  They do so on the float16 matrix core: a matrix is stored as two
// float16 planes, hi = f16(x s) and lo = f16(x s - hi) with a power of two s
// that brings its largest possible value near float16's, 22 bits in all, and a
// product is hi hi + hi lo + lo hi, summed in fp32.  Three float16 products
// take less than a third of the time of one on the fp32 matrix core, whose
// rate is a sixteenth.
//
// A matrix far below the floor 1e-7 starts with |X| far below 1 and grows by at
// most a per step: its planes are scaled up by a further 2^k, k following that
// bound from step to step, so that it loses none of its 22 bits either.
//
// A and A A are symmetric: their tiles on and below the diagonal are computed
// and stored twice.  The planes are padded to whole tiles with zeros, so the
// products have no edge cases.
//
// Eight 1024 x 4096 fp32 matrices: 2.03 ms, per step X X^T 148 us, B 51 us, B X
// 189 us (1090 TFLOP/s of float16 products; a large library product reaches 1190
// on the card).  The symmetric products' 288 tiles leave a second place on most
// CUs empty: 64-wide tiles were slower (191 us for X X^T), and of the 32 tiles beyond
// one per CU split over all CUs the products took 125 us, but adding them 20 more in
// a launch of its own.
#include <algorithm>
#include <utility>

#include "gs_host.h"
#include "gs_matrix.h"
#include "../../include/blitzgs_amd.h"

namespace {

using gs::f16;
using gs::f4;
using gs::Frag;
using gs::Tile;

constexpr float QA = 3.4445f, QB = -4.7750f, QC = 2.0315f;
constexpr float NORM_FLOOR = 1e-7f;
// Scales of the stored planes: 1.21 * 2^14 and 3.5 * 2^13 are below 65504.
constexpr float SX = 16384.0f, SA = 8192.0f;
constexpr int PAD = 64;         // planes are padded to whole tiles of the smaller kind
constexpr int KT = 32;          // depth of a staged tile
constexpr int NORM_PARTS = 64;  // parts of a matrix's sum of squares

// A matrix in two planes: hi at p, lo `plane` elements on.
struct Planes {
    f16* p;
    int64_t plane, stride;   // stride: one matrix of the batch to the next
    int ld;
};

struct ProductArgs {
    Planes l, r, out, add;      // add: the A of B = a I + b A + c A A
    void* final_out;            // the last product's result, or null
    int m, n, k;                // padded
    int rows, cols;             // of the result, unpadded
    int tiles_m, tiles_n;
    int tall;                   // final_out is the transpose
    const float* small;         // -log2 |X| of each matrix at the start
    int step;
    float scale;
    int splits;                 // of the sums' depth
    float* part;                // [tile][split][S x S], in the order of the lanes' registers
};

// X's planes hold X SX 2^k, and A's A SA 4^k, where 2^k |X| <= 1 at this step.
__device__ __forceinline__ int extra_scale(float small, int step)
{
    const float k = small - 1.785f * (float)step;   // log2(3.4445) < 1.785
    return k < 1.0f ? 0 : (int)k;
}

__device__ __forceinline__ void split(float x, f16& hi, f16& lo)
{
    hi = (f16)x;
    lo = (f16)(x - (float)hi);
}

// The squares of elements beyond 2^48 (2^32 elements) to 2^64 (one) pass fp32's range, those
// of SHRINK times them never do.  Where the plain sum does, the matrix is taken times
// SHRINK; what of that falls below fp32's range is less than 2^-60 of the sum.
constexpr float SHRINK = 0x1p-90f;

// What takes G to the planes of X at the start: (G pre) scale, and -log2 |X| there.
struct Start {
    float pre, scale, small;
};

// sum, shrunk: of the squares of G's elements, and of SHRINK times them, which is
// looked at only where sum is infinite
__device__ __forceinline__ Start start_of(float sum, float shrunk)
{
    if (sum == __builtin_inff()) return {SHRINK, SX / __builtin_sqrtf(shrunk), 0.0f};
    const float norm = __builtin_sqrtf(sum), len = norm / (norm + NORM_FLOOR);
    // squares that underflow: the norm is unknown but below 2^-60
    const float small = len > 0.0f ? fminf(-__builtin_log2f(len), 40.0f) : norm == 0.0f ? 20.0f : 0.0f;
    return {1.0f, __builtin_ldexpf(SX, extra_scale(small, 0)) / (norm + NORM_FLOOR), small};
}

// c[v] + a b[v] for operands in two planes; lo lo is below the planes' last bit.
// One plane's products of all v before the next: neighbours do not wait for
// each other's sums.
template <int N>
__device__ __forceinline__ void three(const Frag<f16>& ah, const Frag<f16>& al, const Frag<f16> (&bh)[N],
                                      const Frag<f16> (&bl)[N], f4 (&c)[N])
{
#pragma unroll
    for (int v = 0; v < N; v++) c[v] = gs::mma(al, bh[v], c[v]);
#pragma unroll
    for (int v = 0; v < N; v++) c[v] = gs::mma(ah, bl[v], c[v]);
#pragma unroll
    for (int v = 0; v < N; v++) c[v] = gs::mma(ah, bh[v], c[v]);
}

// ------------------------------------------------------------- the normalised X

// A workgroup's sum over a part of one matrix, in both units: parts holds NORM_PARTS of
// the one and then of the other for each matrix.
template <typename T>
__global__ __launch_bounds__(256) void orth_norm_kernel(const T* __restrict__ g, int64_t size,
                                                        float* __restrict__ parts)
{
    __shared__ float sums[4];
    const T* p = g + (int64_t)blockIdx.y * size;
    constexpr int V = gs::Vec<T>::N;
    const int64_t per = ((size + NORM_PARTS - 1) / NORM_PARTS + V - 1) / V * V;
    const int64_t from = per * blockIdx.x, to = from + per < size ? from + per : size;
    const int64_t whole = to - (to - from) % V;
    auto sum = [&](float pre) __attribute__((always_inline)) {
        float s = 0.0f;
#pragma unroll 4
        for (int64_t i = from + (int64_t)threadIdx.x * V; i < whole; i += 256 * V) {
            const gs::Vec<T> t = gs::load_vec(p + i);
#pragma unroll
            for (int k = 0; k < V; k++) {
                const float x = (float)t.v[k] * pre;
                s = __builtin_fmaf(x, x, s);
            }
        }
        if (from < to && whole + threadIdx.x < to) {
            const float x = (float)p[whole + threadIdx.x] * pre;
            s = __builtin_fmaf(x, x, s);
        }
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d, 64);
        if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
        __syncthreads();
        s = (sums[0] + sums[1]) + (sums[2] + sums[3]);
        __syncthreads();
        return s;
    };
    const float s = sum(1.0f);
    const float shrunk = s == __builtin_inff() ? sum(SHRINK) : s * SHRINK * SHRINK;
    if (threadIdx.x == 0) {
        float* to_parts = parts + blockIdx.y * 2 * NORM_PARTS + blockIdx.x;
        to_parts[0] = s;
        to_parts[NORM_PARTS] = shrunk;
    }
}

// One 64 x 64 tile of X, from G or its transpose, padded with zeros.
template <typename T>
__global__ __launch_bounds__(256) void orth_split_kernel(const T* __restrict__ g, int rows, int cols, int tall,
                                                         const float* __restrict__ parts, float* __restrict__ small,
                                                         Planes x)
{
    __shared__ float tile[64][65];
    const T* p = g + (int64_t)blockIdx.z * rows * cols;
    const float* sums = parts + blockIdx.z * 2 * NORM_PARTS;
    float s = 0.0f, shrunk = 0.0f;
    for (int k = 0; k < NORM_PARTS; k++) s += sums[k];
    if (s == __builtin_inff())
        for (int k = 0; k < NORM_PARTS; k++) shrunk += sums[NORM_PARTS + k];
    const Start start = start_of(s, shrunk);
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) small[blockIdx.z] = start.small;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int y0 = blockIdx.y * 64, x0 = blockIdx.x * 64;   // of the tile in X
    const int gy = tall ? x0 : y0, gx = tall ? y0 : x0;     // in G
    for (int k = wave; k < 64; k += 4)
        tile[k][lane] =
            gy + k < rows && gx + lane < cols
                ? (float)p[(int64_t)(gy + k) * cols + gx + lane] * start.pre * start.scale : 0.0f;
    __syncthreads();
    f16* out = x.p + blockIdx.z * x.stride;
    for (int k = wave; k < 64; k += 4) {
        f16 hi, lo;
        split(tall ? tile[lane][k] : tile[k][lane], hi, lo);
        const int64_t at = (int64_t)(y0 + k) * x.ld + x0 + lane;
        out[at] = hi;
        out[at + x.plane] = lo;
    }
}

// --------------------------------------------------------------------- products

enum Kind { SQUARE, POLY, APPLY };   // A = X X^T;  B = a I + b A + c A A;  X = B X

// Both planes of an operand's next S x KT tile (DOWN: KT x S, k down its rows),
// loaded straight to LDS.  DOWN's rows lie in the order in which Tile::cols
// takes them as k = 8 g + j, each half of its columns as a tile of its own.
template <int S, bool DOWN>
struct Pair {
    static constexpr int CH = S * KT / 8 / 256;                  // chunks per thread and plane
    static constexpr int W = DOWN ? S / 16 : KT / 8;             // chunks per row of a tile
    using L = Tile<f16, 8 * W>;
    const f16* p[CH];
    int64_t plane, step;

    __device__ __forceinline__ void at(const Planes& m, const f16* base, int first)
    {
#pragma unroll
        for (int c = 0; c < CH; c++) {
            // place `id` of the tile holds this chunk of this row
            const int id = threadIdx.x + 256 * c, row = id / W % (DOWN ? KT : S), col = L::chunk(row, id % W) - row * W;
            if constexpr (DOWN) {
                const int k = 8 * (row % 16 / 4) + 4 * (row / 16) + row % 4, half = id / (KT * W);
                p[c] = base + (int64_t)k * m.ld + first + half * (S / 2) + col * 8;
            } else {
                p[c] = base + (int64_t)(first + row) * m.ld + col * 8;
            }
        }
        plane = m.plane;
        step = DOWN ? (int64_t)KT * m.ld : KT;
    }
    __device__ __forceinline__ void skip(int tiles)
    {
#pragma unroll
        for (int c = 0; c < CH; c++) p[c] += tiles * step;
    }
    __device__ __forceinline__ void fetch(uint4* hi, uint4* lo)
    {
        typedef const __attribute__((address_space(1))) void* global_ptr;
        typedef __attribute__((address_space(3))) void* lds_ptr;
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int to = 256 * c + (threadIdx.x & ~63u);   // + 16 bytes per lane
            __builtin_amdgcn_global_load_lds((global_ptr)p[c], (lds_ptr)(hi + to), 16, 0, 0);
            __builtin_amdgcn_global_load_lds((global_ptr)(p[c] + plane), (lds_ptr)(lo + to), 16, 0, 0);
            p[c] += step;
        }
    }
};

// A block computes S x S of the result, four waves a quarter each: columns of
// its matrix-core tiles are rows of the left operand, rows are columns of the
// result, so that a lane holds four neighbours of one row of the result.  With
// splits > 1 a block sums a part of the depth and leaves it in memory as it lies
// in its registers; GATHER then adds a tile's parts in order and finishes it.
template <Kind K, int S, bool GATHER, typename T>
__global__ __launch_bounds__(256, 2) void orth_product_kernel(ProductArgs A)
{
    constexpr int H = S / 2, U = H / 16;
    constexpr int WORDS = S * KT / 8;                // of one operand's plane
    __shared__ uint4 lds[2 * 4 * WORDS];             // [2][left hi, lo, right hi, lo]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
    const uint32_t per = K == APPLY ? (uint32_t)A.tiles_m * A.tiles_n : (uint32_t)A.tiles_m * (A.tiles_m + 1) / 2;
    const uint32_t place = gs::xcd_item(blockIdx.x, gridDim.x), splits = GATHER ? 1u : (uint32_t)A.splits;
    const uint32_t item = place / splits;
    const int batch = (int)(item / per);
    int tm, tn;
    if constexpr (K == APPLY) {
        tm = (int)(item % per) % A.tiles_m;
        tn = (int)(item % per) / A.tiles_m;
    } else {
        const int e = (int)(item % per);   // row tm of the lower triangle starts at tm (tm + 1) / 2
        tm = (int)((__builtin_sqrtf(8.0f * (float)e + 1.0f) - 1.0f) * 0.5f);
        while (tm * (tm + 1) / 2 > e) tm--;
        while ((tm + 1) * (tm + 2) / 2 <= e) tm++;
        tn = e - tm * (tm + 1) / 2;
    }
    const int m0 = tm * S, n0 = tn * S;
    const f16* lp = A.l.p + batch * A.l.stride;
    const f16* rp = A.r.p + batch * A.r.stride;

    const Tile<f16, KT> tile;
    const Tile<f16, H> down;
    const int ml = (wave & 1) * H, nl = (wave >> 1) * H;
    f4 acc[U][U];   // [columns of the result][rows of the result]
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
        for (int v = 0; v < U; v++) acc[u][v] = f4{0, 0, 0, 0};
    f4* part = (f4*)A.part + (int64_t)item * A.splits * (U * U * 256) + threadIdx.x;
    if constexpr (GATHER) {
        for (int p = 0; p < A.splits; p++, part += U * U * 256)
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int v = 0; v < U; v++) acc[u][v] += part[(u * U + v) * 256];
    } else {
        const int all = A.k / KT, split = (int)(place % splits), begin = all * split / A.splits,
                  tiles = all * (split + 1) / A.splits - begin;
        Pair<S, false> sl;
        Pair<S, K == APPLY> sr;
        sl.at(A.l, lp, m0);
        sr.at(A.r, rp, n0);
        sl.skip(begin);
        sr.skip(begin);
        auto fetch = [&](uint4* to) __attribute__((always_inline)) {
            sl.fetch(to, to + WORDS);
            sr.fetch(to + 2 * WORDS, to + 3 * WORDS);
        };
        fetch(lds);
        // two restricted pointers tell the compiler that the loads need not have
        // arrived before the reads
        auto step = [&](int t, const uint4* __restrict__ at, uint4* __restrict__ next) __attribute__((always_inline)) {
            __syncthreads();   // tile t is there for all waves, and all are done with tile t - 1
            if (t + 1 < tiles) fetch(next);
            Frag<f16> lh[U], ll[U];
#pragma unroll
            for (int v = 0; v < U; v++) {
                lh[v] = tile.rows(at + ml * KT / 8, 16 * v, 0);
                ll[v] = tile.rows(at + WORDS + ml * KT / 8, 16 * v, 0);
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                Frag<f16> rh, rl;
                if constexpr (K == APPLY) {
                    rh = down.cols(at + 2 * WORDS + nl * KT / 8, 0, 16 * u);
                    rl = down.cols(at + 3 * WORDS + nl * KT / 8, 0, 16 * u);
                } else {
                    rh = tile.rows(at + 2 * WORDS + nl * KT / 8, 16 * u, 0);
                    rl = tile.rows(at + 3 * WORDS + nl * KT / 8, 16 * u, 0);
                }
                three(rh, rl, lh, ll, acc[u]);
            }
        };
        for (int t = 0; t < tiles; t++)
            step(t, lds + t % 2 * 4 * WORDS, lds + (t + 1) % 2 * 4 * WORDS);
        if (A.splits > 1) {
            part += (int64_t)split * (U * U * 256);
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int v = 0; v < U; v++) part[(u * U + v) * 256] = acc[u][v];
            return;
        }
    }
    const int k = extra_scale(A.small[batch], A.step);
    float scale = A.scale;
    if constexpr (K == POLY) scale = __builtin_ldexpf(scale, -4 * k);
    if constexpr (K == APPLY)
        scale = __builtin_ldexpf(scale, A.final_out != nullptr ? -k : extra_scale(A.small[batch], A.step + 1) - k);
    const float add_scale = __builtin_ldexpf(QB, -2 * k);
    // What leaves goes through LDS and leaves as whole rows of the block (from the
    // lanes' registers it would leave in pieces of 8 bytes, and a transposed
    // block's of 2: 5 us more per launch).
    __syncthreads();
    if constexpr (K == APPLY) {
        if (A.final_out != nullptr) {
            T* f = (T*)A.final_out + (int64_t)batch * A.rows * A.cols;
            float* e = (float*)lds;
            auto at = [](int y, int x) { return y * S + (((x / 4) ^ (y & 15)) * 4) + x % 4; };
            const int y0 = A.tall ? n0 : m0, x0 = A.tall ? m0 : n0, height = A.tall ? A.cols : A.rows,
                      width = A.tall ? A.rows : A.cols;
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int v = 0; v < U; v++) {
                    const int row = ml + 16 * v + i, col = nl + 16 * u + 4 * g;
                    if (A.tall) {
#pragma unroll
                        for (int r = 0; r < 4; r++) e[at(col + r, row)] = acc[u][v][r] * scale;
                    } else {
                        *(f4*)(e + at(row, col)) = acc[u][v] * scale;
                    }
                }
            __syncthreads();
            for (int id = threadIdx.x; id < S * S; id += 256) {
                const int y = id / S, x = id % S;
                if (y0 + y < height && x0 + x < width) f[(int64_t)(y0 + y) * width + x0 + x] = (T)e[at(y, x)];
            }
            return;
        }
    }
    const f16* add = A.add.p + batch * A.add.stride;
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
        for (int v = 0; v < U; v++) {
            acc[u][v] *= scale;
            if constexpr (K == POLY) {
                const int row = m0 + ml + 16 * v + i, col = n0 + nl + 16 * u + 4 * g;
                f16 hi[4], lo[4];
                const f16* p = add + (int64_t)row * A.add.ld + col;
                __builtin_memcpy(hi, p, 8);
                __builtin_memcpy(lo, p + A.add.plane, 8);
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    acc[u][v][r] = __builtin_fmaf(add_scale, (float)hi[r] + (float)lo[r], acc[u][v][r]);
                    if (row == col + r && row < A.rows) acc[u][v][r] += QA * SA;
                }
            }
        }
    f16* out = A.out.p + batch * A.out.stride;
    constexpr int CH = S / 8, LO = S * S;
    f16* eh = (f16*)lds;
    auto at = [](int row, int col) { return row * S + ((col / 8) ^ (row & (CH - 1) & 15)) * 8 + col % 8; };
    auto leave = [&](int row0, int col0) {
        __syncthreads();
#pragma unroll 4
        for (int id = threadIdx.x; id < S * CH; id += 256) {
            const int row = id / CH, col = id % CH * 8;
            f16* p = out + (int64_t)(row0 + row) * A.out.ld + col0 + col;
            *(uint4*)p = *(const uint4*)(eh + at(row, col));
            *(uint4*)(p + A.out.plane) = *(const uint4*)(eh + LO + at(row, col));
        }
    };
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
        for (int v = 0; v < U; v++) {
            f16 hi[4], lo[4];
#pragma unroll
            for (int r = 0; r < 4; r++) split(acc[u][v][r], hi[r], lo[r]);
            f16* p = eh + at(ml + 16 * v + i, nl + 16 * u + 4 * g);
            __builtin_memcpy(p, hi, 8);
            __builtin_memcpy(p + LO, lo, 8);
        }
    leave(m0, n0);
    if (K == APPLY || tm == tn) return;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
        for (int v = 0; v < U; v++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                f16* p = eh + at(nl + 16 * u + 4 * g + r, ml + 16 * v + i);
                split(acc[u][v][r], p[0], p[LO]);
            }
    leave(n0, m0);
}

// ---------------------------------------------------- a small matrix in one CU

// The whole iteration of one matrix whose planes of X and A fit in LDS: X as
// panels of 32 columns, A in the same form, B in A's place.  The launches of the
// products above cost more than the work of such a matrix (250 x 96: 93 us in
// 17 launches).  Eight waves share the 32 x 32 blocks of each product; results
// wait in registers until every wave has read their operands.
constexpr int SMALL_THREADS = 512, SMALL_WAVES = SMALL_THREADS / 64;
constexpr int SMALL_BLOCKS = 5;           // of X per wave
constexpr int SMALL_LDS = 156 * 1024;

// Four neighbours of a row, from column `col` (a multiple of 4), of panels at p.
template <int PANEL>
__device__ __forceinline__ f16* quad(uint4* p, int row, int col)
{
    return (f16*)(p + col / 32 * PANEL + Tile<f16, 32>::chunk(row, col % 32 / 8)) + col % 8;
}

// Block e of the lower triangle, row by row.
__device__ __forceinline__ void corner(int e, int& bm, int& bn)
{
    bm = 0;
    while ((bm + 1) * (bm + 2) / 2 <= e) bm++;
    bn = e - bm * (bm + 1) / 2;
}

// acc = the 32 x 32 block (bm, bn) of Y Y^T, Y's planes in `depth` panels.
template <int PANEL>
__device__ __forceinline__ void square_block(const Tile<f16, 32>& tile, const uint4* hi, const uint4* lo, int depth,
                                             int bm, int bn, f4 (&acc)[2][2])
{
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
        for (int v = 0; v < 2; v++) acc[u][v] = f4{0, 0, 0, 0};
    for (int p = 0; p < depth; p++, hi += PANEL, lo += PANEL) {
        Frag<f16> lh[2], ll[2];
#pragma unroll
        for (int v = 0; v < 2; v++) {
            lh[v] = tile.rows(hi + bm * 128, 16 * v, 0);
            ll[v] = tile.rows(lo + bm * 128, 16 * v, 0);
        }
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const Frag<f16> rh = tile.rows(hi + bn * 128, 16 * u, 0), rl = tile.rows(lo + bn * 128, 16 * u, 0);
            three(rh, rl, lh, ll, acc[u]);
        }
    }
}

// Both planes of four neighbours (row, col ..) of a symmetric matrix, and where
// `both` of (col .., row) too; from and to are a column's place.
template <int PANEL>
__device__ __forceinline__ void store_symmetric(uint4* ph, uint4* pl, int row, int col, int row_to, int col_to,
                                                bool both, f4 x)
{
    f16 hi[4], lo[4];
#pragma unroll
    for (int r = 0; r < 4; r++) split(x[r], hi[r], lo[r]);
    __builtin_memcpy(quad<PANEL>(ph, row, col_to), hi, 8);
    __builtin_memcpy(quad<PANEL>(pl, row, col_to), lo, 8);
    if (!both) return;
#pragma unroll
    for (int r = 0; r < 4; r++) {
        quad<PANEL>(ph, col + r, row_to & ~3)[row_to & 3] = hi[r];
        quad<PANEL>(pl, col + r, row_to & ~3)[row_to & 3] = lo[r];
    }
}

// Where B's column c lies, so that rows() reads it in the order of X's cols().
__device__ __forceinline__ int place(int c) { return c / 32 * 32 + c % 16 / 4 * 8 + c % 32 / 16 * 4 + c % 4; }

template <typename T, int MP>
__global__ __launch_bounds__(SMALL_THREADS) void orth_small_kernel(const T* __restrict__ update, T* __restrict__ result,
                                                                   int m, int n, int tall, int np, int steps)
{
    constexpr int MB = MP / 32, PANEL = MP * 4, SQ = MB * (MB + 1) / 2, PER = (SQ + SMALL_WAVES - 1) / SMALL_WAVES;
    extern __shared__ uint4 lds[];
    const int panels = np / 32, blocks = MB * panels, size = m * n;
    uint4 *xh = lds, *xl = xh + panels * PANEL, *ah = xl + panels * PANEL, *al = ah + MB * PANEL;
    const Tile<f16, 32> tile;
    const int lane = threadIdx.x & 63;
    int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
    const T* src = update + (int64_t)blockIdx.x * size;
    T* dst = result + (int64_t)blockIdx.x * size;

    float* sums = (float*)ah;
    auto sum = [&](float pre) __attribute__((always_inline)) {
        float s = 0.0f;
#pragma unroll 8
        for (int e = threadIdx.x; e < size; e += SMALL_THREADS) {
            const float x = (float)src[e] * pre;
            s = __builtin_fmaf(x, x, s);
        }
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d, 64);
        if (lane == 0) sums[wave] = s;
        __syncthreads();
        s = 0.0f;
#pragma unroll
        for (int w = 0; w < SMALL_WAVES; w++) s += sums[w];
        return s;
    };
    for (int e = threadIdx.x; e < 2 * panels * PANEL; e += SMALL_THREADS) xh[e] = make_uint4(0, 0, 0, 0);
    const float s = sum(1.0f);
    float shrunk = 0.0f;
    if (s == __builtin_inff()) {
        __syncthreads();   // all have read the first sums
        shrunk = sum(SHRINK);
    }
    const Start start = start_of(s, shrunk);
    const float small = start.small;
    // a wave takes rows of G, a lane every 64th element of one
#pragma unroll 2
    for (int r = wave; r < m; r += SMALL_WAVES)
#pragma unroll 4
        for (int c = lane; c < n; c += 64) {
            const int row = tall ? c : r, col = tall ? r : c;
            f16 hi, lo;
            split((float)src[r * n + c] * start.pre * start.scale, hi, lo);
            quad<PANEL>(xh, row, col & ~3)[col & 3] = hi;
            quad<PANEL>(xl, row, col & ~3)[col & 3] = lo;
        }
    __syncthreads();
    for (int step = 0; step < steps; step++) {
        // the blocks' addresses are formed anew in each step: kept, they would not fit the registers
        asm volatile("" : "+s"(wave), "+v"(i), "+v"(g));
        const int k = extra_scale(small, step);
        const bool last = step + 1 == steps;
        f4 acc[PER][2][2];
        // A = X X^T
#pragma unroll
        for (int q = 0; q < PER; q++) {
            int bm, bn;
            corner(wave + q * SMALL_WAVES, bm, bn);
            if (bm >= MB) continue;
            square_block<PANEL>(tile, xh, xl, panels, bm, bn, acc[q]);
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int v = 0; v < 2; v++) {
                    const int row = 32 * bm + 16 * v + i, col = 32 * bn + 16 * u + 4 * g;
                    store_symmetric<PANEL>(ah, al, row, col, row, col, bm != bn, acc[q][u][v] * (SA / (SX * SX)));
                }
        }
        __syncthreads();
        // B = a I + b A + c A A
        const float cc = __builtin_ldexpf(QC / SA, -4 * k), cb = __builtin_ldexpf(QB, -2 * k);
#pragma unroll
        for (int q = 0; q < PER; q++) {
            int bm, bn;
            corner(wave + q * SMALL_WAVES, bm, bn);
            if (bm >= MB) continue;
            square_block<PANEL>(tile, ah, al, MB, bm, bn, acc[q]);
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int v = 0; v < 2; v++) {
                    const int row = 32 * bm + 16 * v + i, col = 32 * bn + 16 * u + 4 * g;
                    f16 hi[4], lo[4];
                    __builtin_memcpy(hi, quad<PANEL>(ah, row, col), 8);
                    __builtin_memcpy(lo, quad<PANEL>(al, row, col), 8);
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const float x = __builtin_fmaf(cb, (float)hi[r] + (float)lo[r], acc[q][u][v][r] * cc);
                        acc[q][u][v][r] = row == col + r ? x + QA * SA : x;
                    }
                }
        }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < PER; q++) {
            int bm, bn;
            corner(wave + q * SMALL_WAVES, bm, bn);
            if (bm >= MB) continue;
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int v = 0; v < 2; v++) {
                    const int row = 32 * bm + 16 * v + i, col = 32 * bn + 16 * u + 4 * g;
                    store_symmetric<PANEL>(ah, al, row, col, place(row), place(col), bm != bn, acc[q][u][v]);
                }
        }
        __syncthreads();
        // X = B X
        f4 xs[SMALL_BLOCKS][2][2];
#pragma unroll
        for (int q = 0; q < SMALL_BLOCKS; q++) {
            const int e = wave + q * SMALL_WAVES, bm = e % MB, bn = e / MB;
            if (e >= blocks) continue;
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int v = 0; v < 2; v++) xs[q][u][v] = f4{0, 0, 0, 0};
#pragma unroll
            for (int p = 0; p < MB; p++) {
                Frag<f16> lh[2], ll[2];
#pragma unroll
                for (int v = 0; v < 2; v++) {
                    lh[v] = tile.rows(ah + p * PANEL + bm * 128, 16 * v, 0);
                    ll[v] = tile.rows(al + p * PANEL + bm * 128, 16 * v, 0);
                }
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const Frag<f16> rh = tile.cols(xh + bn * PANEL, 32 * p, 16 * u);
                    const Frag<f16> rl = tile.cols(xl + bn * PANEL, 32 * p, 16 * u);
                    three(rh, rl, lh, ll, xs[q][u]);
                }
            }
        }
        __syncthreads();
        const float out_scale = last ? __builtin_ldexpf(1.0f / (SA * SX), -k)
                                     : __builtin_ldexpf(1.0f / SA, extra_scale(small, step + 1) - k);
#pragma unroll
        for (int q = 0; q < SMALL_BLOCKS; q++) {
            const int e = wave + q * SMALL_WAVES, bm = e % MB, bn = e / MB;
            if (e >= blocks) continue;
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int v = 0; v < 2; v++) {
                    const int row = 32 * bm + 16 * v + i, col = 32 * bn + 16 * u + 4 * g;
                    const f4 x = xs[q][u][v] * out_scale;
                    if (last) {
#pragma unroll
                        for (int r = 0; r < 4; r++)
                            if (row < (tall ? n : m) && col + r < (tall ? m : n))
                                dst[tall ? (col + r) * n + row : row * n + col + r] = (T)x[r];
                        continue;
                    }
                    f16 hi[4], lo[4];
#pragma unroll
                    for (int r = 0; r < 4; r++) split(x[r], hi[r], lo[r]);
                    __builtin_memcpy(quad<PANEL>(xh, row, col), hi, 8);
                    __builtin_memcpy(quad<PANEL>(xl, row, col), lo, 8);
                }
        }
        __syncthreads();
    }
}

// -------------------------------------------------------------------- launching

int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

// The workspace: partial sums and the matrices' sizes, the planes of X (twice), A
// and B, and the split products' parts.
struct Layout {
    int m, n;               // padded sides, m the shorter
    int64_t parts, x, sq;   // bytes of each piece
    int64_t bytes;
};

// Tiles of 128 do twice the work per byte moved to LDS; 64 where a matrix is
// small (less padding, more workgroups).
int tile_of(int count, int64_t m, int64_t n)
{
    const int64_t pm = up(m, 128), pn = up(n, 128);
    return (int64_t)count * (pm / 128) * (pn / 128) >= 256 ? 128 : 64;
}

// Splits of a product's depth where its tiles leave half of the CUs without work:
// up to two workgroups per CU, none shorter than 16 staged tiles.  One 1024 x 4096
// matrix (36 tiles of X X^T) 818 -> 520 us; with 144 tiles the parts cost more
// than they save (four 1024 x 1024: 484 us whole, 527 split).
int splits_of(int64_t tiles, int depth)
{
    if (tiles >= 128) return 1;
    const int64_t want = (512 + tiles - 1) / tiles, most = depth / KT / 16;
    return (int)(most < 1 ? 1 : want < most ? want : most);
}

Layout layout_of(int count, int m, int n)
{
    Layout L{};
    const int s = m < n ? m : n, l = m < n ? n : m, t = tile_of(count, s, l);
    L.m = (int)up(s, t);
    L.n = (int)up(l, t);
    L.parts = up((int64_t)count * (2 * NORM_PARTS + 1) * 4, 256);
    L.x = up((int64_t)count * L.m * L.n * 4, 256);
    L.sq = up((int64_t)count * L.m * L.m * 4, 256);
    const int64_t tm = L.m / t, tn = L.n / t, sq = count * (tm * (tm + 1) / 2), full = count * tm * tn;
    int64_t most = 0;
    for (const auto& [tiles, depth] : {std::pair<int64_t, int>{sq, L.n}, {sq, L.m}, {full, L.m}}) {
        const int splits = splits_of(tiles, depth);
        if (splits > 1 && tiles * splits > most) most = tiles * splits;
    }
    L.bytes = L.parts + 2 * L.x + 2 * L.sq + most * t * t * 4;
    return L;
}

int check(int type, int count, int m, int n)
{
    GS_REQUIRE(gs::dtype_known(type), "orthogonalise: unknown element type %d", type);
    GS_REQUIRE(count >= 0 && m >= 0 && n >= 0, "orthogonalise: sizes must not be negative");
    GS_REQUIRE(m <= 65536 && n <= 65536, "orthogonalise: a side may have at most 65536 elements");
    GS_REQUIRE(count <= 65535, "orthogonalise: at most 65535 matrices per call");
    return GS_OK;
}

template <Kind K, typename T>
int product(int S, const ProductArgs& A, int count, hipStream_t stream)
{
    const int64_t per = K == APPLY ? (int64_t)A.tiles_m * A.tiles_n : (int64_t)A.tiles_m * (A.tiles_m + 1) / 2;
    GS_REQUIRE(per * count < (1 << 24), "orthogonalise: too many tiles for one launch");
    constexpr const char* name = K == SQUARE ? "orth_square" : K == POLY ? "orth_poly" : "orth_apply";
    ProductArgs P = A;
    P.splits = splits_of(per * count, A.k);
    const dim3 grid((unsigned)(per * count * P.splits));
    if (S == 128)
        GS_TIMED(name, stream,
                 hipLaunchKernelGGL((orth_product_kernel<K, 128, false, T>), grid, dim3(256), 0, stream, P));
    else
        GS_TIMED(name, stream,
                 hipLaunchKernelGGL((orth_product_kernel<K, 64, false, T>), grid, dim3(256), 0, stream, P));
    GS_LAUNCH_CHECK(name);
    if (P.splits == 1) return GS_OK;
    const dim3 tiles((unsigned)(per * count));
    if (S == 128)
        GS_TIMED("orth_gather", stream,
                 hipLaunchKernelGGL((orth_product_kernel<K, 128, true, T>), tiles, dim3(256), 0, stream, P));
    else
        GS_TIMED("orth_gather", stream,
                 hipLaunchKernelGGL((orth_product_kernel<K, 64, true, T>), tiles, dim3(256), 0, stream, P));
    GS_LAUNCH_CHECK("orth_gather");
    return GS_OK;
}

// The padded short side of a matrix that one workgroup takes, 0 if none does.
int small_side(int m, int n)
{
    const int64_t s = up(m < n ? m : n, 32), l = up(m < n ? n : m, 32);
    if (s > 128 || s * (l + s) * 4 > SMALL_LDS || s / 32 * (l / 32) > SMALL_BLOCKS * SMALL_WAVES) return 0;
    return (int)s;
}

template <typename T, int MP>
int orthogonalise_small(int count, int m, int n, const T* g, int steps, T* out, hipStream_t stream)
{
    const int np = (int)up(m < n ? n : m, 32), lds = MP * (np + MP) * 4;
    if (lds > 65536)
        GS_HIP(hipFuncSetAttribute((const void*)orth_small_kernel<T, MP>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                   SMALL_LDS));
    GS_TIMED("orth_small_kernel", stream,
             hipLaunchKernelGGL((orth_small_kernel<T, MP>), dim3((unsigned)count), dim3(SMALL_THREADS), lds, stream, g,
                                out, m, n, (int)(m > n), np, steps));
    GS_LAUNCH_CHECK("orth_small_kernel");
    return GS_OK;
}

template <typename T>
int orthogonalise(int count, int m, int n, const T* g, int steps, T* out, void* workspace, hipStream_t stream)
{
    switch (small_side(m, n)) {
        case 32: return orthogonalise_small<T, 32>(count, m, n, g, steps, out, stream);
        case 64: return orthogonalise_small<T, 64>(count, m, n, g, steps, out, stream);
        case 96: return orthogonalise_small<T, 96>(count, m, n, g, steps, out, stream);
        case 128: return orthogonalise_small<T, 128>(count, m, n, g, steps, out, stream);
    }
    const Layout L = layout_of(count, m, n);
    const int tall = m > n, S = tile_of(count, m < n ? m : n, m < n ? n : m);
    float* parts = (float*)workspace;
    float* small = parts + (int64_t)count * 2 * NORM_PARTS;
    char* at = (char*)workspace + L.parts;
    const int64_t px = (int64_t)L.m * L.n, pa = (int64_t)L.m * L.m;
    Planes x[2] = {{(f16*)at, px, 2 * px, L.n}, {(f16*)(at + L.x), px, 2 * px, L.n}};
    const Planes a{(f16*)(at + 2 * L.x), pa, 2 * pa, L.m}, b{(f16*)(at + 2 * L.x + L.sq), pa, 2 * pa, L.m};
    GS_TIMED("orth_norm_kernel", stream,
             hipLaunchKernelGGL(orth_norm_kernel<T>, dim3(NORM_PARTS, (unsigned)count), dim3(256), 0, stream, g,
                                (int64_t)m * n, parts));
    GS_LAUNCH_CHECK("orth_norm_kernel");
    GS_TIMED("orth_split_kernel", stream,
             hipLaunchKernelGGL(orth_split_kernel<T>, dim3((unsigned)(L.n / 64), (unsigned)(L.m / 64), (unsigned)count),
                                dim3(256), 0, stream, g, m, n, tall, parts, small,
                                x[0]));
    GS_LAUNCH_CHECK("orth_split_kernel");
    ProductArgs A{};
    A.m = L.m;
    A.rows = tall ? n : m;
    A.tall = tall;
    A.small = small;
    A.part = (float*)(at + 2 * L.x + 2 * L.sq);
    A.tiles_m = L.m / S;
    for (int s = 0; s < steps; s++) {
        const bool last = s + 1 == steps;
        A.step = s;
        A.l = A.r = x[s & 1];
        A.add = a;
        A.out = a;
        A.n = L.m;
        A.k = L.n;
        A.cols = A.rows;
        A.tiles_n = A.tiles_m;
        A.scale = SA / (SX * SX);
        A.final_out = nullptr;
        if (int rc = product<SQUARE, T>(S, A, count, stream)) return rc;
        A.l = A.r = a;
        A.out = b;
        A.k = L.m;
        A.scale = QC / SA;
        if (int rc = product<POLY, T>(S, A, count, stream)) return rc;
        A.l = b;
        A.r = x[s & 1];
        A.out = x[~s & 1];
        A.n = L.n;
        A.cols = tall ? m : n;
        A.tiles_n = L.n / S;
        A.scale = last ? 1.0f / (SA * SX) : 1.0f / SA;
        A.final_out = last ? out : nullptr;
        if (int rc = product<APPLY, T>(S, A, count, stream)) return rc;
    }
    return GS_OK;
}

// ------------------------------------------------------- momentum and the step

constexpr int MAX_PARAMS = 32;

struct MomentumBatch {
    void* param[MAX_PARAMS];
    const void* grad[MAX_PARAMS];
    float* momentum[MAX_PARAMS];
};

// Bound by memory, an element per thread.  Eight 1024 x 4096 matrices: 96 us (537 MB, 5.6
// TB/s) and 84 us (403 MB, 4.8) in float32, 94 (5.0) and 77 (3.5: two-byte accesses)
// in bfloat16, beside 2 ms for the products.
// m = beta m + g;  update = nesterov ? g + beta m : m, stacked
template <typename T>
__global__ __launch_bounds__(256) void momentum_kernel(MomentumBatch B, int64_t size, float beta, int nesterov,
                                                       float* __restrict__ update)
{
    const T* grad = (const T*)B.grad[blockIdx.y];
    float *momentum = B.momentum[blockIdx.y], *out = update + blockIdx.y * size;
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < size; e += (int64_t)gridDim.x * 256) {
        const float g = (float)grad[e], m = __builtin_fmaf(beta, momentum[e], g);
        momentum[e] = m;
        out[e] = nesterov ? __builtin_fmaf(beta, m, g) : m;
    }
}

// p = p keep - lr update
template <typename T>
__global__ __launch_bounds__(256) void apply_kernel(MomentumBatch B, int64_t size, float keep, float lr,
                                                    const float* __restrict__ update)
{
    T* param = (T*)B.param[blockIdx.y];
    const float* u = update + blockIdx.y * size;
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < size; e += (int64_t)gridDim.x * 256)
        param[e] = (T)__builtin_fmaf(-lr, u[e], (float)param[e] * keep);
}

dim3 grid_of(int64_t size, int count)
{
    return dim3((unsigned)std::min<int64_t>((size + 255) / 256, 16384), (unsigned)count);
}

}  // namespace

extern "C" size_t gs_orthogonalise_workspace_bytes(int count, int m, int n)
{
    if (check(GS_F32, count, m, n) != GS_OK) return 0;
    if (count == 0 || m == 0 || n == 0 || small_side(m, n) != 0) return 0;
    return (size_t)layout_of(count, m, n).bytes;
}

extern "C" int gs_orthogonalise(int type, int count, int m, int n, const void* update, int steps, void* out,
                                void* workspace, hipStream_t stream)
{
    gs::clear_error();
    if (int rc = check(type, count, m, n)) return rc;
    GS_REQUIRE(steps >= 1 && steps <= 32, "orthogonalise: steps must be in [1, 32], got %d", steps);
    if (count == 0 || m == 0 || n == 0) return GS_OK;
    GS_REQUIRE(update && out, "orthogonalise: update and out must be non-null");
    GS_REQUIRE(workspace || small_side(m, n) != 0, "orthogonalise: this size needs the workspace");
    GS_REQUIRE(((uintptr_t)workspace & 255) == 0, "orthogonalise: the workspace must be 256-byte aligned");
    if (type == GS_F32) return orthogonalise(count, m, n, (const float*)update, steps, (float*)out, workspace, stream);
    if (type == GS_BF16)
        return orthogonalise(count, m, n, (const gs::bf16*)update, steps, (gs::bf16*)out, workspace, stream);
    return orthogonalise(count, m, n, (const f16*)update, steps, (f16*)out, workspace, stream);
}

extern "C" int gs_momentum_update(int type, int count, int64_t size, const void* const* grads, float* const* momenta,
                                  float beta, int nesterov, float* update, hipStream_t stream)
{
    gs::clear_error();
    GS_REQUIRE(gs::dtype_known(type), "momentum: unknown element type %d", type);
    GS_REQUIRE(count >= 0 && count <= MAX_PARAMS, "momentum: at most %d tensors per call", MAX_PARAMS);
    GS_REQUIRE(size >= 0 && size < (1ll << 38), "momentum: size out of range");
    if (count == 0 || size == 0) return GS_OK;
    GS_REQUIRE(grads && momenta && update, "momentum: null argument");
    MomentumBatch B{};
    for (int i = 0; i < count; i++) {
        GS_REQUIRE(grads[i] && momenta[i], "momentum: null tensor %d", i);
        B.grad[i] = grads[i];
        B.momentum[i] = momenta[i];
    }
    const dim3 grid = grid_of(size, count);
    auto run = [&](auto kernel) {
        GS_TIMED("momentum_kernel", stream,
                 hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, B, size, beta, nesterov, update));
    };
    if (type == GS_F32) run(momentum_kernel<float>);
    else if (type == GS_BF16) run(momentum_kernel<gs::bf16>);
    else run(momentum_kernel<f16>);
    GS_LAUNCH_CHECK("momentum_kernel");
    return GS_OK;
}

extern "C" int gs_momentum_apply(int type, int count, int64_t size, void* const* params, float keep, float lr,
                                 const float* update, hipStream_t stream)
{
    gs::clear_error();
    GS_REQUIRE(gs::dtype_known(type), "momentum: unknown element type %d", type);
    GS_REQUIRE(count >= 0 && count <= MAX_PARAMS, "momentum: at most %d tensors per call", MAX_PARAMS);
    GS_REQUIRE(size >= 0 && size < (1ll << 38), "momentum: size out of range");
    if (count == 0 || size == 0) return GS_OK;
    GS_REQUIRE(params && update, "momentum: null argument");
    MomentumBatch B{};
    for (int i = 0; i < count; i++) {
        GS_REQUIRE(params[i], "momentum: null tensor %d", i);
        B.param[i] = params[i];
    }
    const dim3 grid = grid_of(size, count);
    auto run = [&](auto kernel) {
        GS_TIMED("apply_kernel", stream,
                 hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, B, size, keep, lr, update));
    };
    if (type == GS_F32) run(apply_kernel<float>);
    else if (type == GS_BF16) run(apply_kernel<gs::bf16>);
    else run(apply_kernel<f16>);
    GS_LAUNCH_CHECK("apply_kernel");
    return GS_OK;
}
