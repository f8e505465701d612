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
constexpr int NORM_PARTS = 64;  // partial sums of squares per matrix

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

// ------------------------------------------------------------- the normalised X

template <typename T>
__global__ __launch_bounds__(256) void orth_norm_kernel(const T* __restrict__ g, int64_t size, float* __restrict__ parts)
{
    __shared__ float sums[4];
    const T* p = g + (int64_t)blockIdx.y * size;
    constexpr int V = gs::Vec<T>::N;
    const int64_t per = ((size + NORM_PARTS - 1) / NORM_PARTS + V - 1) / V * V;
    const int64_t from = per * blockIdx.x, to = from + per < size ? from + per : size;
    float s = 0.0f;
    const int64_t whole = to - (to - from) % V;
    for (int64_t i = from + (int64_t)threadIdx.x * V; i < whole; i += 256 * V) {
        const gs::Vec<T> t = gs::load_vec(p + i);
#pragma unroll
        for (int k = 0; k < V; k++) s = __builtin_fmaf((float)t.v[k], (float)t.v[k], s);
    }
    if (from < to && whole + threadIdx.x < to) {
        const float t = (float)p[whole + threadIdx.x];
        s = __builtin_fmaf(t, t, s);
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d, 64);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) parts[blockIdx.y * NORM_PARTS + blockIdx.x] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

// One 64 x 64 tile of X, from G or its transpose, padded with zeros.
template <typename T>
__global__ __launch_bounds__(256) void orth_split_kernel(const T* __restrict__ g, int rows, int cols, int tall,
                                                         const float* __restrict__ parts, float* __restrict__ small,
                                                         Planes x)
{
    __shared__ float tile[64][65];
    const T* p = g + (int64_t)blockIdx.z * rows * cols;
    float s = 0.0f;
    for (int k = 0; k < NORM_PARTS; k++) s += parts[blockIdx.z * NORM_PARTS + k];
    const float norm = __builtin_sqrtf(s), len = norm / (norm + NORM_FLOOR);
    // squares that underflow: the norm is unknown but below 2^-60
    const float sm = len > 0.0f ? fminf(-__builtin_log2f(len), 40.0f) : norm == 0.0f ? 20.0f : 0.0f;
    const float scale = __builtin_ldexpf(SX, extra_scale(sm, 0)) / (norm + NORM_FLOOR);
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) small[blockIdx.z] = sm;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int y0 = blockIdx.y * 64, x0 = blockIdx.x * 64;   // of the tile in X
    const int gy = tall ? x0 : y0, gx = tall ? y0 : x0;     // in G
    for (int k = wave; k < 64; k += 4)
        tile[k][lane] = gy + k < rows && gx + lane < cols ? (float)p[(int64_t)(gy + k) * cols + gx + lane] * scale : 0.0f;
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
// result, so that a lane holds four neighbours of one row of the result.
template <Kind K, int S, typename T>
__global__ __launch_bounds__(256, 2) void orth_product_kernel(ProductArgs A)
{
    constexpr int H = S / 2, U = H / 16;
    constexpr int WORDS = S * KT / 8;                // of one operand's plane
    __shared__ uint4 lds[2][4][WORDS];               // left hi, lo, right hi, lo
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
    const uint32_t per = K == APPLY ? (uint32_t)A.tiles_m * A.tiles_n : (uint32_t)A.tiles_m * (A.tiles_m + 1) / 2;
    const uint32_t item = gs::xcd_item(blockIdx.x, gridDim.x);
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

    Pair<S, false> sl;
    Pair<S, K == APPLY> sr;
    sl.at(A.l, lp, m0);
    sr.at(A.r, rp, n0);
    const Tile<f16, KT> tile;
    const Tile<f16, H> down;
    const int ml = (wave & 1) * H, nl = (wave >> 1) * H;
    f4 acc[U][U];   // [columns of the result][rows of the result]
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
        for (int v = 0; v < U; v++) acc[u][v] = f4{0, 0, 0, 0};
    sl.fetch(lds[0][0], lds[0][1]);
    sr.fetch(lds[0][2], lds[0][3]);
    __syncthreads();
    for (int k0 = 0, b = 0; k0 < A.k; k0 += KT, b ^= 1) {
        if (k0 + KT < A.k) {
            sl.fetch(lds[b ^ 1][0], lds[b ^ 1][1]);
            sr.fetch(lds[b ^ 1][2], lds[b ^ 1][3]);
        }
        Frag<f16> lh[U], ll[U];
#pragma unroll
        for (int v = 0; v < U; v++) {
            lh[v] = tile.rows(lds[b][0] + ml * KT / 8, 16 * v, 0);
            ll[v] = tile.rows(lds[b][1] + ml * KT / 8, 16 * v, 0);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            Frag<f16> rh, rl;
            if constexpr (K == APPLY) {
                rh = down.cols(lds[b][2] + nl * KT / 8, 0, 16 * u);
                rl = down.cols(lds[b][3] + nl * KT / 8, 0, 16 * u);
            } else {
                rh = tile.rows(lds[b][2] + nl * KT / 8, 16 * u, 0);
                rl = tile.rows(lds[b][3] + nl * KT / 8, 16 * u, 0);
            }
#pragma unroll
            for (int v = 0; v < U; v++) {
                acc[u][v] = gs::mma(rl, lh[v], acc[u][v]);
                acc[u][v] = gs::mma(rh, ll[v], acc[u][v]);
                acc[u][v] = gs::mma(rh, lh[v], acc[u][v]);
            }
        }
        __syncthreads();
    }
    const int k = extra_scale(A.small[batch], A.step);
    float scale = A.scale;
    if constexpr (K == POLY) scale = __builtin_ldexpf(scale, -4 * k);
    if constexpr (K == APPLY)
        scale = __builtin_ldexpf(scale, A.final_out != nullptr ? -k : extra_scale(A.small[batch], A.step + 1) - k);
    const float add_scale = __builtin_ldexpf(QB, -2 * k);
    f16* out = A.out.p + batch * A.out.stride;
    const f16* add = A.add.p + batch * A.add.stride;
#pragma unroll
    for (int u = 0; u < U; u++) {
#pragma unroll
        for (int v = 0; v < U; v++) {
            const int row = m0 + ml + 16 * v + i, col = n0 + nl + 16 * u + 4 * g;
            f4 x = acc[u][v] * scale;
            if constexpr (K == APPLY) {
                if (A.final_out != nullptr) {
                    T* f = (T*)A.final_out + (int64_t)batch * A.rows * A.cols;
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        if (row < A.rows && col + r < A.cols)
                            f[A.tall ? (int64_t)(col + r) * A.rows + row : (int64_t)row * A.cols + col + r] = (T)x[r];
                    continue;
                }
            }
            if constexpr (K == POLY) {
                f16 hi[4], lo[4];
                const f16* p = add + (int64_t)row * A.add.ld + col;
                __builtin_memcpy(hi, p, 8);
                __builtin_memcpy(lo, p + A.add.plane, 8);
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    x[r] = __builtin_fmaf(add_scale, (float)hi[r] + (float)lo[r], x[r]);
                    if (row == col + r && row < A.rows) x[r] += QA * SA;
                }
            }
            f16 hi[4], lo[4];
#pragma unroll
            for (int r = 0; r < 4; r++) split(x[r], hi[r], lo[r]);
            f16* p = out + (int64_t)row * A.out.ld + col;
            __builtin_memcpy(p, hi, 8);
            __builtin_memcpy(p + A.out.plane, lo, 8);
            if constexpr (K != APPLY) {
                if (tm != tn) {
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        f16* q = out + (int64_t)(col + r) * A.out.ld + row;
                        q[0] = hi[r];
                        q[A.out.plane] = lo[r];
                    }
                }
            }
        }
    }
}

// -------------------------------------------------------------------- launching

int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

// The workspace: partial sums and the matrices' sizes, then the planes of X (twice), A and B.
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

Layout layout_of(int count, int m, int n)
{
    Layout L{};
    const int s = m < n ? m : n, l = m < n ? n : m, t = tile_of(count, s, l);
    L.m = (int)up(s, t);
    L.n = (int)up(l, t);
    L.parts = up((int64_t)count * (NORM_PARTS + 1) * 4, 256);
    L.x = up((int64_t)count * L.m * L.n * 4, 256);
    L.sq = up((int64_t)count * L.m * L.m * 4, 256);
    L.bytes = L.parts + 2 * L.x + 2 * L.sq;
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
    GS_REQUIRE(per * count < 0x7fffffff, "orthogonalise: too many tiles for one launch");
    constexpr const char* name = K == SQUARE ? "orth_square" : K == POLY ? "orth_poly" : "orth_apply";
    const dim3 grid((unsigned)(per * count));
    if (S == 128)
        GS_TIMED(name, stream,
                 hipLaunchKernelGGL((orth_product_kernel<K, 128, T>), grid, dim3(256), 0, stream, A));
    else
        GS_TIMED(name, stream,
                 hipLaunchKernelGGL((orth_product_kernel<K, 64, T>), grid, dim3(256), 0, stream, A));
    GS_LAUNCH_CHECK("orth_product_kernel");
    return GS_OK;
}

template <typename T>
int orthogonalise(int count, int m, int n, const T* g, int steps, T* out, void* workspace, hipStream_t stream)
{
    const Layout L = layout_of(count, m, n);
    const int tall = m > n, S = tile_of(count, m < n ? m : n, m < n ? n : m);
    float* parts = (float*)workspace;
    float* small = parts + (int64_t)count * NORM_PARTS;
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

// m = beta m + g;  update = nesterov ? g + beta m : m, stacked
template <typename T>
__global__ __launch_bounds__(256) void momentum_kernel(MomentumBatch B, int64_t size, float beta, int nesterov,
                                                       float* __restrict__ update)
{
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (e >= size) return;
    const float g = (float)((const T*)B.grad[blockIdx.y])[e];
    float* mp = B.momentum[blockIdx.y] + e;
    const float m = __builtin_fmaf(beta, *mp, g);
    *mp = m;
    update[blockIdx.y * size + e] = nesterov ? __builtin_fmaf(beta, m, g) : m;
}

// p = p keep - lr update
template <typename T>
__global__ __launch_bounds__(256) void apply_kernel(MomentumBatch B, int64_t size, float keep, float lr,
                                                    const float* __restrict__ update)
{
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (e >= size) return;
    T* p = (T*)B.param[blockIdx.y] + e;
    *p = (T)__builtin_fmaf(-lr, update[blockIdx.y * size + e], (float)*p * keep);
}

}  // namespace

extern "C" size_t gs_orthogonalise_workspace_bytes(int count, int m, int n)
{
    if (check(GS_F32, count, m, n) != GS_OK) return 0;
    const Layout L = layout_of(count, m, n);
    return L.bytes < 256 ? 256 : (size_t)L.bytes;
}

extern "C" int gs_orthogonalise(int type, int count, int m, int n, const void* update, int steps, void* out,
                                void* workspace, hipStream_t stream)
{
    gs::clear_error();
    if (int rc = check(type, count, m, n)) return rc;
    GS_REQUIRE(steps >= 1 && steps <= 32, "orthogonalise: steps must be in [1, 32], got %d", steps);
    if (count == 0 || m == 0 || n == 0) return GS_OK;
    GS_REQUIRE(update && out && workspace, "orthogonalise: update, out and workspace must be non-null");
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
    const dim3 grid(gs_div_up((size_t)size, 256), (unsigned)count);
    if (type == GS_F32)
        hipLaunchKernelGGL(momentum_kernel<float>, grid, dim3(256), 0, stream, B, size, beta, nesterov, update);
    else if (type == GS_BF16)
        hipLaunchKernelGGL(momentum_kernel<gs::bf16>, grid, dim3(256), 0, stream, B, size, beta, nesterov, update);
    else hipLaunchKernelGGL(momentum_kernel<f16>, grid, dim3(256), 0, stream, B, size, beta, nesterov, update);
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
    const dim3 grid(gs_div_up((size_t)size, 256), (unsigned)count);
    if (type == GS_F32) hipLaunchKernelGGL(apply_kernel<float>, grid, dim3(256), 0, stream, B, size, keep, lr, update);
    else if (type == GS_BF16)
        hipLaunchKernelGGL(apply_kernel<gs::bf16>, grid, dim3(256), 0, stream, B, size, keep, lr, update);
    else hipLaunchKernelGGL(apply_kernel<f16>, grid, dim3(256), 0, stream, B, size, keep, lr, update);
    GS_LAUNCH_CHECK("apply_kernel");
    return GS_OK;
}
