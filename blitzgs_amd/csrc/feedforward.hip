// The gated feed-forward block, forward and backward.
//
//   a = x G^T, b = x U^T, h = act(a) b, y = h D^T      x (M, W); G, U (H, W); D (O, H)
//   dh = dy D;  da = dh b act'(a), db = dh act(a)
//   dx = da G + db U;  dG = da^T x, dU = db^T x, dD = dy^T h
//
// Nine products of 2 M W H operations where O = W, on the matrix cores; the
// activation, its derivative and the products with them happen in the registers of
// the product before.  One kernel takes them all: C (rows x cols) = sum over k of
// L(row, k) R(col, k), where an operand lies either with k along its rows (x, G, dy
// of dh, ...) or down its rows (D of dh, all of the weights' gradients); the latter
// reaches the matrix cores through transposing LDS reads.
//   HIDDEN  L = x, R = G and U, 16 columns of one and 16 of the other in turn, so
//           that a lane holds a and b of the same elements
//   GRAD    L = dy, R = D (down); leaves da and db
//   SUM     two pairs of operands one after the other along k: dx
//   PLAIN   y, dG, dU, dD
//
// Sums are fp32.  Rounded to the tensors' type: each output once, h, and for the
// backward a, b, da and db, since they are operands of the next product: float16's
// range holds for them too.
#include "gs_host.h"
#include "gs_matrix.h"
#include "../../include/blitzgs_amd.h"

namespace {

using gs::f4;
using gs::Frag;

enum Kind { HIDDEN, GRAD, SUM, PLAIN };

// One product.  Operands' rows (or, down, k) are `ld` elements apart.
struct Product {
    const void* l[2];
    const void* r[2];
    int64_t lld, rld, old;
    int rows, cols, depth;        // of the result, and of each pair of operands
    int tiles_m, tiles_n;
    void* out[3];                 // HIDDEN: h, a, b; GRAD: da, db; else the result
    const void* in[2];            // GRAD: a, b
    int first;                    // workgroup
};

// Products of one kind in one launch.
struct FeedArgs {
    Product p[3];
    int count;
    int act;
    int splits;                   // of the depth
    float* part;
};

__device__ __align__(16) const uint32_t zeros[4] = {0, 0, 0, 0};

// act(a) and its derivative
__device__ __forceinline__ void activation(int act, float a, float& value, float& slope)
{
    if (act == GS_SILU) {
        const float s = 1.0f / (1.0f + expf(-a));
        value = a * s;
        slope = s * __builtin_fmaf(a, 1.0f - s, 1.0f);
    } else {
        // the normal distribution, without cancellation where it is small
        const float phi = 0.5f * erfcf(a * -0.70710678f);
        value = a * phi;
        slope = __builtin_fmaf(a, 0.39894228f * expf(-0.5f * a * a), phi);
    }
}

// An operand's tiles of S rows of the result by KT of the depth, KT elements being
// 128 bytes.  Along: S rows of 128 bytes.  DOWN: KT rows of S elements, as S / KT
// tiles of KT columns, the rows in the order in which Tile::cols takes them as
// k = 8 g + j.
//   DIRECT: straight to LDS, 16 bytes at a time; chunks are whole and aligned.  What
//           lies beyond the depth comes from `zeros`; beyond the last row or column
//           the last one comes again, whose results nobody keeps.
//   else:   through registers, element by element at the edges
template <typename T, int S, bool DOWN, int THREADS, bool DIRECT>
struct Operand {
    static constexpr int KT = 128 / (int)sizeof(T), V = gs::Vec<T>::N, CH = S * 8 / THREADS;
    static_assert(CH >= 1, "a chunk per thread");
    using L = gs::Tile<T, KT>;

    // place `id` of the tile holds k (or the chunk of k from there) and row of the result
    __device__ static __forceinline__ void place(int id, int& row, int& k)
    {
        const int r = DOWN ? id / 8 % KT : id / 8, col = (L::chunk(r, id % 8) - r * 8) * V;
        if constexpr (DOWN) {
            const int q = r % 32;
            row = id / (8 * KT) * KT + col;
            k = r / 32 * 32 + 8 * (q % 16 / 4) + 4 * (q / 16) + q % 4;
        } else {
            row = r;
            k = col;
        }
    }

    // Fetches the tile whose depth begins at k0.  pick(row): the pointer to a row of the result's
    // operand (along), or to its column in row 0 (DOWN).
    template <typename Pick>
    __device__ static __forceinline__ void fetch(uint4* to, int k0, int depth, int limit, int64_t ld, Pick pick)
    {
        typedef const __attribute__((address_space(1))) void* global_ptr;
        typedef __attribute__((address_space(3))) void* lds_ptr;
#pragma unroll
        for (int c = 0; c < CH; c++) {
            int row, k;
            place(threadIdx.x + THREADS * c, row, k);
            k += k0;
            if constexpr (DIRECT) {
                const T* p = DOWN ? pick(row) + (int64_t)k * ld : pick(row) + k;
                const void* from = k < depth ? (const void*)p : (const void*)zeros;
                __builtin_amdgcn_global_load_lds((global_ptr)from, (lds_ptr)(to + THREADS * c + (threadIdx.x & ~63u)),
                                                 16, 0, 0);
            } else {
                gs::Vec<T> v = {};
#pragma unroll
                for (int e = 0; e < V; e++) {
                    if constexpr (DOWN) {
                        if (k < depth && row + e < limit) v.v[e] = pick(row)[(int64_t)k * ld + e];
                    } else {
                        if (k + e < depth && row < limit) v.v[e] = pick(row)[k + e];
                    }
                }
                to[threadIdx.x + THREADS * c] = __builtin_bit_cast(uint4, v);
            }
        }
    }
};

template <typename T, int N>
__device__ __forceinline__ void put(T* p, const float* v, int n)
{
    T t[N];
#pragma unroll
    for (int i = 0; i < N; i++) t[i] = (T)v[i];
    if (n >= N) {
        __builtin_memcpy(p, t, sizeof(t));
    } else {
#pragma unroll
        for (int i = 0; i < N; i++)
            if (i < n) p[i] = t[i];
    }
}

template <typename T, int N>
__device__ __forceinline__ void get(const T* p, float* v, int n)
{
    T t[N] = {};
    if (n >= N) {
        __builtin_memcpy(t, p, sizeof(t));
    } else {
#pragma unroll
        for (int i = 0; i < N; i++)
            if (i < n) t[i] = p[i];
    }
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = (float)t[i];
}

// S x S of the result; waves in a grid of WM x WN.
template <typename T, Kind K, bool LDOWN, bool RDOWN, int S, int WM, int WN, bool DIRECT>
__global__ __launch_bounds__(64 * WM * WN, S == 256 ? 2 : 1) void feed_kernel(FeedArgs A)
{
    constexpr int THREADS = 64 * WM * WN, KT = 128 / (int)sizeof(T), WORDS = S * 8;
    constexpr int HM = S / WM, HN = S / WN, MT = HM / 16, NT = HN / 16;   // of a wave
    using OL = Operand<T, S, LDOWN, THREADS, DIRECT>;
    using OR = Operand<T, S, RDOWN, THREADS, DIRECT>;
    extern __shared__ uint4 lds[];                   // [2][left, right]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
    int which = 0;
    const uint32_t place = gs::xcd_item(blockIdx.x, gridDim.x);
    while (which + 1 < A.count && (int)place >= A.p[which + 1].first) which++;
    const Product& P = A.p[which];
    const int item = (int)place - P.first, tile_item = item / A.splits, split = item % A.splits;
    const int tm = tile_item % P.tiles_m, tn = tile_item / P.tiles_m;
    const int m0 = tm * S, n0 = tn * (K == HIDDEN ? S / 2 : S);
    const int wm = wave % WM * HM, wn = wave / WM * HN;

    f4 acc[NT][MT];
#pragma unroll
    for (int u = 0; u < NT; u++)
#pragma unroll
        for (int v = 0; v < MT; v++) acc[u][v] = f4{0, 0, 0, 0};

    const int per = (P.depth + KT - 1) / KT, all = K == SUM ? 2 * per : per;
    const int begin = (int)((int64_t)all * split / A.splits), end = (int)((int64_t)all * (split + 1) / A.splits);
    const gs::Tile<T, KT> tile;
    auto fetch = [&](int t, uint4* to) __attribute__((always_inline)) {
        const int second = K == SUM && t >= per;
        const int k0 = (t - second * per) * KT;
        const T* l = (const T*)P.l[second];
        const T* r = (const T*)P.r[second];
        OL::fetch(to, k0, P.depth, P.rows - m0, P.lld, [&](int row) {
            const int at = m0 + row;
            if constexpr (LDOWN) return l + (DIRECT ? min(at, P.rows - OL::V) : at);
            else return l + (int64_t)(DIRECT ? min(at, P.rows - 1) : at) * P.lld;
        });
        OR::fetch(to + WORDS, k0, P.depth, K == HIDDEN ? S : P.cols - n0, P.rld, [&](int row) {
            if constexpr (K == HIDDEN) {
                // 16 of the gate's rows, then 16 of up's; rows beyond the last hold the last again
                const int at = min(n0 + row / 32 * 16 + row % 16, P.cols - 1);
                return (const T*)P.r[row / 16 % 2] + (int64_t)at * P.rld;
            } else {
                const int at = n0 + row;
                if constexpr (RDOWN) return r + (DIRECT ? min(at, P.cols - OR::V) : at);
                else return r + (int64_t)(DIRECT ? min(at, P.cols - 1) : at) * P.rld;
            }
        });
    };
    // two restricted pointers tell the compiler that the loads need not have arrived
    // before the reads
    auto step = [&](int t, const uint4* __restrict__ at, uint4* __restrict__ next) __attribute__((always_inline)) {
        __syncthreads();   // tile t is there for all waves, and all are done with tile t - 1
        if (t + 1 < end) fetch(t + 1, next);
#pragma unroll
        for (int k = 0; k < KT; k += 32) {
            Frag<T> l[MT];
#pragma unroll
            for (int v = 0; v < MT; v++) {
                const int row = wm + 16 * v;
                if constexpr (LDOWN) l[v] = tile.cols(at + row / KT * (8 * KT), k, row % KT);
                else l[v] = tile.rows(at, row, k);
            }
#pragma unroll
            for (int u = 0; u < NT; u++) {
                const int row = wn + 16 * u;
                Frag<T> r;
                if constexpr (RDOWN) r = tile.cols(at + WORDS + row / KT * (8 * KT), k, row % KT);
                else r = tile.rows(at + WORDS, row, k);
#pragma unroll
                for (int v = 0; v < MT; v++) acc[u][v] = gs::mma(r, l[v], acc[u][v]);
            }
        }
    };
    if (begin < end) fetch(begin, lds);
    for (int t = begin; t < end; t++)
        step(t, lds + (t - begin) % 2 * 2 * WORDS, lds + (t - begin + 1) % 2 * 2 * WORDS);

    // lane: row 16 v + i of the result, columns 16 u + 4 g .. + 3
    if (A.splits > 1) {
        f4* part = (f4*)A.part + (int64_t)place * (NT * MT * THREADS) + threadIdx.x;
#pragma unroll
        for (int u = 0; u < NT; u++)
#pragma unroll
            for (int v = 0; v < MT; v++) part[(u * MT + v) * THREADS] = acc[u][v];
        return;
    }
#pragma unroll
    for (int v = 0; v < MT; v++) {
        const int row = m0 + wm + 16 * v + i;
        if (row >= P.rows) continue;
#pragma unroll
        for (int u = 0; u < NT; u += K == HIDDEN ? 2 : 1) {
            const int col = K == HIDDEN ? n0 + (wn + 16 * u) / 2 + 4 * g : n0 + wn + 16 * u + 4 * g;
            const int n = P.cols - col;
            if (n <= 0) continue;
            const int64_t at = (int64_t)row * P.old + col;
            float o[4];
            if constexpr (K == HIDDEN) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float value, slope;
                    activation(A.act, acc[u][v][e], value, slope);
                    o[e] = value * acc[u + 1][v][e];
                }
                put<T, 4>((T*)P.out[0] + at, o, n);
                if (P.out[1] != nullptr) {
#pragma unroll
                    for (int w = 0; w < 2; w++) {
#pragma unroll
                        for (int e = 0; e < 4; e++) o[e] = acc[u + w][v][e];
                        put<T, 4>((T*)P.out[1 + w] + at, o, n);
                    }
                }
            } else if constexpr (K == GRAD) {
                float a[4], b[4], d[4];
                get<T, 4>((const T*)P.in[0] + at, a, n);
                get<T, 4>((const T*)P.in[1] + at, b, n);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float value, slope;
                    activation(A.act, a[e], value, slope);
                    o[e] = acc[u][v][e] * b[e] * slope;
                    d[e] = acc[u][v][e] * value;
                }
                put<T, 4>((T*)P.out[0] + at, o, n);
                put<T, 4>((T*)P.out[1] + at, d, n);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) o[e] = acc[u][v][e];
                put<T, 4>((T*)P.out[0] + at, o, n);
            }
        }
    }
}

template <typename T, Kind K, bool LDOWN, bool RDOWN>
int launch_tiles(FeedArgs& A, bool direct, hipStream_t stream)
{
    constexpr int S = 128;
    int blocks = 0;
    for (int i = 0; i < A.count; i++) {
        Product& P = A.p[i];
        P.tiles_m = (P.rows + S - 1) / S;
        P.tiles_n = (P.cols + (K == HIDDEN ? S / 2 : S) - 1) / (K == HIDDEN ? S / 2 : S);
        P.first = blocks;
        const int64_t n = (int64_t)P.tiles_m * P.tiles_n * A.splits;
        GS_REQUIRE(n + blocks < 0x7fffffff, "feed forward: too many tiles");
        blocks += (int)n;
    }
    if (blocks == 0) return GS_OK;
    const size_t lds = 4 * S * 128;
    if (direct)
        GS_TIMED("feed_kernel", stream,
                 hipLaunchKernelGGL((feed_kernel<T, K, LDOWN, RDOWN, S, 2, 2, true>), dim3(blocks), dim3(256), lds,
                                    stream, A));
    else
        GS_TIMED("feed_kernel", stream,
                 hipLaunchKernelGGL((feed_kernel<T, K, LDOWN, RDOWN, S, 2, 2, false>), dim3(blocks), dim3(256), lds,
                                    stream, A));
    GS_LAUNCH_CHECK("feed_kernel");
    return GS_OK;
}

template <Kind K, bool LDOWN, bool RDOWN>
int launch(int type, FeedArgs& A, bool direct, hipStream_t stream)
{
    if (type == GS_F32) return launch_tiles<float, K, LDOWN, RDOWN>(A, direct, stream);
    if (type == GS_BF16) return launch_tiles<gs::bf16, K, LDOWN, RDOWN>(A, direct, stream);
    return launch_tiles<gs::f16, K, LDOWN, RDOWN>(A, direct, stream);
}

constexpr int MAX_SIDE = 1 << 24;

int check(int type, int activation, int64_t rows, int width, int hidden, int out)
{
    GS_REQUIRE(gs::dtype_known(type), "feed forward: unknown element type %d", type);
    GS_REQUIRE(activation == GS_SILU || activation == GS_GELU, "feed forward: unknown activation %d", activation);
    GS_REQUIRE(rows >= 0 && rows < 0x7fff0000, "feed forward: rows must be in [0, 2^31 - 2^16)");
    for (int n : {width, hidden, out})
        GS_REQUIRE(n >= 1 && n <= MAX_SIDE, "feed forward: width, hidden and out must be in [1, 2^24], got %d", n);
    return GS_OK;
}

// Whether rows of `n` elements, `ld` apart from p on, are whole 16-byte pieces
bool whole(const void* p, int64_t ld, int n, int type)
{
    const int v = 16 / gs::dtype_bytes(type);
    return (uintptr_t)p % 16 == 0 && ld % v == 0 && n % v == 0;
}

size_t padded(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace

extern "C" size_t gs_feed_forward_workspace_bytes(int type, int64_t rows, int width, int hidden, int out, int backward)
{
    if (check(type, GS_SILU, rows, width, hidden, out) != GS_OK) return 0;
    if (!backward) return 0;
    return 2 * padded((size_t)rows * hidden * gs::dtype_bytes(type)) + 256;
}

extern "C" int gs_feed_forward(int type, int activation, int64_t rows, int width, int hidden, int out, const void* x,
                               int64_t x_stride, const void* gate, const void* up, const void* down, void* a, void* b,
                               void* h, void* y, void* workspace, hipStream_t stream)
{
    gs::clear_error();
    if (int rc = check(type, activation, rows, width, hidden, out)) return rc;
    GS_REQUIRE((a == nullptr) == (b == nullptr), "feed forward: a and b come together");
    if (rows == 0) return GS_OK;
    GS_REQUIRE(x && gate && up && down && h && y, "feed forward: x, the weights, h and y must be non-null");
    FeedArgs A{};
    A.act = activation;
    A.splits = 1;
    A.count = 1;
    Product& P = A.p[0];
    P.l[0] = x;
    P.lld = x_stride;
    P.r[0] = gate;
    P.r[1] = up;
    P.rld = width;
    P.rows = (int)rows;
    P.cols = hidden;
    P.depth = width;
    P.old = hidden;
    P.out[0] = h;
    P.out[1] = a;
    P.out[2] = b;
    bool direct = whole(x, x_stride, width, type) && whole(gate, width, width, type) && whole(up, width, width, type);
    if (int rc = launch<HIDDEN, false, false>(type, A, direct, stream)) return rc;
    P = Product{};
    P.l[0] = h;
    P.lld = hidden;
    P.r[0] = down;
    P.rld = hidden;
    P.rows = (int)rows;
    P.cols = out;
    P.depth = hidden;
    P.old = out;
    P.out[0] = y;
    direct = whole(h, hidden, hidden, type) && whole(down, hidden, hidden, type);
    return launch<PLAIN, false, false>(type, A, direct, stream);
}

extern "C" int gs_feed_forward_backward(int type, int activation, int64_t rows, int width, int hidden, int out,
                                        const void* x, int64_t x_stride, const void* gate, const void* up,
                                        const void* down, const void* a, const void* b, const void* h, const void* dy,
                                        int64_t dy_stride, void* dx, void* dgate, void* dup, void* ddown,
                                        void* workspace, hipStream_t stream)
{
    gs::clear_error();
    if (int rc = check(type, activation, rows, width, hidden, out)) return rc;
    const bool inner = dx != nullptr || dgate != nullptr || dup != nullptr;
    if (!inner && ddown == nullptr) return GS_OK;
    if (rows > 0) {
        GS_REQUIRE(x && gate && up && down && a && b && h && dy,
                   "feed forward: x, the weights, a, b, h and dy must be non-null");
        GS_REQUIRE(!inner || (workspace != nullptr && (uintptr_t)workspace % 256 == 0),
                   "feed forward: the backward needs its workspace, 256-byte aligned");
    }
    char* da = (char*)workspace;
    char* db = da + padded((size_t)rows * hidden * gs::dtype_bytes(type));
    FeedArgs A{};
    A.act = activation;
    A.splits = 1;
    A.count = 1;
    if (inner && rows > 0) {
        Product& P = A.p[0];
        P.l[0] = dy;
        P.lld = dy_stride;
        P.r[0] = down;
        P.rld = hidden;
        P.rows = (int)rows;
        P.cols = hidden;
        P.depth = out;
        P.old = hidden;
        P.out[0] = da;
        P.out[1] = db;
        P.in[0] = a;
        P.in[1] = b;
        const bool direct = whole(dy, dy_stride, out, type) && whole(down, hidden, hidden, type);
        if (int rc = launch<GRAD, false, true>(type, A, direct, stream)) return rc;
    }
    if (dx != nullptr && rows > 0) {
        Product& P = A.p[0];
        P = Product{};
        P.l[0] = da;
        P.l[1] = db;
        P.lld = hidden;
        P.r[0] = gate;
        P.r[1] = up;
        P.rld = width;
        P.rows = (int)rows;
        P.cols = width;
        P.depth = hidden;
        P.old = width;
        P.out[0] = dx;
        const bool direct = whole(da, hidden, hidden, type) && whole(gate, width, width, type) &&
                            whole(up, width, width, type);
        if (int rc = launch<SUM, false, true>(type, A, direct, stream)) return rc;
    }
    // the weights' gradients, one after the other in one launch
    A.count = 0;
    bool direct = true;
    auto add = [&](const void* l, int64_t lld, int m, const void* r, int64_t rld, int n, void* to) {
        if (to == nullptr) return;
        Product& P = A.p[A.count++];
        P = Product{};
        P.l[0] = l;
        P.lld = lld;
        P.r[0] = r;
        P.rld = rld;
        P.rows = m;
        P.cols = n;
        P.depth = (int)rows;
        P.old = n;
        P.out[0] = to;
        direct = direct && whole(l, lld, m, type) && whole(r, rld, n, type);
    };
    add(da, hidden, hidden, x, x_stride, width, dgate);
    add(db, hidden, hidden, x, x_stride, width, dup);
    add(dy, dy_stride, out, h, hidden, hidden, ddown);
    if (A.count == 0) return GS_OK;
    return launch<PLAIN, true, true>(type, A, direct, stream);
}
