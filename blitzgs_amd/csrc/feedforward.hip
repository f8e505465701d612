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
#include <atomic>

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

// All waves' loads to LDS are there, and all waves are done with what they read: a
// barrier alone waits for neither where the compiler sees that this wave's own reads
// need not.
__device__ __forceinline__ void arrived()
{
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

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
//   else:   through registers, element by element
template <typename T, int S, bool DOWN, int THREADS, bool DIRECT>
struct Operand {
    static constexpr int KT = 128 / (int)sizeof(T), V = gs::Vec<T>::N, CH = S * 8 / THREADS;
    static_assert(CH >= 1 && THREADS % 256 == 0, "a chunk per thread, 32 rows or more per access");
    using L = gs::Tile<T, KT>;
    typedef __attribute__((address_space(3))) void* lds_ptr;

    uint32_t at[CH];   // bytes from the tile's corner

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
    // map(row): the place of the result's row among the operand's rows (DOWN: columns), of which there are `limit`
    template <typename Map>
    __device__ __forceinline__ Operand(int64_t ld, int limit, Map map)
    {
#pragma unroll
        for (int c = 0; c < CH; c++) {
            int row, k;
            place(threadIdx.x + THREADS * c, row, k);
            row = map(row);
            if constexpr (DOWN) at[c] = (uint32_t)(((int64_t)k * ld + min(row, limit - V)) * (int)sizeof(T));
            else at[c] = (uint32_t)(((int64_t)min(row, limit - 1) * ld + k) * (int)sizeof(T));
        }
    }
    // DIRECT: the tile at `from`, of which `depth` is there
    __device__ __forceinline__ void fetch(uint4* to, const T* from, int depth) const
    {
        const char* base = (const char*)from;
        uint4* mine = to + (threadIdx.x & ~63u);   // + 16 bytes per lane
        // As buffer loads: the compiler takes global ones to LDS for accesses of any kind, and
        // waits for all LDS reads while one is under way.  Their offsets are below `span`.
        const __amdgpu_buffer_rsrc_t all = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, -1, 0x27000);
        if (depth >= KT) {
#pragma unroll
            for (int c = 0; c < CH; c++)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(all, (lds_ptr)(mine + THREADS * c), 16, (int)at[c], 0, 0, 0);
        } else {
            const __amdgpu_buffer_rsrc_t none = __builtin_amdgcn_make_buffer_rsrc((void*)zeros, 0, 16, 0x27000);
#pragma unroll
            for (int c = 0; c < CH; c++) {
                int row, k;
                place(threadIdx.x + THREADS * c, row, k);
                if (k < depth)
                    __builtin_amdgcn_raw_ptr_buffer_load_lds(all, (lds_ptr)(mine + THREADS * c), 16, (int)at[c], 0, 0, 0);
                else
                    __builtin_amdgcn_raw_ptr_buffer_load_lds(none, (lds_ptr)(mine + THREADS * c), 16, 0, 0, 0, 0);
            }
        }
    }
    // else: the same, of which `limit` rows (DOWN: columns) are there
    template <typename Map>
    __device__ static __forceinline__ void gather(uint4* to, const T* from, int depth, int64_t ld, int limit, Map map)
    {
#pragma unroll
        for (int c = 0; c < CH; c++) {
            int row, k;
            place(threadIdx.x + THREADS * c, row, k);
            gs::Vec<T> v = {};
#pragma unroll
            for (int e = 0; e < V; e++) {
                if constexpr (DOWN) {
                    if (k < depth && map(row) + e < limit) v.v[e] = from[(int64_t)k * ld + map(row) + e];
                } else {
                    if (k + e < depth && map(row) < limit) v.v[e] = from[(int64_t)map(row) * ld + k + e];
                }
            }
            to[threadIdx.x + THREADS * c] = __builtin_bit_cast(uint4, v);
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

// SM x SN of the result; waves in a grid of WM x WN.
template <typename T, Kind K, bool LDOWN, bool RDOWN, int SM, int SN, int WM, int WN, bool DIRECT>
__global__ __launch_bounds__(64 * WM * WN, 2) void feed_kernel(FeedArgs A)
{
    constexpr int THREADS = 64 * WM * WN, KT = 128 / (int)sizeof(T), LW = SM * 8, RW = SN * 8;
    constexpr int HM = SM / WM, HN = SN / WN, MT = HM / 16, NT = HN / 16;   // of a wave
    using OL = Operand<T, SM, LDOWN, THREADS, DIRECT>;
    using OR = Operand<T, SN, RDOWN, THREADS, DIRECT>;
    extern __shared__ uint4 lds[];                   // [2][left, right]
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int which = 0;
    const uint32_t place = gs::xcd_item(blockIdx.x, gridDim.x);
    while (which + 1 < A.count && (int)place >= A.p[which + 1].first) which++;
    const Product& P = A.p[which];
    const int item = (int)place - P.first, tile_item = item / A.splits, split = item % A.splits;
    // runs of eight rows of tiles: the 32 tiles that an XCD works on at a time are 8 x 4
    const int run = tile_item / (8 * P.tiles_n), high = min(8, P.tiles_m - 8 * run), in_run = tile_item - run * 8 * P.tiles_n;
    const int tm = 8 * run + in_run % high, tn = in_run / high;
    const int m0 = tm * SM, n0 = tn * (K == HIDDEN ? SN / 2 : SN);
    const int wm = wave % WM * HM, wn = wave / WM * HN;

    f4 acc[NT][MT];
#pragma unroll
    for (int u = 0; u < NT; u++)
#pragma unroll
        for (int v = 0; v < MT; v++) acc[u][v] = f4{0, 0, 0, 0};

    const int per = (P.depth + KT - 1) / KT, all = K == SUM ? 2 * per : per;
    const int begin = (int)((int64_t)all * split / A.splits), end = (int)((int64_t)all * (split + 1) / A.splits);
    // 16 rows of the gate, then 16 of up; a wave's eight rows of an access are of one
    const int which_r = K == HIDDEN ? wave / 2 % 2 : 0;
    auto left = [](int row) { return row; };
    auto right = [](int row) { return K == HIDDEN ? row / 32 * 16 + row % 16 : row; };
    const int lrows = P.rows - m0, rrows = P.cols - n0;
    const OL ol(P.lld, lrows, left);
    const OR orr(P.rld, rrows, right);
    // The next tile's corners, how much of the depth is left there, and the steps to the
    // tile after it; held in registers, so that the loop reads no arguments (whose loads
    // would be waited for together with those from LDS).
    const int second = K == SUM && begin >= per, k0 = (begin - second * per) * KT;
    const T* lp = (const T*)P.l[second] + (LDOWN ? (int64_t)k0 * P.lld + m0 : (int64_t)m0 * P.lld + k0);
    const T* rp = (const T*)P.r[second + which_r] + (RDOWN ? (int64_t)k0 * P.rld + n0 : (int64_t)n0 * P.rld + k0);
    const T* lp2 = (const T*)P.l[1] + (LDOWN ? m0 : (int64_t)m0 * P.lld);
    const T* rp2 = (const T*)P.r[1] + (RDOWN ? n0 : (int64_t)n0 * P.rld);
    int64_t lstep = LDOWN ? KT * P.lld : KT, rstep = RDOWN ? KT * P.rld : KT;
    int depth = P.depth, rest = depth - k0;
    if (DIRECT) asm volatile("" : "+s"(lp), "+s"(rp), "+s"(lstep), "+s"(rstep), "+s"(rest));
    if (DIRECT && K == SUM) asm volatile("" : "+s"(lp2), "+s"(rp2), "+s"(depth));
    auto fetch = [&](uint4* to) __attribute__((always_inline)) {
        if constexpr (DIRECT) {
            ol.fetch(to, lp, rest);
            orr.fetch(to + LW, rp, rest);
        } else {
            OL::gather(to, lp, rest, P.lld, lrows, left);
            OR::gather(to + LW, rp, rest, P.rld, rrows, right);
        }
        lp += lstep;
        rp += rstep;
        rest -= KT;
        if (K == SUM && rest <= 0) {
            lp = lp2;
            rp = rp2;
            rest = depth;
        }
    };
    const gs::Tile<T, KT> tile;
    auto get_l = [&](const uint4* at, int k, int v) __attribute__((always_inline)) {
        const int row = wm + 16 * v;
        if constexpr (LDOWN) return tile.cols(at + row / KT * (8 * KT), k, row % KT);
        else return tile.rows(at, row, k);
    };
    auto get_r = [&](const uint4* at, int k, int u) __attribute__((always_inline)) {
        const int row = wn + 16 * u;
        if constexpr (RDOWN) return tile.cols(at + LW + row / KT * (8 * KT), k, row % KT);
        else return tile.rows(at + LW, row, k);
    };
    // A tile is STEPS steps of 32 of the depth and half of the wave's columns.  A step's
    // operands are read from LDS during the step before, its first step's behind the
    // barrier after which the tile is there and the one before it is free; a tile's loads
    // are under way for a whole tile.  Left to itself the compiler reads just before it
    // multiplies.
    constexpr int KS = KT / 32, STEPS = 2 * KS, NH = NT / 2;
    Frag<T> l[2][MT], r[2][NH];
    // Restricted pointers tell the compiler that loads into one need not have arrived
    // before reads of the other.
    auto body = [&](int t, uint4* __restrict__ cur, uint4* __restrict__ next) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            const int k = s / 2, h = s % 2;
            if (s + 1 < STEPS) {
#pragma unroll
                for (int u = 0; u < NH; u++) r[(s + 1) % 2][u] = get_r(cur, (s + 1) / 2 * 32, (s + 1) % 2 * NH + u);
                if (h == 1)
#pragma unroll
                    for (int v = 0; v < MT; v++) l[(k + 1) % 2][v] = get_l(cur, (k + 1) * 32, v);
            } else if (t + 1 < end) {
                arrived();
                if (t + 2 < end) fetch(cur);
#pragma unroll
                for (int u = 0; u < NH; u++) r[(s + 1) % 2][u] = get_r(next, 0, u);
#pragma unroll
                for (int v = 0; v < MT; v++) l[(k + 1) % 2][v] = get_l(next, 0, v);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = 0; u < NH; u++)
#pragma unroll
                for (int v = 0; v < MT; v++)
                    acc[h * NH + u][v] = gs::mma(r[s % 2][u], l[k % 2][v], acc[h * NH + u][v]);
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (KS % 2 == 1) {
#pragma unroll
            for (int v = 0; v < MT; v++) l[0][v] = l[1][v];
        }
    };
    auto walk = [&](uint4* __restrict__ one, uint4* __restrict__ two) __attribute__((always_inline)) {
        fetch(one);
        arrived();
        if (begin + 1 < end) fetch(two);
#pragma unroll
        for (int u = 0; u < NH; u++) r[0][u] = get_r(one, 0, u);
#pragma unroll
        for (int v = 0; v < MT; v++) l[0][v] = get_l(one, 0, v);
        for (int t = begin; t < end; t += 2) {
            body(t, one, two);
            if (t + 1 < end) body(t + 1, two, one);
        }
    };
    if (begin < end) walk(lds, lds + LW + RW);

    // a lane holds row 16 v + i, columns 16 u + 4 g .. + 3
    if (A.splits > 1) {
        f4* part = (f4*)A.part + (int64_t)place * (NT * MT * THREADS) + threadIdx.x;
#pragma unroll
        for (int u = 0; u < NT; u++)
#pragma unroll
            for (int v = 0; v < MT; v++) part[(u * MT + v) * THREADS] = acc[u][v];
        return;
    }
    // Results leave as whole rows, 16 rows of the wave's columns at a time: through LDS,
    // eight neighbours to a lane.  In the lanes' own pieces of 8 bytes the forward's
    // three results and the backward's two, with the two that they read, took as long
    // as the products.
    constexpr int C = (K == HIDDEN ? HN / 2 : HN) / 8, RP = 64 / C, LD = HN + 4;   // lanes and rows of a pass
    static_assert(C >= 4 && C <= 64, "whole rows of lanes");
    float* own = (float*)lds + wave * (16 * LD);
    const int c8 = lane % C * 8, col = (K == HIDDEN ? n0 + wn / 2 : n0 + wn) + c8, n = P.cols - col;
    __syncthreads();   // all waves are done with the tiles
#pragma unroll
    for (int v = 0; v < MT; v++) {
        const int row0 = m0 + wm + 16 * v;
        // before the exchange: what the result is multiplied with
        float in[16 / RP][2][8];
        if constexpr (K == GRAD) {
#pragma unroll
            for (int p = 0; p < 16 / RP; p++) {
                const int row = row0 + p * RP + lane / C;
                const int64_t at = (int64_t)row * P.old + col;
#pragma unroll
                for (int w = 0; w < 2; w++) get<T, 8>((const T*)P.in[w] + at, in[p][w], row < P.rows ? n : 0);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int u = 0; u < NT; u++) *(f4*)(own + i * LD + 16 * u + 4 * g) = acc[u][v];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int p = 0; p < 16 / RP; p++) {
            const int r = p * RP + lane / C, row = row0 + r;
            const float* from = own + r * LD;
            const int64_t at = (int64_t)row * P.old + col;
            const int here = row < P.rows ? n : 0;
            float o[8], d[8];
            if constexpr (K == HIDDEN) {
                // 16 of a and 16 of b in turn
                const float* f = from + c8 / 16 * 32 + c8 % 16;
                float a[8], b[8];
                __builtin_memcpy(a, f, 32);
                __builtin_memcpy(b, f + 16, 32);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    float value, slope;
                    activation(A.act, a[e], value, slope);
                    o[e] = value * b[e];
                }
                put<T, 8>((T*)P.out[0] + at, o, here);
                if (P.out[1] != nullptr) {
                    put<T, 8>((T*)P.out[1] + at, a, here);
                    put<T, 8>((T*)P.out[2] + at, b, here);
                }
            } else if constexpr (K == GRAD) {
                __builtin_memcpy(d, from + c8, 32);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    float value, slope;
                    activation(A.act, in[p][0][e], value, slope);
                    o[e] = d[e] * in[p][1][e] * slope;
                    d[e] = d[e] * value;
                }
                put<T, 8>((T*)P.out[0] + at, o, here);
                put<T, 8>((T*)P.out[1] + at, d, here);
            } else {
                __builtin_memcpy(o, from + c8, 32);
                put<T, 8>((T*)P.out[0] + at, o, here);
            }
        }
    }
}

template <typename T, Kind K, bool LDOWN, bool RDOWN, int SM, int SN, int WM, int WN, bool DIRECT>
int launch_tiles(FeedArgs& A, hipStream_t stream)
{
    int blocks = 0;
    for (int i = 0; i < A.count; i++) {
        Product& P = A.p[i];
        P.tiles_m = (P.rows + SM - 1) / SM;
        P.tiles_n = (P.cols + (K == HIDDEN ? SN / 2 : SN) - 1) / (K == HIDDEN ? SN / 2 : SN);
        P.first = blocks;
        const int64_t n = (int64_t)P.tiles_m * P.tiles_n * A.splits;
        GS_REQUIRE(n + blocks < 0x7fffffff, "feed forward: too many tiles");
        blocks += (int)n;
    }
    if (blocks == 0) return GS_OK;
    constexpr size_t LDS = 2 * (SM + SN) * 128;
    auto kernel = feed_kernel<T, K, LDOWN, RDOWN, SM, SN, WM, WN, DIRECT>;
    if constexpr (LDS > 65536) {
        // on the current device; a driver call, so once a device
        static std::atomic<uint64_t> told{0};
        int device = 0;
        GS_HIP(hipGetDevice(&device));
        const uint64_t bit = 1ull << (device & 63);
        if (!(told.load() & bit)) {
            GS_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS));
            told |= bit;
        }
    }
    GS_TIMED("feed_kernel", stream,
             hipLaunchKernelGGL(kernel, dim3(blocks), dim3(64 * WM * WN), LDS, stream, A));
    GS_LAUNCH_CHECK("feed_kernel");
    return GS_OK;
}

template <typename T, Kind K, bool LDOWN, bool RDOWN>
int launch_shape(FeedArgs& A, bool direct, hipStream_t stream)
{
    if constexpr (sizeof(T) == 2) {
        if (direct) {
            int64_t n = 0;
            for (int i = 0; i < A.count; i++)
                n += (int64_t)((A.p[i].rows + 255) / 256) * ((A.p[i].cols + (K == HIDDEN ? 127 : 255)) / (K == HIDDEN ? 128 : 256));
            if (n >= 160) return launch_tiles<T, K, LDOWN, RDOWN, 256, 256, 4, 2, true>(A, stream);
            if (n >= 64) return launch_tiles<T, K, LDOWN, RDOWN, 256, 128, 4, 2, true>(A, stream);
        }
    }
    if (direct) return launch_tiles<T, K, LDOWN, RDOWN, 128, 128, 2, 2, true>(A, stream);
    return launch_tiles<T, K, LDOWN, RDOWN, 128, 128, 2, 2, false>(A, stream);
}

template <Kind K, bool LDOWN, bool RDOWN>
int launch(int type, FeedArgs& A, bool direct, hipStream_t stream)
{
    if (type == GS_F32) return launch_shape<float, K, LDOWN, RDOWN>(A, direct, stream);
    if (type == GS_BF16) return launch_shape<gs::bf16, K, LDOWN, RDOWN>(A, direct, stream);
    return launch_shape<gs::f16, K, LDOWN, RDOWN>(A, direct, stream);
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
