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
// Sums are fp32.  Rounded to the tensors' type: each output once, and h, da and db, since
// they are operands of the next product: float16's range holds for them too.  The
// backward's a and b are kept in the tensors' type too, with four more bits each in a byte
// of their own: without those the errors of dx and the weights' gradients against 64 bits
// were 1.8 times that of their own rounding (bfloat16 0.0031, 0.0017), with them 1.4.
//
// 8192 rows, 1024 wide, 4096 hidden, bfloat16, forward and backward: 686 us, 900 TFLOP/s (a
// large library product: 1241): HIDDEN 167, GRAD 135, SUM 124, y 64, the weights' gradients
// 196.  One row through 2048 x 8192: 19.5 us, 5.2 TB/s of weights.
#include <atomic>
#include <type_traits>

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
    uint8_t* rest;                // of a and b, or null
    bool pad;                     // the result's rows end with zeros up to a whole piece of 8
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

// All waves' loads to LDS but their last N are there, and all waves are done with what
// they read.  In one piece: the compiler's own barrier waits for all loads.
template <int N>
__device__ __forceinline__ void arrived()
{
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// act(a) and its derivative.  For the 16-bit types, whose results are rounded to 2^-9 and
// more, with the hardware's exponential and reciprocal (off by 2^-20 of the value for |a|
// up to 16, where the sigmoid is 1e-7): the exact ones took a quarter of the backward's
// first product.
template <typename T>
__device__ __forceinline__ void activation(int act, float a, float& value, float& slope)
{
    if (act == GS_SILU) {
        const float s = sizeof(T) == 2 ? __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(a * -1.44269504f))
                                       : 1.0f / (1.0f + expf(-a));
        value = a * s;
        slope = s * __builtin_fmaf(a, 1.0f - s, 1.0f);
    } else {
        // the normal distribution, without cancellation where it is small
        const float phi = 0.5f * erfcf(a * -0.70710678f);
        value = a * phi;
        slope = __builtin_fmaf(a, 0.39894228f * expf(-0.5f * a * a), phi);
    }
}

// An operand's tiles of S rows of the result by KT of the depth, as tiles of rows of W
// elements, 128 bytes.  Along: KT / W tiles of S rows.  DOWN: S / W tiles of KT rows, which
// lie in the order in which Tile::cols takes them as k = 8 g + j.
//   DIRECT: straight to LDS, 16 bytes at a time; chunks are aligned and whole, with zeros
//           behind the last element of an operand's row where its length is no whole
//           number of them.  What lies beyond the depth comes from `zeros`; beyond the
//           last row or column the last one comes again, whose results nobody keeps.
//   else:   through registers, from any address; what lies beyond is zero
template <typename T, int S, int KT, bool DOWN, int THREADS, bool DIRECT>
struct Operand {
    static constexpr int V = gs::Vec<T>::N, W = 128 / (int)sizeof(T), ROWS = DOWN ? KT : S;
    static constexpr int WORDS = S * KT / V, CH = WORDS / THREADS;
    static_assert(WORDS % THREADS == 0 && THREADS % 256 == 0, "whole accesses, of 32 rows or more");
    static_assert(KT % W == 0 && S % (DOWN ? W : 16) == 0, "whole tiles");
    using L = gs::Tile<T, W>;
    typedef __attribute__((address_space(3))) void* lds_ptr;

    uint32_t at[DIRECT ? CH : 1];   // bytes from the tile's corner

    // place `id` of the tile holds k (or the chunk of k from there) and row of the result
    __device__ static __forceinline__ void place(int id, int& row, int& k)
    {
        const int r = id / 8 % ROWS, col = (L::chunk(r, id % 8) - r * 8) * V, sub = id / (8 * ROWS) * W;
        if constexpr (DOWN) {
            const int q = r % 32;
            row = sub + col;
            k = r / 32 * 32 + 8 * (q % 16 / 4) + 4 * (q / 16) + q % 4;
        } else {
            row = r;
            k = sub + col;
        }
    }
    // map(row): the place of the result's row among the operand's rows (DOWN: columns), of which there are `limit`
    template <typename Map>
    __device__ __forceinline__ Operand(int64_t ld, int limit, Map map)
    {
        if constexpr (DIRECT) {
#pragma unroll
            for (int c = 0; c < CH; c++) {
                int row, k;
                place(threadIdx.x + THREADS * c, row, k);
                row = map(row);
                if constexpr (DOWN) at[c] = (uint32_t)(((int64_t)k * ld + min(row, (limit - 1) / V * V)) * (int)sizeof(T));
                else at[c] = (uint32_t)(((int64_t)min(row, limit - 1) * ld + k) * (int)sizeof(T));
            }
        }
    }
    // DIRECT: the tile at `from`, of which `depth` is there.  As buffer loads: the compiler
    // takes global ones to LDS for accesses of any kind, and waits for all LDS reads while
    // one is under way.
    __device__ __forceinline__ void fetch(uint4* to, const T* from, int depth) const
    {
        uint4* mine = to + (threadIdx.x & ~63u);   // + 16 bytes per lane
        const __amdgpu_buffer_rsrc_t all = __builtin_amdgcn_make_buffer_rsrc((void*)from, 0, -1, 0x27000);
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
    // else: the same to registers, of which `limit` rows (DOWN: columns) are there, and from there to LDS
    template <typename Map>
    __device__ static __forceinline__ void gather(gs::Vec<T> (&v)[CH], const T* from, int depth, int64_t ld, int limit,
                                                  Map map)
    {
#pragma unroll
        for (int c = 0; c < CH; c++) {
            int row, k;
            place(threadIdx.x + THREADS * c, row, k);
            row = map(row);
            const T* p = DOWN ? from + (int64_t)k * ld + row : from + (int64_t)row * ld + k;
            const int n = DOWN ? (k < depth ? limit - row : 0) : (row < limit ? depth - k : 0);
            v[c] = {};
            if (n >= V) {
                v[c] = gs::load_vec(p);
            } else {
#pragma unroll
                for (int e = 0; e < V; e++)
                    if (e < n) v[c].v[e] = p[e];
            }
        }
    }
    __device__ static __forceinline__ void settle(const gs::Vec<T> (&v)[CH], uint4* to)
    {
#pragma unroll
        for (int c = 0; c < CH; c++) to[threadIdx.x + THREADS * c] = __builtin_bit_cast(uint4, v[c]);
    }
};

template <typename T, int N>
struct Raw {
    T v[N];
};

// float16 ends at 65504, where a or b may not: beside a small b or a h, y and the gradients are
// within its range, and a slope of infinity is no number.  Such a number is kept, where it has a
// rest, as its sign, an exponent of ones and 14 bits, ten behind the exponent and four in the
// rest: float32's from 2^15 on, to seven of its mantissa.  What is no number is kept so too.
// Lanes look for an exponent of ones in their pieces of eight (case by case in every element
// HIDDEN and GRAD of 8192 x 1024 x 4096 took 25 us more).
__device__ __forceinline__ bool is_far(gs::f16 x) { return (__builtin_bit_cast(uint16_t, x) & 0x7c00u) == 0x7c00u; }
__device__ __forceinline__ bool any_far(const Raw<gs::f16, 8>& a, const Raw<gs::f16, 8>& b)
{
    const uint4 x = __builtin_bit_cast(uint4, a), y = __builtin_bit_cast(uint4, b);
    auto ones = [](uint32_t w) { return (w & 0x7c007c00u) + 0x04000400u; };
    return ((ones(x.x) | ones(x.y) | ones(x.z) | ones(x.w) | ones(y.x) | ones(y.y) | ones(y.z) | ones(y.w)) &
            0x80008000u) != 0;
}
__device__ __forceinline__ gs::f16 far_kept(float x, uint32_t& rest)
{
    const uint32_t code =
        ((x == x ? __float_as_uint(x) & 0x7fffffffu : 0x7fc00000u) - 0x47000000u + 0x8000u) >> 16;
    rest = code & 15u;
    return __builtin_bit_cast(gs::f16, (uint16_t)((__float_as_uint(x) >> 16 & 0x8000u) | 0x7c00u | code >> 4));
}
__device__ __forceinline__ float far_again(gs::f16 x, uint32_t rest)
{
    const uint32_t h = __builtin_bit_cast(uint16_t, x);
    return __uint_as_float((h & 0x8000u) << 16 | (0x47000000u + (((h & 0x3ffu) << 4 | (rest & 15u)) << 16)));
}

// Four bits of what rounding x to T left, in sixteenths of T's last bit, and x again.  As
// integers: numbers of one sign follow one another as their bits do.
template <typename T>
__device__ __forceinline__ uint32_t rest_of(float x)
{
    constexpr int SHIFT = __is_same(T, gs::bf16) ? 12 : 9;
    const uint32_t kept = __float_as_uint((float)(T)x);
    if ((kept & 0x7fffffffu) >= 0x7f800000u) return 0;
    const int q = ((int)(__float_as_uint(x) - kept) + (1 << (SHIFT - 1))) >> SHIFT;
    return (uint32_t)(q > 7 ? 7 : q < -8 ? -8 : q) & 15u;
}
template <typename T>
__device__ __forceinline__ float with_rest(T x, uint32_t rest)
{
    constexpr int SHIFT = __is_same(T, gs::bf16) ? 12 : 9;
    return __uint_as_float(__float_as_uint((float)x) + (uint32_t)(((int)(rest << 28) >> 28) * (1 << SHIFT)));
}

template <typename T, int N>
__device__ __forceinline__ Raw<T, N> rounded(const float* v)
{
    // in pairs, which the conversion instruction takes
    typedef T t2 __attribute__((ext_vector_type(2)));
    typedef float f2 __attribute__((ext_vector_type(2)));
    Raw<T, N> t;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const t2 two = __builtin_convertvector(f2{v[i], v[i + 1]}, t2);
        t.v[i] = two[0];
        t.v[i + 1] = two[1];
    }
    return t;
}

template <typename T, int N, bool WHOLE>
__device__ __forceinline__ void put(T* p, const Raw<T, N>& t, int n)
{
    if (WHOLE || n >= N) {
        __builtin_memcpy(p, &t, sizeof(t));
    } else {
#pragma unroll
        for (int i = 0; i < N; i++)
            if (i < n) p[i] = t.v[i];
    }
}

template <typename T, int N, bool WHOLE>
__device__ __forceinline__ void put(T* p, const float* v, int n)
{
    put<T, N, WHOLE>(p, rounded<T, N>(v), n);
}

template <typename T, int N, bool WHOLE>
__device__ __forceinline__ Raw<T, N> get(const T* p, int n)
{
    Raw<T, N> t = {};
    if (WHOLE || n >= N) {
        __builtin_memcpy(&t, p, sizeof(t));
    } else {
#pragma unroll
        for (int i = 0; i < N; i++)
            if (i < n) t.v[i] = p[i];
    }
    return t;
}

// How 16 rows of a wave's HN columns leave: through LDS, eight neighbours to a lane, as
// whole rows.  In the lanes' own pieces of 8 bytes the forward's three results and the
// backward's two, with the two that they read, took as long as the products.
template <typename T, Kind K, int HN>
struct Leave {
    static constexpr int C = (K == HIDDEN ? HN / 2 : HN) / 8, RP = 64 / C, PASSES = 16 / RP;   // lanes, rows of a pass
    static constexpr int LD = HN + 4;
    static_assert(C >= 4 && C <= 64, "whole rows of lanes");
    struct In {
        Raw<T, 8> v[PASSES][2];
        Raw<uint8_t, 8> rest[PASSES];
    };

    float* own;          // 16 rows of LD floats of the wave's
    int lane, act, rows, n;
    int64_t old;
    T *out0, *out1, *out2;
    const T *in0, *in1;
    uint8_t* rest;
    bool also, pad;

    __device__ __forceinline__ Leave(const Product& P, int act, float* own, int first)
        : own(own), lane(threadIdx.x & 63), act(act), rows(P.rows), old(P.old), also(P.out[1] != nullptr), pad(P.pad)
    {
        const int col = first + lane % C * 8;
        n = P.cols - col;
        out0 = (T*)P.out[0] + col;
        out1 = (T*)P.out[1] + col;
        out2 = (T*)P.out[2] + col;
        in0 = (const T*)P.in[0] + col;
        in1 = (const T*)P.in[1] + col;
        rest = P.rest == nullptr ? nullptr : P.rest + col;
    }
    // elements of this lane's eight that are there; WHOLE: all of the tile are
    template <bool WHOLE>
    __device__ __forceinline__ int here(int row) const
    {
        return WHOLE ? 8 : row < rows ? n : 0;
    }
    // what the rows from row0 on are multiplied with
    template <bool WHOLE>
    __device__ __forceinline__ void ask(In& in, int row0) const
    {
        if constexpr (K == GRAD) {
#pragma unroll
            for (int p = 0; p < PASSES; p++) {
                const int row = row0 + p * RP + lane / C;
                in.v[p][0] = get<T, 8, WHOLE>(in0 + row * old, here<WHOLE>(row));
                in.v[p][1] = get<T, 8, WHOLE>(in1 + row * old, here<WHOLE>(row));
                in.rest[p] = {};
                if (sizeof(T) == 2 && rest != nullptr)
                    in.rest[p] = get<uint8_t, 8, WHOLE>(rest + row * old, here<WHOLE>(row));
            }
        }
    }
    template <bool WHOLE>
    __device__ __forceinline__ void give(const In& in, const f4 (&acc)[HN / 16], int row0) const
    {
        const int i = lane & 15, g = lane >> 4, c8 = lane % C * 8;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int u = 0; u < HN / 16; u++) *(f4*)(own + i * LD + 16 * u + 4 * g) = acc[u];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int p = 0; p < PASSES; p++) {
            const int r = p * RP + lane / C, row = row0 + r, real = here<WHOLE>(row);
            const int count = !WHOLE && pad && real > 0 ? 8 : real;
            const float* from = own + r * LD;
            const int64_t at = row * old;
            float o[8], d[8];
            if constexpr (K == HIDDEN) {
                // 16 of a and 16 of b in turn
                const float* f = from + c8 / 16 * 32 + c8 % 16;
                float a[8], b[8];
                __builtin_memcpy(a, f, 32);
                __builtin_memcpy(b, f + 16, 32);
                if (!WHOLE && pad) {
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        if (e >= real) a[e] = b[e] = 0.0f;
                }
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    float value, slope;
                    activation<T>(act, a[e], value, slope);
                    o[e] = value * b[e];
                }
                put<T, 8, WHOLE>(out0 + at, o, count);
                if (also) {
                    Raw<T, 8> ka = rounded<T, 8>(a), kb = rounded<T, 8>(b);
                    if constexpr (sizeof(T) == 2) {
                        if (rest != nullptr) {
                            Raw<uint8_t, 8> q;
#pragma unroll
                            for (int e = 0; e < 8; e++) q.v[e] = (uint8_t)(rest_of<T>(a[e]) | rest_of<T>(b[e]) << 4);
                            if constexpr (__is_same(T, gs::f16)) {
                                if (any_far(ka, kb)) {
#pragma unroll
                                    for (int e = 0; e < 8; e++) {
                                        uint32_t ra = q.v[e] & 15u, rb = q.v[e] >> 4;
                                        if (is_far(ka.v[e])) ka.v[e] = far_kept(a[e], ra);
                                        if (is_far(kb.v[e])) kb.v[e] = far_kept(b[e], rb);
                                        q.v[e] = (uint8_t)(ra | rb << 4);
                                    }
                                }
                            }
                            put<uint8_t, 8, WHOLE>(rest + at, q, count);
                        }
                    }
                    put<T, 8, WHOLE>(out1 + at, ka, count);
                    put<T, 8, WHOLE>(out2 + at, kb, count);
                }
            } else if constexpr (K == GRAD) {
                __builtin_memcpy(d, from + c8, 32);
                const auto& [ha, hb] = in.v[p];
                float a[8], b[8];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    a[e] = (float)ha.v[e];
                    b[e] = (float)hb.v[e];
                    if constexpr (sizeof(T) == 2) {
                        a[e] = with_rest(ha.v[e], in.rest[p].v[e]);
                        b[e] = with_rest(hb.v[e], in.rest[p].v[e] >> 4);
                    }
                }
                if constexpr (__is_same(T, gs::f16)) {
                    if (rest != nullptr && any_far(ha, hb)) {
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            if (is_far(ha.v[e])) a[e] = far_again(ha.v[e], in.rest[p].v[e]);
                            if (is_far(hb.v[e])) b[e] = far_again(hb.v[e], in.rest[p].v[e] >> 4);
                        }
                    }
                }
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    float value, slope;
                    activation<T>(act, a[e], value, slope);
                    o[e] = d[e] * b[e] * slope;
                    d[e] = d[e] * value;
                    if (!WHOLE && pad && e >= real) o[e] = d[e] = 0.0f;
                }
                put<T, 8, WHOLE>(out0 + at, o, count);
                put<T, 8, WHOLE>(out1 + at, d, count);
            } else {
                __builtin_memcpy(o, from + c8, 32);
                put<T, 8, WHOLE>(out0 + at, o, count);
            }
        }
    }
};

// The product and the tile of it that a workgroup has.  Consecutive tiles are in runs of
// eight rows of tiles, and those of an XCD consecutive: the 32 that it works on at a time
// are 8 x 4, whose operands its L2 holds (the down projection of 8192 x 1024 x 4096 took
// 103 us with whole columns of tiles, 76 so).
struct Place {
    int which, tm, tn, split;
};

__device__ __forceinline__ Place place_of(const FeedArgs& A)
{
    const uint32_t place = gs::xcd_item(blockIdx.x, gridDim.x);
    Place p;
    p.which = 0;
    while (p.which + 1 < A.count && (int)place >= A.p[p.which + 1].first) p.which++;
    const Product& P = A.p[p.which];
    const int item = (int)place - P.first, tile = item / A.splits;
    p.split = item % A.splits;
    const int run = tile / (8 * P.tiles_n), high = min(8, P.tiles_m - 8 * run), in_run = tile - run * 8 * P.tiles_n;
    p.tm = 8 * run + in_run % high;
    p.tn = in_run / high;
    return p;
}

// Where an operand's next tile begins, how much of the depth is left there, and the steps
// to the tile after it; held in registers, so that the loops read no arguments (whose
// loads would be waited for together with those from LDS).
template <typename T, Kind K, int KT, bool LDOWN, bool RDOWN, bool DIRECT>
struct Walk {
    const T *l, *r, *l2, *r2;
    int64_t lstep, rstep;
    int depth, rest;

    __device__ __forceinline__ Walk(const Product& P, int m0, int n0, int which_r, int begin)
    {
        const int per = (P.depth + KT - 1) / KT, second = K == SUM && begin >= per, k0 = (begin - second * per) * KT;
        l = (const T*)P.l[second] + (LDOWN ? (int64_t)k0 * P.lld + m0 : (int64_t)m0 * P.lld + k0);
        r = (const T*)P.r[second + which_r] + (RDOWN ? (int64_t)k0 * P.rld + n0 : (int64_t)n0 * P.rld + k0);
        l2 = (const T*)P.l[1] + (LDOWN ? m0 : (int64_t)m0 * P.lld);
        r2 = (const T*)P.r[1] + (RDOWN ? n0 : (int64_t)n0 * P.rld);
        lstep = LDOWN ? KT * P.lld : KT;
        rstep = RDOWN ? KT * P.rld : KT;
        depth = P.depth;
        rest = depth - k0;
        // without DIRECT the compiler has to see that these point to global memory
        if (DIRECT) asm volatile("" : "+s"(l), "+s"(r), "+s"(lstep), "+s"(rstep), "+s"(rest));
        if (DIRECT && K == SUM) asm volatile("" : "+s"(l2), "+s"(r2), "+s"(depth));
    }
    __device__ __forceinline__ void next()
    {
        l += lstep;
        r += rstep;
        rest -= KT;
        if (K == SUM && rest <= 0) {
            l = l2;
            r = r2;
            rest = depth;
        }
    }
};

// 16-bit types, whole aligned chunks: SM x SN of the result, waves in a grid of WM x WN.
template <typename T, Kind K, bool LDOWN, bool RDOWN, int SM, int SN, int WM, int WN, int BUFFERS>
__global__ __launch_bounds__(64 * WM * WN, 2) void feed_kernel(FeedArgs A)
{
    constexpr int THREADS = 64 * WM * WN, KT = 64;
    constexpr int HM = SM / WM, HN = SN / WN, MT = HM / 16, NT = HN / 16;   // of a wave
    using OL = Operand<T, SM, KT, LDOWN, THREADS, true>;
    using OR = Operand<T, SN, KT, RDOWN, THREADS, true>;
    static_assert((!LDOWN || HM % OL::W == 0) && (!RDOWN || HN % OR::W == 0), "a wave's columns are whole tiles");
    constexpr int LW = OL::WORDS, RW = OR::WORDS, LOADS = OL::CH + OR::CH;
    extern __shared__ uint4 lds[];                   // [BUFFERS][left, right]
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Place at = place_of(A);
    const Product& P = A.p[at.which];
    const int m0 = at.tm * SM, n0 = at.tn * (K == HIDDEN ? SN / 2 : SN);
    const int wm = wave % WM * HM, wn = wave / WM * HN;

    f4 acc[MT][NT];
#pragma unroll
    for (int v = 0; v < MT; v++)
#pragma unroll
        for (int u = 0; u < NT; u++) acc[v][u] = f4{0, 0, 0, 0};

    const int end = (K == SUM ? 2 : 1) * ((P.depth + KT - 1) / KT);
    // 16 rows of the gate, then 16 of up; a wave's eight rows of an access are of one
    const OL ol(P.lld, P.rows - m0, [](int row) { return row; });
    const OR orr(P.rld, P.cols - n0, [](int row) { return K == HIDDEN ? row / 32 * 16 + row % 16 : row; });
    Walk<T, K, KT, LDOWN, RDOWN, true> walk(P, m0, n0, K == HIDDEN ? wave / 2 % 2 : 0, 0);
    auto fetch = [&](uint4* to) __attribute__((always_inline)) {
        ol.fetch(to, walk.l, walk.rest);
        orr.fetch(to + LW, walk.r, walk.rest);
        walk.next();
    };
    const gs::Tile<T, OL::W> tile;
    auto get_l = [&](const uint4* from, int k, int v) __attribute__((always_inline)) {
        const int row = wm + 16 * v;
        if constexpr (LDOWN) return tile.cols(from + row / OL::W * (8 * KT), k, row % OL::W);
        else return tile.rows(from, row, k);
    };
    auto get_r = [&](const uint4* from, int k, int u) __attribute__((always_inline)) {
        const int row = wn + 16 * u;
        if constexpr (RDOWN) return tile.cols(from + LW + row / OR::W * (8 * KT), k, row % OR::W);
        else return tile.rows(from + LW, row, k);
    };
    // A tile is four steps of 32 of the depth and half of the wave's columns.  A step's
    // operands are read from LDS during the step before, its first step's behind the
    // barrier after which the tile is there and the one before it is free: left to itself
    // the compiler reads just before it multiplies.  The loads of the tile BUFFERS on go
    // out there too, all at once: spread between the products they came too late (down
    // projection of 8192 x 1024 x 4096, two buffers, 83 us instead of 72).
    constexpr int STEPS = 4, NH = NT / 2;
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
                if (BUFFERS == 3 && t + 2 < end) arrived<LOADS>(); else arrived<0>();
                if (t + BUFFERS < end) fetch(cur);
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
                    acc[v][h * NH + u] = gs::mma(r[s % 2][u], l[k % 2][v], acc[v][h * NH + u]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto first = [&](const uint4* from) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < NH; u++) r[0][u] = get_r(from, 0, u);
#pragma unroll
        for (int v = 0; v < MT; v++) l[0][v] = get_l(from, 0, v);
    };
    auto walk2 = [&](uint4* __restrict__ one, uint4* __restrict__ two) __attribute__((always_inline)) {
        fetch(one);
        arrived<0>();
        if (1 < end) fetch(two);
        first(one);
        for (int t = 0; t < end; t += 2) {
            body(t, one, two);
            if (t + 1 < end) body(t + 1, two, one);
        }
    };
    auto walk3 = [&](uint4* __restrict__ one, uint4* __restrict__ two, uint4* __restrict__ three)
                     __attribute__((always_inline)) {
        fetch(one);
        if (1 < end) fetch(two);
        if (1 < end) arrived<LOADS>(); else arrived<0>();
        if (2 < end) fetch(three);
        first(one);
        for (int t = 0; t < end; t += 3) {
            body(t, one, two);
            if (t + 1 < end) body(t + 1, two, three);
            if (t + 2 < end) body(t + 2, three, one);
        }
    };
    if constexpr (BUFFERS == 3) walk3(lds, lds + LW + RW, lds + 2 * (LW + RW));
    else walk2(lds, lds + LW + RW);

    using Out = Leave<T, K, HN>;
    const Out out(P, A.act, (float*)lds + wave * (16 * Out::LD), K == HIDDEN ? n0 + wn / 2 : n0 + wn);
    auto finish = [&](auto whole) __attribute__((always_inline)) {
        constexpr bool WHOLE = decltype(whole)::value;
        // two rounds of 16 rows ahead
        typename Out::In in[2];
        out.template ask<WHOLE>(in[0], m0 + wm);
        if (MT > 1) out.template ask<WHOLE>(in[1], m0 + wm + 16);
        arrived<0>();   // all waves are done with the tiles
#pragma unroll
        for (int v = 0; v < MT; v++) {
            out.template give<WHOLE>(in[v % 2], acc[v], m0 + wm + 16 * v);
            if (v + 2 < MT) out.template ask<WHOLE>(in[v % 2], m0 + wm + 16 * (v + 2));
        }
    };
    if (P.rows - m0 >= SM && P.cols - n0 >= (K == HIDDEN ? SN / 2 : SN))
        finish(std::true_type{});
    else
        finish(std::false_type{});
}

// Few tiles, fp32, or chunks that are not whole: 64 x 64 of the result, of whose depth of
// 128 a turn each of four waves takes a quarter, so that a short depth keeps a workgroup
// busy and 64 columns fill its transposing reads.  The waves' sums meet at the end, in
// order.  With splits > 1 a workgroup has a part of the depth and leaves its sums in
// memory for feed_join_kernel.
constexpr int SS = 64, SKT = 128;

template <typename T, Kind K, bool LDOWN, bool RDOWN, bool DIRECT>
__global__ __launch_bounds__(256, 1) void feed_small_kernel(FeedArgs A)
{
    using OL = Operand<T, SS, SKT, LDOWN, 256, DIRECT>;
    using OR = Operand<T, SS, SKT, RDOWN, 256, DIRECT>;
    constexpr int WORDS = OL::WORDS, LOADS = 2 * OL::CH, N = SS / 16;
    constexpr int BUFFERS = DIRECT && sizeof(T) == 2 ? 3 : 2;
    extern __shared__ uint4 lds[];                   // [BUFFERS][left, right]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Place at = place_of(A);
    const Product& P = A.p[at.which];
    const int m0 = at.tm * SS, n0 = at.tn * (K == HIDDEN ? SS / 2 : SS);
    const int all = (K == SUM ? 2 : 1) * ((P.depth + SKT - 1) / SKT);
    const int begin = (int)((int64_t)all * at.split / A.splits), end = (int)((int64_t)all * (at.split + 1) / A.splits);

    f4 acc[N][N];
#pragma unroll
    for (int v = 0; v < N; v++)
#pragma unroll
        for (int u = 0; u < N; u++) acc[v][u] = f4{0, 0, 0, 0};

    auto left = [](int row) { return row; };
    auto right = [](int row) { return K == HIDDEN ? row / 32 * 16 + row % 16 : row; };
    const int lrows = P.rows - m0, rrows = P.cols - n0;
    const OL ol(P.lld, lrows, left);
    const OR orr(P.rld, rrows, right);
    Walk<T, K, SKT, LDOWN, RDOWN, DIRECT> walk(P, m0, n0, K == HIDDEN ? wave / 2 % 2 : 0, begin);
    const int64_t lld = P.lld, rld = P.rld;
    // a wave's quarter of the depth: a tile of 128 bytes, or half of one
    const gs::Tile<T, OL::W> tile;
    const int mine = sizeof(T) == 4 ? 0 : wave & 1 ? tile.row_at[OL::L::RB - 1] : tile.row_at[0];
    auto along = [&](const uint4* from, int v) __attribute__((always_inline)) {
        const uint4* t = from + 32 * wave / OL::W * (8 * SS);
        if constexpr (sizeof(T) == 4) {
            return tile.rows(t, 16 * v, 0);
        } else {
            Frag<T> f;
            f.v = __builtin_bit_cast(gs::s8, t[mine + 16 * v * 8]);
            return f;
        }
    };
    auto down = [&](const uint4* from, int u) __attribute__((always_inline)) {
        return tile.cols(from + 16 * u / OL::W * (8 * SKT) + 32 * 8 * wave, 0, 16 * u % OL::W);
    };
    auto multiply = [&](const uint4* from) __attribute__((always_inline)) {
        Frag<T> l[N], r[N];
#pragma unroll
        for (int v = 0; v < N; v++) {
            if constexpr (LDOWN) l[v] = down(from, v);
            else l[v] = along(from, v);
        }
#pragma unroll
        for (int u = 0; u < N; u++) {
            if constexpr (RDOWN) r[u] = down(from + WORDS, u);
            else r[u] = along(from + WORDS, u);
        }
#pragma unroll
        for (int u = 0; u < N; u++)
#pragma unroll
            for (int v = 0; v < N; v++) acc[v][u] = gs::mma(r[u], l[v], acc[v][u]);
    };
    if constexpr (DIRECT) {
        auto fetch = [&](uint4* to) __attribute__((always_inline)) {
            ol.fetch(to, walk.l, walk.rest);
            orr.fetch(to + WORDS, walk.r, walk.rest);
            walk.next();
        };
        // behind the barrier `cur` is there, and `far`, which the turn before read, is free
        auto body = [&](int t, uint4* __restrict__ cur, uint4* __restrict__ far) __attribute__((always_inline)) {
            if (BUFFERS == 3 && t + 1 < end) arrived<LOADS>(); else arrived<0>();
            if (t + BUFFERS - 1 < end) fetch(far);
            multiply(cur);
        };
        auto walk2 = [&](uint4* __restrict__ one, uint4* __restrict__ two) __attribute__((always_inline)) {
            fetch(one);
            for (int t = begin; t < end; t += 2) {
                body(t, one, two);
                if (t + 1 < end) body(t + 1, two, one);
            }
        };
        auto walk3 = [&](uint4* __restrict__ one, uint4* __restrict__ two, uint4* __restrict__ three)
                         __attribute__((always_inline)) {
            fetch(one);
            if (begin + 1 < end) fetch(two);
            for (int t = begin; t < end; t += 3) {
                body(t, one, three);
                if (t + 1 < end) body(t + 1, two, one);
                if (t + 2 < end) body(t + 2, three, two);
            }
        };
        if (begin < end) {
            if constexpr (BUFFERS == 3) walk3(lds, lds + 2 * WORDS, lds + 4 * WORDS);
            else walk2(lds, lds + 2 * WORDS);
        }
    } else {
        gs::Vec<T> lv[OL::CH], rv[OR::CH];
        auto gather = [&]() __attribute__((always_inline)) {
            OL::gather(lv, walk.l, walk.rest, lld, lrows, left);
            // the right operand's rows of HIDDEN are of two tensors, by the wave
            OR::gather(rv, walk.r, walk.rest, rld, rrows, right);
            walk.next();
        };
        if (begin < end) gather();
        for (int t = begin; t < end; t++) {
            uint4* cur = lds + (t - begin) % 2 * 2 * WORDS;
            OL::settle(lv, cur);
            OR::settle(rv, cur + WORDS);
            __syncthreads();   // the other tile was read before the barrier of the turn before
            if (t + 1 < end) gather();
            multiply(cur);
        }
    }
    // wave w takes the rows 16 w .. 16 w + 15 of all four waves' sums
    f4* meet = (f4*)lds;
    arrived<0>();
#pragma unroll
    for (int v = 0; v < N; v++)
#pragma unroll
        for (int u = 0; u < N; u++) meet[((wave * N + v) * N + u) * 64 + lane] = acc[v][u];
    arrived<0>();
    f4 sum[N];
#pragma unroll
    for (int u = 0; u < N; u++) {
        sum[u] = meet[((0 * N + wave) * N + u) * 64 + lane];
#pragma unroll
        for (int w = 1; w < 4; w++) sum[u] += meet[((w * N + wave) * N + u) * 64 + lane];
    }
    const bool none = m0 + 16 * wave >= P.rows;
    if (A.splits > 1) {
        if (none) return;
        const int64_t tile_of = (int64_t)at.tm * P.tiles_n + at.tn + P.first / A.splits;
        f4* part = (f4*)A.part + (tile_of * A.splits + at.split) * (N * 256) + threadIdx.x;
#pragma unroll
        for (int u = 0; u < N; u++) part[u * 256] = sum[u];
        return;
    }
    arrived<0>();
    if (none) return;
    using Out = Leave<T, K, SS>;
    const Out out(P, A.act, (float*)lds + wave * (16 * Out::LD), n0);
    typename Out::In in;
    out.template ask<false>(in, m0 + 16 * wave);
    out.template give<false>(in, sum, m0 + 16 * wave);
}

// A tile's parts of the depth, added in order: 16 rows of it to a wave.
template <typename T>
__global__ __launch_bounds__(64) void feed_join_kernel(FeedArgs A)
{
    constexpr int N = SS / 16;
    using Out = Leave<T, PLAIN, SS>;
    __shared__ float lds[16 * Out::LD];
    const int item = blockIdx.x / 4, wave = blockIdx.x % 4;
    int which = 0;
    while (which + 1 < A.count && item >= A.p[which + 1].first / A.splits) which++;
    const Product& P = A.p[which];
    const int tile = item - P.first / A.splits, row0 = tile / P.tiles_n * SS + 16 * wave;
    if (row0 >= P.rows) return;
    const f4* part = (const f4*)A.part + (int64_t)item * A.splits * (N * 256) + 64 * wave + threadIdx.x;
    f4 sum[N];
#pragma unroll
    for (int u = 0; u < N; u++) sum[u] = part[u * 256];
#pragma unroll 4
    for (int s = 1; s < A.splits; s++)
#pragma unroll
        for (int u = 0; u < N; u++) sum[u] += part[(int64_t)(s * N + u) * 256];
    const Out out(P, A.act, lds, tile % P.tiles_n * SS);
    typename Out::In in;
    out.template give<false>(in, sum, row0);
}

// HIDDEN or PLAIN of C rows or fewer, whole chunks: C columns of the result to a workgroup,
// operands straight to registers.  A matrix instruction takes 16 / C pieces of the depth at
// once, one to each C of its rows and columns; what it makes of one piece's rows and
// another's columns is left.  Eight waves take steps of the depth in turn, and their sums
// meet in LDS, in order.
template <typename T, Kind K, int C>
__global__ __launch_bounds__(512) void feed_few_kernel(FeedArgs A)
{
    constexpr int WAVES = 8, AHEAD = sizeof(T) == 2 ? 8 : 4, STEP = 32 * (16 / C), N = K == HIDDEN ? 2 : 1;
    __shared__ f4 meet[N][WAVES][64];
    const Product& P = A.p[0];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * C, depth = P.depth, rows = P.rows, cols = P.cols;
    // beyond the last row or column the last one comes again
    const T* l = (const T*)P.l[0] + min(i % C, rows - 1) * P.lld;
    const T* r[N];
    f4 acc[N];
#pragma unroll
    for (int n = 0; n < N; n++) {
        r[n] = (const T*)P.r[n] + min(n0 + i % C, cols - 1) * P.rld;
        acc[n] = f4{0, 0, 0, 0};
    }
    for (int first = wave * STEP; first < depth; first += WAVES * AHEAD * STEP) {
        Raw<T, 8> lv[AHEAD], rv[AHEAD][N];
        bool there[AHEAD];
#pragma unroll
        for (int a = 0; a < AHEAD; a++) {
            const int k = first + a * WAVES * STEP + i / C * 32 + 8 * g;
            there[a] = k < depth;
            const int at = there[a] ? k : 0;
#pragma unroll
            for (int n = 0; n < N; n++) __builtin_memcpy(&rv[a][n], r[n] + at, sizeof(rv[a][n]));
            __builtin_memcpy(&lv[a], l + at, sizeof(lv[a]));
        }
#pragma unroll
        for (int a = 0; a < AHEAD; a++) {
            if (!there[a]) lv[a] = Raw<T, 8>{};
#pragma unroll
            for (int n = 0; n < N; n++) {
                if (!there[a]) rv[a][n] = Raw<T, 8>{};
                acc[n] = gs::mma(__builtin_bit_cast(Frag<T>, rv[a][n]), __builtin_bit_cast(Frag<T>, lv[a]), acc[n]);
            }
        }
    }
#pragma unroll
    for (int n = 0; n < N; n++) meet[n][wave][lane] = acc[n];
    __syncthreads();
    if (threadIdx.x >= C * C) return;
    const int row = threadIdx.x / C, col = threadIdx.x % C;
    if (row >= rows || n0 + col >= (P.pad ? (cols + 7) / 8 * 8 : cols)) return;
    float sum[N] = {};
#pragma unroll
    for (int w = 0; w < WAVES; w++)
#pragma unroll
        for (int piece = 0; piece < 16 / C; piece++) {
            const int j = piece * C + col;
#pragma unroll
            for (int n = 0; n < N; n++) sum[n] += meet[n][w][j / 4 * 16 + piece * C + row][j % 4];
        }
    const int64_t at = row * P.old + n0 + col;
    if (n0 + col >= cols)
#pragma unroll
        for (int n = 0; n < N; n++) sum[n] = 0.0f;
    if constexpr (K == HIDDEN) {
        float value, slope;
        activation<T>(A.act, sum[0], value, slope);
        ((T*)P.out[0])[at] = (T)(value * sum[1]);
        if (P.out[1] != nullptr) {
            T kept[2] = {(T)sum[0], (T)sum[1]};
            if constexpr (sizeof(T) == 2) {
                if (P.rest != nullptr) {
                    uint32_t q[2] = {rest_of<T>(sum[0]), rest_of<T>(sum[1])};
                    if constexpr (__is_same(T, gs::f16))
                        for (int n = 0; n < 2; n++)
                            if (is_far(kept[n])) kept[n] = far_kept(sum[n], q[n]);
                    P.rest[at] = (uint8_t)(q[0] | q[1] << 4);
                }
            }
            ((T*)P.out[1])[at] = kept[0];
            ((T*)P.out[2])[at] = kept[1];
        }
    } else {
        ((T*)P.out[0])[at] = (T)sum[0];
    }
}

// Matrices of a 16-bit type copied to rows of whole 16-byte pieces, zeros behind their ends.
struct PadArgs {
    struct {
        const uint16_t* from;
        uint4* to;
        int64_t ld;
        int rows, cols, pieces;
        unsigned first, blocks;
    } m[5];
    int count;
    unsigned blocks;
};

__global__ __launch_bounds__(256) void feed_pad_kernel(PadArgs A)
{
    int which = 0;
    while (which + 1 < A.count && blockIdx.x >= A.m[which + 1].first) which++;
    const auto& M = A.m[which];
    const int64_t all = (int64_t)M.rows * M.pieces;
    for (int64_t i = (int64_t)(blockIdx.x - M.first) * 256 + threadIdx.x; i < all; i += (int64_t)M.blocks * 256) {
        const int64_t row = i / M.pieces;
        const int col = (int)(i - row * M.pieces) * 8;
        const Raw<uint16_t, 8> v = get<uint16_t, 8, false>(M.from + row * M.ld + col, M.cols - col);
        M.to[i] = __builtin_bit_cast(uint4, v);
    }
}

// Lays the products' tiles of SM x SN out one after the other; the workgroups, or -1 where
// their threads would be 2^32 or more, which no launch takes.
template <Kind K>
int64_t lay_out(FeedArgs& A, int sm, int sn, int threads)
{
    int64_t blocks = 0;
    for (int i = 0; i < A.count; i++) {
        Product& P = A.p[i];
        const int n = K == HIDDEN ? sn / 2 : sn;
        P.tiles_m = (P.rows + sm - 1) / sm;
        P.tiles_n = (P.cols + n - 1) / n;
        P.first = (int)blocks;
        blocks += (int64_t)P.tiles_m * P.tiles_n * A.splits;
        if (blocks * threads > 0xffffffffll) return -1;
    }
    return blocks;
}

// A kernel with more LDS than 64 KB says so once a device.
template <typename F>
int allow_lds(F kernel, size_t bytes, std::atomic<uint64_t>& told)
{
    int device = 0;
    GS_HIP(hipGetDevice(&device));
    const uint64_t bit = 1ull << (device & 63);
    if (device > 63 || !(told.load() & bit)) {
        GS_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
        told |= bit;
    }
    return GS_OK;
}

template <typename T, Kind K, bool LDOWN, bool RDOWN, int SM, int SN, int WM, int WN, int BUFFERS>
int launch_large(FeedArgs& A, hipStream_t stream)
{
    const int64_t blocks = lay_out<K>(A, SM, SN, 64 * WM * WN);
    GS_REQUIRE(blocks >= 0, "feed forward: too many tiles");
    constexpr size_t LDS = (size_t)BUFFERS * (SM + SN) * 128;
    auto kernel = feed_kernel<T, K, LDOWN, RDOWN, SM, SN, WM, WN, BUFFERS>;
    static std::atomic<uint64_t> told{0};
    if (int rc = allow_lds(kernel, LDS, told)) return rc;
    GS_TIMED("feed_kernel", stream,
             hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(64 * WM * WN), LDS, stream, A));
    GS_LAUNCH_CHECK("feed_kernel");
    return GS_OK;
}

template <typename T, Kind K, bool LDOWN, bool RDOWN, bool DIRECT>
int launch_small(FeedArgs& A, hipStream_t stream)
{
    const int64_t blocks = lay_out<K>(A, SS, SS, 256);
    GS_REQUIRE(blocks >= 0, "feed forward: too many tiles");
    constexpr size_t LDS = (size_t)(DIRECT && sizeof(T) == 2 ? 3 : 2) * 2 * SS * SKT * sizeof(T);
    static_assert(LDS >= 4 * SS * SS * sizeof(float), "the waves' sums meet in it");
    auto kernel = feed_small_kernel<T, K, LDOWN, RDOWN, DIRECT>;
    static std::atomic<uint64_t> told{0};
    if (int rc = allow_lds(kernel, LDS, told)) return rc;
    GS_TIMED("feed_small_kernel", stream,
             hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), LDS, stream, A));
    GS_LAUNCH_CHECK("feed_small_kernel");
    if constexpr (K == PLAIN || K == SUM) {
        if (A.splits > 1) {
            GS_TIMED("feed_join_kernel", stream,
                     hipLaunchKernelGGL(feed_join_kernel<T>, dim3((unsigned)(blocks / A.splits * 4)), dim3(64), 0, stream, A));
            GS_LAUNCH_CHECK("feed_join_kernel");
        }
    }
    return GS_OK;
}

template <typename T, Kind K, int C>
int launch_few(const FeedArgs& A, hipStream_t stream)
{
    GS_TIMED("feed_few_kernel", stream,
             hipLaunchKernelGGL((feed_few_kernel<T, K, C>), dim3(gs_div_up((size_t)A.p[0].cols + (A.p[0].pad ? 7 : 0), C)),
                                dim3(512), 0, stream, A));
    GS_LAUNCH_CHECK("feed_few_kernel");
    return GS_OK;
}

constexpr int CUS = 256;

int64_t tiles_of(int64_t m, int64_t n, int sm, int sn) { return (m + sm - 1) / sm * ((n + sn - 1) / sn); }

// Parts of the depth for `tiles` small tiles: while there are fewer than places for them,
// and three turns or more in a part, of which one takes about what adding it up does.  A
// CU has LDS for one workgroup of whole chunks, for two without.
int splits_of(int64_t tiles, int64_t turns, bool direct)
{
    int64_t n = tiles > 0 ? (direct ? CUS : 2 * CUS) / tiles : 1;
    if (n > turns / 3) n = turns / 3;
    return (int)(n < 1 ? 1 : n);
}

// Microseconds that a launch takes with tiles of sm x sn: rounds of tiles, a turn of 64 of
// the depth each, what begins and ends a tile.  Two 128 x 128 workgroups share a CU, so one
// ends while the other multiplies; a 256 x 256 one is alone.  Measured, bfloat16, 8192 x
// 1024 x 4096, with 256 x 256, 256 x 128 (three buffers), 128 x 128 and 64 x 64:
//   HIDDEN 155, 189, 184, 478   GRAD 141, 133, 124, 296   SUM 190, 123, 157, 277
//   y 96, 65, 74, 143           weights' gradients 188, 237, 260, 427
template <Kind K>
double estimate(const FeedArgs& A, int sm, int sn, double turn, double ends)
{
    int64_t tiles = 0;
    for (int i = 0; i < A.count; i++)
        tiles += tiles_of(A.p[i].rows, A.p[i].cols, sm, K == HIDDEN ? sn / 2 : sn);
    const double turns = (K == SUM ? 2 : 1) * ((A.p[0].depth + 63) / 64);
    return (double)((tiles + CUS - 1) / CUS) * (turn * turns + ends);
}

// Columns of a workgroup of feed_few_kernel, or 0 where the tiles of 64 are as fast.  The
// widest that leave every CU rows of weights to read, as many as there are rows of the
// result at least.  Both products of rows x width x hidden x out, us with tiles and so:
//   bfloat16  1 x 2048 x 8192 x 2048   26.0, 20.9    8 rows  26.2, 22.9    16 rows  26.3, 29.2
//             1 x 4096 x 1024 x 16384  26.1, 14.3 with tiles for the second product still; 28.8 for
//             the first still
//   float32   1 x 2048 x 8192 x 2048   73.6, 37.6    16 rows 73.1, 55.6
//   8 x 64 x 16384 x 64, whose second product would have 8 workgroups: bfloat16 18.7, 21.9
template <Kind K>
int few_columns(const Product& P, bool half)
{
    if (P.rows > (half ? 8 : 16) || P.depth % 8) return 0;   // a lane takes eight of the depth
    if (half && K == PLAIN && P.cols >= SS * CUS) return 0;
    const int64_t matrix_rows = (int64_t)(K == HIDDEN ? 2 : 1) * P.cols;
    int c = 16;
    while (c > 4 && c / 2 >= P.rows && matrix_rows < (int64_t)c * CUS) c /= 2;
    return matrix_rows >= 16 * c ? c : 0;
}

template <typename T, Kind K, bool LDOWN, bool RDOWN>
int launch_shape(FeedArgs& A, bool direct, hipStream_t stream)
{
    if constexpr (!LDOWN && !RDOWN) {
        switch (direct ? few_columns<K>(A.p[0], sizeof(T) == 2) : 0) {
        case 4: return launch_few<T, K, 4>(A, stream);
        case 8: return launch_few<T, K, 8>(A, stream);
        case 16: return launch_few<T, K, 16>(A, stream);
        }
    }
    if constexpr (sizeof(T) == 2) {
        if (direct) {
            const double large = estimate<K>(A, 256, 256, 1.4, K == GRAD ? 48 : K == HIDDEN ? 15 : 7),
                         wide = estimate<K>(A, 256, 128, 0.98, K == GRAD ? 18 : K == HIDDEN ? 9 : 5),
                         middle = estimate<K>(A, 128, 128, LDOWN ? 0.68 : 0.58, K == GRAD ? 6 : 2) + 3,
                         small = estimate<K>(A, 64, 64, 0.28, 1.5) / A.splits + (A.splits > 1 ? 7 : 3);
            const int splits = A.splits;
            A.splits = 1;
            if (large <= wide && large <= middle && large <= small)
                return launch_large<T, K, LDOWN, RDOWN, 256, 256, 4, 2, 2>(A, stream);
            if (wide <= middle && wide <= small) return launch_large<T, K, LDOWN, RDOWN, 256, 128, 4, 2, 3>(A, stream);
            if (middle <= small) return launch_large<T, K, LDOWN, RDOWN, 128, 128, 2, 2, 2>(A, stream);
            A.splits = splits;
        }
    }
    if (direct) return launch_small<T, K, LDOWN, RDOWN, true>(A, stream);
    return launch_small<T, K, LDOWN, RDOWN, false>(A, stream);
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
    // a tile's 256 rows are less than 2^31 bytes
    const int v = 16 / gs::dtype_bytes(type);
    return (uintptr_t)p % 16 == 0 && ld % v == 0 && n % v == 0 && ld < 1 << 21;
}

// n up to whole pieces of 8: what rows of h, a, b, their rests, da and db take
int up8(int n) { return (n + 7) / 8 * 8; }

size_t padded(size_t n) { return (n + 255) / 256 * 256; }

// Sets A's parts of the depth.
void split(FeedArgs& A, int64_t turns, bool direct, void* part)
{
    int64_t tiles = 0;
    for (int i = 0; i < A.count; i++) tiles += tiles_of(A.p[i].rows, A.p[i].cols, SS, SS);
    A.splits = splits_of(tiles, turns, direct);
    A.part = (float*)part;
}

int64_t turns_of(int64_t depth) { return (depth + SKT - 1) / SKT; }

// What the parts take: no more of them than places, of any products of a launch.
constexpr size_t PART_BYTES = (size_t)2 * CUS * SS * SS * sizeof(float);

// Whether operands of a 16-bit type whose rows are no whole 16-byte pieces are copied to such rows:
// then the large tiles, straight to LDS, do for them too.  It costs a launch each way and the
// operands' bytes twice.  Forward and backward, bfloat16, us without and with: 8192 x 1023 x
// 3000 2361, 677 (1024 x 3000: 639); 4096 x 511 x 1535 593, 182; 2048 x 255 x 1023 170, 141.
// Smaller blocks take as long as the host does, which pays for the launches, and for fewer
// rows the weights' copies take longer than their products.
bool worth_copies(int type, int64_t rows, int width, int hidden, int out)
{
    return gs::dtype_bytes(type) == 2 && rows >= 256 && rows * hidden * (2.0 * width + out) >= 1 << 30;
}

size_t copy_bytes(int64_t rows, int n) { return padded((size_t)rows * up8(n) * 2); }

// What the copies take: x, the gate and up; down; in the backward dy
size_t copies_bytes(int type, int64_t rows, int width, int hidden, int out, bool backward)
{
    if (!worth_copies(type, rows, width, hidden, out)) return 0;
    return (width % 8 ? copy_bytes(rows, width) + 2 * copy_bytes(hidden, width) : 0) +
           (hidden % 8 ? copy_bytes(out, hidden) : 0) + (backward && out % 8 ? copy_bytes(rows, out) : 0);
}

bool forward_parts(int64_t rows, int hidden, int out)
{
    return splits_of(tiles_of(rows, out, SS, SS), turns_of(hidden), false) > 1;
}

// the weights' gradients are split alone or together, as many as are asked for
bool backward_parts(int64_t rows, int width, int hidden, int out)
{
    return splits_of(tiles_of(rows, width, SS, SS), 2 * turns_of(hidden), false) > 1 ||
           splits_of(tiles_of(hidden, width, SS, SS), turns_of(rows), false) > 1 ||
           splits_of(tiles_of(out, hidden, SS, SS), turns_of(rows), false) > 1;
}

// An operand as the products read it.
struct Matrix {
    const void* p;
    int64_t ld;
    bool direct;
};

struct Copies {
    PadArgs args{};
    int type;
    bool worth;
    char* at;

    Matrix operator()(const void* p, int64_t ld, int64_t rows, int n)
    {
        if (whole(p, ld, n, type)) return {p, ld, true};
        if (!worth || n % 8 == 0 || up8(n) >= 1 << 21) return {p, ld, false};
        auto& m = args.m[args.count++];
        m.from = (const uint16_t*)p;
        m.to = (uint4*)at;
        m.ld = ld;
        m.rows = (int)rows;
        m.cols = n;
        m.pieces = up8(n) / 8;
        m.first = args.blocks;
        const int64_t blocks = (rows * m.pieces + 255) / 256;
        m.blocks = (unsigned)(blocks < 16384 ? blocks : 16384);
        args.blocks += m.blocks;
        const Matrix to{at, up8(n), true};
        at += copy_bytes(rows, n);
        return to;
    }
    int launch(hipStream_t stream)
    {
        if (args.count == 0) return GS_OK;
        GS_TIMED("feed_pad_kernel", stream,
                 hipLaunchKernelGGL(feed_pad_kernel, dim3(args.blocks), dim3(256), 0, stream, args));
        GS_LAUNCH_CHECK("feed_pad_kernel");
        return GS_OK;
    }
};

}  // namespace

extern "C" size_t gs_feed_forward_workspace_bytes(int type, int64_t rows, int width, int hidden, int out, int backward)
{
    if (check(type, GS_SILU, rows, width, hidden, out) != GS_OK) return 0;
    const size_t copies = copies_bytes(type, rows, width, hidden, out, backward != 0);
    if (!backward) return (forward_parts(rows, hidden, out) ? PART_BYTES : 0) + copies;
    return 2 * padded((size_t)rows * up8(hidden) * gs::dtype_bytes(type)) +
           (backward_parts(rows, width, hidden, out) ? PART_BYTES : 256) + copies;
}

extern "C" int gs_feed_forward(int type, int activation, int64_t rows, int width, int hidden, int out, const void* x,
                               int64_t x_stride, const void* gate, const void* up, const void* down, void* a, void* b,
                               void* rest, void* h, void* y, void* workspace, hipStream_t stream)
{
    gs::clear_error();
    if (int rc = check(type, activation, rows, width, hidden, out)) return rc;
    GS_REQUIRE((a == nullptr) == (b == nullptr) && (rest == nullptr || a != nullptr),
               "feed forward: a and b come together, rest with them");
    if (rows == 0) return GS_OK;
    GS_REQUIRE(x_stride >= 0, "feed forward: a stride must not be negative");
    GS_REQUIRE(x && gate && up && down && h && y, "feed forward: x, the weights, h and y must be non-null");
    const bool parts = forward_parts(rows, hidden, out);
    const size_t copied = copies_bytes(type, rows, width, hidden, out, false);
    GS_REQUIRE((!parts && copied == 0) || (workspace != nullptr && (uintptr_t)workspace % 256 == 0),
               "feed forward: these sizes need the workspace, 256-byte aligned");
    Copies copies;
    copies.type = type;
    copies.worth = copied > 0;
    copies.at = (char*)workspace + (parts ? PART_BYTES : 0);
    const Matrix X = copies(x, x_stride, rows, width), G = copies(gate, width, hidden, width),
                 U = copies(up, width, hidden, width), D = copies(down, hidden, out, hidden);
    if (int rc = copies.launch(stream)) return rc;
    FeedArgs A{};
    A.act = activation;
    A.splits = 1;
    A.count = 1;
    Product& P = A.p[0];
    P.l[0] = X.p;
    P.lld = X.ld;
    P.r[0] = G.p;
    P.r[1] = U.p;
    P.rld = G.ld;
    P.rows = (int)rows;
    P.cols = hidden;
    P.depth = width;
    P.old = up8(hidden);
    P.pad = true;
    P.out[0] = h;
    P.out[1] = a;
    P.out[2] = b;
    P.rest = (uint8_t*)rest;
    if (int rc = launch<HIDDEN, false, false>(type, A, X.direct && G.direct && U.direct, stream)) return rc;
    P = Product{};
    P.l[0] = h;
    P.lld = up8(hidden);
    P.r[0] = D.p;
    P.rld = D.ld;
    P.rows = (int)rows;
    P.cols = out;
    P.depth = hidden;
    P.old = out;
    P.out[0] = y;
    const bool direct = D.direct && whole(h, up8(hidden), up8(hidden), type);
    split(A, turns_of(hidden), direct, workspace);
    return launch<PLAIN, false, false>(type, A, direct, stream);
}

extern "C" int gs_feed_forward_backward(int type, int activation, int64_t rows, int width, int hidden, int out,
                                        const void* x, int64_t x_stride, const void* gate, const void* up,
                                        const void* down, const void* a, const void* b, const void* rest, const void* h,
                                        const void* dy,
                                        int64_t dy_stride, void* dx, void* dgate, void* dup, void* ddown,
                                        void* workspace, hipStream_t stream)
{
    gs::clear_error();
    if (int rc = check(type, activation, rows, width, hidden, out)) return rc;
    const bool inner = dx != nullptr || dgate != nullptr || dup != nullptr;
    if (!inner && ddown == nullptr) return GS_OK;
    if (rows > 0) {
        GS_REQUIRE(x_stride >= 0 && dy_stride >= 0, "feed forward: a stride must not be negative");
        GS_REQUIRE(x && gate && up && down && a && b && h && dy,
                   "feed forward: x, the weights, a, b, h and dy must be non-null");
        GS_REQUIRE(workspace != nullptr && (uintptr_t)workspace % 256 == 0,
                   "feed forward: the backward needs its workspace, 256-byte aligned");
    }
    const size_t inner_bytes = padded((size_t)rows * up8(hidden) * gs::dtype_bytes(type));
    char *da = (char*)workspace, *db = da + inner_bytes, *part = db + inner_bytes;
    FeedArgs A{};
    A.act = activation;
    A.splits = 1;
    A.count = 1;
    Copies copies;
    copies.type = type;
    copies.worth = copies_bytes(type, rows, width, hidden, out, true) > 0;
    copies.at = part + (backward_parts(rows, width, hidden, out) ? PART_BYTES : 256);
    const Matrix X = copies(x, x_stride, rows, width), Y = copies(dy, dy_stride, rows, out),
                 G = copies(gate, width, hidden, width), U = copies(up, width, hidden, width),
                 D = copies(down, hidden, out, hidden);
    if (int rc = copies.launch(stream)) return rc;
    const int ld = up8(hidden);
    if (inner && rows > 0) {
        Product& P = A.p[0];
        P.l[0] = Y.p;
        P.lld = Y.ld;
        P.r[0] = D.p;
        P.rld = D.ld;
        P.rows = (int)rows;
        P.cols = hidden;
        P.depth = out;
        P.old = ld;
        P.pad = true;
        P.out[0] = da;
        P.out[1] = db;
        P.in[0] = a;
        P.in[1] = b;
        P.rest = (uint8_t*)const_cast<void*>(rest);
        if (int rc = launch<GRAD, false, true>(type, A, Y.direct && D.direct, stream)) return rc;
    }
    if (dx != nullptr && rows > 0) {
        Product& P = A.p[0];
        P = Product{};
        P.l[0] = da;
        P.l[1] = db;
        P.lld = ld;
        P.r[0] = G.p;
        P.r[1] = U.p;
        P.rld = G.ld;
        P.rows = (int)rows;
        P.cols = width;
        P.depth = hidden;
        P.old = width;
        P.out[0] = dx;
        const bool direct = G.direct && U.direct && whole(da, ld, ld, type);
        split(A, 2 * turns_of(hidden), direct, part);
        if (int rc = launch<SUM, false, true>(type, A, direct, stream)) return rc;
    }
    // the weights' gradients, one after the other in one launch
    A.count = 0;
    bool direct = true;
    auto add = [&](const Matrix& l, int m, const Matrix& r, int n, void* to) {
        if (to == nullptr) return;
        Product& P = A.p[A.count++];
        P = Product{};
        P.l[0] = l.p;
        P.lld = l.ld;
        P.r[0] = r.p;
        P.rld = r.ld;
        P.rows = m;
        P.cols = n;
        P.depth = (int)rows;
        P.old = n;
        P.out[0] = to;
        direct = direct && l.direct && r.direct;
    };
    const bool inner_direct = whole(da, ld, ld, type), h_direct = whole(h, ld, ld, type);
    add(Matrix{da, ld, inner_direct}, hidden, X, width, dgate);
    add(Matrix{db, ld, inner_direct}, hidden, X, width, dup);
    add(Y, out, Matrix{h, ld, h_direct}, hidden, ddown);
    if (A.count == 0) return GS_OK;
    split(A, turns_of(rows), direct, part);
    return launch<PLAIN, true, true>(type, A, direct, stream);
}
