// Matrix-core building blocks of the token operators.
//
// Everything is expressed in one shape, C[16][16] += A[16][32] B[32][16] over a
// wave of 64 lanes, with lane = 16 g + i (g in 0..3, i in 0..15):
//   A: lane holds A[i][k(g, j)], j in 0..7      B: lane holds B[k(g, j)][i]
//   C: lane holds C[4 g + r][i], r in 0..3
// A and B only have to agree on k(g, j).  For the 16-bit types the product is
// one 16x16x32 matrix instruction; for fp32 it is eight 16x16x4 instructions,
// the t-th of which takes the t-th value of every lane.
#pragma once
#include "gs_types.h"

namespace gs {

typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <typename T>
struct Frag {
    s8 v;
};
template <>
struct Frag<float> {
    f4 lo, hi;
};

__device__ __forceinline__ f4 mma(const Frag<bf16>& a, const Frag<bf16>& b, f4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a.v), __builtin_bit_cast(bf16x8, b.v),
                                                   c, 0, 0, 0);
}
__device__ __forceinline__ f4 mma(const Frag<f16>& a, const Frag<f16>& b, f4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a.v), __builtin_bit_cast(f16x8, b.v), c,
                                                  0, 0, 0);
}
__device__ __forceinline__ f4 mma(const Frag<float>& a, const Frag<float>& b, f4 c)
{
#pragma unroll
    for (int t = 0; t < 4; t++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.lo[t], b.lo[t], c, 0, 0, 0);
#pragma unroll
    for (int t = 0; t < 4; t++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.hi[t], b.hi[t], c, 0, 0, 0);
    return c;
}

// The B operand whose k(g, j) is 16 (j / 4) + 4 g + j % 4: two C tiles, one
// above the other, as they lie in their lanes.  No lane exchange.
template <typename T>
__device__ __forceinline__ Frag<T> frag_of_tiles(f4 a, f4 b)
{
    Frag<T> f;
    if constexpr (sizeof(T) == 4) {
        f.lo = a;
        f.hi = b;
    } else {
        T t[8];
#pragma unroll
        for (int r = 0; r < 4; r++) {
            t[r] = (T)a[r];
            t[4 + r] = (T)b[r];
        }
        f.v = __builtin_bit_cast(s8, t);
    }
    return f;
}

// The first n (at most 8) elements at p, the others zero, as an operand whose
// k(g, j) is 8 g + j.  Unless ODD, n is a whole number of 16-byte pieces or
// not positive.
template <typename T, bool ODD>
__device__ __forceinline__ Frag<T> frag_global(const T* p, int n)
{
    constexpr int V = Vec<T>::N;
    Vec<T> v[8 / V] = {};
#pragma unroll
    for (int h = 0; h < 8 / V; h++) {
        if constexpr (ODD) {
#pragma unroll
            for (int e = 0; e < V; e++)
                if (h * V + e < n) v[h].v[e] = p[h * V + e];
        } else {
            if (h * V < n) v[h] = load_vec(p + h * V);
        }
    }
    Frag<T> f;
    if constexpr (sizeof(T) == 4) {
        f.lo = __builtin_bit_cast(f4, v[0]);
        f.hi = __builtin_bit_cast(f4, v[1]);
    } else {
        f.v = __builtin_bit_cast(s8, v[0]);
    }
    return f;
}

// A tile of rows of DP elements in LDS.  A row's 16-byte chunks are permuted by
// an XOR of the row's low bits, so that the two ways it is read meet every
// bank equally: 16 rows at one chunk (row operands), and four neighbouring
// rows at two chunks (column operands).  The XOR repeats every 8 rows and
// every 8 (or 4) chunks, so a lane's addresses are a few numbers, kept in
// registers, plus constants that fit the LDS instructions' offsets.
template <typename T, int DP>
struct Tile {
    static constexpr int CHUNKS = DP * (int)sizeof(T) / 16;
    static constexpr bool EIGHT = CHUNKS % 8 == 0;

    int row_at[2], col_at[sizeof(T) == 4 ? 8 : 4];

    __device__ static __forceinline__ int chunk(int row, int c)
    {
        if constexpr (EIGHT) return row * CHUNKS + (c ^ (((row & 3) << 1) | ((row >> 2) & 1)));
        else return row * CHUNKS + (c ^ ((row & 2) | ((row >> 2) & 1)));
    }

    __device__ __forceinline__ Tile()
    {
        const int i = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int e = 0; e < 2; e++) row_at[e] = chunk(i, 2 * g + e);
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int d = 0; d < 2; d++) col_at[2 * r + d] = chunk(4 * g + r, 4 * d + i / 4) * 4 + i % 4;
        } else {
#pragma unroll
            for (int e = 0; e < 2; e++) row_at[e] = chunk(i, EIGHT ? 4 * e + g : g);
#pragma unroll
            for (int d = 0; d < 4; d++)
                col_at[d] = 2 * chunk(4 * g + i / 4, EIGHT || d < 2 ? 2 * d + (i % 4) / 2 : 0) + i % 2;
        }
    }

    // Rows row + i, k(g, j) = k0 + 8 g + j; row a multiple of 16, k0 of 32.
    __device__ __forceinline__ Frag<T> rows(const uint4* t, int row, int k0) const
    {
        const int c = k0 / 32;
        Frag<T> f;
        if constexpr (sizeof(T) == 4) {
            f.lo = __builtin_bit_cast(f4, t[row_at[0] + row * CHUNKS + 8 * c]);
            f.hi = __builtin_bit_cast(f4, t[row_at[1] + row * CHUNKS + 8 * c]);
        } else {
            f.v = __builtin_bit_cast(
                s8, t[EIGHT ? row_at[c & 1] + row * CHUNKS + 8 * (c >> 1) : row_at[0] + row * CHUNKS + 4 * c]);
        }
        return f;
    }

    // The transposed tile's rows col + i, k(g, j) = row + 16 (j / 4) + 4 g + j % 4:
    // the counterpart of frag_of_tiles; row a multiple of 32, col of 16.  The
    // 16-bit types take it with the transposing LDS read, of which 16 lanes
    // fetch 4 rows of 16 elements.
    __device__ __forceinline__ Frag<T> cols(const uint4* t, int row, int col) const
    {
        const int d = col / 16;
        Frag<T> f;
        if constexpr (sizeof(T) == 4) {
            const float* e = (const float*)t;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                f.lo[r] = e[col_at[2 * r + (d & 1)] + (row * CHUNKS + 8 * (d >> 1)) * 4];
                f.hi[r] = e[col_at[2 * r + (d & 1)] + ((row + 16) * CHUNKS + 8 * (d >> 1)) * 4];
            }
        } else {
            typedef __attribute__((address_space(3))) s4 lds_s4;
            const int at = EIGHT ? col_at[d & 3] + 16 * (d >> 2) : col_at[d & 1] + 8 * (d >> 1);
            const s4* e = (const s4*)t;
            const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(e + at + 2 * row * CHUNKS));
            const s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(e + at + 2 * (row + 16) * CHUNKS));
            f.v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        }
        return f;
    }
};

// ROWS x DP elements on their way from global memory to a Tile: each of the
// block's 256 threads carries CPT chunks in registers.
template <typename T, int DP, int ROWS, bool ODD>
struct Stage {
    static constexpr int CHUNKS = Tile<T, DP>::CHUNKS, CPT = ROWS * CHUNKS / 256, V = Vec<T>::N;
    static_assert(ROWS * CHUNKS % 256 == 0, "a whole number of chunks per thread");
    Vec<T> r[CPT];

    // Rows 0 .. n_rows - 1 at p (the rest zero), `stride` elements apart, of D elements.
    __device__ __forceinline__ void load(const T* p, int64_t stride, int n_rows, int D)
    {
#pragma unroll
        for (int k = 0; k < CPT; k++) {
            const int id = threadIdx.x + 256 * k, row = id / CHUNKS, at = id % CHUNKS * V;
            r[k] = {};
            if constexpr (ODD) {
#pragma unroll
                for (int e = 0; e < V; e++)
                    if (row < n_rows && at + e < D) r[k].v[e] = p[row * stride + at + e];
            } else {
                if (row < n_rows && at < D) r[k] = load_vec(p + row * stride + at);
            }
        }
    }
    __device__ __forceinline__ void store(uint4* t) const
    {
#pragma unroll
        for (int k = 0; k < CPT; k++) {
            const int id = threadIdx.x + 256 * k;
            t[Tile<T, DP>::chunk(id / CHUNKS, id % CHUNKS)] = __builtin_bit_cast(uint4, r[k]);
        }
    }
};

// Neighbouring work items share operands; consecutive workgroups go to
// different XCDs, each with an L2 of its own.  The bijection from workgroup to
// item that gives each XCD one run of consecutive items.
__device__ __forceinline__ uint32_t xcd_item(uint32_t block, uint32_t total)
{
    constexpr uint32_t XCDS = 8;
    const uint32_t x = block % XCDS, per = total / XCDS, rest = total % XCDS;
    return x * per + (x < rest ? x : rest) + block / XCDS;
}

}  // namespace gs
