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

// Eight consecutive elements at p, those from n on zero, as an operand whose
// k(g, j) is 8 g + j.
template <typename T>
__device__ __forceinline__ Frag<T> frag_global(const T* p, int n)
{
    Frag<T> f;
    if constexpr (sizeof(T) == 4) {
        f.lo = n > 0 ? __builtin_bit_cast(f4, load_part(p, n)) : f4{0, 0, 0, 0};
        f.hi = n > 4 ? __builtin_bit_cast(f4, load_part(p + 4, n - 4)) : f4{0, 0, 0, 0};
    } else {
        f.v = n > 0 ? __builtin_bit_cast(s8, load_part(p, n)) : s8{0, 0, 0, 0, 0, 0, 0, 0};
    }
    return f;
}

// A tile of rows of DP elements in LDS.  A row's 16-byte chunks are permuted by
// an XOR of the row's low bits, so that the two ways it is read meet every
// bank equally: 16 rows at one chunk (row operands), and four neighbouring
// rows at two chunks (column operands).
template <typename T, int DP>
struct Tile {
    static constexpr int CHUNKS = DP * (int)sizeof(T) / 16;

    __device__ static __forceinline__ int chunk(int row, int c)
    {
        if constexpr (CHUNKS % 8 == 0) return row * CHUNKS + (c ^ (((row & 3) << 1) | ((row >> 2) & 1)));
        else return row * CHUNKS + (c ^ ((row & 2) | ((row >> 2) & 1)));
    }

    // Rows row + i, k(g, j) = k0 + 8 g + j.
    __device__ static __forceinline__ Frag<T> rows(const uint4* t, int row, int k0)
    {
        const int i = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
        Frag<T> f;
        if constexpr (sizeof(T) == 4) {
            f.lo = __builtin_bit_cast(f4, t[chunk(row + i, k0 / 4 + 2 * g)]);
            f.hi = __builtin_bit_cast(f4, t[chunk(row + i, k0 / 4 + 2 * g + 1)]);
        } else {
            f.v = __builtin_bit_cast(s8, t[chunk(row + i, k0 / 8 + g)]);
        }
        return f;
    }

    // The transposed tile's rows col + i, k(g, j) = row + 16 (j / 4) + 4 g + j % 4:
    // the counterpart of frag_of_tiles.  The 16-bit types take it with the
    // transposing LDS read, of which 16 lanes fetch 4 rows of 16 elements.
    __device__ static __forceinline__ Frag<T> cols(const uint4* t, int row, int col)
    {
        const int i = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
        Frag<T> f;
        if constexpr (sizeof(T) == 4) {
            const float* e = (const float*)t;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                f.lo[r] = e[chunk(row + 4 * g + r, (col + i) / 4) * 4 + i % 4];
                f.hi[r] = e[chunk(row + 16 + 4 * g + r, (col + i) / 4) * 4 + i % 4];
            }
        } else {
            const int r = row + 4 * g + i / 4, c = col / 8 + (i % 4) / 2, half = i % 2;
            typedef __attribute__((address_space(3))) s4 lds_s4;
            const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)((s4*)(t + chunk(r, c)) + half));
            const s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)((s4*)(t + chunk(r + 16, c)) + half));
            f.v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        }
        return f;
    }
};

// ROWS x DP elements on their way from global memory to a Tile: each of the
// block's 256 threads carries CPT chunks in registers.
template <typename T, int DP, int ROWS>
struct Stage {
    static constexpr int CHUNKS = Tile<T, DP>::CHUNKS, CPT = ROWS * CHUNKS / 256;
    static_assert(ROWS * CHUNKS % 256 == 0, "a whole number of chunks per thread");
    uint4 r[CPT];

    // Rows 0 .. n_rows - 1 at p (the rest zero), `stride` elements apart, of D elements.
    __device__ __forceinline__ void load(const T* p, int64_t stride, int n_rows, int D)
    {
#pragma unroll
        for (int k = 0; k < CPT; k++) {
            const int id = threadIdx.x + 256 * k, row = id / CHUNKS, at = id % CHUNKS * Vec<T>::N;
            r[k] = make_uint4(0, 0, 0, 0);
            if (row < n_rows && at < D) r[k] = __builtin_bit_cast(uint4, load_part(p + row * stride + at, D - at));
        }
    }
    __device__ __forceinline__ void store(uint4* t) const
    {
#pragma unroll
        for (int k = 0; k < CPT; k++) {
            const int id = threadIdx.x + 256 * k;
            t[Tile<T, DP>::chunk(id / CHUNKS, id % CHUNKS)] = r[k];
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
