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
        // in pairs, which the conversion instruction takes
        typedef T t2 __attribute__((ext_vector_type(2)));
        typedef float f2 __attribute__((ext_vector_type(2)));
        const t2 t[4] = {__builtin_convertvector(f2{a[0], a[1]}, t2), __builtin_convertvector(f2{a[2], a[3]}, t2),
                         __builtin_convertvector(f2{b[0], b[1]}, t2), __builtin_convertvector(f2{b[2], b[3]}, t2)};
        f.v = __builtin_bit_cast(s8, t);
    }
    return f;
}

// The first n (at most 8) elements at p, the others zero, as an operand whose
// k(g, j) is 8 g + j.  Unless BY_ELEMENT, n is a whole number of 16-byte pieces or
// not positive.
template <typename T, bool BY_ELEMENT>
__device__ __forceinline__ Frag<T> frag_global(const T* p, int n)
{
    constexpr int V = Vec<T>::N;
    Vec<T> v[8 / V] = {};
#pragma unroll
    for (int h = 0; h < 8 / V; h++) {
        if constexpr (BY_ELEMENT) {
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
// an XOR of the row's low bits, so that both ways it is read meet all 64 banks
// equally.  A 16-byte read is served 16 lanes at a time, of which 8 read one
// chunk of rows 0-3 and 12-15 and 8 the next chunk of rows 4-11 (or the other
// way round); the transposing read 32 at a time, two chunks of 8 rows.  With
// chunk c of row r at c ^ x(r) each takes 16 different places of 256 bytes for
//   rows of 256 bytes   x = 2 (r % 8)       of 128 bytes   x = r & 6
//   of 64 or 192 bytes  x = 2 (r / 4 % 2)
// (an XOR of ((r & 3) << 1 | (r >> 2) & 1), which meets 8 lanes' banks equally,
// cost half as many LDS cycles again).  The lane-dependent part of an address
// is one of a few numbers kept in registers; the rest fits the instruction's
// offset.
template <typename T, int DP>
struct Tile {
    static constexpr int CHUNKS = DP * (int)sizeof(T) / 16;
    // chunks that the XOR ranges over, and how many bases rows() and cols() need
    static constexpr int SPAN = CHUNKS % 16 == 0 ? 16 : CHUNKS % 8 == 0 ? 8 : 4;
    static constexpr int RB = sizeof(T) == 4 ? 2 * SPAN / 8 : SPAN / 4, CB = sizeof(T) == 4 ? SPAN : SPAN / 2;

    int row_at[RB], col_at[CB];

    __device__ static __forceinline__ int chunk(int row, int c)
    {
        return row * CHUNKS + (c ^ (SPAN == 16 ? 2 * (row & 7) : SPAN == 8 ? row & 6 : (row >> 1) & 2));
    }

    __device__ __forceinline__ Tile()
    {
        const int i = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int b = 0; b < RB; b++) row_at[b] = chunk(i, 8 * (b >> 1) + 2 * g + (b & 1));
#pragma unroll
            for (int b = 0; b < CB; b++) col_at[b] = chunk(4 * g + (b & 3), 4 * (b >> 2) + i / 4) * 4 + i % 4;
        } else {
#pragma unroll
            for (int b = 0; b < RB; b++) row_at[b] = chunk(i, 4 * b + g);
#pragma unroll
            for (int b = 0; b < CB; b++) col_at[b] = 2 * chunk(4 * g + i / 4, 2 * b + (i % 4) / 2) + i % 2;
        }
    }

    // Rows row + i, k(g, j) = k0 + 8 g + j; row a multiple of 16, k0 of 32.
    __device__ __forceinline__ Frag<T> rows(const uint4* t, int row, int k0) const
    {
        constexpr int STEP = 2 * (int)sizeof(T);   // chunks of 32 k
        const int c = k0 / 32 * STEP, b = c % SPAN / STEP, at = row * CHUNKS + c / SPAN * SPAN;
        Frag<T> f;
        if constexpr (sizeof(T) == 4) {
            f.lo = __builtin_bit_cast(f4, t[row_at[2 * b] + at]);
            f.hi = __builtin_bit_cast(f4, t[row_at[2 * b + 1] + at]);
        } else {
            f.v = __builtin_bit_cast(s8, t[row_at[b] + at]);
        }
        return f;
    }

    // The transposed tile's rows col + i, k(g, j) = row + 16 (j / 4) + 4 g + j % 4:
    // the counterpart of frag_of_tiles; row a multiple of 32, col of 16.  The
    // 16-bit types take it with the transposing LDS read, of which 16 lanes
    // fetch 4 rows of 16 elements.
    __device__ __forceinline__ Frag<T> cols(const uint4* t, int row, int col) const
    {
        constexpr int STEP = (int)sizeof(T);       // chunks of 16 columns
        const int c = col / 16 * STEP, b = c % SPAN / STEP, at = row * CHUNKS + c / SPAN * SPAN;
        Frag<T> f;
        if constexpr (sizeof(T) == 4) {
            const float* e = (const float*)t;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                f.lo[r] = e[col_at[4 * b + r] + 4 * at];
                f.hi[r] = e[col_at[4 * b + r] + 4 * (at + 16 * CHUNKS)];
            }
        } else {
            typedef __attribute__((address_space(3))) s4 lds_s4;
            const s4* e = (const s4*)t + col_at[b] + 2 * at;
            const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)e);
            const s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(e + 2 * 16 * CHUNKS));
            f.v = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
        }
        return f;
    }
};

// How a tile's rows come to LDS.
//   DIRECT  by loads that write LDS themselves: no registers, no LDS stores.
//           Rows are 16-byte aligned, D is a whole number of 16 bytes, and a
//           tile spans less than 2^31 bytes.  Rows beyond the last hold the
//           last one again; clear() has to have zeroed the elements from D on.
//   WHOLE   through registers, 16 bytes at a time, from any address; rows and
//           elements beyond the last are zero
//   ODD     through registers, element by element: D is no multiple of 16 bytes
enum Fill { DIRECT, WHOLE, ODD };

template <typename T, int DP, int ROWS, Fill F>
struct Stage {
    static constexpr int CHUNKS = Tile<T, DP>::CHUNKS, CPT = ROWS * CHUNKS / 256, V = Vec<T>::N;
    static_assert(ROWS * CHUNKS % 256 == 0, "a whole number of chunks per thread");
    Vec<T> r[CPT];

    // Begins to fetch rows 0 .. n_rows - 1 (n_rows >= 1) at p, `stride` elements
    // apart, of D elements, for the tile t.
    __device__ __forceinline__ void fetch(uint4* t, const T* p, int64_t stride, int n_rows, int D)
    {
        if constexpr (F == DIRECT) {
            const int s = (int)stride;
            typedef const __attribute__((address_space(1))) void* global_ptr;
            typedef __attribute__((address_space(3))) void* lds_ptr;
#pragma unroll
            for (int k = 0; k < CPT; k++) {
                // place `id` of the tile holds chunk `at` of its row
                const int id = threadIdx.x + 256 * k, row = id / CHUNKS;
                const int at = Tile<T, DP>::chunk(row, id % CHUNKS) - row * CHUNKS;
                const int from = n_rows >= ROWS ? row : min(row, n_rows - 1);
                uint4* to = t + 256 * k + (threadIdx.x & ~63u);   // + 16 bytes per lane
                if (at * V < D)
                    __builtin_amdgcn_global_load_lds((global_ptr)(p + (from * s + at * V)), (lds_ptr)to, 16, 0, 0);
            }
            return;
        }
#pragma unroll
        for (int k = 0; k < CPT; k++) {
            const int id = threadIdx.x + 256 * k, row = id / CHUNKS, at = id % CHUNKS * V;
            r[k] = {};
            if constexpr (F == ODD) {
#pragma unroll
                for (int e = 0; e < V; e++)
                    if (row < n_rows && at + e < D) r[k].v[e] = p[row * stride + at + e];
            } else {
                if (row < n_rows && at < D) r[k] = load_vec(p + row * stride + at);
            }
        }
    }
    // DIRECT: before the first fetch, for each tile that will be fetched.
    __device__ __forceinline__ static void clear(uint4* t, int D)
    {
        if constexpr (F != DIRECT) return;
        if (D == DP) return;
#pragma unroll
        for (int k = 0; k < CPT; k++) {
            const int id = threadIdx.x + 256 * k, row = id / CHUNKS;
            if ((Tile<T, DP>::chunk(row, id % CHUNKS) - row * CHUNKS) * V >= D) t[id] = make_uint4(0, 0, 0, 0);
        }
    }
    // Ends it; a barrier comes before the tile is read.  With `scrub`, infinities and
    // NaN become zero; whether this thread met one.
    __device__ __forceinline__ bool put(uint4* t, bool scrub = false)
    {
        bool found = false;
        if constexpr (F == DIRECT) {
            if (!scrub) return false;
            // a thread looks at what its own loads bring, once they are there
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
            for (int k = 0; k < CPT; k++) {
                Vec<T> x = __builtin_bit_cast(Vec<T>, t[threadIdx.x + 256 * k]);
                if (finite(x)) continue;
                found = true;
                t[threadIdx.x + 256 * k] = __builtin_bit_cast(uint4, scrubbed(x));
            }
            return found;
        }
#pragma unroll
        for (int k = 0; k < CPT; k++) {
            const int id = threadIdx.x + 256 * k;
            if (scrub && !finite(r[k])) {
                found = true;
                r[k] = scrubbed(r[k]);
            }
            t[Tile<T, DP>::chunk(id / CHUNKS, id % CHUNKS)] = __builtin_bit_cast(uint4, r[k]);
        }
        return found;
    }

private:
    static constexpr uint32_t EXPONENT = sizeof(T) == 4 ? 0x7f800000u : __is_same(T, bf16) ? 0x7f80u : 0x7c00u;

    __device__ __forceinline__ static bool finite(const Vec<T>& x)
    {
        typedef unsigned short us2 __attribute__((ext_vector_type(2)));
        const uint4 w = __builtin_bit_cast(uint4, x);
        if constexpr (sizeof(T) == 4) {
            constexpr uint32_t M = 0x7fffffffu;
            return max(max(w.x & M, w.y & M), max(w.z & M, w.w & M)) < EXPONENT;
        } else {
            constexpr uint32_t M = 0x7fff7fffu;
            auto larger = [](us2 a, us2 b) { return __builtin_elementwise_max(a, b); };
            const us2 top = larger(larger(__builtin_bit_cast(us2, w.x & M), __builtin_bit_cast(us2, w.y & M)),
                                   larger(__builtin_bit_cast(us2, w.z & M), __builtin_bit_cast(us2, w.w & M)));
            return max(top[0], top[1]) < EXPONENT;
        }
    }
    __device__ __forceinline__ static Vec<T> scrubbed(Vec<T> x)
    {
#pragma unroll
        for (int e = 0; e < V; e++)
            if (!(__builtin_fabsf((float)x.v[e]) < __builtin_inff())) x.v[e] = (T)0.0f;
        return x;
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
