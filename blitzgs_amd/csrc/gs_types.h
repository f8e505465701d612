// Element types of the token operators (layer norm, attention, the
// orthogonalised update): tensors in 32 bits, bfloat16 or float16, all
// arithmetic in fp32.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace gs {

typedef __bf16 bf16;
typedef _Float16 f16;

// The C ABI's codes (GS_F32 ...) and the bytes of one element.
inline bool dtype_known(int t) { return t >= 0 && t <= 2; }
inline int dtype_bytes(int t) { return t == 0 ? 4 : 2; }

// Sixteen bytes of elements, and an access to them at any element's address:
// rows of odd widths and views with odd strides start at any multiple of the
// element, which gfx950's global memory instructions take as they are.
template <typename T>
struct Vec {
    static constexpr int N = 16 / (int)sizeof(T);
    T v[N];
};

template <typename T>
__device__ __forceinline__ Vec<T> load_vec(const T* p)
{
    Vec<T> r;
    __builtin_memcpy(&r, p, 16);
    return r;
}

template <typename T>
__device__ __forceinline__ void store_vec(T* p, const Vec<T>& r)
{
    __builtin_memcpy(p, &r, 16);
}

// The first n elements (0..N) at p, the others zero.
template <typename T>
__device__ __forceinline__ Vec<T> load_part(const T* p, int n)
{
    if (n >= Vec<T>::N) return load_vec(p);
    Vec<T> r;
#pragma unroll
    for (int i = 0; i < Vec<T>::N; i++) r.v[i] = i < n ? p[i] : (T)0.0f;
    return r;
}

template <typename T>
__device__ __forceinline__ void store_part(T* p, const Vec<T>& r, int n)
{
    if (n >= Vec<T>::N) {
        store_vec(p, r);
        return;
    }
#pragma unroll
    for (int i = 0; i < Vec<T>::N; i++)
        if (i < n) p[i] = r.v[i];
}

}  // namespace gs
