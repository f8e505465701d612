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
// views with odd strides start at any multiple of the element, which gfx950's
// global memory instructions take as they are.  Rows whose width is not a whole
// number of these go through kernels of their own: a partial access beside a
// whole one in the same loop costs the whole one its single instruction.
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

}  // namespace gs
