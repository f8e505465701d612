// One AdamW step over many tensors, moments in 32 bits or in 8.
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
//   p = p (1 - lr decay) - lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps)
//
// Every element is read and written once, so the step is bound by memory: 28
// bytes an element with all in fp32, 16 with 8-bit moments, 10 with 16-bit
// parameters beside them.  A launch takes up to MAX_TENSORS tensors, whose
// addresses travel in its arguments; a workgroup finds its tensor by their first
// workgroups and walks CHUNK elements at a time, eight neighbours to a lane.
//
// 8 bits.  BLOCK_8 neighbours share a power of two 2^e, that of the largest.  A
// number over it is below 2 and is held as a small float with three bits of
// mantissa: m with a sign and a 4-bit exponent (1 is exponent 14), v, which is
// never negative, with a 5-bit one (1 is exponent 30).  b2 = 0.999 moves v by a
// thousandth a step where a code's neighbours are a sixteenth away: to nearest it
// would never move, so the rest is rounded up with its own probability, by 16
// bits of a hash of the tensor's key and the element's index.  A code of all ones
// (bar the sign) is NaN, which infinities become too; they leave their block's
// power of two alone.  The step itself uses m and v before they are rounded.
//
// A v that is not zero never becomes zero: its root's smallest step is 2^-16 of the block's,
// as m's is, and an m that was rounded up beside a v that was rounded away is divided by next
// to nothing a step later (a block's elements of 1e-5 of its largest took updates of up to 1500
// lr).  So elements whose root of v is below 2^-16 of their block's largest are stepped as if it
// were that: by less than AdamW does on average, in single steps by up to 2.4 lr.
//
// A code shifted to fp32's exponent is the number up to a power of two, below the
// smallest exponent too, where both are subnormal: decoding and encoding change an
// exponent, without cases.  NaN and infinities, which would need some, have a path that a
// wave takes only where it meets one.
//
// 122M elements in fp32: 651 us, 3.42 GB at 5.25 TB/s (a large copy: 5.15).  183M bfloat16
// elements with 8-bit moments: 361 us, 1.83 GB at 5.1 TB/s (472 us before the instructions
// of an element were 87 and are about 50); their moments' values 180 us.
#include <math.h>

#include <algorithm>
#include <memory>
#include <new>

#include "gs_host.h"
#include "gs_types.h"
#include "../../include/blitzgs_amd.h"

namespace {

constexpr int MAX_TENSORS = 48;
constexpr int THREADS = 256;
constexpr int V = 8;                       // elements of a lane
constexpr int CHUNK = THREADS * V;
constexpr int BLOCK_8 = 128;               // elements that share a power of two: 16 lanes
constexpr int TOP_M = 14, TOP_V = 30;      // exponent codes of 1
constexpr uint64_t MAX_GROUPS = (1u << 24) - 1;   // a launch has fewer than 2^32 threads

struct Tensor {
    void* p;
    const void* g;
    void* m;
    void* v;
    uint8_t* ms;
    uint8_t* vs;
    int64_t size;
    uint32_t key;
    uint32_t first;                        // workgroup
};

struct AdamArgs {
    Tensor t[MAX_TENSORS];
    int count;
    int chunks;                            // of a workgroup
    float b1, c1, b2, c2;                  // c = 1 - b
    float keep, rate, root, eps;           // 1 - lr decay, lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
};

__host__ __device__ inline uint32_t scrambled(uint32_t x)
{
    // xor-shifts between products with the fractional parts of sqrt(2) and sqrt(3)
    x ^= x >> 16;
    x *= 0x6A09E667u;
    x ^= x >> 15;
    x *= 0xBB67AE85u;
    return x ^ (x >> 16);
}
constexpr uint32_t PHI = 0x9E3779B9u;      // of the golden ratio

struct Bytes {
    uint8_t b[V];
};

// Eight codes.
struct Codes {
    uint32_t w[2];

    __device__ __forceinline__ uint32_t at(int i) const { return w[i / 4] >> (i % 4 * 8) & 255u; }
    // whether one of them is NaN's: all ones, the sign (bit 7) apart
    template <bool SIGN>
    __device__ __forceinline__ bool special() const
    {
        uint32_t found = 0;
#pragma unroll
        for (int k = 0; k < 2; k++)
            found |= ((w[k] & 0x7f7f7f7fu) + 0x01010101u) & (SIGN ? 0x80808080u : w[k] & 0x80808080u);
        return found != 0;
    }
};

// The number that a code stands for, in a block of scale 2^(biased - 127); NaN only with SPECIAL.
template <int TOP, bool SIGN, bool SPECIAL>
__device__ __forceinline__ float decoded(uint32_t code, int biased)
{
    constexpr uint32_t ONES = SIGN ? 127u : 255u;
    const uint32_t c = code & ONES, sign = SIGN ? (code & 128u) << 24 : 0u;
    const float x = __builtin_ldexpf(__uint_as_float(c << 20 | sign), biased - TOP);
    return SPECIAL && c == ONES ? __builtin_nanf("") : x;
}

// x over its block's power of two, rounded up where its rest and draw / 2^16 make a step; NaN,
// infinities and what could be rounded up to one only with SPECIAL
template <int TOP, bool SIGN, bool SPECIAL>
__device__ __forceinline__ uint32_t encoded(float x, int biased, uint32_t draw)
{
    constexpr uint32_t ONES = SIGN ? 127u : 255u;
    const float size = __builtin_ldexpf(__builtin_fabsf(x), TOP - biased);
    uint32_t c = (__float_as_uint(size) + (draw << 4)) >> 20;
    // no number is above 2^128
    if (SPECIAL && biased == 254) c = min(c, 8u * TOP + 7u);
    if (SPECIAL && !(__builtin_fabsf(x) < __builtin_inff())) c = ONES;
    return SIGN ? c | (__float_as_uint(x) >> 24 & 128u) : c;
}

// The hardware's square root, and its reciprocal in the step, are off by one last bit, of
// an update that is a small part of its parameter; with 8-bit moments there is little room for
// instructions: with the exact ones 183M bfloat16 elements took 55 us more.  The hardware's
// root takes no subnormals, which matter only beside an eps that is one, or none.
template <bool TINY>
__device__ __forceinline__ float root_of(float v)
{
    if constexpr (!TINY) return __builtin_amdgcn_sqrtf(v);
    const bool tiny = v < 0x1p-96f;
    const float r = __builtin_amdgcn_sqrtf(tiny ? v * 0x1p96f : v);
    return tiny ? r * 0x1p-48f : r;
}

// The largest finite of eight numbers' bits, without their signs.
template <bool SPECIAL>
__device__ __forceinline__ uint32_t largest_of(const float (&x)[V], int n)
{
    uint32_t l = 0;
#pragma unroll
    for (int i = 0; i < V; i++) {
        const uint32_t a = __float_as_uint(x[i]) & 0x7fffffffu;
        l = max(l, i < n && (!SPECIAL || a < 0x7f800000u) ? a : 0u);
    }
    return l;
}

template <bool SPECIAL>
__device__ __forceinline__ void keep(const Tensor& t, int64_t at, int n, const float (&m)[V], float (&v)[V],
                                     Codes& cm, Codes& cv, uint32_t& em, uint32_t& ev)
{
    uint32_t lm = largest_of<SPECIAL>(m, n), lv = largest_of<SPECIAL>(v, n);
#pragma unroll
    for (int d = 1; d < BLOCK_8 / V; d <<= 1) {
        lm = max(lm, (uint32_t)__shfl_xor((int)lm, d, 64));
        lv = max(lv, (uint32_t)__shfl_xor((int)lv, d, 64));
    }
    em = lm >> 23;
    ev = lv >> 23;
    // v > 0 is not below the smallest code's value.  Only lanes with one that is look for it (in every
    // element's encoding this took 20 of 387 us for 183M elements).
    uint32_t least = __float_as_uint(v[0]);
#pragma unroll
    for (int i = 1; i < V; i++) least = min(least, __float_as_uint(v[i]));
    if (least < (ev > 33u ? ev - 32u : 1u) << 23) {
        const float smallest = __builtin_ldexpf(1.0f, (int)ev - 127 - 32);
#pragma unroll
        for (int i = 0; i < V; i++)
            if (v[i] != 0.0f && v[i] < smallest) v[i] = smallest;
    }
    uint32_t place = (uint32_t)at * PHI + t.key + (uint32_t)(at >> 32) * 0x6A09E667u;
    cm = cv = Codes{};
#pragma unroll
    for (int i = 0; i < V; i++, place += PHI) {
        const uint32_t draw = scrambled(place);
        cm.w[i / 4] |= encoded<TOP_M, true, SPECIAL>(m[i], (int)em, draw & 0xffffu) << (i % 4 * 8);
        cv.w[i / 4] |= encoded<TOP_V, false, SPECIAL>(v[i], (int)ev, draw >> 16) << (i % 4 * 8);
    }
}

template <typename T, int BITS, bool TINY, bool WHOLE>
__device__ __forceinline__ void step(const AdamArgs& A, const Tensor& t, int64_t at)
{
    T* p = (T*)t.p + at;
    const T* g = (const T*)t.g + at;
    const int n = WHOLE ? V : (int)(t.size - at < V ? t.size - at : V);   // may be negative
    auto get = [&](const auto* from, auto& to) __attribute__((always_inline)) {
        if constexpr (WHOLE) {
            __builtin_memcpy(&to, from, sizeof(to));
        } else {
#pragma unroll
            for (int i = 0; i < V; i++)
                if (i < n) to[i] = from[i];
        }
    };
    auto put = [&](auto* to, const auto& from) __attribute__((always_inline)) {
        if constexpr (WHOLE) {
            __builtin_memcpy(to, &from, sizeof(from));
        } else {
#pragma unroll
            for (int i = 0; i < V; i++)
                if (i < n) to[i] = from[i];
        }
    };
    T tp[V] = {}, tg[V] = {};
    float m[V] = {}, v[V] = {};
    get((const T*)p, tp);
    get(g, tg);
    const int64_t block = at / BLOCK_8;
    if constexpr (BITS == 32) {
        get((const float*)t.m + at, m);
        get((const float*)t.v + at, v);
    } else {
        uint8_t bm[V] = {}, bv[V] = {};
        get((const uint8_t*)t.m + at, bm);
        get((const uint8_t*)t.v + at, bv);
        const Codes cm = __builtin_bit_cast(Codes, bm), cv = __builtin_bit_cast(Codes, bv);
        const int um = n > 0 ? t.ms[block] : 0, uv = n > 0 ? t.vs[block] : 0;
        // the whole wave one way or the other
        const bool special = __any(cm.special<true>() || cv.special<false>());
#pragma unroll
        for (int i = 0; i < V; i++) {
            m[i] = decoded<TOP_M, true, false>(cm.at(i), um);
            v[i] = decoded<TOP_V, false, false>(cv.at(i), uv);
        }
        if (special) {
#pragma unroll
            for (int i = 0; i < V; i++) {
                m[i] = decoded<TOP_M, true, true>(cm.at(i), um);
                v[i] = decoded<TOP_V, false, true>(cv.at(i), uv);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < V; i++) {
        const float gi = (float)tg[i];
        m[i] = __builtin_fmaf(A.b1, m[i], A.c1 * gi);
        v[i] = __builtin_fmaf(A.b2, v[i], A.c2 * gi * gi);
        const float by = __builtin_fmaf(root_of<TINY>(v[i]), A.root, A.eps);
        tp[i] = (T)__builtin_fmaf((float)tp[i], A.keep, -(A.rate * (m[i] * __builtin_amdgcn_rcpf(by))));
    }
    put(p, tp);
    if constexpr (BITS == 32) {
        put((float*)t.m + at, m);
        put((float*)t.v + at, v);
    } else {
        Codes cm, cv;
        uint32_t em, ev;
        // NaN and infinities have larger bits than any number, and 1.875 2^127 is the last below a code of 2^128
        const int there = WHOLE ? V : n;
        const bool special = max(largest_of<false>(m, there), largest_of<false>(v, there)) >= 0x7f700000u;
        if (__any(special)) keep<true>(t, at, there, m, v, cm, cv, em, ev);
        else keep<false>(t, at, there, m, v, cm, cv, em, ev);
        put((uint8_t*)t.m + at, __builtin_bit_cast(Bytes, cm).b);
        put((uint8_t*)t.v + at, __builtin_bit_cast(Bytes, cv).b);
        if (n > 0 && at % BLOCK_8 == 0) {
            t.ms[block] = (uint8_t)em;
            t.vs[block] = (uint8_t)ev;
        }
    }
}

template <typename T, int BITS, bool TINY>
__global__ __launch_bounds__(THREADS) void adamw_kernel(AdamArgs A)
{
    int lo = 0, hi = A.count - 1;          // the last tensor that begins at or before this workgroup
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (A.t[mid].first <= blockIdx.x) lo = mid; else hi = mid - 1;
    }
    const Tensor t = A.t[lo];
    const int64_t begin = (int64_t)(blockIdx.x - t.first) * A.chunks * CHUNK;
    for (int c = 0; c < A.chunks; c++) {
        const int64_t from = begin + (int64_t)c * CHUNK;
        if (from >= t.size) return;
        // the lanes of a block of 128 go the same way
        if (from + CHUNK <= t.size)
            step<T, BITS, TINY, true>(A, t, from + threadIdx.x * V);
        else
            step<T, BITS, TINY, false>(A, t, from + threadIdx.x * V);
    }
}

template <typename T>
__global__ __launch_bounds__(THREADS) void adamw_values_kernel(int64_t size, const uint8_t* __restrict__ m,
                                                               const uint8_t* __restrict__ v,
                                                               const uint8_t* __restrict__ ms,
                                                               const uint8_t* __restrict__ vs, T* __restrict__ mo,
                                                               T* __restrict__ vo)
{
    for (int64_t at = ((int64_t)blockIdx.x * THREADS + threadIdx.x) * V; at < size;
         at += (int64_t)gridDim.x * CHUNK) {
        const int um = ms[at / BLOCK_8], uv = vs[at / BLOCK_8];
        if (at + V <= size) {
            Codes cm, cv;
            __builtin_memcpy(&cm, m + at, V);
            __builtin_memcpy(&cv, v + at, V);
            T tm[V], tv[V];
#pragma unroll
            for (int i = 0; i < V; i++) {
                tm[i] = (T)decoded<TOP_M, true, false>(cm.at(i), um);
                tv[i] = (T)decoded<TOP_V, false, false>(cv.at(i), uv);
            }
            if (__any(cm.special<true>() || cv.special<false>())) {
#pragma unroll
                for (int i = 0; i < V; i++) {
                    tm[i] = (T)decoded<TOP_M, true, true>(cm.at(i), um);
                    tv[i] = (T)decoded<TOP_V, false, true>(cv.at(i), uv);
                }
            }
            __builtin_memcpy(mo + at, tm, sizeof(tm));
            __builtin_memcpy(vo + at, tv, sizeof(tv));
        } else {
            for (int64_t i = at; i < size; i++) {
                mo[i] = (T)decoded<TOP_M, true, true>(m[i], um);
                vo[i] = (T)decoded<TOP_V, false, true>(v[i], uv);
            }
        }
    }
}

template <typename T, bool TINY>
void launch(int bits, const AdamArgs& A, unsigned blocks, hipStream_t stream)
{
    if (bits == 32)
        GS_TIMED("adamw_kernel", stream,
                 hipLaunchKernelGGL((adamw_kernel<T, 32, TINY>), dim3(blocks), dim3(THREADS), 0, stream, A));
    else
        GS_TIMED("adamw_kernel", stream,
                 hipLaunchKernelGGL((adamw_kernel<T, 8, TINY>), dim3(blocks), dim3(THREADS), 0, stream, A));
}

template <typename T>
void launch(int bits, const AdamArgs& A, unsigned blocks, hipStream_t stream)
{
    // a root that is missing a subnormal is off by 1e-19
    if (A.eps >= 1e-12f) launch<T, false>(bits, A, blocks, stream);
    else launch<T, true>(bits, A, blocks, stream);
}

struct Range {
    uintptr_t from, to;
};

// Tensors that are written lie apart from each other and from the gradients: of an overlap
// the step would leave what its last workgroup wrote.
int check_apart(int type, int bits, int count, const int64_t* sizes, void* const* params, const void* const* grads,
                void* const* exp_avgs, void* const* exp_avg_sqs, uint8_t* const* exp_avg_scales,
                uint8_t* const* exp_avg_sq_scales)
{
    const int64_t of_p = gs::dtype_bytes(type), of_m = bits / 8;
    std::unique_ptr<Range[]> all(new (std::nothrow) Range[5 * (size_t)count]);
    GS_REQUIRE(all != nullptr, "adamw: no memory for the addresses of %d tensors", count);
    size_t n = 0;
    auto add = [&](const void* p, int64_t bytes) { all[n++] = Range{(uintptr_t)p, (uintptr_t)p + (uintptr_t)bytes}; };
    for (int i = 0; i < count; i++) {
        if (sizes[i] == 0) continue;
        add(params[i], sizes[i] * of_p);
        add(exp_avgs[i], sizes[i] * of_m);
        add(exp_avg_sqs[i], sizes[i] * of_m);
        if (bits == 32) continue;
        const int64_t blocks = (sizes[i] + BLOCK_8 - 1) / BLOCK_8;
        add(exp_avg_scales[i], blocks);
        add(exp_avg_sq_scales[i], blocks);
    }
    Range* end = all.get() + n;
    std::sort(all.get(), end, [](const Range& a, const Range& b) { return a.from < b.from; });
    for (size_t i = 1; i < n; i++)
        GS_REQUIRE(all[i - 1].to <= all[i].from, "adamw: a tensor may not come twice in a call or overlap another");
    for (int i = 0; i < count; i++) {
        if (sizes[i] == 0) continue;
        const uintptr_t from = (uintptr_t)grads[i], to = from + (uintptr_t)(sizes[i] * of_p);
        // the first that ends behind the gradient's begin
        const Range* r = std::partition_point(all.get(), end, [&](const Range& a) { return a.to <= from; });
        GS_REQUIRE(r == end || r->from >= to, "adamw: gradient %d overlaps a tensor that is written", i);
    }
    return GS_OK;
}

}  // namespace

extern "C" int gs_adamw_update(int type, int bits, int count, const int64_t* sizes, void* const* params,
                               const void* const* grads, void* const* exp_avgs, void* const* exp_avg_sqs,
                               uint8_t* const* exp_avg_scales, uint8_t* const* exp_avg_sq_scales,
                               const gs_adamw_settings* settings, hipStream_t stream)
{
    gs::clear_error();
    GS_REQUIRE(gs::dtype_known(type), "adamw: unknown element type %d", type);
    GS_REQUIRE(bits == 8 || bits == 32, "adamw: moments have 8 or 32 bits, not %d", bits);
    GS_REQUIRE(count >= 0, "adamw: count must not be negative");
    GS_REQUIRE(settings != nullptr, "adamw: the settings must be non-null");
    const double lr = settings->lr, beta1 = settings->beta1, beta2 = settings->beta2;
    GS_REQUIRE(settings->step >= 1, "adamw: step must be at least 1");
    GS_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "adamw: the betas must be in [0, 1)");
    GS_REQUIRE(lr >= 0.0 && settings->eps >= 0.0 && settings->weight_decay >= 0.0,
               "adamw: lr, eps and weight_decay must not be negative");
    if (count == 0) return GS_OK;
    GS_REQUIRE(sizes && params && grads && exp_avgs && exp_avg_sqs, "adamw: the arrays must be non-null");
    GS_REQUIRE(bits == 32 || (exp_avg_scales && exp_avg_sq_scales), "adamw: 8-bit moments need their scales");
    for (int i = 0; i < count; i++) {
        GS_REQUIRE(sizes[i] >= 0 && sizes[i] < (1ll << 40), "adamw: tensor %d has an impossible size", i);
        if (sizes[i] == 0) continue;
        GS_REQUIRE(params[i] && grads[i] && exp_avgs[i] && exp_avg_sqs[i], "adamw: tensor %d has a null pointer", i);
        GS_REQUIRE(bits == 32 || (exp_avg_scales[i] && exp_avg_sq_scales[i]), "adamw: tensor %d has no scales", i);
    }
    if (int rc = check_apart(type, bits, count, sizes, params, grads, exp_avgs, exp_avg_sqs, exp_avg_scales,
                             exp_avg_sq_scales))
        return rc;
    AdamArgs A;
    A.b1 = (float)beta1;
    A.c1 = (float)(1.0 - beta1);
    A.b2 = (float)beta2;
    A.c2 = (float)(1.0 - beta2);
    A.keep = (float)(1.0 - lr * settings->weight_decay);
    A.rate = (float)(lr / (1.0 - pow(beta1, (double)settings->step)));
    A.root = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)settings->step)));
    A.eps = (float)settings->eps;
    const uint32_t start = scrambled((uint32_t)settings->step * PHI + settings->seed);
    int64_t largest = 0;
    for (int i = 0; i < count; i++) largest = std::max(largest, sizes[i]);
    A.chunks = 1 + (int)((uint64_t)largest / (MAX_GROUPS * CHUNK));
    for (int i = 0; i < count;) {
        uint64_t blocks = 0;
        A.count = 0;
        for (; i < count && A.count < MAX_TENSORS; i++) {
            if (sizes[i] == 0) continue;
            const uint64_t n = ((uint64_t)sizes[i] + (uint64_t)A.chunks * CHUNK - 1) / ((uint64_t)A.chunks * CHUNK);
            if (A.count > 0 && blocks + n > MAX_GROUPS) break;
            Tensor& t = A.t[A.count++];
            t.p = params[i];
            t.g = grads[i];
            t.m = exp_avgs[i];
            t.v = exp_avg_sqs[i];
            t.ms = bits == 8 ? exp_avg_scales[i] : nullptr;
            t.vs = bits == 8 ? exp_avg_sq_scales[i] : nullptr;
            t.size = sizes[i];
            t.key = scrambled((uint32_t)i * PHI + start);
            t.first = (uint32_t)blocks;
            blocks += n;
        }
        if (blocks == 0) continue;
        if (type == GS_F32)
            launch<float>(bits, A, (unsigned)blocks, stream);
        else if (type == GS_BF16)
            launch<gs::bf16>(bits, A, (unsigned)blocks, stream);
        else
            launch<gs::f16>(bits, A, (unsigned)blocks, stream);
        GS_LAUNCH_CHECK("adamw_kernel");
    }
    return GS_OK;
}

extern "C" int gs_adamw_values(int type, int64_t size, const uint8_t* exp_avg, const uint8_t* exp_avg_sq,
                               const uint8_t* exp_avg_scale, const uint8_t* exp_avg_sq_scale, void* exp_avg_out,
                               void* exp_avg_sq_out, hipStream_t stream)
{
    gs::clear_error();
    GS_REQUIRE(type == GS_F32 || type == GS_BF16, "adamw: values are float32 or bfloat16, not type %d", type);
    GS_REQUIRE(size >= 0, "adamw: size must not be negative");
    if (size == 0) return GS_OK;
    GS_REQUIRE(exp_avg && exp_avg_sq && exp_avg_scale && exp_avg_sq_scale && exp_avg_out && exp_avg_sq_out,
               "adamw: the moments and their values must be non-null");
    const int64_t n = (size + CHUNK - 1) / CHUNK;
    const dim3 blocks((unsigned)(n < 65536 ? n : 65536));
    if (type == GS_F32)
        GS_TIMED("adamw_values_kernel", stream,
                 hipLaunchKernelGGL((adamw_values_kernel<float>), blocks, dim3(THREADS), 0, stream, size, exp_avg,
                                    exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, (float*)exp_avg_out,
                                    (float*)exp_avg_sq_out));
    else
        GS_TIMED("adamw_values_kernel", stream,
                 hipLaunchKernelGGL((adamw_values_kernel<gs::bf16>), blocks, dim3(THREADS), 0, stream, size, exp_avg,
                                    exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, (gs::bf16*)exp_avg_out,
                                    (gs::bf16*)exp_avg_sq_out));
    GS_LAUNCH_CHECK("adamw_values_kernel");
    return GS_OK;
}
