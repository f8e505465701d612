// Rotary positions of queries and keys, alone or after the RMS norm of every
// head, forward and backward.
//
//   phase  = position * frequency  mod 2^64, in 2^-64ths of a turn
//   c, s   = cos, sin(2 pi phase / 2^64), times the magnitude
//   norm   r = 1 / sqrt(mean(x^2) + eps), z = x r, u = w z      (else u = x)
//   y1 = u1 c - u2 s,  y2 = u1 s + u2 c  for each of the N = axes * pairs pairs:
//          elements (i, i + N), or (2i, 2i + 1) where interleaved; the rest is u
//   backward   g = dy rotated by -phase, h = g w, dx = r (h - z mean(h z)),
//              dw = sum over rows of g z                        (else dx = g)
//
// An integer product modulo a turn loses nothing however far the position: a
// float32 angle at position 2^20 would be off by 2^-4.  Its cosine and sine are
// formed once per token and pair by the workgroup, left in LDS and used for all
// heads of the token.
//
// Both passes are bound by memory and touch each element once.  A row (one head
// of one token) is held by `lpr` neighbouring lanes, each with one or two items:
// V elements and the V that they are paired with, so that a rotation needs no
// exchange, and a norm's sums are lane exchanges inside a wave.  The weights'
// gradients are column sums: a thread meets the same columns in every row, adds
// them in registers, a workgroup stores one partial row, and a second kernel adds
// those in a fixed order.  All sums are fp32, each output is rounded once.
//
// Forward and backward, bfloat16: 16384 tokens of 20 heads of 128, rotation alone, 75 us, 4.5
// TB/s; 32768 tokens of 24 heads of 64 with norm and weights, 107 us, 4.7 TB/s (a large copy:
// 5.15).  27567 rows of 75 float elements, 41 MB: 38 us, a chain of loads, exchanges and stores
// at few rows a CU.
#include "gs_host.h"
#include "gs_types.h"
#include "../../include/blitzgs_amd.h"

namespace {

constexpr int BLOCK = 256;
constexpr int MAX_DIM = 256;
constexpr int MAX_TABLE = 2048;       // pairs of the tokens of a workgroup's turn: 16 KB of LDS
constexpr int MAX_BLOCKS = 1 << 20;
constexpr int MAX_PARTS = 1024;       // partial rows of a weight's gradient

struct Side {                         // the queries or the keys
    const void* x;                    // the rows that are normed; backward without norm: null
    const void* dy;                   // backward
    const void* w;
    void* out;                        // forward: y, backward: dx
    float* parts;                     // backward: [blocks][D], or null
    int64_t xs[3], dys[3], outs[3];   // strides of batch, head, token
    int heads;
    int tokens;                       // of a workgroup's turn
    unsigned blocks;
};

struct RotaryArgs {
    Side side[2];
    const void* positions;
    int64_t ps[3];                    // strides of batch, token, axis
    const uint64_t* frequencies;
    int64_t n_tokens;                 // B T
    int T, D, pairs, N;               // N = axes * pairs
    int lpr;                          // lanes a row, a power of two
    int wide;                         // positions have 64 bits
    int w32;                          // weights are float32
    float magnitude, eps, inv_d;
};

// x in [-pi/4, pi/4]: the series to x^9 and x^10, whose next terms are below 3e-9
// and 5e-10.
__device__ __forceinline__ void cos_sin(uint64_t phase, float& c, float& s)
{
    const uint32_t quarter = (uint32_t)((phase + (1ull << 61)) >> 62);
    const int64_t rest = (int64_t)(phase - ((uint64_t)quarter << 62));
    const float x = (float)rest * (float)(6.283185307179586 / 18446744073709551616.0), q = x * x;
    float a = __builtin_fmaf(q, 2.7557319e-6f, -1.9841270e-4f);
    a = __builtin_fmaf(q, a, 8.3333333e-3f);
    a = __builtin_fmaf(q, a, -1.6666667e-1f);
    const float sx = __builtin_fmaf(q * x, a, x);
    float b = __builtin_fmaf(q, -2.7557319e-7f, 2.4801587e-5f);
    b = __builtin_fmaf(q, b, -1.3888889e-3f);
    b = __builtin_fmaf(q, b, 4.1666667e-2f);
    b = __builtin_fmaf(q, b, -0.5f);
    const float cx = __builtin_fmaf(q, b, 1.0f);
    c = quarter & 1 ? sx : cx;
    s = quarter & 1 ? cx : sx;
    if (quarter == 1 || quarter == 2) c = -c;
    if (quarter >= 2) s = -s;
}

template <typename T, int V>
__device__ __forceinline__ void load(const T* p, float* to)
{
    T t[V];
    __builtin_memcpy(t, p, sizeof(t));
#pragma unroll
    for (int i = 0; i < V; i++) to[i] = (float)t[i];
}

template <typename T, int V>
__device__ __forceinline__ void store(T* p, const float* from)
{
    T t[V];
#pragma unroll
    for (int i = 0; i < V; i++) t[i] = (T)from[i];
    __builtin_memcpy(p, t, sizeof(t));
}

// An item of a row: n_lo elements from lo on and n_hi from hi on, of the pairs from `pair`
// on, or of none (pair < 0).  All are V or none but where the row is RAGGED: a last item of
// the pairs and a last one of what is not rotated have fewer.
struct Item {
    int lo, hi, pair;
    int n_lo, n_hi;
};

template <int V, bool IL>
__device__ __forceinline__ Item item_of(int i, int N, int D)
{
    Item t;
    const int pair = i * V, last = (N + V - 1) / V;
    if (i < last) {
        t.lo = IL ? 2 * pair : pair;
        t.hi = IL ? 2 * pair + V : pair + N;
        t.pair = pair;
        t.n_lo = t.n_hi = min(V, N - pair);
    } else {
        t.lo = 2 * N + (i - last) * 2 * V;
        t.hi = t.lo + V;
        t.pair = -1;
        t.n_lo = max(0, min(V, D - t.lo));
        t.n_hi = max(0, min(V, D - t.hi));
    }
    return t;
}

// Whether the item's register i holds an element
template <int V, bool IL>
__device__ __forceinline__ bool holds(const Item& t, int i)
{
    return IL ? i < t.n_lo + t.n_hi : i < V ? i < t.n_lo : i - V < t.n_hi;
}

template <typename T, int V, bool RAGGED>
__device__ __forceinline__ void load_part(const T* p, int n, float* to)
{
    if (n == V) {
        load<T, V>(p, to);
    } else if (RAGGED && n > 0) {
        // without branches, so that all are under way together
        T t[V];
#pragma unroll
        for (int i = 0; i < V; i++) t[i] = p[min(i, n - 1)];
#pragma unroll
        for (int i = 0; i < V; i++) to[i] = i < n ? (float)t[i] : 0.0f;
    }
}

template <typename T, int V, bool RAGGED>
__device__ __forceinline__ void store_part(T* p, int n, const float* from)
{
    if (n == V) {
        store<T, V>(p, from);
    } else if (RAGGED) {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i < n) p[i] = (T)from[i];
    }
}

// Where pairs are neighbours an item is one piece of 2 V elements, of which the rest of a row may be half.
template <typename T, int V, bool IL, bool RAGGED>
__device__ __forceinline__ void load_item(const T* row, const Item& t, float (&v)[2 * V])
{
#pragma unroll
    for (int i = 0; i < 2 * V; i++) v[i] = 0.0f;
    if constexpr (IL) {
        load_part<T, 2 * V, RAGGED>(row + t.lo, t.n_lo + t.n_hi, v);
    } else {
        load_part<T, V, RAGGED>(row + t.lo, t.n_lo, v);
        load_part<T, V, RAGGED>(row + t.hi, t.n_hi, v + V);
    }
}

template <typename T, int V, bool IL, bool RAGGED>
__device__ __forceinline__ void store_item(T* row, const Item& t, const float (&v)[2 * V])
{
    if constexpr (IL) {
        store_part<T, 2 * V, RAGGED>(row + t.lo, t.n_lo + t.n_hi, v);
    } else {
        store_part<T, V, RAGGED>(row + t.lo, t.n_lo, v);
        store_part<T, V, RAGGED>(row + t.hi, t.n_hi, v + V);
    }
}

// The rotation by the table's angles, or back.
template <int V, bool IL, bool BACK, bool RAGGED>
__device__ __forceinline__ void turn(float (&v)[2 * V], const float2* cs, int n)
{
#pragma unroll
    for (int j = 0; j < V; j++) {
        if (RAGGED && j >= n) break;
        float& a = v[IL ? 2 * j : j];
        float& b = v[IL ? 2 * j + 1 : V + j];
        const float c = cs[j].x, s = BACK ? -cs[j].y : cs[j].y;
        const float y1 = __builtin_fmaf(a, c, -(b * s)), y2 = __builtin_fmaf(a, s, b * c);
        a = y1;
        b = y2;
    }
}

template <typename T, int V, int NC, bool IL, bool RAGGED, bool NORM, bool BWD>
__global__ __launch_bounds__(BLOCK) void rotary_kernel(RotaryArgs A)
{
    extern __shared__ uint64_t lds[];
    const Side& S = A.side[blockIdx.y];
    if (blockIdx.x >= S.blocks) return;
    // [tokens][4] offsets of x, dy, out and the positions; then [tokens][N] of cosine and sine
    int64_t* offset = (int64_t*)lds;
    float2* table = (float2*)(lds + 4 * S.tokens);
    const int lpr = A.lpr, lane = threadIdx.x & (lpr - 1), group = threadIdx.x / lpr, groups = BLOCK / lpr;
    const int N = A.N, D = A.D;

    Item items[NC];
    float w[NC][2 * V], dw[NC][2 * V];
#pragma unroll
    for (int c = 0; c < NC; c++) {
        items[c] = item_of<V, IL>(c * lpr + lane, N, D);
#pragma unroll
        for (int i = 0; i < 2 * V; i++) {
            w[c][i] = 1.0f;
            dw[c][i] = 0.0f;
        }
        if (NORM && S.w != nullptr) {
            if (A.w32)
                load_item<float, V, IL, RAGGED>((const float*)S.w, items[c], w[c]);
            else
                load_item<T, V, IL, RAGGED>((const T*)S.w, items[c], w[c]);
        }
    }
    // a group's rows are `groups` apart, a thread's pairs BLOCK: no divisions in the loops
    const int step_token = groups / S.heads, step_head = groups % S.heads;
    const int first_head = group % S.heads, first_token = group / S.heads;
    const int table_token = threadIdx.x / N, table_pair = threadIdx.x - table_token * N;
    const int table_tokens = BLOCK / N, table_pairs = BLOCK - table_tokens * N;

    for (int64_t first = (int64_t)blockIdx.x * S.tokens; first < A.n_tokens; first += (int64_t)S.blocks * S.tokens) {
        const int here = A.n_tokens - first < S.tokens ? (int)(A.n_tokens - first) : S.tokens;
        if (threadIdx.x < here) {
            const int64_t b = (first + threadIdx.x) / A.T, t = (first + threadIdx.x) - b * A.T;
            offset[4 * threadIdx.x] = b * S.xs[0] + t * S.xs[2];
            offset[4 * threadIdx.x + 1] = b * S.dys[0] + t * S.dys[2];
            offset[4 * threadIdx.x + 2] = b * S.outs[0] + t * S.outs[2];
            offset[4 * threadIdx.x + 3] = b * A.ps[0] + t * A.ps[1];
        }
        __syncthreads();
        for (int token = table_token, pair = table_pair; token < here;) {
            int64_t at = offset[4 * token + 3];
            if (A.pairs < N) at += pair / A.pairs * A.ps[2];
            const int64_t position = A.wide ? ((const int64_t*)A.positions)[at] : ((const int*)A.positions)[at];
            float c, s;
            cos_sin((uint64_t)position * A.frequencies[pair], c, s);
            table[token * N + pair] = make_float2(c * A.magnitude, s * A.magnitude);
            token += table_tokens;
            pair += table_pairs;
            if (pair >= N) {
                pair -= N;
                token++;
            }
        }
        __syncthreads();
        // the lanes of a row leave the loop together
        int token = first_token, head = first_head;
        while (token < here) {
            const T* x = (const T*)S.x + offset[4 * token] + head * S.xs[1];
            const T* dy = (const T*)S.dy + offset[4 * token + 1] + head * S.dys[1];
            T* out = (T*)S.out + offset[4 * token + 2] + head * S.outs[1];
            const float2* cs = table + token * N;
            float v[NC][2 * V], g[NC][2 * V];
            float r = 1.0f, up = 1.0f;
#pragma unroll
            for (int c = 0; c < NC; c++) {
                if constexpr (!BWD || NORM) load_item<T, V, IL, RAGGED>(x, items[c], v[c]);
                if constexpr (BWD) load_item<T, V, IL, RAGGED>(dy, items[c], g[c]);
            }
            if constexpr (NORM) {
                // of what is multiplied by a power of two
                auto mean_of_squares = [&](float by) __attribute__((always_inline)) {
                    float sum = 0.0f;
#pragma unroll
                    for (int c = 0; c < NC; c++)
#pragma unroll
                        for (int i = 0; i < 2 * V; i++) {
                            const float x = v[c][i] * by;
                            sum = __builtin_fmaf(x, x, sum);
                        }
                    for (int d = lpr / 2; d > 0; d >>= 1) sum += __shfl_xor(sum, d, 64);
                    return __builtin_fmaf(sum, A.inv_d, A.eps * by * by);
                };
                const float mean = mean_of_squares(1.0f);
                r = 1.0f / __builtin_sqrtf(mean);
                // Squares that fp32 does not hold, or not to its last bit: a row's lanes go together
                if (mean > 0x1p100f) {
                    r = 0x1p-96f / __builtin_sqrtf(mean_of_squares(0x1p-96f));
                } else if (mean < 0x1p-100f) {
                    // beside such a row 1 / r may pass fp32's range, so that the row itself grows
                    up = 0x1p96f;
                    r = 1.0f / __builtin_sqrtf(mean_of_squares(up));
#pragma unroll
                    for (int c = 0; c < NC; c++)
#pragma unroll
                        for (int i = 0; i < 2 * V; i++) v[c][i] *= up;
                }
            }
            if constexpr (!BWD) {
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    if constexpr (NORM) {
#pragma unroll
                        for (int i = 0; i < 2 * V; i++) v[c][i] = v[c][i] * r * w[c][i];
                    }
                    if (items[c].pair >= 0) turn<V, IL, false, RAGGED>(v[c], cs + items[c].pair, items[c].n_lo);
                }
            } else {
                float sum = 0.0f;
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    if (items[c].pair >= 0) turn<V, IL, true, RAGGED>(g[c], cs + items[c].pair, items[c].n_lo);
                    if constexpr (NORM) {
#pragma unroll
                        for (int i = 0; i < 2 * V; i++) {
                            v[c][i] *= r;                       // z
                            dw[c][i] = __builtin_fmaf(g[c][i], v[c][i], dw[c][i]);
                            g[c][i] *= w[c][i];                 // h
                            sum = __builtin_fmaf(g[c][i], v[c][i], sum);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 2 * V; i++) v[c][i] = g[c][i];
                    }
                }
                if constexpr (NORM) {
                    for (int d = lpr / 2; d > 0; d >>= 1) sum += __shfl_xor(sum, d, 64);
                    const float mean = sum * A.inv_d;
#pragma unroll
                    for (int c = 0; c < NC; c++)
#pragma unroll
                        for (int i = 0; i < 2 * V; i++) v[c][i] = r * __builtin_fmaf(-v[c][i], mean, g[c][i]);
                    if (up != 1.0f) {
#pragma unroll
                        for (int c = 0; c < NC; c++)
#pragma unroll
                            for (int i = 0; i < 2 * V; i++) v[c][i] *= up;
                    }
                }
            }
#pragma unroll
            for (int c = 0; c < NC; c++) store_item<T, V, IL, RAGGED>(out, items[c], v[c]);
            head += step_head;
            token += step_token;
            if (head >= S.heads) {
                head -= S.heads;
                token++;
            }
        }
        __syncthreads();   // the table is free
    }
    if constexpr (NORM && BWD) {
        if (S.parts == nullptr) return;
        float* sums = (float*)lds;      // [2 V][BLOCK]
        float* part = S.parts + (size_t)blockIdx.x * D;
#pragma unroll
        for (int c = 0; c < NC; c++) {
#pragma unroll
            for (int i = 0; i < 2 * V; i++) sums[i * BLOCK + threadIdx.x] = dw[c][i];
            __syncthreads();
            for (int e = threadIdx.x; e < 2 * V * lpr; e += BLOCK) {
                const int l = e & (lpr - 1), i = e / lpr;
                float s = 0.0f;
                for (int k = 0; k < groups; k++) s += sums[i * BLOCK + k * lpr + l];
                const Item t = item_of<V, IL>(c * lpr + l, N, D);
                if (holds<V, IL>(t, i)) part[i < V ? t.lo + i : t.hi + i - V] = s;
            }
            __syncthreads();
        }
    }
}

// A weight's gradient from the partial rows: 64 columns per block, 16 waves that
// each add every 16th partial row.
struct ColumnArgs {
    const float* parts[2];
    void* dw[2];
    unsigned n_parts[2];
    int D;
};

template <typename W>
__global__ __launch_bounds__(1024) void rotary_columns_kernel(ColumnArgs A)
{
    __shared__ float sums[16][64];
    const float* parts = A.parts[blockIdx.y];
    W* dw = (W*)A.dw[blockIdx.y];
    if (dw == nullptr) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = blockIdx.x * 64 + lane;
    float s = 0.0f;
    if (col < A.D) {
#pragma unroll 8
        for (unsigned p = wave; p < A.n_parts[blockIdx.y]; p += 16) s += parts[(size_t)p * A.D + col];
    }
    sums[wave][lane] = s;
    __syncthreads();
    if (wave != 0 || col >= A.D) return;
#pragma unroll
    for (int i = 1; i < 16; i++) s += sums[i][lane];
    dw[col] = (W)s;
}

struct Plan {
    int v, lpr, nc, tokens;
    bool ragged;
    unsigned blocks;
};

constexpr int RAGGED_V = 4;

// Elements per access: 16 bytes, or 8, where pairs and the rest of a row are a whole number
// of them.  Else four from any element on, with last items of fewer, or one by one where those
// leave half of the lanes idle.  196608 rows of queries and 98304 of keys, forward with norm,
// us with four and with one:
//   75 of 37 pairs, interleaved   float 46, 73    bfloat16 45, 78
//   33 of 16 pairs                float 29, 41    bfloat16 26, 40
//   129 of 64 pairs (17 of 32 lanes)   float 119, 96    255 of 127 (33 of 64)   float 256, 124
void lanes_of(Plan& p, int type, int N, int D)
{
    const int full = 16 / gs::dtype_bytes(type);
    auto lanes = [&](int v) {
        const int items = (N + v - 1) / v + (D - 2 * N + 2 * v - 1) / (2 * v);
        for (p.lpr = 1; p.lpr < 64 && p.lpr < items; p.lpr *= 2) {}
        p.nc = (items + p.lpr - 1) / p.lpr;
        p.v = v;
        return items;
    };
    p.ragged = false;
    for (int v : {full, full / 2})
        if (N % v == 0 && (D - 2 * N) % (2 * v) == 0) {
            lanes(v);
            return;
        }
    p.ragged = true;
    const int items = lanes(RAGGED_V);
    if (items * 16 < p.lpr * 9) lanes(1);
}

Plan plan_of(int type, int64_t n_tokens, int heads, int D, int N, bool parts)
{
    Plan p;
    lanes_of(p, type, N, D);
    // Four rows a group, or fewer where that would leave CUs without work: the angles of one
    // workgroup are formed while others move rows (32768 tokens of 24 heads of 64, forward
    // and backward: 103 us, with eight rows 111).
    const int64_t rows = BLOCK / p.lpr;
    int64_t tokens = (4 * rows + heads - 1) / heads;
    while (tokens > 1 && (n_tokens + tokens - 1) / tokens < 1024) tokens = (tokens + 1) / 2;
    const int64_t fit = MAX_TABLE / N < BLOCK ? MAX_TABLE / N : BLOCK;
    p.tokens = (int)(tokens < fit ? tokens : fit);
    const int64_t blocks = (n_tokens + p.tokens - 1) / p.tokens;
    const int64_t most = parts ? MAX_PARTS : MAX_BLOCKS;
    p.blocks = (unsigned)(blocks < most ? blocks : most);
    return p;
}

template <typename T, int V, int NC, bool RAGGED, bool NORM, bool BWD>
void launch_layout(const RotaryArgs& A, bool interleaved, dim3 grid, size_t lds, hipStream_t stream)
{
    if (interleaved)
        GS_TIMED(BWD ? "rotary_bwd_kernel" : "rotary_fwd_kernel", stream,
                 hipLaunchKernelGGL((rotary_kernel<T, V, NC, true, RAGGED, NORM, BWD>), grid, dim3(BLOCK), lds, stream,
                                    A));
    else
        GS_TIMED(BWD ? "rotary_bwd_kernel" : "rotary_fwd_kernel", stream,
                 hipLaunchKernelGGL((rotary_kernel<T, V, NC, false, RAGGED, NORM, BWD>), grid, dim3(BLOCK), lds, stream,
                                    A));
}

template <typename T, bool NORM, bool BWD>
void launch_vec(const RotaryArgs& A, const Plan& p, bool interleaved, dim3 grid, size_t lds, hipStream_t stream)
{
    constexpr int V = gs::Vec<T>::N;
    if (!p.ragged) {
        if (p.v == V) return launch_layout<T, V, 1, false, NORM, BWD>(A, interleaved, grid, lds, stream);
        return launch_layout<T, V / 2, 1, false, NORM, BWD>(A, interleaved, grid, lds, stream);
    }
    if (p.v == RAGGED_V) return launch_layout<T, RAGGED_V, 1, true, NORM, BWD>(A, interleaved, grid, lds, stream);
    if (p.nc == 1) return launch_layout<T, 1, 1, true, NORM, BWD>(A, interleaved, grid, lds, stream);
    return launch_layout<T, 1, 2, true, NORM, BWD>(A, interleaved, grid, lds, stream);
}

template <bool NORM, bool BWD>
void launch(int type, const RotaryArgs& A, const Plan& p, bool interleaved, dim3 grid, size_t lds, hipStream_t stream)
{
    if (type == GS_F32) return launch_vec<float, NORM, BWD>(A, p, interleaved, grid, lds, stream);
    if (type == GS_BF16) return launch_vec<gs::bf16, NORM, BWD>(A, p, interleaved, grid, lds, stream);
    return launch_vec<gs::f16, NORM, BWD>(A, p, interleaved, grid, lds, stream);
}

int check(int type, int param_type, int B, int Hq, int Hk, int T, int D, int axes, int pairs)
{
    GS_REQUIRE(gs::dtype_known(type), "rotary: unknown element type %d", type);
    GS_REQUIRE(param_type == type || param_type == GS_F32, "rotary: the weights have the rows' type or float32");
    GS_REQUIRE(B >= 0 && T >= 0 && Hq >= 0 && Hk >= 0, "rotary: sizes must not be negative");
    GS_REQUIRE(Hq <= 65536 && Hk <= 65536, "rotary: at most 65536 heads");
    GS_REQUIRE(D >= 1 && D <= MAX_DIM, "rotary: the head dimension must be in [1, %d], got %d", MAX_DIM, D);
    GS_REQUIRE(axes >= 1 && pairs >= 1 && axes <= D && pairs <= D && 2 * axes * pairs <= D,
               "rotary: %d axes of %d pairs do not fit a head dimension of %d", axes, pairs, D);
    return GS_OK;
}

void copy3(int64_t (&to)[3], const int64_t* from)
{
    for (int i = 0; i < 3; i++) to[i] = from[i];
}

// Fills in what both directions share and the two sides' plans; the LDS that a workgroup needs.
size_t fill(RotaryArgs& A, Plan (&plan)[2], int type, int param_type, int B, const int (&heads)[2], int T, int D,
            int axes, int pairs, float magnitude, float eps, const void* positions, int wide,
            const int64_t* position_strides, const int64_t* frequencies, bool parts)
{
    A.positions = positions;
    copy3(A.ps, position_strides);
    A.frequencies = (const uint64_t*)frequencies;
    A.n_tokens = (int64_t)B * T;
    A.T = T;
    A.D = D;
    A.pairs = pairs;
    A.N = axes * pairs;
    A.wide = wide;
    A.w32 = param_type == GS_F32;
    A.magnitude = magnitude;
    A.eps = eps;
    A.inv_d = 1.0f / (float)D;
    size_t lds = 0;
    for (int i = 0; i < 2; i++) {
        plan[i] = plan_of(type, A.n_tokens, heads[i] > 0 ? heads[i] : 1, D, A.N, parts);
        A.lpr = plan[i].lpr;
        A.side[i].heads = heads[i];
        A.side[i].tokens = plan[i].tokens;
        A.side[i].blocks = heads[i] > 0 && A.side[i].out != nullptr ? plan[i].blocks : 0;
        size_t n = (size_t)plan[i].tokens * (4 * sizeof(int64_t) + A.N * sizeof(float2));
        if (parts && n < 2u * plan[i].v * BLOCK * sizeof(float)) n = 2u * plan[i].v * BLOCK * sizeof(float);
        if (A.side[i].blocks > 0 && n > lds) lds = n;
    }
    return lds;
}

}  // namespace

extern "C" int gs_rotary_forward(int type, int param_type, int B, int Hq, int Hk, int T, int D, int axes, int pairs,
                                 int interleaved, float magnitude, int norm, float eps, const void* q,
                                 const int64_t* q_strides, const void* k, const int64_t* k_strides,
                                 const void* q_weight, const void* k_weight, const void* positions, int wide,
                                 const int64_t* position_strides, const int64_t* frequencies, void* q_out,
                                 const int64_t* q_out_strides, void* k_out, const int64_t* k_out_strides,
                                 hipStream_t stream)
{
    gs::clear_error();
    if (int rc = check(type, param_type, B, Hq, Hk, T, D, axes, pairs)) return rc;
    GS_REQUIRE(!norm || eps >= 0.0f, "rotary: eps must not be negative");
    if (B == 0 || T == 0 || (Hq == 0 && Hk == 0)) return GS_OK;
    GS_REQUIRE(positions && position_strides && frequencies, "rotary: positions and frequencies must be given");
    GS_REQUIRE(Hq == 0 || (q && q_strides && q_out && q_out_strides), "rotary: q, its output and strides must be given");
    GS_REQUIRE(Hk == 0 || (k && k_strides && k_out && k_out_strides), "rotary: k, its output and strides must be given");
    RotaryArgs A{};
    const void* in[2] = {q, k};
    const void* weight[2] = {q_weight, k_weight};
    void* out[2] = {q_out, k_out};
    const int64_t *is[2] = {q_strides, k_strides}, *os[2] = {q_out_strides, k_out_strides};
    const int heads[2] = {Hq, Hk};
    for (int i = 0; i < 2; i++) {
        if (heads[i] == 0) continue;
        A.side[i].x = in[i];
        A.side[i].w = weight[i];
        A.side[i].out = out[i];
        copy3(A.side[i].xs, is[i]);
        copy3(A.side[i].outs, os[i]);
    }
    Plan plan[2];
    const size_t lds = fill(A, plan, type, param_type, B, heads, T, D, axes, pairs, magnitude, eps, positions, wide,
                            position_strides, frequencies, false);
    const unsigned blocks = A.side[0].blocks > A.side[1].blocks ? A.side[0].blocks : A.side[1].blocks;
    if (norm)
        launch<true, false>(type, A, plan[0], interleaved != 0, dim3(blocks, 2), lds, stream);
    else
        launch<false, false>(type, A, plan[0], interleaved != 0, dim3(blocks, 2), lds, stream);
    GS_LAUNCH_CHECK("rotary_fwd_kernel");
    return GS_OK;
}

extern "C" size_t gs_rotary_workspace_bytes(int type, int B, int Hq, int Hk, int T, int D, int axes, int pairs)
{
    if (check(type, type, B, Hq, Hk, T, D, axes, pairs) != GS_OK) return 0;
    const int64_t n = (int64_t)B * T;
    size_t rows = 0;
    for (int heads : {Hq, Hk})
        if (heads > 0) rows += plan_of(type, n, heads, D, axes * pairs, true).blocks;
    return rows * D * sizeof(float);
}

extern "C" int gs_rotary_backward(int type, int param_type, int B, int Hq, int Hk, int T, int D, int axes, int pairs,
                                  int interleaved, float magnitude, int norm, float eps, const void* q,
                                  const int64_t* q_strides, const void* k, const int64_t* k_strides,
                                  const void* q_weight, const void* k_weight, const void* positions, int wide,
                                  const int64_t* position_strides, const int64_t* frequencies, const void* dq_out,
                                  const int64_t* dq_out_strides, const void* dk_out, const int64_t* dk_out_strides,
                                  void* dq, const int64_t* dq_strides, void* dk, const int64_t* dk_strides,
                                  void* dq_weight, void* dk_weight, void* workspace, hipStream_t stream)
{
    gs::clear_error();
    if (int rc = check(type, param_type, B, Hq, Hk, T, D, axes, pairs)) return rc;
    GS_REQUIRE(!norm || eps >= 0.0f, "rotary: eps must not be negative");
    const bool parts = norm && (dq_weight != nullptr || dk_weight != nullptr);
    const bool rows = B > 0 && T > 0 && (Hq > 0 || Hk > 0);
    GS_REQUIRE(!parts || !rows || workspace != nullptr, "rotary: the weights' gradients need the workspace");
    const void* in[2] = {q, k};
    const void* weight[2] = {q_weight, k_weight};
    const void* grad[2] = {dq_out, dk_out};
    void* out[2] = {dq, dk};
    void* dw[2] = {dq_weight, dk_weight};
    const int64_t *is[2] = {q_strides, k_strides}, *gs_[2] = {dq_out_strides, dk_out_strides},
                  *os[2] = {dq_strides, dk_strides};
    const int heads[2] = {Hq, Hk};
    RotaryArgs A{};
    ColumnArgs C{};
    C.D = D;
    C.dw[0] = dq_weight;
    C.dw[1] = dk_weight;
    if (rows) {
        GS_REQUIRE(positions && position_strides && frequencies, "rotary: positions and frequencies must be given");
        bool any = false;
        for (int i = 0; i < 2; i++) {
            if (heads[i] == 0) continue;
            GS_REQUIRE(dw[i] == nullptr || out[i] != nullptr, "rotary: a weight's gradient comes with its rows'");
            if (out[i] == nullptr) continue;
            GS_REQUIRE(grad[i] && gs_[i] && os[i] && (!norm || (in[i] && is[i])),
                       "rotary: the gradients' tensors and strides must be given");
            any = true;
            if (norm) {
                A.side[i].x = in[i];
                copy3(A.side[i].xs, is[i]);
            }
            A.side[i].w = weight[i];
            A.side[i].dy = grad[i];
            A.side[i].out = out[i];
            copy3(A.side[i].dys, gs_[i]);
            copy3(A.side[i].outs, os[i]);
        }
        Plan plan[2];
        const size_t lds = fill(A, plan, type, param_type, B, heads, T, D, axes, pairs, magnitude, eps, positions,
                                wide, position_strides, frequencies, parts);
        float* p = (float*)workspace;
        for (int i = 0; i < 2; i++) {
            if (heads[i] == 0) continue;
            if (dw[i] != nullptr) {
                A.side[i].parts = p;
                C.parts[i] = p;
                C.n_parts[i] = A.side[i].blocks;
            }
            if (parts) p += (size_t)plan[i].blocks * D;
        }
        const unsigned blocks = A.side[0].blocks > A.side[1].blocks ? A.side[0].blocks : A.side[1].blocks;
        // without rows to write a weight of no heads has its gradient, zero, to come
        if (any && norm)
            launch<true, true>(type, A, plan[0], interleaved != 0, dim3(blocks, 2), lds, stream);
        else if (any)
            launch<false, true>(type, A, plan[0], interleaved != 0, dim3(blocks, 2), lds, stream);
        GS_LAUNCH_CHECK("rotary_bwd_kernel");
    }
    if (parts) {
        const dim3 grid(gs_div_up((size_t)D, 64), 2);
        if (param_type == GS_F32)
            GS_TIMED("rotary_columns_kernel", stream,
                     hipLaunchKernelGGL(rotary_columns_kernel<float>, grid, dim3(1024), 0, stream, C));
        else if (param_type == GS_BF16)
            GS_TIMED("rotary_columns_kernel", stream,
                     hipLaunchKernelGGL(rotary_columns_kernel<gs::bf16>, grid, dim3(1024), 0, stream, C));
        else
            GS_TIMED("rotary_columns_kernel", stream,
                     hipLaunchKernelGGL(rotary_columns_kernel<gs::f16>, grid, dim3(1024), 0, stream, C));
        GS_LAUNCH_CHECK("rotary_columns_kernel");
    }
    return GS_OK;
}
