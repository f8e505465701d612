// Layer normalisation of rows, forward and backward.
//
//   forward    mean = sum(x) / n,  rstd = 1 / sqrt(sum((x - mean)^2) / n + eps)
//              z = (x - mean) rstd,  y = w z + b
//   backward   h = dy w,  dx = rstd (h - mean(h) - z mean(h z))
//              dw = sum over rows of dy z,  db = sum over rows of dy
//
// Both passes are bound by memory: the forward reads x and writes y, the
// backward reads x and dy and writes dx, and each touches every element once.
// A row is held in the registers of the LPR threads that share it (NC chunks
// of 16 bytes each), so that the centred second pass over the squares, and
// the backward's use of x after its two row sums, cost no second read.  Up to
// 64 threads a row's sums are lane exchanges inside a wave, without barrier.
//
// The weight's and the bias's gradients are column sums over all rows.  A
// thread owns the same columns in every row it visits, so it carries their
// partial sums in registers over the whole strided loop; a block adds its
// rows' threads in LDS and stores one partial row, and a second kernel adds
// the partial rows in a fixed order.  No atomics: the same inputs give the
// same bits.  All sums and statistics are fp32 whatever the tensors' type;
// each output is rounded to its type once.
//
// 65536 x 1024 bfloat16, fp32 parameters: forward 53 us (268 MB, 5.0 TB/s),
// backward 83 us (403 MB, 4.8 TB/s) and 4 us for the partial rows; a large copy
// reaches 5.15 TB/s.  10007 x 513 float32, one element per access: 12, 17 and 4 us
// (103 MB, 20 us at that rate).
#include "gs_host.h"
#include "gs_types.h"
#include "../../include/blitzgs_amd.h"

namespace {

constexpr int BLOCK = 256;
constexpr int MAX_WIDTH = 32768;
// Partial rows of the column sums: two blocks per CU, enough waves in flight
// to cover memory latency and few enough partial rows to add up quickly.
constexpr int MAX_PARTS = 512;
constexpr int MAX_BLOCKS = 1 << 20;   // of the forward: more rows are walked with that stride

template <int V, typename W>
__device__ __forceinline__ void load_params(const W* p, int at, float (&out)[V], float none)
{
    if (p == nullptr) {
#pragma unroll
        for (int i = 0; i < V; i++) out[i] = none;
        return;
    }
    W t[V];
    __builtin_memcpy(t, p + at, V * sizeof(W));
#pragma unroll
    for (int i = 0; i < V; i++) out[i] = (float)t[i];
}

template <typename T, int V>
struct Chunk {
    T v[V];
};

// The sum of v over the LPR threads of a row, in every one of them.  Rows of
// more than a wave meet in LDS (`meet`, one slot per wave; two barriers).
template <int LPR>
__device__ __forceinline__ float row_sum(float v, float* meet)
{
#pragma unroll
    for (int d = (LPR < 64 ? LPR : 64) / 2; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
    if constexpr (LPR > 64) {
        if ((threadIdx.x & 63) == 0) meet[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int i = 0; i < LPR / 64; i++) v += meet[i];
        __syncthreads();
    }
    return v;
}

struct NormArgs {
    const void* x;
    const void* dy;
    const void* w;
    const void* b;
    void* y;            // forward: y, backward: dx
    float* mean;
    float* rstd;
    float* parts;       // backward: [blocks][2][width], or null
    int64_t rows;
    int64_t xs, dys;    // row strides in elements
    int width;
    float eps;
};

template <typename T, typename W, int V, int LPR, int NC>
__global__ __launch_bounds__(LPR > BLOCK ? LPR : BLOCK) void norm_fwd_kernel(NormArgs A)
{
    constexpr int RPB = LPR > BLOCK ? 1 : BLOCK / LPR;
    __shared__ float meet[LPR > 64 ? LPR / 64 : 1];
    const int l = threadIdx.x % LPR;
    const float inv_n = 1.0f / (float)A.width;
    // whole rows leave the loop together: with LPR > 64 the block has one row
    for (int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / LPR; row < A.rows; row += (int64_t)gridDim.x * RPB) {
        const T* x = (const T*)A.x + row * A.xs;
        T* y = (T*)A.y + row * A.width;
        float v[NC][V];
        float s = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const int at = (c * LPR + l) * V;
            Chunk<T, V> t{};
            if (at < A.width) __builtin_memcpy(&t, x + at, sizeof(t));
#pragma unroll
            for (int i = 0; i < V; i++) {
                v[c][i] = (float)t.v[i];
                s += v[c][i];
            }
        }
        const float mean = row_sum<LPR>(s, meet) * inv_n;
        float q = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const bool in = (c * LPR + l) * V < A.width;
#pragma unroll
            for (int i = 0; i < V; i++) {
                v[c][i] = in ? v[c][i] - mean : 0.0f;
                q = __builtin_fmaf(v[c][i], v[c][i], q);
            }
        }
        const float rstd = 1.0f / __builtin_sqrtf(row_sum<LPR>(q, meet) * inv_n + A.eps);
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const int at = (c * LPR + l) * V;
            if (at >= A.width) continue;
            float w[V], b[V];
            load_params<V>((const W*)A.w, at, w, 1.0f);
            load_params<V>((const W*)A.b, at, b, 0.0f);
            Chunk<T, V> t;
#pragma unroll
            for (int i = 0; i < V; i++) t.v[i] = (T)__builtin_fmaf(v[c][i] * rstd, w[i], b[i]);
            __builtin_memcpy(y + at, &t, sizeof(t));
        }
        if (l == 0 && A.mean != nullptr) {
            A.mean[row] = mean;
            A.rstd[row] = rstd;
        }
    }
}

template <typename T, typename W, int V, int LPR, int NC>
__global__ __launch_bounds__(LPR > BLOCK ? LPR : BLOCK) void norm_bwd_kernel(NormArgs A)
{
    constexpr int THREADS = LPR > BLOCK ? LPR : BLOCK, RPB = THREADS / LPR;
    __shared__ float meet[LPR > 64 ? LPR / 64 : 1];
    __shared__ float sums[RPB > 1 ? (RPB - 1) * LPR * V : 1];
    const int l = threadIdx.x % LPR, sub = threadIdx.x / LPR;
    const float inv_n = 1.0f / (float)A.width;
    float w[NC][V], dw[NC][V], db[NC][V];
#pragma unroll
    for (int c = 0; c < NC; c++) {
        const int at = (c * LPR + l) * V;
#pragma unroll
        for (int i = 0; i < V; i++) w[c][i] = dw[c][i] = db[c][i] = 0.0f;
        if (at < A.width) load_params<V>((const W*)A.w, at, w[c], 1.0f);
    }
    // a row's threads leave the loop together: its barriers are met by whole rows
    for (int64_t row = (int64_t)blockIdx.x * RPB + sub; row < A.rows; row += (int64_t)gridDim.x * RPB) {
        const T* x = (const T*)A.x + row * A.xs;
        const T* dy = (const T*)A.dy + row * A.dys;
        T* dx = (T*)A.y + row * A.width;
        const float mean = A.mean[row], rstd = A.rstd[row];
        float z[NC][V], h[NC][V];
        float sh = 0.0f, shz = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const int at = (c * LPR + l) * V;
            const bool in = at < A.width;
            Chunk<T, V> tx{}, tg{};
            if (in) {
                __builtin_memcpy(&tx, x + at, sizeof(tx));
                __builtin_memcpy(&tg, dy + at, sizeof(tg));
            }
#pragma unroll
            for (int i = 0; i < V; i++) {
                const float g = (float)tg.v[i];
                z[c][i] = in ? ((float)tx.v[i] - mean) * rstd : 0.0f;
                h[c][i] = g * w[c][i];
                sh += h[c][i];
                shz = __builtin_fmaf(h[c][i], z[c][i], shz);
                dw[c][i] = __builtin_fmaf(g, z[c][i], dw[c][i]);
                db[c][i] += g;
            }
        }
        const float mh = row_sum<LPR>(sh, meet) * inv_n, mhz = row_sum<LPR>(shz, meet) * inv_n;
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const int at = (c * LPR + l) * V;
            if (at >= A.width) continue;
            Chunk<T, V> t;
#pragma unroll
            for (int i = 0; i < V; i++) t.v[i] = (T)(rstd * (h[c][i] - mh - z[c][i] * mhz));
            __builtin_memcpy(dx + at, &t, sizeof(t));
        }
    }
    if (A.parts == nullptr) return;
    float* part = A.parts + (size_t)blockIdx.x * 2 * A.width;
#pragma unroll
    for (int k = 0; k < 2; k++) {
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const int at = (c * LPR + l) * V;
            float (&acc)[V] = k == 0 ? dw[c] : db[c];
            if constexpr (RPB > 1) {
                __syncthreads();
                if (sub > 0) {
#pragma unroll
                    for (int i = 0; i < V; i++) sums[((sub - 1) * V + i) * LPR + l] = acc[i];
                }
                __syncthreads();
                if (sub == 0) {
#pragma unroll 1
                    for (int r = 0; r < RPB - 1; r++) {
#pragma unroll
                        for (int i = 0; i < V; i++) acc[i] += sums[(r * V + i) * LPR + l];
                    }
                }
            }
            if (sub == 0) {
#pragma unroll
                for (int i = 0; i < V; i++)
                    if (at + i < A.width) part[(size_t)k * A.width + at + i] = acc[i];
            }
        }
    }
}

// dw and db from the partial rows: 64 columns of [dw | db] per block, 16 waves
// that each add every 16th partial row.
template <typename W>
__global__ __launch_bounds__(1024) void norm_columns_kernel(const float* __restrict__ parts, int n_parts, int width,
                                                            W* __restrict__ dw, W* __restrict__ db)
{
    __shared__ float sums[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = blockIdx.x * 64 + lane;
    float s = 0.0f;
    if (col < 2 * width) {
#pragma unroll 8
        for (int p = wave; p < n_parts; p += 16) s += parts[(size_t)p * 2 * width + col];
    }
    sums[wave][lane] = s;
    __syncthreads();
    if (wave != 0 || col >= 2 * width) return;
#pragma unroll
    for (int i = 1; i < 16; i++) s += sums[i][lane];
    if (col < width) {
        if (dw != nullptr) dw[col] = (W)s;
    } else if (db != nullptr) {
        db[col - width] = (W)s;
    }
}

// Elements per access (16 bytes; one where the width is no multiple of that),
// threads per row and accesses per thread: the fewest threads that hold the
// row in one access each, then a wave with up to 32 elements per lane, then 4
// and 16 waves.  More elements per lane would spill the backward's five
// values per element, as 16 waves do already, which leave a lane 128 registers
// (widths above 8192: up to 656 bytes of scratch a lane backward).  Rows of
// single elements step from 8 accesses to 12 before 16: 10007 rows of 513 float32
// take 19.4 us backward with 12 and 21.1 with 16, of 767 22.6 and 25.0; of 513
// bfloat16 24.8 and 27.4.  6 and 24 have not been tried.
struct Shape {
    int v, lpr, nc;
};

Shape shape_of(int width, int vec)
{
    const int v = width % vec == 0 ? vec : 1, chunks = width / v;
    if (v == 1) {
        for (int lpr = 64; lpr <= 1024; lpr *= 4)
            for (int nc : {1, 2, 4, 8, 12, 16, 32})
                if ((lpr == 64 || nc >= 16) && chunks <= lpr * nc) return {v, lpr, nc};
    } else {
        for (int lpr = 8; lpr <= 64; lpr *= 2)
            if (chunks <= lpr) return {v, lpr, 1};
        for (int lpr = 64; lpr <= 1024; lpr *= 4)
            for (int nc = 2; nc <= 32 / v; nc *= 2)
                if (chunks <= lpr * nc) return {v, lpr, nc};
    }
    return {};
}

int rows_per_block(const Shape& s) { return s.lpr >= BLOCK ? 1 : BLOCK / s.lpr; }

int parts_of(int64_t rows, const Shape& s)
{
    const int64_t n = (rows + rows_per_block(s) - 1) / rows_per_block(s);
    return (int)(n < MAX_PARTS ? n : MAX_PARTS);
}

template <typename T, typename W, bool BWD, int V, int LPR, int NC>
void launch_one(const NormArgs& A, unsigned blocks, hipStream_t stream)
{
    const dim3 threads(LPR > BLOCK ? LPR : BLOCK);
    if constexpr (BWD)
        GS_TIMED("norm_bwd_kernel", stream,
                 hipLaunchKernelGGL((norm_bwd_kernel<T, W, V, LPR, NC>), dim3(blocks), threads, 0, stream, A));
    else
        GS_TIMED("norm_fwd_kernel", stream,
                 hipLaunchKernelGGL((norm_fwd_kernel<T, W, V, LPR, NC>), dim3(blocks), threads, 0, stream, A));
}

template <typename T, typename W, bool BWD>
void launch_shape(const Shape& s, const NormArgs& A, unsigned blocks, hipStream_t stream)
{
    constexpr int V = gs::Vec<T>::N;
#define GS_NORM_CASE(v, L, C) \
    case L * 64 + C: return launch_one<T, W, BWD, v, L, C>(A, blocks, stream)
    if (s.v == 1) {
        switch (s.lpr * 64 + s.nc) {
            GS_NORM_CASE(1, 64, 1);
            GS_NORM_CASE(1, 64, 2);
            GS_NORM_CASE(1, 64, 4);
            GS_NORM_CASE(1, 64, 8);
            GS_NORM_CASE(1, 64, 12);
            GS_NORM_CASE(1, 64, 16);
            GS_NORM_CASE(1, 64, 32);
            GS_NORM_CASE(1, 256, 16);
            GS_NORM_CASE(1, 256, 32);
            GS_NORM_CASE(1, 1024, 16);
            GS_NORM_CASE(1, 1024, 32);
        }
        return;
    }
    switch (s.lpr * 64 + s.nc) {
        GS_NORM_CASE(V, 8, 1);
        GS_NORM_CASE(V, 16, 1);
        GS_NORM_CASE(V, 32, 1);
        GS_NORM_CASE(V, 64, 1);
        GS_NORM_CASE(V, 64, 2);
        GS_NORM_CASE(V, 64, 4);
        GS_NORM_CASE(V, 256, 2);
        GS_NORM_CASE(V, 256, 4);
        GS_NORM_CASE(V, 1024, 2);
        GS_NORM_CASE(V, 1024, 4);
    }
    if constexpr (V == 4) {
        switch (s.lpr * 64 + s.nc) {
            GS_NORM_CASE(V, 64, 8);
            GS_NORM_CASE(V, 256, 8);
            GS_NORM_CASE(V, 1024, 8);
        }
    }
#undef GS_NORM_CASE
}

template <bool BWD>
void launch(int type, int param_type, const Shape& s, const NormArgs& A, unsigned blocks, hipStream_t stream)
{
    if (type == GS_F32) return launch_shape<float, float, BWD>(s, A, blocks, stream);
    if (type == GS_BF16) {
        if (param_type == GS_F32) return launch_shape<gs::bf16, float, BWD>(s, A, blocks, stream);
        return launch_shape<gs::bf16, gs::bf16, BWD>(s, A, blocks, stream);
    }
    if (param_type == GS_F32) return launch_shape<gs::f16, float, BWD>(s, A, blocks, stream);
    return launch_shape<gs::f16, gs::f16, BWD>(s, A, blocks, stream);
}

// Checks shared by both directions; GS_OK or an error that is set.
int check(int type, int param_type, int64_t rows, int width, int64_t stride)
{
    GS_REQUIRE(gs::dtype_known(type), "layer norm: unknown element type %d", type);
    GS_REQUIRE(param_type == type || param_type == GS_F32,
               "layer norm: the parameters have the rows' type or float32");
    GS_REQUIRE(rows >= 0 && rows <= 0x7fffffff, "layer norm: rows must be in [0, 2^31)");
    GS_REQUIRE(width >= 1 && width <= MAX_WIDTH, "layer norm: width must be in [1, %d], got %d", MAX_WIDTH, width);
    GS_REQUIRE(stride >= width || stride == 0 || rows <= 1,
               "layer norm: rows may not overlap (stride %lld below the width %d)", (long long)stride, width);
    return GS_OK;
}

}  // namespace

extern "C" int gs_layer_norm_forward(int type, int param_type, int64_t rows, int width, const void* x,
                                     int64_t x_stride, const void* weight, const void* bias, float eps, void* y,
                                     float* mean, float* rstd, hipStream_t stream)
{
    gs::clear_error();
    if (int rc = check(type, param_type, rows, width, x_stride)) return rc;
    GS_REQUIRE(eps >= 0.0f, "layer norm: eps must not be negative");
    GS_REQUIRE((mean == nullptr) == (rstd == nullptr), "layer norm: mean and rstd come together");
    if (rows == 0) return GS_OK;
    GS_REQUIRE(x != nullptr && y != nullptr, "layer norm: x and y must be non-null");
    const Shape s = shape_of(width, 16 / gs::dtype_bytes(type));
    NormArgs A{};
    A.x = x;
    A.w = weight;
    A.b = bias;
    A.y = y;
    A.mean = mean;
    A.rstd = rstd;
    A.rows = rows;
    A.xs = x_stride;
    A.width = width;
    A.eps = eps;
    const int64_t blocks = (rows + rows_per_block(s) - 1) / rows_per_block(s);
    launch<false>(type, param_type, s, A, (unsigned)(blocks < MAX_BLOCKS ? blocks : MAX_BLOCKS), stream);
    GS_LAUNCH_CHECK("norm_fwd_kernel");
    return GS_OK;
}

extern "C" size_t gs_layer_norm_workspace_bytes(int type, int64_t rows, int width)
{
    if (check(type, type, rows, width, width) != GS_OK) return 0;
    const Shape s = shape_of(width, 16 / gs::dtype_bytes(type));
    const size_t n = (size_t)parts_of(rows, s) * 2 * (size_t)width * sizeof(float);
    return n < 256 ? 256 : n;
}

extern "C" int gs_layer_norm_backward(int type, int param_type, int64_t rows, int width, const void* x,
                                      int64_t x_stride, const void* weight, const float* mean, const float* rstd,
                                      const void* dy, int64_t dy_stride, void* dx, void* dweight, void* dbias,
                                      void* workspace, hipStream_t stream)
{
    gs::clear_error();
    if (int rc = check(type, param_type, rows, width, x_stride)) return rc;
    if (int rc = check(type, param_type, rows, width, dy_stride)) return rc;
    const bool columns = dweight != nullptr || dbias != nullptr;
    GS_REQUIRE(!columns || workspace != nullptr, "layer norm: the parameters' gradients need the workspace");
    const Shape s = shape_of(width, 16 / gs::dtype_bytes(type));
    const int parts = parts_of(rows, s);
    if (rows > 0) {
        GS_REQUIRE(x && dy && dx && mean && rstd, "layer norm: x, dy, dx, mean and rstd must be non-null");
        NormArgs A{};
        A.x = x;
        A.dy = dy;
        A.w = weight;
        A.y = dx;
        A.mean = const_cast<float*>(mean);
        A.rstd = const_cast<float*>(rstd);
        A.parts = columns ? (float*)workspace : nullptr;
        A.rows = rows;
        A.xs = x_stride;
        A.dys = dy_stride;
        A.width = width;
        launch<true>(type, param_type, s, A, (unsigned)parts, stream);
        GS_LAUNCH_CHECK("norm_bwd_kernel");
    }
    if (columns) {
        const dim3 grid(gs_div_up(2 * (size_t)width, 64));
        const float* p = (const float*)workspace;
        if (param_type == GS_F32)
            GS_TIMED("norm_columns_kernel", stream,
                     hipLaunchKernelGGL(norm_columns_kernel<float>, grid, dim3(1024), 0, stream, p, parts, width,
                                        (float*)dweight, (float*)dbias));
        else if (param_type == GS_BF16)
            GS_TIMED("norm_columns_kernel", stream,
                     hipLaunchKernelGGL(norm_columns_kernel<gs::bf16>, grid, dim3(1024), 0, stream, p, parts, width,
                                        (gs::bf16*)dweight, (gs::bf16*)dbias));
        else
            GS_TIMED("norm_columns_kernel", stream,
                     hipLaunchKernelGGL(norm_columns_kernel<gs::f16>, grid, dim3(1024), 0, stream, p, parts, width,
                                        (gs::f16*)dweight, (gs::f16*)dbias));
        GS_LAUNCH_CHECK("norm_columns_kernel");
    }
    return GS_OK;
}
