// card_norm.hip - root-mean-square norm of rows, with the residual's addition before it and 8 bits after it.
//
//   h = x + residual,  y = h * rstd * w,  rstd = 1 / sqrt(mean(h^2) + eps)
//   8 bits: amax = max |y| of the row, scale = amax / 448, q = e4m3(y * 448 / amax)     (y itself is never stored)
//   backward, from the h that forward stored:  gw = g * w,  dx = rstd * (gw - h * rstd^2 * mean(gw * h)) + gh,
//   dw = sum over rows of g * h * rstd;  the residual's gradient is dx.
//
// Everything between a load and a store is 32 bits (rows of at most 64 columns: 64 bits in backward, see there); h and y are
// rounded once, and y comes from the h that is not rounded yet.  A row is read once and lives in registers: V vectors of
// 16 bytes in each of TPR threads.
#include "card_layers.h"

using namespace card;

namespace {

constexpr int kThreads = 256;                      // of a workgroup whose rows take 256 threads or less
constexpr float kE4m3Max = 448.0f;

struct NormArgs {
    const void* x;
    const void* residual;
    const void* w;              // NULL: ones
    void* h;
    void* y;
    float* scale;
    long long rows;
    int cols;
    int w_f32;                  // w holds floats whatever x holds
    float eps;
    // backward
    const void* g;              // NULL: zeros
    const void* gh;             // NULL: zeros
    float* part;                // (workgroups, cols) partial dw, or NULL
};

__device__ __forceinline__ float max_nan(float a, float b) {          // for values >= 0: their bits order them, NaN above all
    return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b)));
}

// all-reduce over the TPR threads of a row; `buf` holds two floats per wave of the workgroup's row, `turn` alternates
template <int TPR, typename F, typename Op> __device__ __forceinline__ F row_reduce(F v, F* buf, Op op) {
#pragma unroll
    for (int o = 1; o < (TPR < 64 ? TPR : 64); o <<= 1) v = op(v, __shfl_xor(v, o, 64));
    if constexpr (TPR > 64) {
        constexpr int W = TPR / 64;
        if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
        __syncthreads();
        v = buf[0];
#pragma unroll
        for (int k = 1; k < W; ++k) v = op(v, buf[k]);
    }
    return v;
}

template <int N, typename T> __device__ __forceinline__ void load_w(const NormArgs& a, int c, int n, float (&w)[N]) {
    if (!a.w) {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = 1.0f;
    } else if (a.w_f32) {
        load_n<N>((const float*)a.w + c, n, w);
    } else {
        load_n<N>((const T*)a.w + c, n, w);
    }
}

// four floats as e4m3 bytes, round to nearest even
__device__ __forceinline__ int pack_e4m3(float a, float b, float c, float d) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}

template <typename T, int TPR, int V, bool Q>
__global__ __launch_bounds__(TPR > kThreads ? TPR : kThreads) void rms_norm_kernel(const NormArgs a) {
    constexpr int N = 16 / sizeof(T), T_WG = TPR > kThreads ? TPR : kThreads, RPW = T_WG / TPR;
    __shared__ float buf[2][TPR > 64 ? TPR / 64 : 1];
    const int t = threadIdx.x % TPR;
    for (long long r0 = (long long)blockIdx.x * RPW; r0 < a.rows; r0 += (long long)gridDim.x * RPW) {
        const long long row = r0 + threadIdx.x / TPR;
        const bool live = row < a.rows;
        float h[V][N];
        float ss = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c = (v * TPR + t) * N, n = live ? a.cols - c : 0;
            load_n<N>((const T*)a.x + row * a.cols + c, n, h[v]);
            if (a.residual) {
                float r[N];
                load_n<N>((const T*)a.residual + row * a.cols + c, n, r);
#pragma unroll
                for (int i = 0; i < N; ++i) h[v][i] += r[i];
                if (n > 0) store_n<N>((T*)a.h + row * a.cols + c, n, h[v]);
            }
#pragma unroll
            for (int i = 0; i < N; ++i) ss += h[v][i] * h[v][i];
        }
        ss = row_reduce<TPR>(ss, buf[0], [](float p, float q) { return p + q; });
        const float rstd = 1.0f / sqrtf(ss / (float)a.cols + a.eps);
        float amax = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c = (v * TPR + t) * N, n = live ? a.cols - c : 0;
            float w[N];
            load_w<N, T>(a, c, n, w);
#pragma unroll
            for (int i = 0; i < N; ++i) h[v][i] = h[v][i] * rstd * w[i];
            if constexpr (Q) {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (i < n) amax = max_nan(amax, fabsf(h[v][i]));
            } else {
                if (n > 0) store_n<N>((T*)a.y + row * a.cols + c, n, h[v]);
            }
        }
        if constexpr (Q) {
            amax = row_reduce<TPR>(amax, buf[1], max_nan);
            // a row of zeros (or of values below 448 / FLT_MAX) must not divide by zero; NaN stays NaN
            const float inv = amax < 1.4e-36f ? 3.0e38f : kE4m3Max / amax;
            if (live && t == 0) a.scale[row] = amax / kE4m3Max;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int c = (v * TPR + t) * N, n = live ? a.cols - c : 0;
                unsigned char* q = (unsigned char*)a.y + row * a.cols + c;
                int word[N / 4];
#pragma unroll
                for (int k = 0; k < N / 4; ++k)
                    word[k] = pack_e4m3(h[v][4 * k] * inv, h[v][4 * k + 1] * inv, h[v][4 * k + 2] * inv, h[v][4 * k + 3] * inv);
                if (n >= N) {
                    memcpy(q, word, N);
                } else {
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        if (i < n) q[i] = (unsigned char)(word[i / 4] >> (8 * (i % 4)));
                }
            }
        }
        if constexpr (TPR > 64) __syncthreads();            // buf is free for the next row
    }
}

// F: in rows of a few columns the two terms of dx all but cancel (at one column to eps * rstd^2 of either), so there the
// row's numbers and the difference are formed in 64 bits.
template <typename T, typename F, int TPR, int V>
__global__ __launch_bounds__(TPR > kThreads ? TPR : kThreads) void rms_norm_backward_kernel(const NormArgs a) {
    constexpr int N = 16 / sizeof(T), T_WG = TPR > kThreads ? TPR : kThreads, RPW = T_WG / TPR;
    __shared__ F buf[2][TPR > 64 ? TPR / 64 : 1];
    __shared__ float join[RPW > 1 ? RPW * TPR * V * N : 1];
    const int t = threadIdx.x % TPR;
    float dw[V][N] = {};
    for (long long r0 = (long long)blockIdx.x * RPW; r0 < a.rows; r0 += (long long)gridDim.x * RPW) {
        const long long row = r0 + threadIdx.x / TPR;
        const bool live = row < a.rows;
        float h[V][N], g[V][N];
        F ss = 0, sg = 0;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c = (v * TPR + t) * N, n = live ? a.cols - c : 0;
            float w[N];
            load_n<N>((const T*)a.x + row * a.cols + c, n, h[v]);
            load_n<N>((const T*)a.g + row * a.cols + c, a.g ? n : 0, g[v]);
            load_w<N, T>(a, c, n, w);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                ss += (F)h[v][i] * h[v][i];
                sg += (F)g[v][i] * w[i] * h[v][i];
            }
        }
        auto add = [](F p, F q) { return p + q; };
        ss = row_reduce<TPR>(ss, buf[0], add);
        sg = row_reduce<TPR>(sg, buf[1], add);
        const F rstd2 = (F)1 / (ss / (F)a.cols + (F)a.eps), rstd = sqrt(rstd2), k = rstd2 * sg / (F)a.cols;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c = (v * TPR + t) * N, n = live ? a.cols - c : 0;
            float w[N], gh[N], d[N];
            load_w<N, T>(a, c, n, w);
            load_n<N>((const T*)a.gh + row * a.cols + c, a.gh ? n : 0, gh);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                d[i] = (float)(rstd * ((F)g[v][i] * w[i] - h[v][i] * k) + gh[i]);
                dw[v][i] += g[v][i] * (float)(h[v][i] * rstd);
            }
            if (n > 0) store_n<N>((T*)a.y + row * a.cols + c, n, d);
        }
        if constexpr (TPR > 64) __syncthreads();
    }
    if (!a.part) return;
    float* part = a.part + (long long)blockIdx.x * a.cols;
    if constexpr (RPW > 1) {             // the rows of a workgroup join before they leave it
        constexpr int L = TPR * V * N;
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int i = 0; i < N; ++i) join[(threadIdx.x / TPR) * L + (v * TPR + t) * N + i] = dw[v][i];
        __syncthreads();
        for (int c = threadIdx.x; c < a.cols; c += T_WG) {
            float s = 0.0f;
            for (int k = 0; k < RPW; ++k) s += join[k * L + c];
            part[c] = s;
        }
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c = (v * TPR + t) * N;
            if (c < a.cols) store_n<N>(part + c, a.cols - c, dw[v]);
        }
    }
}

// dw[c] = sum of n partial rows, four threads a column, joined in a fixed order
__global__ __launch_bounds__(kThreads) void dw_join_kernel(const float* part, int n, int cols, float* dw32, void* dw16, int bf16) {
    __shared__ float s[4][64];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), k = threadIdx.x >> 6;
    float v = 0.0f;
    if (c < cols)
        for (int i = k; i < n; i += 4) v += part[(long long)i * cols + c];
    s[k][threadIdx.x & 63] = v;
    __syncthreads();
    if (k || c >= cols) return;
    v = (s[0][threadIdx.x] + s[1][threadIdx.x]) + (s[2][threadIdx.x] + s[3][threadIdx.x]);
    if (dw32) dw32[c] = v;
    else if (bf16) ((bf16_t*)dw16)[c] = (bf16_t)v;
    else ((f16_t*)dw16)[c] = (f16_t)v;
}

constexpr int kMaxCols = CARD_NORM_MAX_COLS;
constexpr int kBackwardGroups = 1024;      // at most so many partial rows of dw

struct Form { int tpr, v; };               // threads per row, vectors per thread: the smallest that holds a row
Form form_of(int64_t cols, int n) {
    const int64_t vecs = (cols + n - 1) / n;
    const Form all[] = {{8, 1}, {64, 1}, {64, 2}, {256, 1}, {256, 2}, {256, 4}, {1024, 2}, {1024, 4}, {1024, 8}, {1024, 16}};
    for (const Form& f : all)
        if ((int64_t)f.tpr * f.v >= vecs) return f;
    return {0, 0};
}
long long groups(const Form& f, int64_t rows, long long most) {
    const long long rpw = f.tpr < kThreads ? kThreads / f.tpr : 1, g = (rows + rpw - 1) / rpw;
    return g < most ? g : most;
}

template <typename T, bool Q> int forward(const NormArgs& a, hipStream_t st) {
    constexpr int N = 16 / sizeof(T);
    const Form f = form_of(a.cols, N);
    const unsigned grid = (unsigned)groups(f, a.rows, 1 << 20);
#define CARD_NORM_CASE(TPR, V) \
    if (f.tpr == TPR && f.v == V) rms_norm_kernel<T, TPR, V, Q><<<grid, TPR > kThreads ? TPR : kThreads, 0, st>>>(a)
    CARD_NORM_CASE(8, 1); CARD_NORM_CASE(64, 1); CARD_NORM_CASE(64, 2); CARD_NORM_CASE(256, 1); CARD_NORM_CASE(256, 2);
    CARD_NORM_CASE(256, 4); CARD_NORM_CASE(1024, 2); CARD_NORM_CASE(1024, 4); CARD_NORM_CASE(1024, 8);
    if constexpr (sizeof(T) == 4) CARD_NORM_CASE(1024, 16);
#undef CARD_NORM_CASE
    HIP_TRY(hipGetLastError());
    return CARD_OK;
}

template <typename T> int backward(const NormArgs& a, hipStream_t st) {
    constexpr int N = 16 / sizeof(T);
    const Form f = form_of(a.cols, N);
    const unsigned grid = (unsigned)groups(f, a.rows, kBackwardGroups);
#define CARD_NORM_CASE(F, TPR, V) \
    if (f.tpr == TPR && f.v == V) rms_norm_backward_kernel<T, F, TPR, V><<<grid, TPR > kThreads ? TPR : kThreads, 0, st>>>(a)
    CARD_NORM_CASE(double, 8, 1); CARD_NORM_CASE(float, 64, 1); CARD_NORM_CASE(float, 64, 2); CARD_NORM_CASE(float, 256, 1);
    CARD_NORM_CASE(float, 256, 2); CARD_NORM_CASE(float, 256, 4); CARD_NORM_CASE(float, 1024, 2); CARD_NORM_CASE(float, 1024, 4);
    CARD_NORM_CASE(float, 1024, 8);
    if constexpr (sizeof(T) == 4) CARD_NORM_CASE(float, 1024, 16);
#undef CARD_NORM_CASE
    HIP_TRY(hipGetLastError());
    return CARD_OK;
}

int check(const char* who, int32_t dtype, int32_t w_dtype, int64_t rows, int64_t cols, double eps) {
    if (dtype != CARD_DTYPE_F32 && dtype != CARD_DTYPE_BF16 && dtype != CARD_DTYPE_F16)
        return card_fail(CARD_E_INVALID, "%s: dtype %d is none of CARD_DTYPE_F32, _BF16, _F16", who, dtype);
    if (w_dtype != dtype && w_dtype != CARD_DTYPE_F32)
        return card_fail(CARD_E_INVALID, "%s: weight dtype %d is neither CARD_DTYPE_F32 nor the rows' type %d", who, w_dtype, dtype);
    if (rows < 0 || cols < 1) return card_fail(CARD_E_INVALID, "%s: rows=%lld < 0 or cols=%lld < 1", who, (long long)rows, (long long)cols);
    if (cols > kMaxCols) return card_fail(CARD_E_UNSUPPORTED, "%s: cols=%lld > %d", who, (long long)cols, kMaxCols);
    if (rows > INT64_MAX / 8 / cols) return card_fail(CARD_E_INVALID, "%s: more bytes than 63 bits count", who);
    if (!(eps >= 0.0) || isinf(eps)) return card_fail(CARD_E_INVALID, "%s: eps=%g is not a finite number >= 0", who, eps);
    return CARD_OK;
}

}  // namespace

extern "C" CARD_API int card_rms_norm(const void* x, const void* residual, const void* weight, int32_t dtype, int32_t weight_dtype,
                                      int64_t rows, int64_t cols, double eps, void* h, void* y, int32_t y_dtype, float* scale,
                                      void* stream) {
    const int rc = check("card_rms_norm", dtype, weight_dtype, rows, cols, eps);
    if (rc != CARD_OK) return rc;
    if (y_dtype != dtype && y_dtype != CARD_DTYPE_E4M3)
        return card_fail(CARD_E_INVALID, "card_rms_norm: y_dtype %d is neither the rows' type %d nor CARD_DTYPE_E4M3", y_dtype, dtype);
    if (rows == 0) return CARD_OK;
    if (!x || !y) return card_fail(CARD_E_INVALID, "card_rms_norm: null x / y");
    if ((residual == nullptr) != (h == nullptr)) return card_fail(CARD_E_INVALID, "card_rms_norm: residual and h come together");
    if ((scale != nullptr) != (y_dtype == CARD_DTYPE_E4M3)) return card_fail(CARD_E_INVALID, "card_rms_norm: scale goes with y_dtype CARD_DTYPE_E4M3");
    NormArgs a;
    memset(&a, 0, sizeof(a));
    a.x = x; a.residual = residual; a.w = weight; a.h = h; a.y = y; a.scale = scale;
    a.rows = rows; a.cols = (int)cols; a.w_f32 = weight_dtype == CARD_DTYPE_F32; a.eps = (float)eps;
    hipStream_t st = (hipStream_t)stream;
    if (scale) return dtype == CARD_DTYPE_F32 ? forward<float, true>(a, st) : dtype == CARD_DTYPE_BF16 ? forward<bf16_t, true>(a, st) : forward<f16_t, true>(a, st);
    return dtype == CARD_DTYPE_F32 ? forward<float, false>(a, st) : dtype == CARD_DTYPE_BF16 ? forward<bf16_t, false>(a, st) : forward<f16_t, false>(a, st);
}

extern "C" CARD_API int card_rms_norm_backward_workspace_bytes(int32_t dtype, int64_t rows, int64_t cols, uint64_t* bytes) {
    const int rc = check("card_rms_norm_backward_workspace_bytes", dtype, dtype, rows, cols, 0.0);
    if (rc != CARD_OK) return rc;
    if (!bytes) return card_fail(CARD_E_INVALID, "card_rms_norm_backward_workspace_bytes: null argument");
    *bytes = (uint64_t)groups(form_of(cols, 16 / (int)card_dtype_bytes(dtype)), rows, kBackwardGroups) * (uint64_t)cols * sizeof(float);
    return CARD_OK;
}

extern "C" CARD_API int card_rms_norm_backward(const void* h, const void* weight, const void* g, const void* gh, int32_t dtype,
                                               int32_t weight_dtype, int64_t rows, int64_t cols, double eps, void* dx, void* dweight,
                                               void* workspace, uint64_t workspace_bytes, void* stream) {
    const char* who = "card_rms_norm_backward";
    const int rc = check(who, dtype, weight_dtype, rows, cols, eps);
    if (rc != CARD_OK) return rc;
    if (rows > 0 && (!h || !dx)) return card_fail(CARD_E_INVALID, "%s: null h / dx", who);
    if (dweight && !weight) return card_fail(CARD_E_INVALID, "%s: dweight without a weight", who);
    const int n = (int)groups(form_of(cols, 16 / (int)card_dtype_bytes(dtype)), rows, kBackwardGroups);
    if (dweight && rows > 0 && (!workspace || workspace_bytes < (uint64_t)n * (uint64_t)cols * sizeof(float)))
        return card_fail(CARD_E_INVALID, "%s: workspace of %llu bytes, need %llu", who, (unsigned long long)workspace_bytes,
                         (unsigned long long)((uint64_t)n * (uint64_t)cols * sizeof(float)));
    if (dweight && ((uintptr_t)workspace & 15)) return card_fail(CARD_E_INVALID, "%s: workspace is not 16-byte aligned", who);
    hipStream_t st = (hipStream_t)stream;
    if (rows > 0) {
        NormArgs a;
        memset(&a, 0, sizeof(a));
        a.x = h; a.w = weight; a.y = dx; a.g = g; a.gh = gh; a.rows = rows; a.cols = (int)cols;
        a.w_f32 = weight_dtype == CARD_DTYPE_F32; a.eps = (float)eps; a.part = dweight ? (float*)workspace : nullptr;
        const int e = dtype == CARD_DTYPE_F32 ? backward<float>(a, st) : dtype == CARD_DTYPE_BF16 ? backward<bf16_t>(a, st) : backward<f16_t>(a, st);
        if (e != CARD_OK) return e;
    }
    if (dweight) {
        const bool f32 = weight_dtype == CARD_DTYPE_F32;
        dw_join_kernel<<<(unsigned)((cols + 63) / 64), kThreads, 0, st>>>((const float*)workspace, n, (int)cols, f32 ? (float*)dweight : nullptr,
                                                                         f32 ? nullptr : dweight, weight_dtype == CARD_DTYPE_BF16);
        HIP_TRY(hipGetLastError());
    }
    return CARD_OK;
}
