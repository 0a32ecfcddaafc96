// card_dropout.hip - dropout whose mask is a function of (seed, element, draw) and is never stored.
//
//   y[r, z, c] = residual[r, z, c] + keep(e) * x[r, c] / (1 - p),   e = elem_offset + ((r * n_z + z) * cols + c)
//   dx[r, c]   = sum over z of keep(e) * g[r, z, c] / (1 - p)       (the residual's gradient is g itself)
//
// Backward makes the same mask again from the same numbers: nothing of the forward pass is kept but the seed.
#include "card_layers.h"

using namespace card;

int drop_rule(const char* who, double p, uint64_t seed, uint64_t elem_offset, const uint64_t* state, int32_t draw, DropRule* d) {
    if (!(p >= 0.0 && p <= 1.0)) return card_fail(CARD_E_INVALID, "%s: p=%g outside [0, 1]", who, p);
    if (draw < 0) return card_fail(CARD_E_INVALID, "%s: draw=%d < 0", who, draw);
    if (elem_offset >> 63) return card_fail(CARD_E_INVALID, "%s: elem_offset beyond 2^63", who);
    const double t = nearbyint(p * 4294967296.0);
    d->seed = seed; d->elem_offset = elem_offset; d->state = (const unsigned long long*)state; d->draw = (uint32_t)draw;
    d->none = t >= 4294967296.0;
    d->threshold = d->none ? 0xFFFFFFFFu : (uint32_t)t;
    d->scale = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.0f;
    return CARD_OK;
}

namespace {

constexpr int kThreads = 256;

// n / d for 0 <= n < 2^31 by a multiply and a shift (n + n 2^-32 m' never passes 32 bits); 64-bit division beyond
struct Divisor {
    long long d;
    uint32_t m, s;
    __host__ void set(long long by) {
        d = by;
        s = 0;
        while (s < 31 && (1ll << s) < by) ++s;
        m = by < 1ll << 31 ? (uint32_t)(((1ull << 32) * ((1ull << s) - (unsigned long long)by)) / (unsigned long long)by + 1) : 0;
    }
    __device__ __forceinline__ long long of(long long n, bool small) const {
        return small ? (long long)((__umulhi(m, (uint32_t)n) + (uint32_t)n) >> s) : n / d;
    }
};

struct Shape {
    long long cols;        // of a row of x
    long long total;       // elements of the output: rows * n_z * cols
    long long rows;
    int n_z;
    int small;             // every index is below 2^31
    Divisor by_cols, by_nz;
};

// One thread per 16 bytes of the output that begin with a whole block of the generator, wherever that is in memory: every
// block of four words is made once.  n_z > 1: the thread's first element tells row and column, and only where a row ends
// within the thread's elements are they taken one by one.
template <typename T, bool STREAM>
__global__ __launch_bounds__(kThreads) void dropout_kernel(const Shape s, const DropRule d, const T* x, const T* residual, T* out) {
    constexpr int N = 16 / sizeof(T);
    const long long id = (long long)blockIdx.x * kThreads + threadIdx.x;
    unsigned long long seed, off;
    drop_key(d, seed, off);
    const int lead = (int)(off % N);                 // elements ahead of the tensor in its first block's vector
    const long long at = id * N - lead;
    const int from = at < 0 ? lead : 0, n = s.total - at < N ? (int)(s.total - at) : N;          // elements from ... n - 1 are the thread's
    if (n <= from) return;
    float v[N], r[N];
    const bool whole = from == 0 && n == N;
    if (s.n_z == 1) {
        if (whole) {
            load_n<N, STREAM>(x + at, N, v);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = i >= from && i < n ? (float)x[at + i] : 0.0f;
        }
    } else {
        const long long rz = s.by_cols.of(at + from, s.small), c = at + from - rz * s.cols, row = s.by_nz.of(rz, s.small);
        if (whole && c + N <= s.cols) {
            load_n<N>(x + row * s.cols + c, N, v);
        } else if (whole && s.cols >= N) {           // one row ends among the elements
            const int k = (int)(s.cols - c);
            const T *p = x + row * s.cols + c, *q = x + s.by_nz.of(rz + 1, s.small) * s.cols - k;
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = (float)*(i < k ? p + i : q + i);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                v[i] = 0.0f;
                if (i >= from && i < n) {
                    const long long q = s.by_cols.of(at + i, s.small);
                    v[i] = (float)x[s.by_nz.of(q, s.small) * s.cols + (at + i - q * s.cols)];
                }
            }
        }
    }
    if (residual) {
        if (whole) {
            load_n<N, STREAM>(residual + at, N, r);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) r[i] = i >= from && i < n ? (float)residual[at + i] : 0.0f;
        }
    }
    drop<N>(d, seed, (off - (unsigned long long)lead + (unsigned long long)(id * N)) >> 2, v);
    if (residual) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += r[i];
    }
    if (whole) {
        store_n<N>(out + at, N, v);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i >= from && i < n) out[at + i] = (T)v[i];
    }
}

// n_z > 1: lanes_z threads of a workgroup share 16 bytes of dx, each takes every lanes_z-th mask, and their sums are joined in
// a fixed order.
template <typename T>
__global__ __launch_bounds__(kThreads) void dropout_backward_kernel(const Shape s, const Divisor by_chunks, const DropRule d, const T* g, T* dx, int lanes_z) {
    constexpr int N = 16 / sizeof(T);
    __shared__ float part[kThreads][N + 1];
    const int per_wg = kThreads / lanes_z, sub = threadIdx.x / per_wg;
    const long long id = (long long)blockIdx.x * per_wg + threadIdx.x % per_wg;
    const bool live = id < s.rows * by_chunks.d;
    unsigned long long seed, off;
    drop_key(d, seed, off);
    float sum[N] = {};
    const long long row = live ? by_chunks.of(id, s.small) : 0, c = live ? (id - row * by_chunks.d) * N : 0, n = s.cols - c;
    if (live) {
        for (int z = sub; z < s.n_z; z += lanes_z) {
            const long long at = (row * s.n_z + z) * s.cols + c;
            float v[N];
            load_n<N>(g + at, n, v);
            const uint32_t m = keep_bits<N>(d, seed, off + (unsigned long long)at, n < N ? (int)n : N);
#pragma unroll
            for (int i = 0; i < N; ++i) sum[i] += (m >> i) & 1 ? v[i] : 0.0f;
        }
    }
    if (lanes_z > 1) {
#pragma unroll
        for (int i = 0; i < N; ++i) part[threadIdx.x][i] = sum[i];
        __syncthreads();
        if (sub == 0)
            for (int k = 1; k < lanes_z; ++k)
#pragma unroll
                for (int i = 0; i < N; ++i) sum[i] += part[threadIdx.x + k * per_wg][i];
    }
    if (!live || sub) return;
#pragma unroll
    for (int i = 0; i < N; ++i) sum[i] *= d.scale;
    store_n<N>(dx + row * s.cols + c, n, sum);
}

int shape_of(const char* who, int32_t dtype, int64_t rows, int64_t cols, int32_t n_z, Shape* s) {
    const int64_t eb = card_dtype_bytes(dtype);
    if (dtype == CARD_DTYPE_E4M3 || !eb) return card_fail(CARD_E_INVALID, "%s: dtype %d is none of CARD_DTYPE_F32, _BF16, _F16", who, dtype);
    if (rows < 0 || cols < 0) return card_fail(CARD_E_INVALID, "%s: rows=%lld or cols=%lld < 0", who, (long long)rows, (long long)cols);
    if (n_z < 1) return card_fail(CARD_E_INVALID, "%s: n_z=%d < 1", who, n_z);
    int64_t all;
    if (__builtin_mul_overflow(rows, cols, &all) || __builtin_mul_overflow(all, (int64_t)n_z * eb, &all))
        return card_fail(CARD_E_INVALID, "%s: more bytes than 63 bits count", who);
    s->cols = cols; s->rows = rows; s->n_z = n_z; s->total = rows * cols * n_z;
    s->small = s->total < (1ll << 31) - 64;
    s->by_cols.set(cols > 0 ? cols : 1);
    s->by_nz.set(n_z);
    // a launch has fewer than 2^32 threads, and the last workgroup is rounded up
    if (all / 16 > (1ll << 32) - 4 * kThreads) return card_fail(CARD_E_UNSUPPORTED, "%s: more than 2^24 workgroups (16 bytes a thread)", who);
    return CARD_OK;
}

template <typename T> int forward(const Shape& s, const DropRule& d, const void* x, const void* residual, void* out, hipStream_t stream) {
    constexpr int N = 16 / sizeof(T);
    const bool past = (s.total * (residual ? 2 : 1) + s.rows * s.cols) * (long long)sizeof(T) > kStreamBytes;
    // as many vectors as the output has, and one more where the first one begins ahead of it
    const long long vectors = s.total / N + 2;
    const unsigned grid = (unsigned)((vectors + kThreads - 1) / kThreads);
    if (past) dropout_kernel<T, true><<<grid, kThreads, 0, stream>>>(s, d, (const T*)x, (const T*)residual, (T*)out);
    else dropout_kernel<T, false><<<grid, kThreads, 0, stream>>>(s, d, (const T*)x, (const T*)residual, (T*)out);
    HIP_TRY(hipGetLastError());
    return CARD_OK;
}

template <typename T> int backward(const Shape& s, const DropRule& d, const void* g, void* dx, hipStream_t stream) {
    if (s.n_z == 1) return forward<T>(s, d, g, nullptr, dx, stream);
    constexpr int N = 16 / sizeof(T);
    Divisor by_chunks;
    by_chunks.set((s.cols + N - 1) / N);
    const long long chunks = s.rows * by_chunks.d;
    // threads share a vector's masks until 2048 waves are there, eight to a CU (16 x 4096 bf16, 64 masks: one thread each 48 us,
    // up to 1024 waves 9.3, 2048 7.1, 8192 10.5; 64 x 100 fp32, 100 masks: 30 us and 5.5)
    int lanes = 1;
    while (lanes < 64 && 2 * lanes <= s.n_z && chunks * lanes < 1 << 17) lanes *= 2;
    const long long per_wg = kThreads / lanes, grid = (chunks + per_wg - 1) / per_wg;
    if (grid >= 1 << 24) return card_fail(CARD_E_UNSUPPORTED, "card_dropout_backward: more than 2^24 workgroups");
    dropout_backward_kernel<T><<<(unsigned)grid, kThreads, 0, stream>>>(s, by_chunks, d, (const T*)g, (T*)dx, lanes);
    HIP_TRY(hipGetLastError());
    return CARD_OK;
}

}  // namespace

extern "C" CARD_API int card_dropout(const void* x, const void* residual, void* out, int32_t dtype, int64_t rows, int64_t cols,
                                     int32_t n_z, double p, uint64_t seed, uint64_t elem_offset, const uint64_t* state,
                                     int32_t draw, void* stream) {
    Shape s;
    DropRule d;
    int rc = shape_of("card_dropout", dtype, rows, cols, n_z, &s);
    if (rc == CARD_OK) rc = drop_rule("card_dropout", p, seed, elem_offset, state, draw, &d);
    if (rc != CARD_OK || s.total == 0) return rc;
    if (!x || !out) return card_fail(CARD_E_INVALID, "card_dropout: null x / out");
    hipStream_t st = (hipStream_t)stream;
    return dtype == CARD_DTYPE_F32 ? forward<float>(s, d, x, residual, out, st)
         : dtype == CARD_DTYPE_BF16 ? forward<bf16_t>(s, d, x, residual, out, st) : forward<f16_t>(s, d, x, residual, out, st);
}

extern "C" CARD_API int card_dropout_backward(const void* g, void* dx, int32_t dtype, int64_t rows, int64_t cols, int32_t n_z,
                                              double p, uint64_t seed, uint64_t elem_offset, const uint64_t* state, int32_t draw,
                                              void* stream) {
    Shape s;
    DropRule d;
    int rc = shape_of("card_dropout_backward", dtype, rows, cols, n_z, &s);
    if (rc == CARD_OK) rc = drop_rule("card_dropout_backward", p, seed, elem_offset, state, draw, &d);
    if (rc != CARD_OK || s.total == 0) return rc;
    if (!g || !dx) return card_fail(CARD_E_INVALID, "card_dropout_backward: null g / dx");
    hipStream_t st = (hipStream_t)stream;
    return dtype == CARD_DTYPE_F32 ? backward<float>(s, d, g, dx, st)
         : dtype == CARD_DTYPE_BF16 ? backward<bf16_t>(s, d, g, dx, st) : backward<f16_t>(s, d, g, dx, st);
}
