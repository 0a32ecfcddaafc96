// card_norm.hip - root-mean-square norm of rows, with the residual's addition before it and 8 bits after it.
//
//   h = x + residual,  y = h * rstd * w,  rstd = 1 / sqrt(mean(h^2) + eps)
//   8 bits: amax = max |y| of the row, scale = max(amax / 448, 2^-140), q = e4m3(y / scale)     (y itself is never stored)
//   backward, from the h that forward stored:  gw = g * w,  dx = rstd * (gw - h * rstd^2 * mean(gw * h)) + gh,
//   dw = sum over rows of g * h * rstd;  the residual's gradient is dx.
//
// Everything between a load and a store is 32 bits (rows of at most 8 vectors: 64 bits in backward, see there); h and y are
// rounded once, and y comes from the h that is not rounded yet.
//
// What bounds it is memory: a row is read once and lives in registers, V vectors of 16 bytes in each thread of a workgroup
// of as many waves as the row needs (up to 64 vectors: 8, 16, 32 or 64 lanes).  A workgroup walks over rows with the weight in
// registers and asks for the next row before it joins the sums of this one, so loads are on their way all the time.  Long
// rows do not fit wholly: forward spills 14 to 87 registers to scratch where rows pass 64 KB (fp32 without e4m3: 128 KB), backward
// 18 for 8193 to 16384 columns in 16 bits.
// 8192 x 6144 bf16 with residual: forward 60 us (6.7 TB/s), backward 68 us (6.0 TB/s) and 4 us to join dw; 8192 x 4096 to e4m3
// 44 us back to back (5.3 TB/s); one row of 4096 2.5 us.  A large copy reaches 5.5 TB/s on this card.
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
    bool stream;                // x, residual, g and gh are read past the caches
    float eps;
    // backward
    const void* g;              // NULL: zeros
    const void* gh;             // NULL: zeros
    float* part;                // (workgroups, cols) partial dw, or NULL
};

__device__ __forceinline__ float max_nan(float a, float b) {          // for values >= 0: their bits order them, NaN above all
    return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b)));
}

// v of the lane o away in the exchange that makes 2 o lanes alike once o are: quads by quad_perm, 8 and 16 lanes by mirrors,
// 32 and 64 by swapping rows of lanes -- all on the vector unit, where a shuffle through LDS takes some 60 cycles a step
template <int O> __device__ __forceinline__ float partner(float v) {
    const int i = __builtin_bit_cast(int, v);
    if constexpr (O == 1) return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(i, 0xB1, 0xF, 0xF, true));
    else if constexpr (O == 2) return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(i, 0x4E, 0xF, 0xF, true));
    else if constexpr (O == 4) return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(i, 0x141, 0xF, 0xF, true));
    else return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(i, 0x140, 0xF, 0xF, true));
}
// the same value in all lanes of each group of L: op over the group
template <int L, typename Op> __device__ __forceinline__ float lanes_reduce(float v, Op op) {
    v = op(v, partner<1>(v));
    v = op(v, partner<2>(v));
    v = op(v, partner<4>(v));
    if constexpr (L >= 16) v = op(v, partner<8>(v));
    if constexpr (L >= 32) {
        const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = op(__uint_as_float(p[0]), __uint_as_float(p[1]));
    }
    if constexpr (L >= 64) {
        const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = op(__uint_as_float(p[0]), __uint_as_float(p[1]));
    }
    return v;
}
template <int L, typename Op> __device__ __forceinline__ double lanes_reduce(double v, Op op) {
#pragma unroll
    for (int o = 1; o < L; o <<= 1) v = op(v, __shfl_xor(v, o, 64));
    return v;
}
// op over a workgroup's waves, whose values are in `buf` behind the barrier; absent waves hold 0 (clear_buf)
template <typename Op> __device__ __forceinline__ float waves_reduce(const float* buf, Op op) {
    return lanes_reduce<16>(buf[threadIdx.x & 15], op);
}
// all-reduce over the threads of a row: L lanes of a wave, or (L = 0) the workgroup through `buf`, 16 floats that are not
// written again before another barrier
template <int L, typename Op> __device__ __forceinline__ float row_reduce(float v, float* buf, Op op) {
    v = lanes_reduce<L ? L : 64>(v, op);
    if constexpr (L == 0) {
        if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
        __syncthreads();
        v = waves_reduce(buf, op);
    }
    return v;
}
template <int L, int K> __device__ __forceinline__ void clear_buf(float (&buf)[K]) {
    if constexpr (L == 0) {
        if (threadIdx.x < K) buf[threadIdx.x] = 0.0f;          // a workgroup has K threads at least
        __syncthreads();
    }
}

// a thread's vectors of one row as they lie in memory
template <typename T, int V, bool STREAM> struct RowRaw {
    typename Vec<T, 16 / sizeof(T)>::type v[V];
    __device__ __forceinline__ void load(const T* row, int cols, int t, int threads, bool live) {
        constexpr int N = 16 / sizeof(T);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const int c = (k * threads + t) * N, n = live ? cols - c : 0;
            if (n >= N) {
                v[k] = load_vec<STREAM, N>(row + c);
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) v[k][i] = i < n ? row[c + i] : (T)0.0f;
            }
        }
    }
};

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

// L lanes per row (0: the workgroup), V vectors per thread
template <typename T, int L, int V, bool Q, bool STREAM>
__global__ __launch_bounds__(L ? kThreads : 1024) void rms_norm_kernel(const NormArgs a) {
    constexpr int N = 16 / sizeof(T);
    constexpr bool kAhead = V <= 2;                       // longer rows fill the registers by themselves
    __shared__ __align__(16) float bufs[64];
    float(*const buf)[2][16] = (float(*)[2][16])bufs;
    clear_buf<L>(bufs);
    const int threads = L ? L : blockDim.x, t = L ? threadIdx.x % L : threadIdx.x, rpw = L ? kThreads / L : 1;
    const long long step = (long long)gridDim.x * rpw;
    long long row = (long long)blockIdx.x * rpw + (L ? threadIdx.x / L : 0);
    const long long last = L ? (a.rows + rpw - 1) / rpw * rpw : a.rows;          // all lanes of a wave take the same number of turns
    float w[V][N];
    if constexpr (kAhead) {
#pragma unroll
        for (int v = 0; v < V; ++v) load_w<N, T>(a, (v * threads + t) * N, a.cols - (v * threads + t) * N, w[v]);
    }
    RowRaw<T, V, STREAM> x, r;
    auto fetch = [&](long long at) {
        x.load((const T*)a.x + at * a.cols, a.cols, t, threads, at < a.rows);
        if (a.residual) r.load((const T*)a.residual + at * a.cols, a.cols, t, threads, at < a.rows);
    };
    if (kAhead && row < last) fetch(row);
    for (int turn = 0; row < last; row += step, turn ^= 1) {
        const bool live = row < a.rows;
        float h[V][N];
        float ss = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c = (v * threads + t) * N, n = live ? a.cols - c : 0;
            if constexpr (kAhead) {
#pragma unroll
                for (int i = 0; i < N; ++i) h[v][i] = (float)x.v[v][i];
            } else {
                load_n<N>((const T*)a.x + row * a.cols + c, n, h[v]);
            }
            if (a.residual) {
                float rv[N];
                if constexpr (kAhead) {
#pragma unroll
                    for (int i = 0; i < N; ++i) rv[i] = (float)r.v[v][i];
                } else {
                    load_n<N>((const T*)a.residual + row * a.cols + c, n, rv);
                }
#pragma unroll
                for (int i = 0; i < N; ++i) h[v][i] += rv[i];
                if (n > 0) store_n<N>((T*)a.h + row * a.cols + c, n, h[v]);
            }
#pragma unroll
            for (int i = 0; i < N; ++i) ss += h[v][i] * h[v][i];
        }
        if (kAhead && row + step < last) fetch(row + step);
        ss = row_reduce<L>(ss, buf[turn][0], [](float p, float q) { return p + q; });
        const float rstd = 1.0f / sqrtf(ss / (float)a.cols + a.eps);
        float amax = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c = (v * threads + t) * N, n = live ? a.cols - c : 0;
            if constexpr (!kAhead) load_w<N, T>(a, c, n, w[v]);
#pragma unroll
            for (int i = 0; i < N; ++i) h[v][i] = h[v][i] * rstd * w[v][i];
            if constexpr (Q) {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (i < n) amax = max_nan(amax, fabsf(h[v][i]));
            } else {
                if (n > 0) store_n<N>((T*)a.y + row * a.cols + c, n, h[v]);
            }
        }
        if constexpr (Q) {
            amax = row_reduce<L>(amax, buf[turn][1], max_nan);
            // scale is 2^-140 at least, which a float holds to 2^-10 and where the smallest of them, 2^-149, is still a number of 8
            // bits.  448 / amax passes the largest float in rows below 1.4e-36: those are lifted by 2^100 first, which is exact, and
            // divided by the scale as it was rounded.  (A row of zeros has scale 0; NaN stays NaN.)
            const float scale = amax > 0.0f ? fmaxf(amax / kE4m3Max, 0x1p-140f) : amax;
            float inv = kE4m3Max / amax;
            if (amax < 1.4e-36f) {
                inv = amax > 0.0f ? 1.0f / (scale * 0x1p100f) : 0.0f;
#pragma unroll
                for (int v = 0; v < V; ++v)
#pragma unroll
                    for (int i = 0; i < N; ++i) h[v][i] *= 0x1p100f;
            }
            if (live && t == 0) a.scale[row] = scale;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int c = (v * threads + t) * N, n = live ? a.cols - c : 0;
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
    }
}

// Six waves to a SIMD (80 registers) are worth more than the last registers: 40000 x 1000 bf16 71 us against 89.  The 64-bit form
// (90 registers in fp32, 120 in 16 bits) and the one of two vectors a thread (106 and 128) run five and four.
// F: in rows of a few columns the two terms of dx all but cancel (at one column to eps * rstd^2 of either), so there the
// row's numbers and the difference are formed in 64 bits.
template <typename T, typename F, int L, int V, bool STREAM>
__global__ __launch_bounds__(L ? kThreads : 1024, V == 1 && sizeof(F) == 4 ? 6 : 4) void rms_norm_backward_kernel(const NormArgs a) {
    constexpr int N = 16 / sizeof(T), RPW = L ? kThreads / L : 1;
    static_assert(V <= 2, "longer rows: rms_norm_backward_long_kernel");
    __shared__ __align__(16) float bufs[64];
    float(*const buf)[2][16] = (float(*)[2][16])bufs;
    clear_buf<L>(bufs);
    __shared__ float join[L ? RPW * L * V * N : 1];
    const int threads = L ? L : blockDim.x, t = L ? threadIdx.x % L : threadIdx.x;
    const long long step = (long long)gridDim.x * RPW;
    long long row = (long long)blockIdx.x * RPW + (L ? threadIdx.x / L : 0);
    const long long last = L ? (a.rows + RPW - 1) / RPW * RPW : a.rows;
    float w[V][N], dw[V][N] = {};
#pragma unroll
    for (int v = 0; v < V; ++v) load_w<N, T>(a, (v * threads + t) * N, a.cols - (v * threads + t) * N, w[v]);
    RowRaw<T, V, STREAM> rh, rg, rgh;
    auto fetch = [&](long long at) {
        rh.load((const T*)a.x + at * a.cols, a.cols, t, threads, at < a.rows);
        rg.load((const T*)a.g + at * a.cols, a.cols, t, threads, a.g && at < a.rows);
        rgh.load((const T*)a.gh + at * a.cols, a.cols, t, threads, a.gh && at < a.rows);
    };
    if (row < last) fetch(row);
    for (int turn = 0; row < last; row += step, turn ^= 1) {
        const bool live = row < a.rows;
        const RowRaw<T, V, STREAM> h = rh, g = rg, gh = rgh;
        F ss = 0, sg = 0;
#pragma unroll
        for (int v = 0; v < V; ++v) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const F hv = (F)(float)h.v[v][i];
                ss += hv * hv;
                sg += (F)(float)g.v[v][i] * w[v][i] * hv;
            }
        }
        if (row + step < last) fetch(row + step);
        auto add = [](F p, F q) { return p + q; };
        ss = lanes_reduce<L ? L : 64>(ss, add);
        sg = lanes_reduce<L ? L : 64>(sg, add);
        if constexpr (L == 0) {                           // both sums behind one barrier; the other turn's buffers are free by then
            if ((threadIdx.x & 63) == 0) {
                buf[turn][0][threadIdx.x >> 6] = ss;
                buf[turn][1][threadIdx.x >> 6] = sg;
            }
            __syncthreads();
            ss = waves_reduce(buf[turn][0], add);
            sg = waves_reduce(buf[turn][1], add);
        }
        // a place behind the last row holds zeros, whose root is infinite where eps is 0: it adds nothing to dw
        const F rstd2 = live ? (F)1 / (ss / (F)a.cols + (F)a.eps) : (F)0, rstd = sqrt(rstd2), k = rstd2 * sg / (F)a.cols;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c = (v * threads + t) * N, n = live ? a.cols - c : 0;
            float d[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float hv = (float)h.v[v][i], gv = (float)g.v[v][i];
                d[i] = (float)(rstd * ((F)gv * w[v][i] - hv * k) + (F)(float)gh.v[v][i]);
                dw[v][i] += gv * (float)(hv * rstd);
            }
            if (n > 0) store_n<N>((T*)a.y + row * a.cols + c, n, d);
        }
    }
    if (!a.part) return;
    float* part = a.part + (long long)blockIdx.x * a.cols;
    if constexpr (L != 0) {              // the rows of a workgroup join before they leave it
        constexpr int S = L * V * N;
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int i = 0; i < N; ++i) join[(threadIdx.x / L) * S + (v * L + t) * N + i] = dw[v][i];
        __syncthreads();
        for (int c = threadIdx.x; c < a.cols; c += kThreads) {
            float s = 0.0f;
            for (int k = 0; k < RPW; ++k) s += join[k * S + c];
            part[c] = s;
        }
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c = (v * threads + t) * N;
            if (c < a.cols) store_n<N>(part + c, a.cols - c, dw[v]);
        }
    }
}

// Rows of more than 2 x 1024 vectors do not stay in registers: h and g are read again (from the caches, as far as they hold
// them) once the row's sums are there, and the workgroup's partial dw lies in memory.
template <typename T>
__global__ __launch_bounds__(1024) void rms_norm_backward_long_kernel(const NormArgs a) {
    constexpr int N = 16 / sizeof(T);
    __shared__ __align__(16) float bufs[64];
    float(*const buf)[2][16] = (float(*)[2][16])bufs;
    clear_buf<0>(bufs);
    float* const part = a.part ? a.part + (long long)blockIdx.x * a.cols : nullptr;
    auto add = [](float p, float q) { return p + q; };
    int turn = 0;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
        const T *hr = (const T*)a.x + row * a.cols, *gr = (const T*)a.g + row * a.cols, *ghr = (const T*)a.gh + row * a.cols;
        float ss = 0.0f, sg = 0.0f;
#pragma unroll 2
        for (int c = threadIdx.x * N; c < a.cols; c += 1024 * N) {
            const int n = a.cols - c;
            float h[N], g[N], w[N];
            load_n<N>(hr + c, n, h);
            load_n<N>(gr + c, a.g ? n : 0, g);
            load_w<N, T>(a, c, n, w);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                ss += h[i] * h[i];
                sg += g[i] * w[i] * h[i];
            }
        }
        ss = lanes_reduce<64>(ss, add);
        sg = lanes_reduce<64>(sg, add);
        if ((threadIdx.x & 63) == 0) {
            buf[turn][0][threadIdx.x >> 6] = ss;
            buf[turn][1][threadIdx.x >> 6] = sg;
        }
        __syncthreads();
        ss = waves_reduce(buf[turn][0], add);
        sg = waves_reduce(buf[turn][1], add);
        const float rstd2 = 1.0f / (ss / (float)a.cols + a.eps), rstd = sqrtf(rstd2), k = rstd2 * sg / (float)a.cols;
#pragma unroll 2
        for (int c = threadIdx.x * N; c < a.cols; c += 1024 * N) {
            const int n = a.cols - c;
            float h[N], g[N], w[N], gh[N], d[N];
            load_n<N>(hr + c, n, h);
            load_n<N>(gr + c, a.g ? n : 0, g);
            load_n<N>(ghr + c, a.gh ? n : 0, gh);
            load_w<N, T>(a, c, n, w);
#pragma unroll
            for (int i = 0; i < N; ++i) d[i] = rstd * (g[i] * w[i] - h[i] * k) + gh[i];
            store_n<N>((T*)a.y + row * a.cols + c, n, d);
            if (part) {
                load_n<N>(part + c, row == blockIdx.x ? 0 : n, d);
#pragma unroll
                for (int i = 0; i < N; ++i) d[i] += g[i] * (h[i] * rstd);
                store_n<N>(part + c, n, d);
            }
        }
    }
}

// dw[c] = sum of n partial rows: 32 columns to a workgroup, 8 lanes of four columns, the rows over the other 128 threads;
// a fixed order throughout
constexpr int kJoinCols = 32, kJoinThreads = 1024;
__global__ __launch_bounds__(kJoinThreads) void dw_join_kernel(const float* part, int n, int cols, float* dw32, void* dw16, int bf16) {
    constexpr int R = kJoinThreads / 8;
    __shared__ float s[R][kJoinCols + 1];
    const int lane = threadIdx.x & 7, k = threadIdx.x >> 3, c = blockIdx.x * kJoinCols + lane * 4;
    float v[4] = {};
    for (int i = k; i < n; i += R) {
        float p[4];
        load_n<4>(part + (long long)i * cols + c, cols - c, p);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += p[j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) s[k][lane * 4 + j] = v[j];
    __syncthreads();
    const int col = threadIdx.x & 31, q = threadIdx.x >> 5;          // 32 threads per column, four partial sums each
    float sum = (s[q][col] + s[q + 32][col]) + (s[q + 64][col] + s[q + 96][col]);
    __syncthreads();
    s[q][col] = sum;
    __syncthreads();
    if (q || blockIdx.x * kJoinCols + col >= cols) return;
#pragma unroll
    for (int j = 1; j < 32; ++j) sum += s[j][col];
    const int o = blockIdx.x * kJoinCols + col;
    if (dw32) dw32[o] = sum;
    else if (bf16) ((bf16_t*)dw16)[o] = (bf16_t)sum;
    else ((f16_t*)dw16)[o] = (f16_t)sum;
}

constexpr int kMaxCols = CARD_NORM_MAX_COLS;
constexpr int kCus = 256;
// Waves to a CU that workgroups are launched for: what the forms of one vector a thread have registers for.  With more vectors and
// in the 64-bit form a CU holds 16 to 20, and the workgroups past those start when the first ones end.
constexpr int kForwardWaves = 32, kBackwardWaves = 24;

struct Form { int lanes, v, threads; };    // lanes per row (0: a workgroup of `threads`), vectors per thread
Form form_of(int64_t cols, int n) {
    const int vecs = (int)((cols + n - 1) / n);
    for (int lanes = 8; lanes <= 64; lanes *= 2)
        if (vecs <= lanes) return {lanes, 1, kThreads};
    int v = 1;
    while ((int64_t)v * 1024 < vecs) v *= 2;
    const int waves = (vecs + 64 * v - 1) / (64 * v);
    return {0, v, 64 * waves};
}
// workgroups that walk over the rows
long long groups(const Form& f, int64_t rows, int waves) {
    const long long rpw = f.lanes ? kThreads / f.lanes : 1, g = (rows + rpw - 1) / rpw, per_cu = waves / (f.threads / 64);
    const long long most = kCus * (per_cu > 0 ? per_cu : 1);
    return g < most ? g : most;
}

long long backward_groups(int32_t dtype, int64_t rows, int64_t cols) {
    return groups(form_of(cols, 16 / (int)card_dtype_bytes(dtype)), rows, kBackwardWaves);
}

template <typename T, bool Q> int forward(const NormArgs& a, hipStream_t st) {
    constexpr int N = 16 / sizeof(T);
    const Form f = form_of(a.cols, N);
    const unsigned grid = (unsigned)groups(f, a.rows, kForwardWaves);
#define CARD_NORM_CASE(L, V, STREAM) \
    if (f.lanes == L && f.v == V && (V > 2 || a.stream == STREAM)) rms_norm_kernel<T, L, V, Q, STREAM><<<grid, f.threads, 0, st>>>(a)
#define CARD_NORM_BOTH(L, V) CARD_NORM_CASE(L, V, false); CARD_NORM_CASE(L, V, true)
    CARD_NORM_BOTH(8, 1); CARD_NORM_BOTH(16, 1); CARD_NORM_BOTH(32, 1); CARD_NORM_BOTH(64, 1); CARD_NORM_BOTH(0, 1); CARD_NORM_BOTH(0, 2);
    CARD_NORM_CASE(0, 4, false); CARD_NORM_CASE(0, 8, false);
    if constexpr (sizeof(T) == 4) CARD_NORM_CASE(0, 16, false);
#undef CARD_NORM_BOTH
#undef CARD_NORM_CASE
    HIP_TRY(hipGetLastError());
    return CARD_OK;
}

template <typename T> int backward(const NormArgs& a, hipStream_t st) {
    constexpr int N = 16 / sizeof(T);
    const Form f = form_of(a.cols, N);
    const unsigned grid = (unsigned)backward_groups(sizeof(T) == 4 ? CARD_DTYPE_F32 : CARD_DTYPE_BF16, a.rows, a.cols);
#define CARD_NORM_CASE(F, L, V, STREAM) \
    if (f.lanes == L && f.v == V && a.stream == STREAM) rms_norm_backward_kernel<T, F, L, V, STREAM><<<grid, f.threads, 0, st>>>(a)
#define CARD_NORM_BOTH(F, L, V) CARD_NORM_CASE(F, L, V, false); CARD_NORM_CASE(F, L, V, true)
    CARD_NORM_BOTH(double, 8, 1); CARD_NORM_BOTH(float, 16, 1); CARD_NORM_BOTH(float, 32, 1); CARD_NORM_BOTH(float, 64, 1);
    CARD_NORM_BOTH(float, 0, 1); CARD_NORM_BOTH(float, 0, 2);
#undef CARD_NORM_BOTH
    if (f.v > 2) rms_norm_backward_long_kernel<T><<<grid, 1024, 0, st>>>(a);
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
    if (rows > INT64_MAX / 16 / cols) return card_fail(CARD_E_INVALID, "%s: more bytes than 63 bits count", who);
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
    const int64_t eb = card_dtype_bytes(dtype);
    a.stream = rows * cols * (eb * (residual ? 3 : 1) + (scale ? 1 : eb)) > kStreamBytes;
    hipStream_t st = (hipStream_t)stream;
    if (scale) return dtype == CARD_DTYPE_F32 ? forward<float, true>(a, st) : dtype == CARD_DTYPE_BF16 ? forward<bf16_t, true>(a, st) : forward<f16_t, true>(a, st);
    return dtype == CARD_DTYPE_F32 ? forward<float, false>(a, st) : dtype == CARD_DTYPE_BF16 ? forward<bf16_t, false>(a, st) : forward<f16_t, false>(a, st);
}

extern "C" CARD_API int card_rms_norm_backward_workspace_bytes(int32_t dtype, int64_t rows, int64_t cols, uint64_t* bytes) {
    const int rc = check("card_rms_norm_backward_workspace_bytes", dtype, dtype, rows, cols, 0.0);
    if (rc != CARD_OK) return rc;
    if (!bytes) return card_fail(CARD_E_INVALID, "card_rms_norm_backward_workspace_bytes: null argument");
    *bytes = (uint64_t)backward_groups(dtype, rows, cols) * (uint64_t)cols * sizeof(float);
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
    const int n = (int)backward_groups(dtype, rows, cols);
    if (dweight && rows > 0 && (!workspace || workspace_bytes < (uint64_t)n * (uint64_t)cols * sizeof(float)))
        return card_fail(CARD_E_INVALID, "%s: workspace of %llu bytes, need %llu", who, (unsigned long long)workspace_bytes,
                         (unsigned long long)((uint64_t)n * (uint64_t)cols * sizeof(float)));
    if (dweight && ((uintptr_t)workspace & 15)) return card_fail(CARD_E_INVALID, "%s: workspace is not 16-byte aligned", who);
    hipStream_t st = (hipStream_t)stream;
    if (rows > 0) {
        NormArgs a;
        memset(&a, 0, sizeof(a));
        a.x = h; a.w = weight; a.y = dx; a.g = g; a.gh = gh; a.rows = rows; a.cols = (int)cols;
        a.stream = rows * cols * card_dtype_bytes(dtype) * (2 + (g != nullptr) + (gh != nullptr)) > kStreamBytes;
        a.w_f32 = weight_dtype == CARD_DTYPE_F32; a.eps = (float)eps; a.part = dweight ? (float*)workspace : nullptr;
        const int e = dtype == CARD_DTYPE_F32 ? backward<float>(a, st) : dtype == CARD_DTYPE_BF16 ? backward<bf16_t>(a, st) : backward<f16_t>(a, st);
        if (e != CARD_OK) return e;
    }
    if (dweight) {
        const bool f32 = weight_dtype == CARD_DTYPE_F32;
        dw_join_kernel<<<(unsigned)((cols + kJoinCols - 1) / kJoinCols), kJoinThreads, 0, st>>>((const float*)workspace, n, (int)cols, f32 ? (float*)dweight : nullptr,
                                                                         f32 ? nullptr : dweight, weight_dtype == CARD_DTYPE_BF16);
        HIP_TRY(hipGetLastError());
    }
    return CARD_OK;
}
