// card_linear4.hip - products of few rows with 4-bit weights and a scale (and zero point) per group of columns.
//
//   y[m, o] = act(gamma[o] * (x_scale[m] * sum_k (q[o, k] - zero[o, k / group]) * scale[o, k / group] * x[m, k] + bias[o]))
//   act(v) = v > 0 ? v : slope * v
//
// The differences q - zero are small integers, exact in every type; products and sums are fp32, y is rounded once.
#include <new>

#include "card_layers.h"

using namespace card;

struct card_linear4 {
    int in, out, group, groups, device;
    int words;                 // 32-bit words of a packed row: ceil(in / 8)
    uint32_t* q;               // (out, words): nibble i of a word is column 8 * word + i
    float* scale;              // (out, groups)
    uint8_t* zero;             // (out, groups)
    float* bias;               // (out)
};

namespace {

constexpr int kThreads = 256, kRows = 8;

__global__ void pack_kernel(const uint8_t* q, int in, int words, long long n, uint32_t* out) {
    const long long id = (long long)blockIdx.x * kThreads + threadIdx.x;
    if (id >= n) return;
    const long long o = id / words;
    const int k = (int)(id - o * words) * 8;
    uint32_t w = 0;
    for (int i = 0; i < 8; ++i)
        if (k + i < in) w |= (uint32_t)(q[o * in + k + i] & 15u) << (4 * i);
    out[id] = w;
}
__global__ void side_kernel(const float* scale, const uint8_t* zero, const float* bias, long long n, int out_f, float* s, uint8_t* z, float* b) {
    const long long id = (long long)blockIdx.x * kThreads + threadIdx.x;
    if (id < n) {
        s[id] = scale[id];
        z[id] = zero ? zero[id] & 15u : 8u;
    }
    if (id < out_f) b[id] = bias ? bias[id] : 0.0f;
}

// one wave per (row o of the weights, group of columns): q = round(w / scale) + zero with scale = (max - min) / 15 over the
// group's values and zero
__global__ __launch_bounds__(kThreads) void quantize_kernel(const float* W, int in, int group, int groups, long long n, uint8_t* q,
                                                            float* scale, uint8_t* zero) {
    const long long id = (long long)blockIdx.x * (kThreads / 64) + threadIdx.x / 64;
    if (id >= n) return;
    const int lane = threadIdx.x & 63;
    const long long o = id / groups;
    const int k0 = (int)(id - o * groups) * group, k1 = k0 + group < in ? k0 + group : in;
    float lo = 0.0f, hi = 0.0f;
    for (int k = k0 + lane; k < k1; k += 64) { lo = fminf(lo, W[o * in + k]); hi = fmaxf(hi, W[o * in + k]); }
    for (int s = 1; s < 64; s <<= 1) { lo = fminf(lo, __shfl_xor(lo, s, 64)); hi = fmaxf(hi, __shfl_xor(hi, s, 64)); }
    const float sc = (hi - lo) / 15.0f, inv = sc > 0.0f ? 1.0f / sc : 0.0f;
    const float z = fminf(fmaxf(rintf(-lo * inv), 0.0f), 15.0f);
    if (lane == 0) { scale[id] = sc; zero[id] = (uint8_t)z; }
    for (int k = k0 + lane; k < k1; k += 64) q[o * in + k] = (uint8_t)fminf(fmaxf(rintf(W[o * in + k] * inv) + z, 0.0f), 15.0f);
}

struct Args {
    const uint32_t* q;
    const float* scale;
    const uint8_t* zero;
    const float* bias;
    const float* x_scale;
    const float* gamma;
    float slope;
    int in, out, group, groups, words;
    int rows;
};

__device__ __forceinline__ float e4m3_at(const uint8_t* p) { return __builtin_amdgcn_cvt_f32_fp8((int)*p, 0); }
__device__ __forceinline__ float as_float(const float* p) { return *p; }
__device__ __forceinline__ float as_float(const bf16_t* p) { return (float)*p; }
__device__ __forceinline__ float as_float(const f16_t* p) { return (float)*p; }
__device__ __forceinline__ float as_float(const uint8_t* p) { return e4m3_at(p); }

// one wave per output column and kRows rows of x
template <typename X, typename Y>
__global__ __launch_bounds__(kThreads) void linear4_kernel(const Args a, const X* x, Y* y) {
    const int o = blockIdx.x * (kThreads / 64) + threadIdx.x / 64, lane = threadIdx.x & 63, m0 = blockIdx.y * kRows;
    if (o >= a.out) return;
    float acc[kRows] = {};
    for (int w = lane; w < a.words; w += 64) {
        const uint32_t q = a.q[(long long)o * a.words + w];
        const long long g = (long long)o * a.groups + w * 8 / a.group;
        const float s = a.scale[g], z = a.zero[g];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (w * 8 + i >= a.in) break;
            const float v = ((float)((q >> (4 * i)) & 15u) - z) * s;
#pragma unroll
            for (int m = 0; m < kRows; ++m)
                if (m0 + m < a.rows) acc[m] += v * as_float(x + (long long)(m0 + m) * a.in + w * 8 + i);
        }
    }
#pragma unroll
    for (int m = 0; m < kRows; ++m)
        for (int s = 1; s < 64; s <<= 1) acc[m] += __shfl_xor(acc[m], s, 64);
    if (lane) return;
#pragma unroll
    for (int m = 0; m < kRows; ++m) {
        if (m0 + m >= a.rows) continue;
        float v = (a.x_scale ? acc[m] * a.x_scale[m0 + m] : acc[m]) + a.bias[o];
        if (a.gamma) v *= a.gamma[o];
        y[(long long)(m0 + m) * a.out + o] = (Y)(v > 0.0f ? v : v * a.slope);
    }
}

template <typename X, typename Y> int launch(const Args& a, const void* x, void* y, hipStream_t st) {
    linear4_kernel<X, Y><<<dim3((a.out + 3) / 4, (a.rows + kRows - 1) / kRows), kThreads, 0, st>>>(a, (const X*)x, (Y*)y);
    HIP_TRY(hipGetLastError());
    return CARD_OK;
}
template <typename X> int by_y(const Args& a, const void* x, void* y, int y_dtype, hipStream_t st) {
    return y_dtype == CARD_DTYPE_F32 ? launch<X, float>(a, x, y, st) : y_dtype == CARD_DTYPE_BF16 ? launch<X, bf16_t>(a, x, y, st)
                                                                                                 : launch<X, f16_t>(a, x, y, st);
}

}  // namespace

extern "C" CARD_API int card_linear4_quantize(const float* W, int32_t out_features, int32_t in_features, int32_t group, uint8_t* q,
                                              float* scale, uint8_t* zero, void* stream) {
    const char* who = "card_linear4_quantize";
    if (out_features < 1 || in_features < 1) return card_fail(CARD_E_INVALID, "%s: %d x %d features", who, out_features, in_features);
    if (group != 32 && group != 64 && group != 128) return card_fail(CARD_E_UNSUPPORTED, "%s: group=%d is none of 32, 64, 128", who, group);
    if (!W || !q || !scale || !zero) return card_fail(CARD_E_INVALID, "%s: null argument", who);
    const int groups = (in_features + group - 1) / group;
    const long long n = (long long)out_features * groups, grid = (n + kThreads / 64 - 1) / (kThreads / 64);
    if (grid > 0x7fffffff) return card_fail(CARD_E_UNSUPPORTED, "%s: more than 2^31 workgroups", who);
    quantize_kernel<<<(unsigned)grid, kThreads, 0, (hipStream_t)stream>>>(W, in_features, group, groups, n, q, scale, zero);
    HIP_TRY(hipGetLastError());
    return CARD_OK;
}

extern "C" CARD_API int card_linear4_create(const card_linear4_desc* d, void* stream, card_linear4** out) {
    const char* who = "card_linear4_create";
    if (!d || !out) return card_fail(CARD_E_INVALID, "%s: null argument", who);
    *out = nullptr;
    if (d->struct_bytes != (int32_t)sizeof(card_linear4_desc))
        return card_fail(CARD_E_INVALID, "%s: struct_bytes %d != %zu", who, d->struct_bytes, sizeof(card_linear4_desc));
    if (d->in_features < 1 || d->out_features < 1) return card_fail(CARD_E_INVALID, "%s: %d x %d features", who, d->out_features, d->in_features);
    if (d->in_features > CARD_LINEAR4_MAX_FEATURES || d->out_features > CARD_LINEAR4_MAX_FEATURES)
        return card_fail(CARD_E_UNSUPPORTED, "%s: %d x %d features, at most %d each", who, d->out_features, d->in_features, CARD_LINEAR4_MAX_FEATURES);
    if (d->group != 32 && d->group != 64 && d->group != 128)
        return card_fail(CARD_E_UNSUPPORTED, "%s: group=%d is none of 32, 64, 128", who, d->group);
    if (!d->q || !d->scale) return card_fail(CARD_E_INVALID, "%s: null q / scale", who);
    card_linear4* s = new (std::nothrow) card_linear4();
    if (!s) return card_fail(CARD_E_NOMEM, "%s: out of host memory", who);
    s->in = d->in_features; s->out = d->out_features; s->group = d->group; s->groups = (s->in + s->group - 1) / s->group;
    s->words = (s->in + 7) / 8;
    hipStream_t st = (hipStream_t)stream;
    const long long nw = (long long)s->out * s->words, ng = (long long)s->out * s->groups;
    hipError_t e = hipGetDevice(&s->device);
    if (e == hipSuccess) e = hipMalloc(&s->q, nw * sizeof(uint32_t));
    if (e == hipSuccess) e = hipMalloc(&s->scale, ng * sizeof(float));
    if (e == hipSuccess) e = hipMalloc(&s->zero, ng);
    if (e == hipSuccess) e = hipMalloc(&s->bias, s->out * sizeof(float));
    if (e == hipSuccess) {
        pack_kernel<<<(unsigned)((nw + kThreads - 1) / kThreads), kThreads, 0, st>>>(d->q, s->in, s->words, nw, s->q);
        side_kernel<<<(unsigned)((ng + kThreads - 1) / kThreads), kThreads, 0, st>>>(d->scale, d->zero, d->bias, ng, s->out, s->scale, s->zero, s->bias);
        e = hipGetLastError();
    }
    if (e != hipSuccess) {
        card_linear4_destroy(s);
        return card_fail(e == hipErrorOutOfMemory ? CARD_E_NOMEM : CARD_E_HIP, "%s: %s", who, hipGetErrorString(e));
    }
    *out = s;
    return CARD_OK;
}

extern "C" CARD_API void card_linear4_destroy(card_linear4* s) {
    if (!s) return;
    if (s->q) (void)hipFree(s->q);
    if (s->scale) (void)hipFree(s->scale);
    if (s->zero) (void)hipFree(s->zero);
    if (s->bias) (void)hipFree(s->bias);
    delete s;
}

extern "C" CARD_API int card_linear4_forward(const card_linear4* s, const void* x, int32_t x_dtype, const float* x_scale, int64_t rows,
                                             const float* gamma, float slope, void* y, int32_t y_dtype, void* stream) {
    const char* who = "card_linear4_forward";
    if (!s) return card_fail(CARD_E_INVALID, "%s: null handle", who);
    if (!card_dtype_bytes(x_dtype)) return card_fail(CARD_E_INVALID, "%s: x_dtype %d is no card_dtype", who, x_dtype);
    if (!card_dtype_bytes(y_dtype) || y_dtype == CARD_DTYPE_E4M3)
        return card_fail(CARD_E_INVALID, "%s: y_dtype %d is none of CARD_DTYPE_F32, _BF16, _F16", who, y_dtype);
    if (rows < 0) return card_fail(CARD_E_INVALID, "%s: rows=%lld < 0", who, (long long)rows);
    if (rows > CARD_LINEAR4_MAX_ROWS) return card_fail(CARD_E_UNSUPPORTED, "%s: rows=%lld > %d", who, (long long)rows, CARD_LINEAR4_MAX_ROWS);
    if (!(fabsf(slope) <= 3.0e38f)) return card_fail(CARD_E_INVALID, "%s: slope is not finite", who);
    if (rows == 0) return CARD_OK;
    if ((x_scale != nullptr) != (x_dtype == CARD_DTYPE_E4M3)) return card_fail(CARD_E_INVALID, "%s: x_scale goes with x_dtype CARD_DTYPE_E4M3", who);
    if (!x || !y) return card_fail(CARD_E_INVALID, "%s: null x / y", who);
    int device = -1;
    HIP_TRY(hipGetDevice(&device));
    if (device != s->device) return card_fail(CARD_E_INVALID, "%s: the weights are on device %d, the current device is %d", who, s->device, device);
    Args a;
    a.q = s->q; a.scale = s->scale; a.zero = s->zero; a.bias = s->bias; a.x_scale = x_scale; a.gamma = gamma; a.slope = slope;
    a.in = s->in; a.out = s->out; a.group = s->group; a.groups = s->groups; a.words = s->words; a.rows = (int)rows;
    hipStream_t st = (hipStream_t)stream;
    switch (x_dtype) {
        case CARD_DTYPE_F32: return by_y<float>(a, x, y, y_dtype, st);
        case CARD_DTYPE_BF16: return by_y<bf16_t>(a, x, y, y_dtype, st);
        case CARD_DTYPE_F16: return by_y<f16_t>(a, x, y, y_dtype, st);
        default: return by_y<uint8_t>(a, x, y, y_dtype, st);
    }
}
