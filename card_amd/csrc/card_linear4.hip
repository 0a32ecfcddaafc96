// card_linear4.hip - products of few rows with 4-bit weights and a scale (and zero point) per group of columns.
//
//   y[m, o] = act(gamma[o] * (x_scale[m] * sum_k (q[o, k] - zero[o, k / group]) * scale[o, k / group] * x[m, k] + bias[o]))
//   act(v) = v > 0 ? v : slope * v
//
// The differences q - zero are small integers, exact in every type; products and sums are fp32, y is rounded once.  Sums that are
// not finite on the way are formed again from these differences (plain_sum).
#include <new>

#include "card_layers.h"

using namespace card;

struct card_linear4 {
    int in, out, group, device;
    int blocks;                // blocks of kBlock columns: ceil(in / kBlock)
    int tiles;                 // tiles of 16 outputs: ceil(out / 16)
    uint4* q;                  // (tiles, blocks, 64): see pack_kernel
    float* scale;              // (tiles, blocks, kBlock / group, 16)
    uint8_t* zero;             // likewise
    float* bias;               // (out)
};

namespace {

constexpr int kThreads = 256, kBlock = 128;

// Weights in the order in which the matrix instruction takes them.  Of a tile of 16 outputs and a block of 128 columns lane l
// holds 16 bytes: word s has the eight values of output l % 16 at the columns 32 s + 8 (l / 16) ... + 7 of the block.  The
// value of column 2 j + h sits in the word's field j + 4 h; field 0 begins at bit 3 and field 7 wraps around.  A mask then
// leaves two neighbouring columns as the mantissas of two bf16 numbers 16 + q (bf16_of below) and three shifts give the rest.
__global__ void pack_kernel(const uint8_t* q, int in, int out_f, int blocks, long long n, uint4* out) {
    for (long long id = (long long)blockIdx.x * kThreads + threadIdx.x; id < n; id += (long long)gridDim.x * kThreads) {
        const int l = (int)(id & 63), block = (int)((id >> 6) % blocks);
        const long long o = (id >> 6) / blocks * 16 + (l & 15);
        uint32_t w[4];
        for (int s = 0; s < 4; ++s) {
            uint32_t u = 0;
            for (int i = 0; i < 8; ++i) {
                const int k = block * kBlock + 32 * s + 8 * (l >> 4) + i;
                if (o < out_f && k < in) u |= (uint32_t)(q[o * in + k] & 15u) << (4 * (i / 2 + 4 * (i & 1)));
            }
            w[s] = u << 3 | u >> 29;
        }
        out[id] = make_uint4(w[0], w[1], w[2], w[3]);
    }
}
__global__ void side_kernel(const float* scale, const uint8_t* zero, const float* bias, int group, int groups, int blocks, int out_f,
                            long long n, float* s, uint8_t* z, float* b) {
    const int per = kBlock / group;
    for (long long id = (long long)blockIdx.x * kThreads + threadIdx.x; id < n; id += (long long)gridDim.x * kThreads) {          // n >= out_f
        if (id < out_f) b[id] = bias ? bias[id] : 0.0f;
        const long long at = id >> 4, o = at / per / blocks * 16 + (id & 15), g = at % ((long long)per * blocks);
        const bool real = o < out_f && g < groups;
        s[id] = real ? scale[o * groups + g] : 0.0f;
        z[id] = real && zero ? zero[o * groups + g] & 15u : 8u;
    }
}

// one wave per (row o of the weights, group of columns): q = round(w / scale) + zero with scale = (max - min) / 15 over the
// group's values and zero.  A NaN or an infinity makes the scale NaN or infinite, and so the group: q - zero is 0 then.
__global__ __launch_bounds__(kThreads) void quantize_kernel(const float* W, int in, int group, int groups, long long n, uint8_t* q,
                                                            float* scale, uint8_t* zero) {
    const int lane = threadIdx.x & 63;
    for (long long id = (long long)blockIdx.x * (kThreads / 64) + threadIdx.x / 64; id < n; id += (long long)gridDim.x * (kThreads / 64)) {
        const long long o = id / groups;
        const int k0 = (int)(id - o * groups) * group, k1 = k0 + group < in ? k0 + group : in;
        float lo = 0.0f, hi = 0.0f;
        bool nan = false;
        for (int k = k0 + lane; k < k1; k += 64) {
            const float w = W[o * in + k];
            nan |= w != w;
            lo = fminf(lo, w);
            hi = fmaxf(hi, w);
        }
        for (int s = 1; s < 64; s <<= 1) { lo = fminf(lo, __shfl_xor(lo, s, 64)); hi = fmaxf(hi, __shfl_xor(hi, s, 64)); }
        float sc = (hi - lo) / 15.0f;
        if (isinf(sc)) sc = hi / 15.0f - lo / 15.0f;                      // the span alone may pass the largest float
        if (__any(nan)) sc = __builtin_nanf("");
        const float inv = sc > 0.0f ? 1.0f / sc : 0.0f;
        const bool tiny = isinf(inv);                                     // a scale whose reciprocal is no float: divide
        const float z = fminf(fmaxf(rintf(tiny ? -lo / sc : -lo * inv), 0.0f), 15.0f);
        if (lane == 0) { scale[id] = sc; zero[id] = (uint8_t)z; }
        for (int k = k0 + lane; k < k1; k += 64) {
            const float w = W[o * in + k];
            q[o * in + k] = (uint8_t)(isfinite(sc) ? fminf(fmaxf(rintf(tiny ? w / sc : w * inv) + z, 0.0f), 15.0f) : z);
        }
    }
}

// a launch has fewer than 2^32 threads: what prepares weights walks over them with fewer
unsigned walkers(long long workgroups) { return (unsigned)(workgroups < 1 << 20 ? workgroups : 1 << 20); }

struct Args {
    const uint4* q;
    const float* scale;
    const uint8_t* zero;
    const float* bias;
    const float* x_scale;
    const float* gamma;
    float slope;
    int in, out, blocks, tiles;
    int rows;
    int y_dtype;
    float* partial;            // (splits, rows, out): sums of a share of the columns each, or NULL: one share
    int splits;
};

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// eight 4-bit values as 16 + q, in bf16 (exponent of 16, q in mantissa bits 3-6) or fp16 (bits 6-9): no conversion, and exact.
// `sixteen` holds the two exponents and comes from sixteen_of, in a vector register: an instruction takes one literal, and
// with the mask as that one a word's pair is a single v_and_or_b32.
template <int X> __device__ __forceinline__ uint32_t sixteen_of() {
    uint32_t c;
    asm("v_mov_b32 %0, %1" : "=v"(c) : "i"(X == CARD_DTYPE_F16 ? 0x4C004C00 : 0x41804180));
    return c;
}
template <int X> __device__ __forceinline__ u32x4 ints_of(uint32_t w, uint32_t sixteen) {
    if constexpr (X == CARD_DTYPE_F16) {
        const uint32_t m = 0x03C003C0u;
        return u32x4{(__builtin_amdgcn_alignbit(w, w, 29) & m) | sixteen, ((w >> 1) & m) | sixteen, ((w >> 5) & m) | sixteen,
                     (__builtin_amdgcn_alignbit(w, w, 9) & m) | sixteen};
    } else {
        const uint32_t m = 0x00780078u;
        return u32x4{(w & m) | sixteen, ((w >> 4) & m) | sixteen, ((w >> 8) & m) | sixteen, (__builtin_amdgcn_alignbit(w, w, 12) & m) | sixteen};
    }
}
template <int X> __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (X == CARD_DTYPE_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// eight values of x as they lie in memory, and as operands: one of 16 bits each, or for fp32 three bf16 operands whose sum is
// exactly x (8 + 8 + 8 of its 24 significant bits)
template <int X> struct Row8;
template <> struct Row8<CARD_DTYPE_BF16> {
    typedef uint16_t elem;
    static constexpr int kParts = 1, kWords = 4;
};
template <> struct Row8<CARD_DTYPE_F16> {
    typedef uint16_t elem;
    static constexpr int kParts = 1, kWords = 4;
};
template <> struct Row8<CARD_DTYPE_F32> {
    typedef uint32_t elem;
    static constexpr int kParts = 3, kWords = 8;
};
template <> struct Row8<CARD_DTYPE_E4M3> {
    typedef uint8_t elem;
    static constexpr int kParts = 1, kWords = 2;
};
template <int X> struct Raw { uint32_t w[Row8<X>::kWords]; };

template <int X> __device__ __forceinline__ Raw<X> load_x(const typename Row8<X>::elem* p) {
    typedef uint32_t words __attribute__((ext_vector_type(Row8<X>::kWords)));
    typedef words loose __attribute__((aligned(sizeof(typename Row8<X>::elem))));
    const words v = *reinterpret_cast<const loose*>(p);
    Raw<X> r;
#pragma unroll
    for (int i = 0; i < Row8<X>::kWords; ++i) r.w[i] = v[i];
    return r;
}
// columns col ... col + 7 of a row of `in`, zeros behind its end: whole vectors where rows end with one, else element by
// element.  No load waits for another: all are asked for, at the last one's place where there is none.
template <int X> __device__ __forceinline__ Raw<X> load_tail(const typename Row8<X>::elem* row, int col, int in) {
    typedef typename Row8<X>::elem E;
    constexpr int per = 4 / sizeof(E);
    Raw<X> r;
    if (in % 8 == 0) {
        r = load_x<X>(row + (col < in ? col : in - 8));
#pragma unroll
        for (int i = 0; i < Row8<X>::kWords; ++i) r.w[i] = col < in ? r.w[i] : 0u;
    } else {
        uint32_t e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = row[col + i < in ? col + i : in - 1];
#pragma unroll
        for (int i = 0; i < Row8<X>::kWords; ++i) {
            r.w[i] = 0;
#pragma unroll
            for (int j = 0; j < per; ++j) r.w[i] |= (col + i * per + j < in ? e[i * per + j] : 0u) << (j * 8 * sizeof(E) % 32);
        }
    }
    return r;
}
template <int X> __device__ __forceinline__ void parts_of(const Raw<X>& r, u32x4 (&a)[Row8<X>::kParts]) {
    if constexpr (X == CARD_DTYPE_F32) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t h[2], m[2], l[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float v = __uint_as_float(r.w[2 * j + i]);
                h[i] = r.w[2 * j + i] & 0xFFFF0000u;
                const float v1 = v - __uint_as_float(h[i]);
                m[i] = __float_as_uint(v1) & 0xFFFF0000u;
                l[i] = __float_as_uint(v1 - __uint_as_float(m[i]));
            }
            a[0][j] = h[0] >> 16 | h[1];
            a[1][j] = m[0] >> 16 | m[1];
            a[2][j] = l[0] >> 16 | (l[1] & 0xFFFF0000u);
        }
    } else if constexpr (X == CARD_DTYPE_E4M3) {
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            a[0][2 * j] = __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r.w[j], 1.0f, false));
            a[0][2 * j + 1] = __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r.w[j], 1.0f, true));
        }
    } else {
        a[0] = u32x4{r.w[0], r.w[1], r.w[2], r.w[3]};
    }
}

// a block of weights of NT tiles on its way
template <int G, int NT, bool STREAM> struct Weights {
    u32x4 q[NT];
    float s[NT][G];
    uint32_t z[NT][G];
    // at: the block's index, the same for all lanes
    __device__ __forceinline__ void load(const Args& a, const long long (&at)[NT], int b) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const long long i = at[t] + b;
            const u32x4* p = (const u32x4*)(a.q + i * 64) + lane;
            q[t] = STREAM ? __builtin_nontemporal_load(p) : *p;
#pragma unroll
            for (int g = 0; g < G; ++g) {
                s[t][g] = (a.scale + (i * G + g) * 16)[lane & 15];
                z[t][g] = (a.zero + (i * G + g) * 16)[lane & 15];
            }
        }
    }
};

// acc += one block: per group of columns the matrix pipe forms P = sum (16 + q) x and, against ones, S = sum x (for all NT
// tiles), the vector pipe adds scale * (P - (16 + zero) S).  part(m, s, p): the parts of step s of rows 16 m ...
// fp32 rows: P and S are some five times their difference, and sums over a group lose that much at their last bit.  So the
// first part's P and S, products of 13 bits, are taken for 32 columns each, where next to nothing is rounded; only the smaller
// parts' run over the group.  Off by (root mean square) 6.7e-8 instead of 5.6e-7 at 465 columns, 1.1e-7 and 9.1e-7 at 4096, a
// plain fp32 product 1.9e-7 and 5.8e-7; it costs 16 rows of 8192 x 28672 52.6 us for 44.5, of 4096 x 4096 8.9 for 8.3.  Shorter
// rows are as exact without: bf16 and e4m3 products have 13 bits at most (fp32 results off by 4e-8 to 1.1e-7 at 70 to 12000
// columns), fp16's 16 (1.2e-7 to 1.9e-7).
template <int X, int G, int MT, int NT, bool STREAM, typename F>
__device__ __forceinline__ void add_block(const Weights<G, NT, STREAM>& w, uint32_t sixteen, f32x4 (&acc)[MT][NT], F part) {
    constexpr int P = Row8<X>::kParts, S = 4 / G;          // S steps of 32 columns in a group
    const uint32_t one = X == CARD_DTYPE_F16 ? 0x3C003C00u : 0x3F803F80u;
    const u32x4 ones = {one, one, one, one};
#pragma unroll
    for (int g = 0; g < G; ++g) {
        f32x4 sum[MT], prod[MT][NT];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            sum[m] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int t = 0; t < NT; ++t) prod[m][t] = f32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int s = g * S; s < (g + 1) * S; ++s) {
            u32x4 v[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) v[t] = ints_of<X>(w.q[t][s], sixteen);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                u32x4 p[P];
                part(m, s, p);
#pragma unroll
                for (int k = P - 1; k >= (P > 1); --k) {
#pragma unroll
                    for (int t = 0; t < NT; ++t) prod[m][t] = mfma<X>(p[k], v[t], prod[m][t]);
                    sum[m] = mfma<X>(p[k], ones, sum[m]);
                }
                if constexpr (P > 1) {
                    const f32x4 none = {0, 0, 0, 0}, s0 = mfma<X>(p[0], ones, none);
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        const float off = -16.0f - (float)w.z[t][g];
                        const f32x4 p0 = mfma<X>(p[0], v[t], none);
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[m][t][r] = fmaf(w.s[t][g], fmaf(off, s0[r], p0[r]), acc[m][t][r]);
                    }
                }
            }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const float off = -16.0f - (float)w.z[t][g], sc = w.s[t][g];
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[m][t][r] = fmaf(sc, fmaf(off, sum[m][r], prod[m][t][r]), acc[m][t][r]);
        }
    }
}

__device__ __forceinline__ float epilogue(const Args& a, float v, float x_scale, float bias, float gamma) {
    v = (v * x_scale + bias) * gamma;
    return v > 0.0f ? v : v * a.slope;
}
__device__ __forceinline__ void store_y(const Args& a, void* y, long long at, float v) {
    if (a.y_dtype == CARD_DTYPE_F32) ((float*)y)[at] = v;
    else if (a.y_dtype == CARD_DTYPE_BF16) ((bf16_t*)y)[at] = (bf16_t)v;
    else ((f16_t*)y)[at] = (f16_t)v;
}

template <int X> __device__ __forceinline__ float value_of(typename Row8<X>::elem v) {
    if constexpr (X == CARD_DTYPE_F32) return __uint_as_float(v);
    else if constexpr (X == CARD_DTYPE_BF16) return __uint_as_float((uint32_t)v << 16);
    else if constexpr (X == CARD_DTYPE_F16) return (float)__builtin_bit_cast(_Float16, v);
    else return __builtin_amdgcn_cvt_f32_fp8((int)v, 0);
}
// One sum as it is defined, weight by weight, where the sum by P and S is not finite: an infinite x makes both infinite and
// their difference NaN, and x of 2^115 and more passes the largest float there.  A thread to an output, 128 columns at a time;
// a NaN ends it.
template <int X, int G> __device__ float plain_sum(const Args& a, const typename Row8<X>::elem* x, int row, long long o) {
    const typename Row8<X>::elem* xr = x + (long long)row * a.in;
    float sum = 0.0f;
    for (int b = 0; b < a.blocks && sum == sum; ++b) {
        const long long i = (o >> 4) * a.blocks + b;
        float part = 0.0f;
#pragma unroll 4
        for (int c = 0; c < 16; ++c) {                   // columns 8 c ... of the block: lanes 16 (c % 4) ..., word c / 4
            const long long at = (i * G + c * G / 16) * 16 + (o & 15);
            const uint32_t w = ((const uint32_t*)a.q)[(i * 64 + 16 * (c & 3) + (o & 15)) * 4 + (c >> 2)], u = w >> 3 | w << 29;
            const float s = a.scale[at], z = (float)a.zero[at];
            const int k = b * kBlock + 8 * c;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float v = value_of<X>(xr[k + j < a.in ? k + j : a.in - 1]), n = (float)(u >> (4 * (j / 2 + 4 * (j & 1))) & 15u);
                part += k + j < a.in ? (n - z) * s * v : 0.0f;
            }
        }
        sum += part;
    }
    return sum;
}

// What the epilogue multiplies and adds for one output: asked for at the start, so that it has come by the end.
struct Out {
    int row;
    long long o;
    float x_scale, bias, gamma;
    bool real;
    template <int MT> __device__ __forceinline__ void ask(const Args& a, int id, int tile0, int m0) {
        const int l = id & 63, r = (id >> 6) & 3, m = (id >> 8) % MT, t = (id >> 8) / MT;
        row = m0 + 16 * m + 4 * (l >> 4) + r;
        o = (long long)(tile0 + t) * 16 + (l & 15);
        real = row < a.rows && o < a.out;
        x_scale = real && a.x_scale ? a.x_scale[row] : 1.0f;
        bias = real ? a.bias[o] : 0.0f;
        gamma = real && a.gamma ? a.gamma[o] : 1.0f;
    }
};

// The waves join through LDS in a fixed order, and the epilogue.
template <int X, int G, int MT, int NT>
__device__ __forceinline__ void finish(const Args& a, const typename Row8<X>::elem* x, const f32x4 (&acc)[MT][NT], float* join, int tile0, int m0, Out out, void* y) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) join[((wave * NT + t) * MT + m) * 256 + r * 64 + lane] = acc[m][t][r];
    __syncthreads();
    constexpr int n = NT * MT * 256;
    for (int id = threadIdx.x; id < n; id += blockDim.x) {
        if (id >= (int)blockDim.x) out.ask<MT>(a, id, tile0, m0);
        if (!out.real) continue;
        float v = join[id];
        for (int w = 1; w < waves; ++w) v += join[w * n + id];
        const long long at = (long long)out.row * a.out + out.o;
        if (a.partial) {
            a.partial[(long long)blockIdx.z * a.rows * a.out + at] = v;
        } else {
            if (!__builtin_isfinite(v)) v = plain_sum<X, G>(a, x, out.row, out.o);
            store_y(a, y, at, epilogue(a, v, out.x_scale, out.bias, out.gamma));
        }
    }
}

// the shares of the columns join in a fixed order
template <int X, int G>
__global__ __launch_bounds__(kThreads) void linear4_join_kernel(const Args a, const typename Row8<X>::elem* x, void* y) {
    const long long id = (long long)blockIdx.x * kThreads + threadIdx.x, n = (long long)a.rows * a.out;
    if (id >= n) return;
    const int row = (int)(id / a.out), o = (int)(id - (long long)row * a.out);
    float v = a.partial[id];
#pragma unroll 4
    for (int k = 1; k < a.splits; ++k) v += a.partial[k * n + id];
    if (!__builtin_isfinite(v)) v = plain_sum<X, G>(a, x, row, o);
    store_y(a, y, id, epilogue(a, v, a.x_scale ? a.x_scale[row] : 1.0f, a.bias[o], a.gamma ? a.gamma[o] : 1.0f));
}

// One workgroup: 16 MT rows of x by 16 NT outputs; each of its waves takes a run of blocks of columns.
//
// The matrix instruction wants row l % 16 of x in lane l.  Asked for like that, 16 neighbouring lanes read 16 rows and every
// load costs 64 cycles of the cache's address path (42 us for 16 rows of 8192 columns, 28672 outputs, against 31.5).  So lane l
// asks for row l / 4 -- four lanes share a row's 64 bytes -- and ds_bpermute hands the values over where they are used; LDS
// between them took as long and needs barriers.  U blocks of weights and of x are on their way while one is used: the loop
// over them has no branch, or every wait in it would be for all of them.  A last block that is not full comes after the loop.
template <int X, int G, int MT, int NT, int U, bool STREAM, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void linear4_kernel(const Args a, const typename Row8<X>::elem* x, void* y) {
    extern __shared__ float join[];                  // (waves, NT, MT, 4, 64)
    constexpr int W = Row8<X>::kWords;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int tile0 = blockIdx.x * NT, m0 = blockIdx.y * (16 * MT);
    const int s0 = a.blocks * blockIdx.z / gridDim.z, n = a.blocks * (blockIdx.z + 1) / gridDim.z - s0;          // this share's blocks
    const bool tail = a.in % kBlock != 0 && wave == waves - 1 && blockIdx.z == gridDim.z - 1;
    const int b0 = s0 + n * wave / waves, b1 = s0 + n * (wave + 1) / waves - tail;
    const int lrow = lane >> 2, lcol = 8 * (lane & 3), from = 4 * (4 * (lane & 15) + (lane >> 4));
    const typename Row8<X>::elem* xr[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int row = m0 + 16 * m + lrow;
        xr[m] = x + (long long)(row < a.rows ? row : a.rows - 1) * a.in + lcol;
    }
    long long at[NT];                                // a tile behind the last one repeats it and is not stored
#pragma unroll
    for (int t = 0; t < NT; ++t) at[t] = (long long)(tile0 + t < a.tiles ? tile0 + t : a.tiles - 1) * a.blocks;
    struct Stage {
        Weights<G, NT, STREAM> w;
        Raw<X> x[MT][4];
    } st[U];
    auto fetch = [&](Stage& g, int b) {
        g.w.load(a, at, b);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int s = 0; s < 4; ++s) g.x[m][s] = load_x<X>(xr[m] + b * kBlock + 32 * s);
    };
    Out out = {};
    if (threadIdx.x < NT * MT * 256) out.ask<MT>(a, threadIdx.x, tile0, m0);
    const uint32_t sixteen = sixteen_of<X>();
    f32x4 acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[m][t] = f32x4{0, 0, 0, 0};
    auto use = [&](const Stage& g) {
        add_block<X, G, MT, NT, STREAM>(g.w, sixteen, acc, [&](int m, int s, u32x4 (&p)[Row8<X>::kParts]) {
            Raw<X> r = g.x[m][s];
#pragma unroll
            for (int i = 0; i < W; ++i) r.w[i] = (uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)r.w[i]);
            parts_of<X>(r, p);
        });
    };
    int b = b0;
    if (b1 - b0 >= 2 * U) {
#pragma unroll
        for (int u = 0; u < U; ++u) fetch(st[u], b + u);
        for (; b + 2 * U <= b1; b += U) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                use(st[u]);
                fetch(st[u], b + u + U);
            }
        }
    } else {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (b + u < b1) fetch(st[u], b + u);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (b + u < b1) use(st[u]);
        if (b + u + U < b1) fetch(st[u], b + u + U);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (b + u + U < b1) use(st[u]);
    if (tail) {
        st[0].w.load(a, at, b1);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int s = 0; s < 4; ++s) st[0].x[m][s] = load_tail<X>(xr[m] - lcol, b1 * kBlock + 32 * s + lcol, a.in);
        use(st[0]);
    }
    finish<X, G, MT, NT>(a, x, acc, join, tile0, m0, out, y);
}

template <int X, int G, int MT, int NT, int U, bool STREAM, int WAVES> int launch(const Args& a, const void* x, void* y, hipStream_t st) {
    int waves = 1;                                   // a block of columns for each at least
    while (waves < WAVES && a.blocks / a.splits >= 2 * waves) waves *= 2;
    const dim3 grid((a.tiles + NT - 1) / NT, (a.rows + 16 * MT - 1) / (16 * MT), a.splits);
    const typename Row8<X>::elem* xe = (const typename Row8<X>::elem*)x;
    linear4_kernel<X, G, MT, NT, U, STREAM, WAVES><<<grid, 64 * waves, waves * NT * MT * 256 * sizeof(float), st>>>(a, xe, y);
    HIP_TRY(hipGetLastError());
    if (a.partial) {
        linear4_join_kernel<X, G><<<(unsigned)(((long long)a.rows * a.out + kThreads - 1) / kThreads), kThreads, 0, st>>>(a, xe, y);
        HIP_TRY(hipGetLastError());
    }
    return CARD_OK;
}
// Shares of the columns, where there are too few tiles for the chip and a workgroup would be long at its columns: one for every
// eight blocks (a block for each of its waves) while the chip has CUs for them.  The second launch costs some 3 us, so it has to
// be long: a wave's blocks, weighted by the row tiles and by fp32's three operands, are 24 or more (12000 columns, 100 outputs:
// 30 rows fp32 33 us in one share and 13.5 in eleven, 30 rows bf16 12.9 and 9.2; below, 16 rows fp16 8.6 and 8.7, 8000 columns
// of 30 rows e4m3 8.5 and 9.4).
int splits_of(int tiles, int blocks, int64_t rows, int x_dtype) {
    const int row_tiles = rows <= 16 ? 1 : 2, work = (blocks + 7) / 8 * row_tiles * (x_dtype == CARD_DTYPE_F32 ? 3 : 1);
    const int64_t groups = tiles * ((rows + 16 * row_tiles - 1) / (16 * row_tiles));
    if (tiles > 128 || work < 24) return 1;
    const int64_t most = 256 / groups, s = blocks / 8 < most ? blocks / 8 : most;
    return s > 1 ? (int)s : 1;
}
// Several tiles share the values of x where there are more tiles than CUs (24 rows, 6144 outputs: 9.8 us with two against
// 10.3).  From 1024 tiles on the weights pass by the caches, which cannot hold them (16 rows of 8192 columns, 28672 outputs:
// 29.7 us against 31.5; but 5.8 against 5.1 for 4096 x 4096, whose weights stay in L2 from call to call), and workgroups are
// plenty: four tiles and four waves with one block on its way, workgroups small enough that a CU holds several: up to 16 rows
// three or two in 16 bits (152 to 175 registers), four to two in e4m3, two in fp32; 17 rows and more two, but one in e4m3 with
// groups of 64 (263 registers).  8192 columns, 28672 outputs: 16 rows bf16 30.2 us against 34.8 with two tiles, eight waves and
// two blocks, 32 rows e4m3 40.0 and 51.1.  Up to 16 rows of e4m3, half of bf16's x to read, need only three tiles to share them,
// and smaller workgroups even out the last ones (28672 outputs 29.4 us against 29.9 with four, 17000 outputs of 4096 columns 12.2
// and 14.5; but bf16 33.0 against 30.2).  All of these were measured with groups of 128.
constexpr int kCus = 256, kStreamTiles = 1024;
template <int X, int G, int MT> int by_tiles(const Args& a, const void* x, void* y, hipStream_t st) {
    // blocks on their way: one where rows are wide -- more than 16, or fp32 with its three operands -- for the registers' sake
    constexpr int U = X == CARD_DTYPE_F32 || MT > 1 ? 1 : 2;
    if (a.tiles <= kCus) return launch<X, G, MT, 1, U, false, 8>(a, x, y, st);
    if (a.tiles < kStreamTiles) return launch<X, G, MT, 2, U, false, 8>(a, x, y, st);
    return launch<X, G, MT, X == CARD_DTYPE_E4M3 && MT == 1 ? 3 : 4, 1, true, 4>(a, x, y, st);
}
template <int X, int G> int by_rows(const Args& a, const void* x, void* y, hipStream_t st) {
    return a.rows <= 16 ? by_tiles<X, G, 1>(a, x, y, st) : by_tiles<X, G, 2>(a, x, y, st);
}
template <int X> int by_group(const Args& a, int group, const void* x, void* y, hipStream_t st) {
    return group == 128 ? by_rows<X, 1>(a, x, y, st) : group == 64 ? by_rows<X, 2>(a, x, y, st) : by_rows<X, 4>(a, x, y, st);
}

}  // namespace

extern "C" CARD_API int card_linear4_quantize(const float* W, int32_t out_features, int32_t in_features, int32_t group, uint8_t* q,
                                              float* scale, uint8_t* zero, void* stream) {
    const char* who = "card_linear4_quantize";
    if (out_features < 1 || in_features < 1) return card_fail(CARD_E_INVALID, "%s: %d x %d features", who, out_features, in_features);
    if (group != 32 && group != 64 && group != 128) return card_fail(CARD_E_UNSUPPORTED, "%s: group=%d is none of 32, 64, 128", who, group);
    if (!W || !q || !scale || !zero) return card_fail(CARD_E_INVALID, "%s: null argument", who);
    const int groups = (in_features + group - 1) / group;
    const long long n = (long long)out_features * groups;
    quantize_kernel<<<walkers((n + kThreads / 64 - 1) / (kThreads / 64)), kThreads, 0, (hipStream_t)stream>>>(W, in_features, group, groups, n, q, scale, zero);
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
    s->in = d->in_features; s->out = d->out_features; s->group = d->group;
    s->blocks = (s->in + kBlock - 1) / kBlock; s->tiles = (s->out + 15) / 16;
    hipStream_t st = (hipStream_t)stream;
    const long long nw = (long long)s->tiles * s->blocks * 64, ng = (long long)s->tiles * s->blocks * (kBlock / s->group) * 16;
    hipError_t e = hipGetDevice(&s->device);
    if (e == hipSuccess) e = hipMalloc(&s->q, nw * sizeof(uint4));
    if (e == hipSuccess) e = hipMalloc(&s->scale, ng * sizeof(float));
    if (e == hipSuccess) e = hipMalloc(&s->zero, ng);
    if (e == hipSuccess) e = hipMalloc(&s->bias, s->out * sizeof(float));
    if (e == hipSuccess) {
        pack_kernel<<<walkers((nw + kThreads - 1) / kThreads), kThreads, 0, st>>>(d->q, s->in, s->out, s->blocks, nw, s->q);
        side_kernel<<<walkers((ng + kThreads - 1) / kThreads), kThreads, 0, st>>>(d->scale, d->zero, d->bias, s->group, (s->in + s->group - 1) / s->group,
                                                                                  s->blocks, s->out, ng, s->scale, s->zero, s->bias);
        e = hipGetLastError();
    }
    if (e != hipSuccess) {
        (void)hipGetLastError();                         // or the next launch's check would find it
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

extern "C" CARD_API int card_linear4_workspace_bytes(const card_linear4* s, int32_t x_dtype, int64_t rows, uint64_t* bytes) {
    const char* who = "card_linear4_workspace_bytes";
    if (!s || !bytes) return card_fail(CARD_E_INVALID, "%s: null argument", who);
    if (!card_dtype_bytes(x_dtype)) return card_fail(CARD_E_INVALID, "%s: x_dtype %d is no card_dtype", who, x_dtype);
    if (rows < 0) return card_fail(CARD_E_INVALID, "%s: rows=%lld < 0", who, (long long)rows);
    if (rows > CARD_LINEAR4_MAX_ROWS) return card_fail(CARD_E_UNSUPPORTED, "%s: rows=%lld > %d", who, (long long)rows, CARD_LINEAR4_MAX_ROWS);
    const int n = rows ? splits_of(s->tiles, s->blocks, rows, x_dtype) : 1;
    *bytes = n > 1 ? (uint64_t)n * (uint64_t)rows * (uint64_t)s->out * sizeof(float) : 0;
    return CARD_OK;
}

extern "C" CARD_API int card_linear4_forward(const card_linear4* s, const void* x, int32_t x_dtype, const float* x_scale, int64_t rows,
                                             const float* gamma, float slope, void* y, int32_t y_dtype, void* workspace,
                                             uint64_t workspace_bytes, void* stream) {
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
    a.in = s->in; a.out = s->out; a.blocks = s->blocks; a.tiles = s->tiles; a.rows = (int)rows; a.y_dtype = y_dtype;
    a.splits = splits_of(s->tiles, s->blocks, rows, x_dtype);
    a.partial = a.splits > 1 ? (float*)workspace : nullptr;
    if (a.splits > 1) {
        const uint64_t need = (uint64_t)a.splits * (uint64_t)rows * (uint64_t)s->out * sizeof(float);
        if (!workspace || workspace_bytes < need)
            return card_fail(CARD_E_INVALID, "%s: workspace of %llu bytes, need %llu", who, (unsigned long long)workspace_bytes, (unsigned long long)need);
        if ((uintptr_t)workspace & 15) return card_fail(CARD_E_INVALID, "%s: workspace is not 16-byte aligned", who);
    }
    hipStream_t st = (hipStream_t)stream;
    switch (x_dtype) {
        case CARD_DTYPE_F32: return by_group<CARD_DTYPE_F32>(a, s->group, x, y, st);
        case CARD_DTYPE_BF16: return by_group<CARD_DTYPE_BF16>(a, s->group, x, y, st);
        case CARD_DTYPE_F16: return by_group<CARD_DTYPE_F16>(a, s->group, x, y, st);
        default: return by_group<CARD_DTYPE_E4M3>(a, s->group, x, y, st);
    }
}
