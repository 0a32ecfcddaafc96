// card_layers.h - device helpers of the layer operators (card_dropout.hip, card_norm.hip, card_linear4.hip): element types,
// vector loads that ask for no more than the element's own alignment, and the dropout mask.
#ifndef CARD_LAYERS_H
#define CARD_LAYERS_H
#include "card_common.h"

namespace card {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <typename T, int N> struct Vec {
    typedef T type __attribute__((ext_vector_type(N)));
    // rows of an odd width start anywhere: gfx950 loads and stores 16 bytes at any element's address
    typedef type loose __attribute__((aligned(sizeof(T))));
};

// n <= N values at p as floats, the rest of v zero
template <int N, typename T> __device__ __forceinline__ void load_n(const T* p, long long n, float (&v)[N]) {
    if (n >= N) {
        const typename Vec<T, N>::type t = *reinterpret_cast<const typename Vec<T, N>::loose*>(p);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (float)t[i];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = i < n ? (float)p[i] : 0.0f;
    }
}

template <int N, typename T> __device__ __forceinline__ void store_n(T* p, long long n, const float (&v)[N]) {
    typename Vec<T, N>::type t;
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = (T)v[i];          // round to nearest even
    if (n >= N) {
        *reinterpret_cast<typename Vec<T, N>::loose*>(p) = t;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < n) p[i] = t[i];
    }
}

// ------------------------------------------------------------------------------------------------
// The dropout mask: element e of mask `draw` takes word e & 3 of Philox4x32-10 at the counter (e >> 2, draw, 1) -- the
// sampler's normals use (element, draw block, 0), so one seed serves both -- and is kept when that word is >= threshold.
// ------------------------------------------------------------------------------------------------
struct DropRule {
    unsigned long long seed, elem_offset;
    const unsigned long long* state;     // not NULL: {seed, element offset} in device memory, instead of seed; the offsets add
    uint32_t threshold;                  // round(p * 2^32)
    uint32_t draw;
    float scale;                         // 1 / (1 - p)
    int none;                            // p = 1: nothing is kept
};
__device__ __forceinline__ void drop_key(const DropRule& d, unsigned long long& seed, unsigned long long& off) {
    seed = d.state ? d.state[0] : d.seed;
    off = d.elem_offset + (d.state ? d.state[1] : 0ull);
}
// bit j: element e + j is kept, j < n <= N (bits from n on may be anything)
template <int N>
__device__ __forceinline__ uint32_t keep_bits(const DropRule& d, unsigned long long seed, unsigned long long e, int n) {
    const unsigned long long b = e >> 2;
    const int s = (int)(e & 3);
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k <= N / 4; ++k) {
        if (4 * k < s + n) {
            uint32_t r[4];
            const unsigned long long c = b + k;
            philox4x32_10((uint32_t)c, (uint32_t)(c >> 32), d.draw, 1u, (uint32_t)seed, (uint32_t)(seed >> 32), r);
#pragma unroll
            for (int w = 0; w < 4; ++w) m |= (r[w] >= d.threshold ? 1u : 0u) << (4 * k + w);
        }
    }
    return d.none ? 0u : m >> s;
}

}  // namespace card

// host side (card_dropout.hip): checks p and fills the rule; 0 or a card_status
int drop_rule(const char* who, double p, uint64_t seed, uint64_t elem_offset, const uint64_t* state, int32_t draw, card::DropRule* out);
inline int64_t card_dtype_bytes(int32_t dtype) {
    return dtype == CARD_DTYPE_F32 ? 4 : dtype == CARD_DTYPE_BF16 || dtype == CARD_DTYPE_F16 ? 2 : dtype == CARD_DTYPE_E4M3 ? 1 : 0;
}
#endif
