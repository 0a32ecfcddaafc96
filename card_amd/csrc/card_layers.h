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

// Calls that move more than this read past the caches (`stream`): the last level holds 256 MB, and what a larger call leaves
// there is gone before it is asked for again.  8192 x 6144 bf16, norm with residual: forward 75 us without and 60 us with,
// backward 93 and 68; 16384 x 8192 bf16 dropout with residual 141 and 128.  Smaller calls lose by it: 1000 x 4096 norm 6.6 and 7.6.
constexpr long long kStreamBytes = 300000000;
// (A choice at compile time: of two loads behind a branch the compiler makes one.)
template <bool STREAM, int N, typename T> __device__ __forceinline__ typename Vec<T, N>::type load_vec(const T* p) {
    const typename Vec<T, N>::loose* q = reinterpret_cast<const typename Vec<T, N>::loose*>(p);
    if constexpr (STREAM) return __builtin_nontemporal_load(q);
    else return *q;
}

// n <= N values at p as floats, the rest of v zero
template <int N, bool STREAM = false, typename T> __device__ __forceinline__ void load_n(const T* p, long long n, float (&v)[N]) {
    if (n >= N) {
        const typename Vec<T, N>::type t = load_vec<STREAM, N>(p);
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
// Philox4x32-10 of the block (c, draw, 1): card_common.h's generator in 20 multiplies that give both halves and 20 three-way
// xors; the keys are the same for all lanes and step on the scalar unit.  A stream of bf16 elements is bound by these
// instructions and not by memory: 8192 x 4096, forward or backward, 43 us with two multiplies and two xors for one, 33 us so.
__device__ __forceinline__ void drop_words(const DropRule& d, unsigned long long seed, unsigned long long c, uint32_t (&r)[4]) {
    uint32_t c0 = (uint32_t)c, c1 = (uint32_t)(c >> 32), c2 = d.draw, c3 = 1u, k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int i = 0; i < 10; ++i) {
        unsigned long long p0, p1, cc;
        asm("v_mad_u64_u32 %0, %1, %2, %3, 0" : "=v"(p0), "=s"(cc) : "v"(c0), "s"(0xD2511F53u));
        asm("v_mad_u64_u32 %0, %1, %2, %3, 0" : "=v"(p1), "=s"(cc) : "v"(c2), "s"(0xCD9E8D57u));
        const uint32_t h0 = (uint32_t)(p0 >> 32), l0 = (uint32_t)p0, h1 = (uint32_t)(p1 >> 32), l1 = (uint32_t)p1;
        c0 = __builtin_amdgcn_bitop3_b32(h1, c1, k0, 0x96);
        c2 = __builtin_amdgcn_bitop3_b32(h0, c3, k1, 0x96);
        c1 = l1; c3 = l0;
        k0 += 0x9E3779B9u; k1 += 0xBB67AE85u;
    }
    r[0] = c0; r[1] = c1; r[2] = c2; r[3] = c3;
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
            drop_words(d, seed, b + k, r);
#pragma unroll
            for (int w = 0; w < 4; ++w) m |= (r[w] >= d.threshold ? 1u : 0u) << (4 * k + w);
        }
    }
    return d.none ? 0u : m >> s;
}
// v[j] = kept ? v[j] * scale : 0 for the N elements of whole blocks from block b on: the words decide as they come
template <int N> __device__ __forceinline__ void drop(const DropRule& d, unsigned long long seed, unsigned long long b, float (&v)[N]) {
#pragma unroll
    for (int k = 0; k < N / 4; ++k) {
        uint32_t r[4];
        drop_words(d, seed, b + k, r);
#pragma unroll
        for (int w = 0; w < 4; ++w) v[4 * k + w] = r[w] >= d.threshold && !d.none ? v[4 * k + w] * d.scale : 0.0f;
    }
}

}  // namespace card

// host side (card_dropout.hip): checks p and fills the rule; 0 or a card_status
int drop_rule(const char* who, double p, uint64_t seed, uint64_t elem_offset, const uint64_t* state, int32_t draw, card::DropRule* out);
inline int64_t card_dtype_bytes(int32_t dtype) {
    return dtype == CARD_DTYPE_F32 ? 4 : dtype == CARD_DTYPE_BF16 || dtype == CARD_DTYPE_F16 ? 2 : dtype == CARD_DTYPE_E4M3 ? 1 : 0;
}
#endif
