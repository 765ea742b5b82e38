// Device code that the kernels of the 4-bit KV cache's attention share: loads and
// stores of value types, hi / lo splits, and code words as fp16.
#pragma once

#include <cuda_bf16.h>

#include "jl_kv4.cuh"

namespace jl {

// Weights times V's scales enter the second product as fp16 hi and lo parts: 22 bits of
// a product of 2^-2 and more, down to steps of 2^-24 below. So the largest product of a
// row has to be near the top of fp16's range whatever the scales are, in each 64-value
// group by itself (kv4_ref): products are kept at or below 2^kTop, and a new reference
// puts the largest at 2^(kTop - kHeadroom), so that the sums are not rescaled at every
// new maximum (most units of a short run have one in some row).
//
// How large the products of a block are: its largest score times its largest scale is a
// bound, at most 2^kSpread above the truth when the scales of all its positions and
// groups are within that (kv4_spread), and then costs nothing. Else, and in blocks that
// not all rows see whole, the maximum is taken over the products that the row has.
constexpr float kTop = 15.0f, kHeadroom = 4.0f, kLeast = -40.0f;  // 2^kLeast: taken for products of 0
constexpr int kSpread = 10;

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

// Four values.
__device__ __forceinline__ void put4(float* p, const float* x) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ void put4(__half* p, const float* x) {
    const __half2 u = __floats2half2_rn(x[0], x[1]), v = __floats2half2_rn(x[2], x[3]);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&u), *reinterpret_cast<const uint32_t*>(&v));
}
__device__ __forceinline__ void put4(__nv_bfloat16* p, const float* x) {
    const __nv_bfloat162 u = __floats2bfloat162_rn(x[0], x[1]), v = __floats2bfloat162_rn(x[2], x[3]);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&u), *reinterpret_cast<const uint32_t*>(&v));
}

__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
    const uint4 w = *reinterpret_cast<const uint4*>(p);
    const T* h = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = to_f32(h[j]);
}
__device__ __forceinline__ void put8(float* p, const float (&x)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void put8(__half* p, const float (&x)[8]) {
    __half2 h[4];
#pragma unroll
    for (int j = 0; j < 4; j++) h[j] = __floats2half2_rn(x[2 * j], x[2 * j + 1]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(h);
}
__device__ __forceinline__ void put8(__nv_bfloat16* p, const float (&x)[8]) {
    __nv_bfloat162 h[4];
#pragma unroll
    for (int j = 0; j < 4; j++) h[j] = __floats2bfloat162_rn(x[2 * j], x[2 * j + 1]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(h);
}
__device__ __forceinline__ void put1(float* p, float x) { *p = x; }
__device__ __forceinline__ void put1(__half* p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void put1(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 2^e is above x >= 0 (by at most 2): e, at least kLeast.
__device__ __forceinline__ float exponent_of(float x) {
    return fmaxf((float)((int)(__float_as_uint(x) >> 23) - 126), kLeast);
}

// From the largest and smallest scale's bits: the exponent that bounds them, and whether
// some are zero, subnormal or smaller by more than 2^kSpread.
__device__ __forceinline__ float kv4_top(uint32_t most) { return (float)((int)(most >> 10) - 14); }
__device__ __forceinline__ bool kv4_spread(uint32_t most, uint32_t least) {
    return least < 1024 || most - least > (uint32_t)kSpread << 10;
}

// A row's references: weights are 2^(score - ref), and those of a head's second group
// (G1) may take a power of two more into the product, so that each group's largest
// product is near the top: 2^lift would bring it there, and lifts of 0 to kNoLift are
// left out: `ref` goes by the larger group unless the second is larger by more, so
// that ordinary rows have no other. `ref` is a score plus a whole number.
constexpr float kNoLift = 8.0f;
template <bool G1>
struct kv4_ref {
    float ref, lift;
    __device__ __forceinline__ void clear() { ref = -INFINITY, lift = 0.0f; }
    __device__ __forceinline__ bool lifted() const { return G1 && !(lift >= 0.0f && lift <= kNoLift); }
    __device__ __forceinline__ float log_more() const { return lifted() ? lift : 0.0f; }
    // the second group's factor, and what brings its sums to a scale without it
    __device__ __forceinline__ float more() const { return __uint_as_float((uint32_t)((int)log_more() + 127) << 23); }
    __device__ __forceinline__ float less() const { return __uint_as_float((uint32_t)(127 - (int)log_more()) << 23); }
    __device__ __forceinline__ float minus() const { return ref == -INFINITY ? 0.0f : -ref; }
    // Does a product of at most 2^(b0 + score - mx) of group 0, or 2^(b1 + ...) of group 1, pass the limit?
    __device__ __forceinline__ bool past(float mx, float b0, float b1) const {
        return (mx - ref) + (G1 ? fmaxf(b0, b1 + log_more()) : b0) > kTop;
    }
    // Brings the references to a row's largest score mx (its products below 2^b0 and 2^b1 of
    // that weight) and returns the factors of the sums: of the weights and group 0, of group 1.
    // A reference that fp32 cannot hold to within 1 (scores past 2^24) is the score itself.
    __device__ __forceinline__ float2 move(float mx, float b0, float b1) {
        const float old = ref, was = log_more(), b = G1 && b1 - b0 <= kNoLift ? fmaxf(b0, b1) : b0;
        if ((mx - ref) + b > kTop) {
            const float k = ceilf(b - (kTop - kHeadroom));
            ref = mx + k;
            if (!(fabsf((ref - mx) - k) <= 1.0f)) ref = mx;
        }
        const float al = ex2(old - ref);  // the first time: 0
        if (!G1) return make_float2(al, al);
        const float at = (mx - ref) + b1, most = floorf((kTop - kHeadroom) - at);
        lift = old == -INFINITY ? most : lift + floorf(ref - old);
        if (at + log_more() > kTop) lift = most;
        lift = fminf(fmaxf(lift, -100.0f), 100.0f);
        return make_float2(al, ex2((old - ref) + (log_more() - was)));
    }
};

// A sum of weights that keeps what its additions round off: added one after the other
// for a whole history, equal weights all round the same way (1e-4 after 23,000).
struct kv4_sum {
    float s, rest;
    __device__ __forceinline__ void clear() { s = rest = 0.0f; }
    __device__ __forceinline__ void add(float2 x) {
        const float b = x.x + x.y, t = __fadd_rn(s, b), z = __fsub_rn(t, s);
        rest = __fadd_rn(rest, __fadd_rn(__fsub_rn(s, __fsub_rn(t, z)), __fsub_rn(b, z)));
        s = t;
    }
    __device__ __forceinline__ void scale(float f) { s *= f, rest *= f; }
    __device__ __forceinline__ float total() const { return s + rest; }
};

__device__ __forceinline__ uint32_t h2bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }

// A pair as fp16 pairs, hi the nearest and lo what hi misses: 22 bits of values of 2^-2
// and more, steps of 2^-24 of smaller ones (the callers' largest are 2^1 and more: a
// row's q by a power of two, products by kv4_ref).
__device__ __forceinline__ void split2(float2 x, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __float22half2_rn(x);
    const float2 f = __half22float2(h);
    hi = h2bits(h);
    lo = h2bits(__float22half2_rn(__fadd2_rn(x, make_float2(-f.x, -f.y))));
}

__device__ __forceinline__ float2 f2(float x) { return make_float2(x, x); }

// n - 8 of the nibbles at bits 0-3 (even) or 4-7 (odd) of both halves, exactly,
// as fp16: 1024 + n (1024 + 16 n) by its bits, then one packed sum (FMA). The
// and-or is one instruction only when written as lop3 (measured: 256 fewer of
// 1,590 instructions per block, on the pipe that is busiest).
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t m, uint32_t o) {
    uint32_t y;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(x), "r"(m), "r"(o));
    return y;
}
__device__ __forceinline__ uint32_t code_even(uint32_t x) {
    x = and_or(x, 0x000F000Fu, 0x64006400u);
    return h2bits(__hsub2(*reinterpret_cast<__half2*>(&x), __floats2half2_rn(1032.0f, 1032.0f)));
}
__device__ __forceinline__ uint32_t code_odd(uint32_t x) {
    x = and_or(x, 0x00F000F0u, 0x64006400u);
    return h2bits(__hfma2(*reinterpret_cast<__half2*>(&x), __floats2half2_rn(0.0625f, 0.0625f),
                          __floats2half2_rn(-72.0f, -72.0f)));
}

constexpr int kKvUnit = kKv4Rows;  // positions taken at a time: a cache block

// Units of sequence b (0 when its slot or length is outside the cache), and
// what it counts in the cut: its units, or 1 when segments are not cut.
struct kv4_seqs {
    const int* slots;
    const int* lens;
    int len_add, longest, nslots, whole;
    __device__ int len(int b) const {
        const int n = __ldg(lens + b) + len_add, s = __ldg(slots + b);
        return s >= 0 && s < nslots && n >= 0 && n <= longest ? n : -1;
    }
    __device__ int units(int b) const { return (max(0, len(b)) + kKvUnit - 1) / kKvUnit; }
    __device__ int weight(int b) const { return whole ? len(b) > 0 : units(b); }
};

}  // namespace jl
