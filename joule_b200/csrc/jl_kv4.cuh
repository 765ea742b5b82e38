// Layout of the 4-bit KV cache and the device code that writes its records.
//
// A cache is [slots][L][n_kv][blocks] blocks of kKv4Rows positions of one kv
// head; one block is one contiguous run of 68 * hd bytes (8,704 at hd = 128),
// so that a consumer fetches the K and V records of 64 positions by a single
// bulk copy:
//
//   [K codes 64 x hd/2][K scales 64 x hd/64][V codes 64 x hd/2][V scales 64 x hd/64]
//
// A record is a Q4 record (q4_store.py:40-55): groups of 64 values, fp16 scale
// s = max|x| / 7, code n = clip(rint(x / s), -8, 7) + 8, value (n - 8) * s,
// value 2i of a group in the low nibble of byte i. In the cache the 4-byte
// words (8 values) of a row's groups are interleaved (word u of group g at
// word u * ng + g, ng = hd / 64), and V row r lies at place vplace(r) with its
// word u at u ^ (r & 4): the attention kernel's fragments of the matrix
// instruction are then 16-byte (K) and 8-byte (V) shared-memory loads without
// bank conflicts, straight from the copied block.
#pragma once

#include "jl_common.cuh"

namespace jl {

constexpr int kKv4Rows = 64;        // positions per block
constexpr int kErrKvIndex = 8;      // a slot, position or length outside the cache (status bit)

// All offsets in bytes; hd is 64 or 128.
__host__ __device__ constexpr int kv4_block_bytes(int hd) { return 68 * hd; }
__host__ __device__ constexpr int kv4_kscale(int hd) { return 32 * hd; }
__host__ __device__ constexpr int kv4_vcode(int hd) { return 34 * hd; }
__host__ __device__ constexpr int kv4_vscale(int hd) { return 66 * hd; }
__host__ __device__ constexpr int kv4_vplace(int r) { return (r & ~7) | ((r & 1) << 2) | ((r >> 1) & 3); }

// Code word u (8 values) of group g of row r; `is_v` selects the section.
__host__ __device__ constexpr int kv4_word_off(int hd, int is_v, int r, int g, int u) {
    return is_v ? kv4_vcode(hd) + kv4_vplace(r) * (hd / 2) + ((u ^ (r & 4)) * (hd / 64) + g) * 4
                : r * (hd / 2) + (u * (hd / 64) + g) * 4;
}
__host__ __device__ constexpr int kv4_scale_off(int hd, int is_v, int r, int g) {
    return (is_v ? kv4_vscale(hd) : kv4_kscale(hd)) + (r * (hd / 64) + g) * 2;
}

// Base of (slot, layer, head)'s run of blocks.
struct kv4_dims {
    uint8_t* base;
    int slots, L, KH, hd, nb, maxT;
    __host__ __device__ uint8_t* run(int slot, int l, int h) const {
        return base + (((size_t)slot * L + l) * KH + h) * (size_t)nb * kv4_block_bytes(hd);
    }
};

// Codes of eight values of a group with scale s (the nearest steps of the exact
// quotients, ties to even): an IEEE division each.
inline __device__ __noinline__ uint32_t kv4_codes_div(float4 x, float4 y, float s) {
    const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float q = rintf(__fdiv_rn(v[j], s));
        const int n = q != q ? 8 : (int)fminf(fmaxf(q, -8.0f), 7.0f) + 8;
        w |= (uint32_t)n << (4 * j);
    }
    return w;
}

// max of |a|, |b| and m that keeps a NaN.
__device__ __forceinline__ float kv4_max_nan(float m, float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(fabsf(a)), "f"(fabsf(b)));
    return r;
}

// Quantises a group of 64 values held by 8 / W consecutive lanes (a lane has the W words
// from u on: values 8u .. 8u + 8W - 1) and stores it as (row r, group g) of block
// `blk` when `store`. A code is the step nearest to the exact x / s, ties to even. Its
// first guess k is the product with about 1 / s, rounded by adding 1.5 * 2^23 + 8; it
// stands when what is left, x - k s, is below half a step. That remainder is exact
// (11 by 4 bits from a value of the same size), so a value past half or at half of a
// step moves by one (one bf16 value in 700 is at half). The lane divides for a NaN, an infinity, and a
// scale past the largest or of less than 8 of fp16's smallest steps, whose rounding can
// leave amax above 7.5 steps. amax / 7 is the product with 1 / 7 corrected once by its
// exact remainder (Markstein's correction; equal to the IEEE quotient for every
// significand). Beyond the record's own rules: a scale that fp16 cannot hold stays at
// its largest number (values past 7 * 65504 saturate) and a NaN becomes zero, so what
// the cache holds is always finite. All lanes of the warp call it.
template <int W>
__device__ __forceinline__ void kv4_store_group(uint8_t* blk, int hd, int is_v, int r, int g, int u, const float4 (&x)[2 * W],
                                                bool store) {
    float2 v[4 * W];
#pragma unroll
    for (int j = 0; j < 2 * W; j++) v[2 * j] = make_float2(x[j].x, x[j].y), v[2 * j + 1] = make_float2(x[j].z, x[j].w);
    float amax = 0.0f;
#pragma unroll
    for (int j = 0; j < 4 * W; j++) amax = fmaxf(amax, fmaxf(fabsf(v[j].x), fabsf(v[j].y)));
#pragma unroll
    for (int o = 4 / W; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    amax = fmaxf(amax, 1e-12f);
    const float seventh = 1.0f / 7.0f, q0 = amax * seventh;  // (an infinity becomes a NaN, and the largest scale)
    const __half sh = __float2half_rn(fminf(fmaf(fmaf(-7.0f, q0, amax), seventh, q0), 65504.0f));
    const float s = __half2float(sh);
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
    const float2 inv2 = make_float2(inv, inv), s2 = make_float2(s, s), magic = make_float2(12582920.0f, 12582920.0f);
    float2 d[4 * W];  // -k
    float left = s >= 0x1p-21f && s < 65504.0f ? 0.0f : INFINITY;  // (others can be more than 7.5 steps)
#pragma unroll
    for (int j = 0; j < 4 * W; j++) {
        d[j] = __ffma2_rn(__ffma2_rn(v[j], inv2, magic), make_float2(-1.0f, -1.0f), magic);
        const float2 e = __ffma2_rn(d[j], s2, v[j]);
        left = kv4_max_nan(left, e.x, e.y);
    }
    // four codes k + 8 as the low 16 bits of 2^23 + 0x8888 + sum of 16^j k
    auto four = [](float2 a, float2 b) {
        const float f = fmaf(fmaf(fmaf(b.y, 16.0f, b.x), 16.0f, a.y), 16.0f, a.x);
        return __float_as_uint(8388608.0f + 34952.0f - f);
    };
    if (!(left <= 0.499998f * s) && left <= s) {  // near a tie: one step on from past half, and from half to even
        const float half = 0.5f * s;
        auto nearest = [&](float& d, float v) {
            const float e = fmaf(d, s, v), a = fabsf(e);
            if (a > half || (a == half && (__float_as_uint(magic.x - d) & 1))) d -= copysignf(1.0f, e);
        };
#pragma unroll
        for (int j = 0; j < 4 * W; j++) nearest(d[j].x, v[j].x), nearest(d[j].y, v[j].y);
    }
    const bool divide = !(left <= s);
#pragma unroll
    for (int i = 0; i < W; i++) {
        uint32_t w = __byte_perm(four(d[4 * i], d[4 * i + 1]), four(d[4 * i + 2], d[4 * i + 3]), 0x5410);
        if (divide) w = kv4_codes_div(x[2 * i], x[2 * i + 1], s);
        if (store) *reinterpret_cast<uint32_t*>(blk + kv4_word_off(hd, is_v, r, g, u + i)) = w;
    }
    if (store && u == 0) *reinterpret_cast<uint16_t*>(blk + kv4_scale_off(hd, is_v, r, g)) = __half_as_ushort(sh);
}

}  // namespace jl
