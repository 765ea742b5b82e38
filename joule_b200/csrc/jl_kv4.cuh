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

// Quantises a group of 64 values held by 8 consecutive lanes (lane u of the 8 has
// word u: values 8u .. 8u + 7, x then y) and stores it as (row r, group g) of block
// `blk` when `store`. A code is the step nearest to the exact x / s. Its first guess
// is the product with 1 / s, rounded by adding 1.5 * 2^23 + 8; the guess n stands when
// what is left, x - (n - 8) s (exact: 11 by 4 bits from a value of the same size), is
// clearly below half a step, and the lane divides when it is not (a tie or nearly one,
// a NaN, an infinity, a scale of 0, a value past the largest scale). Beyond the
// record's own rules: a scale that fp16 cannot hold stays at its largest number
// (values past 7 * 65504 saturate) and a NaN becomes zero, so what the cache holds is
// always finite. All lanes of the warp call it.
__device__ __forceinline__ void kv4_store_group(uint8_t* blk, int hd, int is_v, int r, int g, int u, float4 x, float4 y,
                                                bool store) {
    const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    float amax = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) amax = fmaxf(amax, fabsf(v[j]));
#pragma unroll
    for (int o = 4; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const __half sh = __float2half_rn(fminf(__fdiv_rn(fmaxf(amax, 1e-12f), 7.0f), 65504.0f));
    const float s = __half2float(sh), inv = __frcp_rn(s), bound = 0.4999f * s;
    uint32_t w = 0;
    bool sure = s >= 0x1p-21f && s < 65504.0f;  // (others can leave values past 7.5 steps)
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float q = fmaf(v[j], inv, 12582920.0f);
        const float left = fmaf(12582920.0f - q, s, v[j]);
        sure = sure && fabsf(left) <= bound;
        w |= (__float_as_uint(q) & 15u) << (4 * j);
    }
    if (!sure) w = kv4_codes_div(x, y, s);
    if (!store) return;
    *reinterpret_cast<uint32_t*>(blk + kv4_word_off(hd, is_v, r, g, u)) = w;
    if (u == 0) *reinterpret_cast<uint16_t*>(blk + kv4_scale_off(hd, is_v, r, g)) = __half_as_ushort(sh);
}

}  // namespace jl
