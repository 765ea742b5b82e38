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

// Quantises one group of 64 values held by 16 consecutive lanes (lane i of the
// 16 holds values 4i..4i+3) and stores it as (row r, group g) of block `blk`.
// The quotient is an IEEE division, so a code is the nearest step to the exact
// x / s. Beyond the record's own rules: a scale that fp16 cannot hold stays at
// its largest number (values past 7 * 65504 saturate) and a NaN becomes zero,
// so what the cache holds is always finite. All 16 lanes of the group call it.
__device__ __forceinline__ void kv4_store_group(uint8_t* blk, int hd, int is_v, int r, int g, float4 x, int i,
                                                uint32_t mask) {
    float amax = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
#pragma unroll
    for (int o = 8; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(mask, amax, o));
    const __half sh = __float2half_rn(fminf(__fdiv_rn(fmaxf(amax, 1e-12f), 7.0f), 65504.0f));
    const float s = __half2float(sh);
    const float v[4] = {x.x, x.y, x.z, x.w};
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float q = rintf(__fdiv_rn(v[j], s));
        const int n = q != q ? 8 : (int)fminf(fmaxf(q, -8.0f), 7.0f) + 8;
        w |= (uint32_t)n << (4 * j);
    }
    w |= __shfl_down_sync(mask, w, 1) << 16;  // the odd lane's four values
    if ((i & 1) == 0) *reinterpret_cast<uint32_t*>(blk + kv4_word_off(hd, is_v, r, g, i >> 1)) = w;
    if (i == 0) *reinterpret_cast<uint16_t*>(blk + kv4_scale_off(hd, is_v, r, g)) = __half_as_ushort(sh);
}

}  // namespace jl
