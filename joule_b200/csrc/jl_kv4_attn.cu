// Attention over the 4-bit KV cache (layout: jl_kv4.cuh).
//
// out[b, i, h] = sum_t softmax_t(scale * q[b, i, h] . K_t) V_t over the first
// lens[b] - T + 1 + i cached positions of sequence b's slot.
#include <cuda_bf16.h>

#include "jl_internal.h"
#include "jl_kv4.cuh"

namespace jl {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_f32(float* p, float x) { *p = x; }
__device__ __forceinline__ void from_f32(__half* p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void from_f32(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// Block = one query row (b, i, h): four warps take every fourth position with a
// running maximum and sum each and meet in shared memory.
template <int HD, typename T>
__global__ void __launch_bounds__(128) k_kv4_attn_row(kv4_dims c, int l, jl_kv4_attn_args a) {
    griddep_wait();
    griddep_launch_dependents();
    constexpr int NG = HD / 64, PL = HD / 32;  // groups, values per lane
    const int h = blockIdx.x % a.H, i = blockIdx.x / a.H % a.T, b = blockIdx.x / a.H / a.T;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, kh = h / (a.H / c.KH);
    const int slot = a.slots[b], len = a.lens[b] + a.len_add;
    bool ok = slot >= 0 && slot < c.slots && len >= 0 && len <= a.longest;
    if (!ok && threadIdx.x == 0 && a.err) atomicOr(a.err, kErrKvIndex);
    const int n = ok ? max(0, len - a.T + 1 + i) : 0;
    const T* q = static_cast<const T*>(a.q) + ((long long)b * a.T + i) * a.q_stride + h * HD;
    float qv[PL], o[PL], m = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int e = 0; e < PL; e++) qv[e] = to_f32(q[lane * PL + e]) * a.scale, o[e] = 0.0f;
    const int d0 = lane * PL, g = d0 / 64, u = d0 % 64 / 8, sh = d0 % 8 * 4;
    const uint8_t* run = c.run(ok ? slot : 0, l, kh);
    for (int t = warp; t < n; t += 4) {
        const uint8_t* blk = run + (size_t)(t / kKv4Rows) * kv4_block_bytes(HD);
        const int r = t % kKv4Rows;
        const uint32_t kw = *reinterpret_cast<const uint32_t*>(blk + kv4_word_off(HD, 0, r, g, u)) >> sh;
        const uint32_t vw = *reinterpret_cast<const uint32_t*>(blk + kv4_word_off(HD, 1, r, g, u)) >> sh;
        const float ks = half_bits_to_f32(*reinterpret_cast<const uint16_t*>(blk + kv4_scale_off(HD, 0, r, g)));
        const float vs = half_bits_to_f32(*reinterpret_cast<const uint16_t*>(blk + kv4_scale_off(HD, 1, r, g)));
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < PL; e++) s += qv[e] * ((float)((int)(kw >> (4 * e) & 15u) - 8) * ks);
#pragma unroll
        for (int w = 16; w; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
        const float m1 = fmaxf(m, s), alpha = __expf(m - m1), p = __expf(s - m1);
        sum = sum * alpha + p;
        m = m1;
#pragma unroll
        for (int e = 0; e < PL; e++) o[e] = o[e] * alpha + p * ((float)((int)(vw >> (4 * e) & 15u) - 8) * vs);
    }
    __shared__ float so[4][HD], sm[4], ss[4];
#pragma unroll
    for (int e = 0; e < PL; e++) so[warp][d0 + e] = o[e];
    if (lane == 0) sm[warp] = m, ss[warp] = sum;
    __syncthreads();
    float M = -INFINITY, S = 0.0f;
    for (int w = 0; w < 4; w++) M = fmaxf(M, sm[w]);
    float f[4];
    for (int w = 0; w < 4; w++) {
        f[w] = sm[w] == -INFINITY ? 0.0f : __expf(sm[w] - M);
        S += ss[w] * f[w];
    }
    for (int d = threadIdx.x; d < HD; d += 128) {
        float x = 0.0f;
        for (int w = 0; w < 4; w++) x += so[w][d] * f[w];
        x = S == 0.0f ? 0.0f : x / S;
        const long long row = (long long)b * a.T + i;
        from_f32(static_cast<T*>(a.out) + (row * a.H + h) * HD + d, x);
        if (a.outT) a.outT[((size_t)h * HD + d) * a.outT_ld + row] = x;
    }
}

}  // namespace jl

long long jl_kv4_attn_ws_bytes(const jl::kv4_dims&, int, int, int) { return 0; }

namespace {

template <int HD>
int launch_hd(const jl::kv4_dims& c, int l, const jl_kv4_attn_args& a, cudaStream_t s) {
    using namespace jl;
    const dim3 grid((unsigned)(a.B * a.T * a.H)), block(128);
    if (a.dtype == JL_F32) return launch(k_kv4_attn_row<HD, float>, grid, block, 0, s, c, l, a);
    if (a.dtype == JL_F16) return launch(k_kv4_attn_row<HD, __half>, grid, block, 0, s, c, l, a);
    return launch(k_kv4_attn_row<HD, __nv_bfloat16>, grid, block, 0, s, c, l, a);
}

}  // namespace

int jl_launch_kv4_attn(const jl::kv4_dims& c, int l, const jl_kv4_attn_args& a, cudaStream_t s) {
    return c.hd == 64 ? launch_hd<64>(c, l, a, s) : launch_hd<128>(c, l, a, s);
}
