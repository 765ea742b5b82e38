// The 4-bit KV cache: rows quantised as they are appended, read back, and the
// entry points of the attention over it (jl_kv4_attn.cu). Layout: jl_kv4.cuh.
#include <cuda_bf16.h>

#include <climits>
#include <cmath>

#include "jl_internal.h"
#include "jl_kv4.cuh"

namespace jl {

constexpr int kKvThreads = 256;

__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 load4(const __half* p) {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
    return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ float4 load4(const __nv_bfloat16* p) {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    return make_float4(bf16_to_f32(w.x & 0xFFFFu), bf16_to_f32(w.x >> 16), bf16_to_f32(w.y & 0xFFFFu),
                       bf16_to_f32(w.y >> 16));
}

// Append: 16 lanes per (row, head, K or V, group) read 4 values each, reduce
// the group's maximum by shuffles and store its record. Bound by HBM (each
// value read once, an eighth of its fp32 size written).
template <typename T>
__global__ void __launch_bounds__(kKvThreads) k_kv4_append(kv4_dims c, int l, const T* __restrict__ k,
                                                           const T* __restrict__ v, long long ks, long long vs,
                                                           const int* __restrict__ slots,
                                                           const int* __restrict__ positions, long long ntask,
                                                           int* err) {
    griddep_wait();
    griddep_launch_dependents();
    const int i = threadIdx.x & 15, ng = c.hd / 64, per = c.KH * 2 * ng;
    const uint32_t mask = 0xFFFFu << (threadIdx.x & 16);
    const long long task = ((long long)blockIdx.x * kKvThreads + threadIdx.x) >> 4;
    if (task >= ntask) return;
    const long long n = task / per;
    const int rest = (int)(task - n * per), is_v = rest / (c.KH * ng), h = rest % (c.KH * ng) / ng, g = rest % ng;
    const int slot = slots[n], pos = positions[n];
    if (slot < 0 || slot >= c.slots || pos < 0 || pos >= c.maxT) {
        if (rest == 0 && i == 0 && err) atomicOr(err, kErrKvIndex);
        return;
    }
    const T* src = (is_v ? v + n * vs : k + n * ks) + h * c.hd + g * 64 + 4 * i;
    uint8_t* blk = c.run(slot, l, h) + (size_t)(pos / kKv4Rows) * kv4_block_bytes(c.hd);
    kv4_store_group(blk, c.hd, is_v, pos % kKv4Rows, g, load4(src), i, mask);
}

__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store8(__half* p, const float (&x)[8]) {
    __half2 h[4];
#pragma unroll
    for (int j = 0; j < 4; j++) h[j] = __floats2half2_rn(x[2 * j], x[2 * j + 1]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(h);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&x)[8]) {
    __nv_bfloat162 h[4];
#pragma unroll
    for (int j = 0; j < 4; j++) h[j] = __floats2bfloat162_rn(x[2 * j], x[2 * j + 1]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(h);
}

// Read back: thread = one code word (8 values) of (row, head, K or V, group);
// (n - 8) * s is exact in fp32 (4 by 11 bits), rounded once to a 16-bit type.
// A row outside the cache reads as zeros. Bound by HBM (the values written).
template <typename T>
__global__ void __launch_bounds__(kKvThreads) k_kv4_read(kv4_dims c, int l, T* __restrict__ k, T* __restrict__ v,
                                                         const int* __restrict__ slots,
                                                         const int* __restrict__ positions, long long ntask,
                                                         int* err) {
    griddep_wait();
    griddep_launch_dependents();
    const int ng = c.hd / 64, per = c.KH * 2 * ng * 8;
    const long long task = (long long)blockIdx.x * kKvThreads + threadIdx.x;
    if (task >= ntask) return;
    const long long n = task / per;
    const int rest = (int)(task - n * per), is_v = rest / (c.KH * ng * 8), hg = rest % (c.KH * ng * 8) / 8;
    const int u = rest % 8, h = hg / ng, g = hg % ng;
    const int slot = slots[n], pos = positions[n];
    float x[8] = {};
    if (slot < 0 || slot >= c.slots || pos < 0 || pos >= c.maxT) {
        if (rest == 0 && err) atomicOr(err, kErrKvIndex);
    } else {
        const uint8_t* blk = c.run(slot, l, h) + (size_t)(pos / kKv4Rows) * kv4_block_bytes(c.hd);
        const int r = pos % kKv4Rows;
        const uint32_t w = *reinterpret_cast<const uint32_t*>(blk + kv4_word_off(c.hd, is_v, r, g, u));
        const float s = half_bits_to_f32(*reinterpret_cast<const uint16_t*>(blk + kv4_scale_off(c.hd, is_v, r, g)));
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = __fmul_rn((float)((int)(w >> (4 * j) & 15u) - 8), s);
    }
    store8((is_v ? v : k) + (n * c.KH + h) * c.hd + g * 64 + 8 * u, x);
}

}  // namespace jl

namespace {

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

int jl_kv4_view(const jl_kv4* c, int l, jl::kv4_dims* out) {
    if (!c || !c->base || !aligned16(c->base) || (c->hd != 64 && c->hd != 128)) return JL_ERR_INVALID;
    if (c->slots < 1 || c->L < 1 || c->n_kv < 1 || c->maxT < 1 || l < 0 || l >= c->L) return JL_ERR_INVALID;
    if (c->maxT > INT_MAX - jl::kKv4Rows) return JL_ERR_INVALID;
    out->base = static_cast<uint8_t*>(c->base);
    out->slots = c->slots, out->L = c->L, out->KH = c->n_kv, out->hd = c->hd, out->maxT = c->maxT;
    out->nb = (c->maxT + jl::kKv4Rows - 1) / jl::kKv4Rows;
    return JL_OK;
}

extern "C" long long jl_kv4_bytes(const jl_kv4* c) {
    if (!c || (c->hd != 64 && c->hd != 128) || c->slots < 1 || c->L < 1 || c->n_kv < 1 || c->maxT < 1) return -1;
    const long long nb = ((long long)c->maxT + jl::kKv4Rows - 1) / jl::kKv4Rows;
    long long n = 0;
    if (__builtin_mul_overflow((long long)c->slots * c->L, (long long)c->n_kv, &n) ||
        __builtin_mul_overflow(n, nb * jl::kv4_block_bytes(c->hd), &n))
        return -1;
    return n;
}

namespace {

template <typename T>
int launch_append(const jl::kv4_dims& c, int l, const void* k, const void* v, long long ks, long long vs,
                  const int* slots, const int* positions, int N, int* err, cudaStream_t s) {
    using namespace jl;
    const long long ntask = (long long)N * c.KH * 2 * (c.hd / 64);
    const long long blocks = (ntask * 16 + kKvThreads - 1) / kKvThreads;
    if (blocks > INT_MAX) return JL_ERR_INVALID;
    return launch(k_kv4_append<T>, dim3((unsigned)blocks), dim3(kKvThreads), 0, s, c, l, (const T*)k, (const T*)v, ks,
                  vs, slots, positions, ntask, err);
}

template <typename T>
int launch_read(const jl::kv4_dims& c, int l, const int* slots, const int* positions, int N, void* k, void* v,
                int* err, cudaStream_t s) {
    using namespace jl;
    const long long ntask = (long long)N * c.KH * 2 * (c.hd / 64) * 8;
    const long long blocks = (ntask + kKvThreads - 1) / kKvThreads;
    if (blocks > INT_MAX) return JL_ERR_INVALID;
    return launch(k_kv4_read<T>, dim3((unsigned)blocks), dim3(kKvThreads), 0, s, c, l, (T*)k, (T*)v, slots, positions,
                  ntask, err);
}

}  // namespace

extern "C" int jl_kv4_append(const jl_kv4* c, int l, const void* k, const void* v, int dtype, long long k_stride,
                             long long v_stride, const int* slots, const int* positions, int N, int* dev_status,
                             void* stream) {
    jl::kv4_dims d;
    const int rc = jl_kv4_view(c, l, &d);
    if (rc) return rc;
    if (N < 0 || dtype < JL_F32 || dtype > JL_BF16) return JL_ERR_INVALID;
    if (N == 0) return JL_OK;
    const long long unit = dtype == JL_F32 ? 4 : 8, row = (long long)d.KH * d.hd;
    if (!k || !v || !slots || !positions || !aligned16(k) || !aligned16(v) || k_stride % unit || v_stride % unit ||
        (N > 1 && (k_stride < row || v_stride < row)))
        return JL_ERR_INVALID;
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == JL_F32) return launch_append<float>(d, l, k, v, k_stride, v_stride, slots, positions, N, dev_status, s);
    if (dtype == JL_F16) return launch_append<__half>(d, l, k, v, k_stride, v_stride, slots, positions, N, dev_status, s);
    return launch_append<__nv_bfloat16>(d, l, k, v, k_stride, v_stride, slots, positions, N, dev_status, s);
}

extern "C" int jl_kv4_read(const jl_kv4* c, int l, const int* slots, const int* positions, int N, void* k, void* v,
                           int dtype, int* dev_status, void* stream) {
    jl::kv4_dims d;
    const int rc = jl_kv4_view(c, l, &d);
    if (rc) return rc;
    if (N < 0 || dtype < JL_F32 || dtype > JL_BF16) return JL_ERR_INVALID;
    if (N == 0) return JL_OK;
    if (!k || !v || !slots || !positions || !aligned16(k) || !aligned16(v)) return JL_ERR_INVALID;
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == JL_F32) return launch_read<float>(d, l, slots, positions, N, k, v, dev_status, s);
    if (dtype == JL_F16) return launch_read<__half>(d, l, slots, positions, N, k, v, dev_status, s);
    return launch_read<__nv_bfloat16>(d, l, slots, positions, N, k, v, dev_status, s);
}

extern "C" long long jl_kv4_attn_ws(const jl_kv4* c, int B, int T, int H) {
    jl::kv4_dims d;
    if (jl_kv4_view(c, 0, &d) || B < 0 || T < 1 || H < 1 || H % d.KH) return -1;
    return jl_kv4_attn_ws_bytes(d, B, T, H);
}

extern "C" int jl_kv4_attn(const jl_kv4* c, int l, const void* q, int dtype, long long q_stride, const int* slots,
                           const int* lens, int longest, int B, int T, int H, float scale, void* out, void* ws,
                           long long ws_bytes, int* dev_status, void* stream) {
    jl::kv4_dims d;
    const int rc = jl_kv4_view(c, l, &d);
    if (rc) return rc;
    if (B < 0 || T < 1 || H < 1 || H % d.KH || dtype < JL_F32 || dtype > JL_BF16 || !std::isfinite(scale) ||
        longest < 0 || longest > d.maxT)
        return JL_ERR_INVALID;
    if ((long long)B * T > INT_MAX / H) return JL_ERR_INVALID;
    if (B == 0) return JL_OK;
    const long long unit = dtype == JL_F32 ? 4 : 8, row = (long long)H * d.hd;
    if (!q || !slots || !lens || !out || !aligned16(q) || !aligned16(out) || q_stride % unit ||
        ((long long)B * T > 1 && q_stride < row))
        return JL_ERR_INVALID;
    const long long need = jl_kv4_attn_ws_bytes(d, B, T, H);
    if (need > 0 && (!ws || !aligned16(ws) || ws_bytes < need)) return JL_ERR_INVALID;
    jl_kv4_attn_args a;
    a.q = q, a.dtype = dtype, a.q_stride = q_stride, a.slots = slots, a.lens = lens, a.len_add = 0;
    a.longest = longest ? longest : d.maxT, a.B = B, a.T = T, a.H = H, a.scale = scale, a.out = out, a.outT = nullptr;
    a.outT_ld = 0, a.ws = ws, a.err = dev_status;
    return jl_launch_kv4_attn(d, l, a, (cudaStream_t)stream);
}
