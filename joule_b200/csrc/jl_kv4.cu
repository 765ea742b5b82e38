// The 4-bit KV cache: rows quantised as they are appended, read back, and the
// entry points of the attention over it (jl_kv4_attn.cu). Layout: jl_kv4.cuh.
#include <cuda_bf16.h>

#include <algorithm>
#include <climits>
#include <cmath>

#include "jl_internal.h"
#include "jl_kv4.cuh"

namespace jl {

constexpr int kKvThreads = 256;

// Eight values as they lie, and as fp32 (apart: a conversion among the loads would
// wait for each before the next is issued). STREAM: first to leave L2 (a long call's
// rows, read once).
template <typename T>
struct kv4_eight {
    uint4 w;
};
template <>
struct kv4_eight<float> {
    float4 x, y;
};
template <bool STREAM, typename V>
__device__ __forceinline__ V load_from(const void* p) {
    return STREAM ? __ldcs(static_cast<const V*>(p)) : *static_cast<const V*>(p);
}
template <bool STREAM>
__device__ __forceinline__ void load8(const float* p, kv4_eight<float>& v) {
    v.x = load_from<STREAM, float4>(p);
    v.y = load_from<STREAM, float4>(p + 4);
}
template <bool STREAM, typename T>
__device__ __forceinline__ void load8(const T* p, kv4_eight<T>& v) {
    v.w = load_from<STREAM, uint4>(p);
}
__device__ __forceinline__ void to_fp32(const kv4_eight<float>& v, float4& x, float4& y) { x = v.x, y = v.y; }
__device__ __forceinline__ void to_fp32(const kv4_eight<__half>& v, float4& x, float4& y) {
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v.w.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&v.w.y));
    const float2 c = __half22float2(*reinterpret_cast<const __half2*>(&v.w.z));
    const float2 d = __half22float2(*reinterpret_cast<const __half2*>(&v.w.w));
    x = make_float4(a.x, a.y, b.x, b.y);
    y = make_float4(c.x, c.y, d.x, d.y);
}
__device__ __forceinline__ void to_fp32(const kv4_eight<__nv_bfloat16>& v, float4& x, float4& y) {
    auto lo = [](uint32_t w) { return __uint_as_float(w << 16); };
    auto hi = [](uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); };
    x = make_float4(lo(v.w.x), hi(v.w.x), lo(v.w.y), hi(v.w.y));
    y = make_float4(lo(v.w.z), hi(v.w.z), lo(v.w.w), hi(v.w.w));
}

// Append and read back: block (row chunk, K or V of a head; a chunk's heads next to one
// another, or rows of many heads are fetched in pieces: append 29 -> 26 us), a row's
// head by HD / values-per-lane lanes, several rows of a lane in flight. (An index of one
// flat item per lane took three times the instructions and bound both kernels by
// issue: 8,179 rows x 16 heads 65 + 47 us under ncu.) Rows in flight in long calls:
// append 4 of fp32 at head dim 128 (8 by registers 35 us against 26, 2 27.5), else 2 (4:
// bf16 27 us against 23, fp32 at head dim 64 16.3 against 14.7), read 8 (4: 27 against 24).
constexpr int kKvReadRows = 8;
template <int HD, typename T>
constexpr int kKvAppendRows = HD * sizeof(T) == 512 ? 4 : 2;

// Append: a lane has 32 bytes of a row, W code words (8 values each); the 8 / W lanes of
// a group reduce its maximum by shuffles and store its record. 8,179 rows of 16 heads of 128: fp32 26 us
// (23 at the copy rate), bound by HBM and issue alike; bf16 23 us (13), by issue (a word
// a lane: 27).
template <int HD, typename T, int STEPS>
__global__ void __launch_bounds__(kKvThreads) k_kv4_append(kv4_dims c, int l, const T* __restrict__ k,
                                                           const T* __restrict__ v, long long ks, long long vs,
                                                           const int* __restrict__ slots,
                                                           const int* __restrict__ positions, int N, int* err) {
    constexpr int W = 4 / sizeof(T), LPR = HD / (8 * W), ROWS = kKvThreads / LPR;  // lanes per row, rows per step
    griddep_wait();
    griddep_launch_dependents();
    const int hv = blockIdx.x % (2 * c.KH), chunk = blockIdx.x / (2 * c.KH);
    const int is_v = hv & 1, h = hv >> 1, w = threadIdx.x % LPR * W, g = w / 8, u = w % 8;
    const long long stride = is_v ? vs : ks;
    const int n0 = chunk * ROWS * STEPS + threadIdx.x / LPR;
    const T* src = (is_v ? v : k) + h * HD + 8 * w;
    kv4_eight<T> raw[STEPS][W];
    int slot[STEPS], pos[STEPS];
#pragma unroll
    for (int j = 0; j < STEPS; j++) {  // (rows past the last: the last, not stored)
        const int n = min(n0 + j * ROWS, N - 1);
        slot[j] = __ldg(slots + n), pos[j] = __ldg(positions + n);
#pragma unroll
        for (int i = 0; i < W; i++) load8<(STEPS > 1)>(src + n * stride + 8 * i, raw[j][i]);
    }
    uint8_t* base = c.run(0, l, h);
    const size_t per_slot = (size_t)c.L * c.KH * c.nb * kv4_block_bytes(HD);
#pragma unroll
    for (int j = 0; j < STEPS; j++) {
        const bool in = n0 + j * ROWS < N, ok = in && (unsigned)slot[j] < (unsigned)c.slots && (unsigned)pos[j] < (unsigned)c.maxT;
        if (in && !ok && hv == 0 && w == 0 && err) atomicOr(err, kErrKvIndex);
        uint8_t* blk = base + (unsigned)slot[j] * per_slot + (size_t)((unsigned)pos[j] / kKv4Rows) * kv4_block_bytes(HD);
        float4 x[2 * W];
#pragma unroll
        for (int i = 0; i < W; i++) to_fp32(raw[j][i], x[2 * i], x[2 * i + 1]);
        kv4_store_group<W>(blk, HD, is_v, pos[j] % kKv4Rows, g, u, x, ok);
    }
}

// 16 bytes of values. STREAM: first to leave L2 (outputs of long calls, which would
// push out the cache's records and one another: 30,000 rows x 4 heads 33 -> 26 us).
template <bool STREAM>
__device__ __forceinline__ void store16(void* p, uint4 v) {
    if (STREAM) __stcs(reinterpret_cast<uint4*>(p), v);
    else *reinterpret_cast<uint4*>(p) = v;
}
template <bool STREAM>
__device__ __forceinline__ void store_values(float* p, const float (&x)[4]) {
    store16<STREAM>(p, make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])));
}
template <bool STREAM>
__device__ __forceinline__ void store_values(__half* p, const float (&x)[8]) {
    __half2 h[4];
#pragma unroll
    for (int j = 0; j < 4; j++) h[j] = __floats2half2_rn(x[2 * j], x[2 * j + 1]);
    store16<STREAM>(p, *reinterpret_cast<uint4*>(h));
}
template <bool STREAM>
__device__ __forceinline__ void store_values(__nv_bfloat16* p, const float (&x)[8]) {
    __nv_bfloat162 h[4];
#pragma unroll
    for (int j = 0; j < 4; j++) h[j] = __floats2bfloat162_rn(x[2 * j], x[2 * j + 1]);
    store16<STREAM>(p, *reinterpret_cast<uint4*>(h));
}

// Read back: a lane writes 16 bytes (half a code word's values in fp32, a word's in
// 16 bits); (n - 8) * s is exact in fp32 (4 by 11 bits), rounded once to a 16-bit
// type. A row outside the cache reads as zeros. Bound by HBM (the values written):
// 8,179 rows of 16 heads of 128 in fp32 24 us, 23 at the copy rate.
template <int HD, typename T, int STEPS>
__global__ void __launch_bounds__(kKvThreads) k_kv4_read(kv4_dims c, int l, T* __restrict__ k, T* __restrict__ v,
                                                         const int* __restrict__ slots,
                                                         const int* __restrict__ positions, int N, int* err) {
    constexpr int VPT = 16 / sizeof(T), LPR = HD / VPT, ROWS = kKvThreads / LPR;
    griddep_wait();
    griddep_launch_dependents();
    const int hv = blockIdx.x % (2 * c.KH), chunk = blockIdx.x / (2 * c.KH);
    const int is_v = hv & 1, h = hv >> 1, e = threadIdx.x % LPR * VPT, g = e / 64, u = e % 64 / 8;
    const int n0 = chunk * ROWS * STEPS + threadIdx.x / LPR;
    const uint8_t* base = c.run(0, l, h);
    const size_t per_slot = (size_t)c.L * c.KH * c.nb * kv4_block_bytes(HD);
    uint32_t word[STEPS];
    uint16_t scale[STEPS];
    int slot[STEPS], pos[STEPS];
#pragma unroll
    for (int j = 0; j < STEPS; j++) {  // (rows past the last: the last, not stored)
        const int n = min(n0 + j * ROWS, N - 1);
        slot[j] = __ldg(slots + n), pos[j] = __ldg(positions + n);
    }
#pragma unroll
    for (int j = 0; j < STEPS; j++) {
        const bool ok = (unsigned)slot[j] < (unsigned)c.slots && (unsigned)pos[j] < (unsigned)c.maxT;
        if (!ok) {
            if (hv == 0 && e == 0 && err) atomicOr(err, kErrKvIndex);
            slot[j] = 0, pos[j] = -1;  // some record, read as zeros
        }
        const unsigned at = max(pos[j], 0);
        const uint8_t* blk = base + (unsigned)slot[j] * per_slot + (size_t)(at / kKv4Rows) * kv4_block_bytes(HD);
        word[j] = *reinterpret_cast<const uint32_t*>(blk + kv4_word_off(HD, is_v, at % kKv4Rows, g, u));
        scale[j] = *reinterpret_cast<const uint16_t*>(blk + kv4_scale_off(HD, is_v, at % kKv4Rows, g));
    }
    T* dst = (is_v ? v : k) + ((size_t)n0 * c.KH + h) * HD + e;
#pragma unroll
    for (int j = 0; j < STEPS; j++) {
        if (n0 + j * ROWS >= N) break;
        const float s = pos[j] < 0 ? 0.0f : half_bits_to_f32(scale[j]);
        if (pos[j] < 0) word[j] = 0x88888888u;
        // nibble q of a half word left in place in 2^23's mantissa: 2^23 + 16^q n, then n - 8 by an exact FMA
        float x[VPT];
#pragma unroll
        for (int q = 0; q < VPT; q++) {
            const uint32_t half = VPT == 4 ? word[j] >> (e % 8 * 4) : q < 4 ? word[j] : word[j] >> 16;
            const float unit = q % 4 == 0 ? 1.0f : q % 4 == 1 ? 0.0625f : q % 4 == 2 ? 0.00390625f : 0.000244140625f;
            x[q] = __fmul_rn(fmaf(__uint_as_float((half & (15u << (4 * (q % 4)))) | 0x4B000000u), unit, -8388608.0f * unit - 8.0f), s);
        }
        store_values<(STEPS > 1)>(dst + (size_t)j * ROWS * c.KH * HD, x);
    }
}

}  // namespace jl

namespace {

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

int jl_kv4_view(const jl_kv4* c, int l, jl::kv4_dims* out) {
    if (!c || !c->base || !aligned16(c->base) || (c->hd != 64 && c->hd != 128)) return JL_ERR_INVALID;
    if (c->slots < 1 || c->L < 1 || c->n_kv < 1 || c->maxT < 1 || l < 0 || l >= c->L) return JL_ERR_INVALID;
    if (c->maxT > INT_MAX - jl::kKv4Rows || c->n_kv > 4096) return JL_ERR_INVALID;
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

// Several rows of a lane in flight for calls that fill the device with blocks all
// the same, one row for short ones.
template <int HD, typename T, int VPT, int STEPS, typename K1, typename K, typename... Args>
int launch_rows(K1 one, K many, int KH, int N, cudaStream_t s, Args... args) {
    using namespace jl;
    const int rows = kKvThreads / (HD / VPT);
    const bool big = (long long)N * KH >= (long long)rows * 1024;
    const int per = big ? rows * STEPS : rows;
    const long long blocks = ((long long)N + per - 1) / per * 2 * KH;
    if (blocks > INT_MAX) return JL_ERR_INVALID;
    const dim3 grid((unsigned)blocks);
    return big ? launch(many, grid, dim3(kKvThreads), 0, s, args...) : launch(one, grid, dim3(kKvThreads), 0, s, args...);
}

template <int HD, typename T>
int launch_append(const jl::kv4_dims& c, int l, const void* k, const void* v, long long ks, long long vs,
                  const int* slots, const int* positions, int N, int* err, cudaStream_t s) {
    using namespace jl;
    return launch_rows<HD, T, 32 / sizeof(T), kKvAppendRows<HD, T>>(k_kv4_append<HD, T, 1>, k_kv4_append<HD, T, kKvAppendRows<HD, T>>, c.KH, N, s, c, l, (const T*)k,
                                 (const T*)v, ks, vs, slots, positions, N, err);
}

template <int HD, typename T>
int launch_read(const jl::kv4_dims& c, int l, const int* slots, const int* positions, int N, void* k, void* v,
                int* err, cudaStream_t s) {
    using namespace jl;
    return launch_rows<HD, T, 16 / sizeof(T), kKvReadRows>(k_kv4_read<HD, T, 1>, k_kv4_read<HD, T, kKvReadRows>, c.KH, N, s, c, l, (T*)k,
                                              (T*)v, slots, positions, N, err);
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
    const bool wide = d.hd == 128;
    if (dtype == JL_F32) return (wide ? launch_append<128, float> : launch_append<64, float>)(d, l, k, v, k_stride, v_stride, slots, positions, N, dev_status, s);
    if (dtype == JL_F16) return (wide ? launch_append<128, __half> : launch_append<64, __half>)(d, l, k, v, k_stride, v_stride, slots, positions, N, dev_status, s);
    return (wide ? launch_append<128, __nv_bfloat16> : launch_append<64, __nv_bfloat16>)(d, l, k, v, k_stride, v_stride, slots, positions, N, dev_status, s);
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
    const bool wide = d.hd == 128;
    if (dtype == JL_F32) return (wide ? launch_read<128, float> : launch_read<64, float>)(d, l, slots, positions, N, k, v, dev_status, s);
    if (dtype == JL_F16) return (wide ? launch_read<128, __half> : launch_read<64, __half>)(d, l, slots, positions, N, k, v, dev_status, s);
    return (wide ? launch_read<128, __nv_bfloat16> : launch_read<64, __nv_bfloat16>)(d, l, slots, positions, N, k, v, dev_status, s);
}

extern "C" long long jl_kv4_attn_ws(const jl_kv4* c, int B, int T, int H, int longest) {
    jl::kv4_dims d;
    if (jl_kv4_view(c, 0, &d) || B < 0 || T < 1 || H < 1 || H % d.KH || (long long)B * T > INT_MAX / H || longest < 0 ||
        longest > d.maxT)
        return -1;
    return B ? jl_kv4_attn_ws_bytes(d, B, T, H, longest ? longest : d.maxT) : 0;
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
    if ((long long)B * T > INT_MAX / H || H > INT_MAX / d.hd) return JL_ERR_INVALID;  // rows, and a row's values
    if (B == 0) return JL_OK;
    const long long unit = dtype == JL_F32 ? 4 : 8, row = (long long)H * d.hd;
    if (!q || !slots || !lens || !out || !aligned16(q) || !aligned16(out) || q_stride % unit ||
        ((long long)B * T > 1 && q_stride < row))
        return JL_ERR_INVALID;
    // out takes intermediate sums in some forms, and rows of q are read more than once
    const long long n = (long long)B * T, esize = dtype == JL_F32 ? 4 : 2;
    const char *q0 = static_cast<const char*>(q), *o0 = static_cast<const char*>(out);
    if (q0 < o0 + n * row * esize && o0 < q0 + ((n > 1 ? (n - 1) * q_stride : 0) + row) * esize) return JL_ERR_INVALID;
    const long long need = jl_kv4_attn_ws_bytes(d, B, T, H, longest ? longest : d.maxT);
    if (need > 0 && (!ws || !aligned16(ws) || ws_bytes < need)) return JL_ERR_INVALID;
    jl_kv4_attn_args a;
    a.q = q, a.dtype = dtype, a.q_stride = q_stride, a.slots = slots, a.lens = lens, a.len_add = 0;
    a.longest = longest ? longest : d.maxT, a.B = B, a.T = T, a.H = H, a.scale = scale, a.out = out, a.outT = nullptr;
    a.outT_ld = 0, a.ws = ws, a.err = dev_status;
    return jl_launch_kv4_attn(d, l, a, (cudaStream_t)stream);
}
