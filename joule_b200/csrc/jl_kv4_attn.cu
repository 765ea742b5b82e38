// Attention over the 4-bit KV cache (layout: jl_kv4.cuh).
//
// out[b, i, h] = sum_t softmax_t(scale * q[b, i, h] . K_t) V_t over the first
// lens[b] - T + 1 + i cached positions of sequence b's slot.
//
// The query rows (i, h) of one (sequence, kv head) form tiles of 8 rows (one
// group of 8 heads in a decode step). A segment is one tile over the blocks of
// its (sequence, kv head); all segments' blocks in a row are cut into equal
// runs, one per warp, whatever the lengths are (the cut is computed on the
// device from lens, so captured graphs follow growing sequences). A segment
// that one warp covers is written by it; the parts of the others meet in
// k_kv4_merge.
#include <cuda_bf16.h>

#include <algorithm>
#include <climits>

#include "jl_internal.h"
#include "jl_kv4.cuh"

namespace jl {

constexpr int kKvRing = 2;     // cache blocks in a warp's ring
constexpr int kKvTile = 8;     // query rows of a tile
constexpr float kLoScale = 2048.0f;
// A new reference is 2^kHeadroom above the largest score, so that weights stay
// at or below 1 without a rescaling of the sums at every new maximum (most blocks
// of a short run have one in some row).
constexpr float kHeadroom = 4.0f;

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

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

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t h2bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }

__device__ __forceinline__ float2 f2(float x) { return make_float2(x, x); }

// A pair as fp16 pairs: hi = the nearest, lo = 2048 times what hi misses, so
// that hi + lo / 2048 holds 22 bits and lo does not underflow before hi does.
__device__ __forceinline__ void split2(float2 x, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __float22half2_rn(x);
    hi = h2bits(h);
    lo = h2bits(__float22half2_rn(__ffma2_rn(__half22float2(h), f2(-kLoScale), __fmul2_rn(x, f2(kLoScale)))));
}

// The scales of positions r, r + 1 of a section: per group a pair over the two.
template <int NG>
__device__ __forceinline__ void scale_pairs(const uint8_t* section, int r, float2 (&sc)[NG]) {
    const uint8_t* p = section + r * 2 * NG;
    if (NG == 2) {
        const uint2 w = *reinterpret_cast<const uint2*>(p);
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x));
        const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
        sc[0] = make_float2(a.x, b.x);
        sc[NG - 1] = make_float2(a.y, b.y);
    } else {
        sc[0] = __half22float2(*reinterpret_cast<const __half2*>(p));
    }
}

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

// Blocks of sequence b (0 when its slot or length is outside the cache), and
// what it counts in the cut: its blocks, or 1 when segments are not cut.
struct kv4_seqs {
    const int* slots;
    const int* lens;
    int len_add, longest, nslots, whole;
    __device__ int len(int b) const {
        const int n = __ldg(lens + b) + len_add, s = __ldg(slots + b);
        return s >= 0 && s < nslots && n >= 0 && n <= longest ? n : -1;
    }
    __device__ int blocks(int b) const { return (max(0, len(b)) + kKv4Rows - 1) / kKv4Rows; }
    __device__ int weight(int b) const { return whole ? len(b) > 0 : blocks(b); }
};

// The sum of weights over all sequences, and the sequence that holds unit u
// when a sequence has S segments of its weight: b and the unit's offset in it
// (b = B when u is past the end). Called by a whole warp.
__device__ __forceinline__ uint32_t warp_total(const kv4_seqs& q, int B) {
    uint32_t n = 0;
    for (int b = threadIdx.x & 31; b < B; b += 32) n += q.weight(b);
#pragma unroll
    for (int o = 16; o; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    return n;
}
__device__ __forceinline__ void warp_find(const kv4_seqs& q, int B, uint32_t S, uint32_t u, int& b_out, uint32_t& off) {
    const int lane = threadIdx.x & 31;
    uint32_t base = 0;
    for (int b0 = 0; b0 < B; b0 += 32) {
        const uint32_t n = b0 + lane < B ? q.weight(b0 + lane) * S : 0;
        uint32_t inc = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, base + inc > u);
        if (past) {
            const int w = __ffs(past) - 1;
            b_out = b0 + w;
            off = u - (base + __shfl_sync(0xffffffffu, inc - n, w));
            return;
        }
        base += __shfl_sync(0xffffffffu, inc, 31);
    }
    b_out = B;
    off = 0;
}

// n units in `parts` runs whose sizes differ by one at most, the longer first:
// run i begins at start(i), and unit u is in run of(u). No run is empty when
// parts <= n.
struct kv4_split {
    uint32_t parts, q, r;
    __device__ kv4_split(uint32_t n, uint32_t parts_) : parts(parts_), q(n / parts_), r(n - n / parts_ * parts_) {}
    __device__ uint32_t start(uint32_t i) const { return i * q + min(i, r); }
    __device__ uint32_t of(uint32_t u) const { return u < r * (q + 1) ? u / (q + 1) : r + (u - r * (q + 1)) / q; }
};

// The cut of U units over at most `blocks` blocks of NW warps: ctas blocks take
// a share each and nw of a block's warps share that alike, in order (few units
// spread over all blocks first). U >= 1.
struct kv4_cut {
    uint32_t ctas, nw;
    kv4_split by_block;
    __device__ kv4_cut(uint32_t U, uint32_t blocks, uint32_t NW)
        : ctas(min(blocks, U)), nw(min(NW, U / min(blocks, U))), by_block(U, min(blocks, U)) {}
    __device__ uint32_t start(uint32_t c) const { return by_block.start(c); }
    __device__ kv4_split by_warp(uint32_t c) const { return kv4_split(start(c + 1) - start(c), nw); }
    __device__ uint32_t warp_of(uint32_t u) const {  // nw * block + warp
        const uint32_t c = by_block.of(u);
        return c * nw + by_warp(c).of(u - start(c));
    }
};

// A partial result in the workspace: O [8][HD], m [8], l [8] (fp32, base-2
// exponents). Warp w's part 0 belongs to the segment that began before its run,
// part 1 to the one that begins in it and goes on past it. Where all warps of a
// block are inside one segment, the block's first warp holds their sum.
__host__ __device__ constexpr int kv4_part_floats(int hd) { return kKvTile * hd + 2 * kKvTile; }

// Warps of a block (one block per SM): as many as the registers of a tile's
// sums and the ring of whole blocks allow. 128: 12 warps of 168 registers, 209 KB.
__host__ __device__ constexpr int kv4_warps(int hd) { return hd == 128 ? 12 : 16; }
template <int HD>
struct kv4_smem {
    static constexpr int BLK = 68 * HD, NW = kv4_warps(HD);
    static constexpr int bars = NW * kKvRing * BLK;
    static constexpr int stat = bars + NW * kKvRing * 8;      // m, l [NW][8] of the block's sum
    static constexpr int total = stat + NW * 2 * kKvTile * 4;
    static_assert(kKvRing * BLK >= kKvTile * HD * 4, "a warp's ring holds its sums");
};

// One warp's running state for the segment it is in. The matrix instruction's
// 16 rows are the tile's 8 query rows twice: rows 0-7 the hi parts of q (and of
// the weights), rows 8-15 the lo parts, so a 22-bit operand costs no further
// instruction. Thread (g, t) = (lane / 4, lane % 4) holds row g.
template <int HD>
struct kv4_state {
    static constexpr int NG = HD / 64;
    uint32_t qf[NG * 4][4];   // q fragments per k step of 16 values
    float f;                  // accumulator -> score in base 2 (a power of two)
    float o[NG][8][4];        // o[g][j][c], [2 + c]: hi, lo sums of value 64 g + 8 (2 t + c) + j
    float m;                  // reference of the exponents, in the accumulator's units: no score is above it
    float2 l;                 // this thread's sum of weights
    int n;                    // positions that row g sees
};

template <int HD, typename T>
__device__ __forceinline__ void kv4_load_q(kv4_state<HD>& st, const T* q, float scale) {
    constexpr int NG = HD / 64;
    const int t = threadIdx.x & 3;
    float x[NG][2][8], mx = 0.0f;
#pragma unroll
    for (int g = 0; g < NG; g++)
#pragma unroll
        for (int w = 0; w < 2; w++) {
            load8(q + g * 64 + 16 * t + 8 * w, x[g][w]);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                x[g][w][j] *= scale * 1.4426950408889634f;
                mx = fmaxf(mx, fabsf(x[g][w][j]));
            }
        }
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    // q by a power of two so that its largest value is in [1, 2): fp16 has room for the rest
    int e = (int)(__float_as_uint(mx) >> 23);
    e = e == 0 ? 127 : min(e, 253);
    const float inv = __uint_as_float((uint32_t)(254 - e) << 23);
    st.f = __uint_as_float((uint32_t)e << 23);
#pragma unroll
    for (int g = 0; g < NG; g++) {
#pragma unroll
        for (int w = 0; w < 2; w++) {
            float (&v)[8] = x[g][w];
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] *= inv;
            // nibbles j and j + 4 of a word share a half pair
#pragma unroll
            for (int s = 0; s < 2; s++) {
                uint32_t (&a)[4] = st.qf[g * 4 + w * 2 + s];
                split2(make_float2(v[2 * s], v[2 * s + 4]), a[0], a[1]);
                split2(make_float2(v[2 * s + 1], v[2 * s + 5]), a[2], a[3]);
            }
        }
#pragma unroll
        for (int j = 0; j < 8; j++)
#pragma unroll
            for (int c = 0; c < 4; c++) st.o[g][j][c] = 0.0f;
    }
    st.m = -INFINITY;
    st.l = f2(0.0f);
}

// One block of 64 positions (j0 = its first) against the tile.
//
// Codes become n - 8 exactly, by one AND-OR into 1024's mantissa and one packed
// fp16 sum per two values (the offset's own sum would be far larger than the
// results'). K's scale multiplies the accumulated group, V's the weight, both in
// fp32.
// MASK: the block reaches past what some row sees; pieces of it that no row sees
// (n_max) are passed over.
template <int HD, bool MASK>
__device__ __forceinline__ void kv4_block(kv4_state<HD>& st, const uint8_t* blk, int j0, int n_max) {
    constexpr int NG = HD / 64, ROW = HD / 2;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    float2 s[8];
#pragma unroll
    for (int nt = 0; nt < 8; nt++) {
        if (MASK && j0 + nt * 8 >= n_max) {
            s[nt] = f2(-INFINITY);
            continue;
        }
        float acc[NG][4];
        uint32_t kw[NG * 2];
        const uint8_t* kp = blk + (nt * 8 + g) * ROW + t * 8 * NG;
        if (NG == 2) {
            const uint4 w = *reinterpret_cast<const uint4*>(kp);
            kw[0] = w.x, kw[1] = w.y, kw[NG] = w.z, kw[2 * NG - 1] = w.w;
        } else {
            const uint2 w = *reinterpret_cast<const uint2*>(kp);
            kw[0] = w.x, kw[1] = w.y;
        }
#pragma unroll
        for (int gr = 0; gr < NG; gr++) acc[gr][0] = acc[gr][1] = acc[gr][2] = acc[gr][3] = 0.0f;
#pragma unroll
        for (int w = 0; w < 2; w++)
#pragma unroll
            for (int sh = 0; sh < 2; sh++)
#pragma unroll
                for (int gr = 0; gr < NG; gr++) {
                    const uint32_t x = sh ? kw[w * NG + gr] >> 8 : kw[w * NG + gr];
                    const uint32_t (&a)[4] = st.qf[gr * 4 + w * 2 + sh];
                    mma16816(acc[gr], a[0], a[1], a[2], a[3], code_even(x), code_odd(x));
                }
        float2 sc[NG];
        scale_pairs<NG>(blk + kv4_kscale(HD), nt * 8 + 2 * t, sc);
        s[nt] = __fmul2_rn(sc[0], __ffma2_rn(make_float2(acc[0][2], acc[0][3]), f2(1.0f / kLoScale),
                                             make_float2(acc[0][0], acc[0][1])));
        if (NG == 2)
            s[nt] = __ffma2_rn(sc[NG - 1], __ffma2_rn(make_float2(acc[NG - 1][2], acc[NG - 1][3]), f2(1.0f / kLoScale),
                                                      make_float2(acc[NG - 1][0], acc[NG - 1][1])), s[nt]);
        if (MASK) {
            if (j0 + nt * 8 + 2 * t >= st.n) s[nt].x = -INFINITY;
            if (j0 + nt * 8 + 2 * t + 1 >= st.n) s[nt].y = -INFINITY;
        }
    }
    float m = fmaxf(s[0].x, s[0].y);
#pragma unroll
    for (int nt = 1; nt < 8; nt++) m = fmaxf(m, fmaxf(s[nt].x, s[nt].y));
    if (__any_sync(0xffffffffu, m > st.m)) {  // a score past the reference: all lanes of the row take a new one
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
        if (m > st.m) {
            m = fmaf(kHeadroom, 1.0f / st.f, m);
            const float al = ex2((st.m - m) * st.f);  // st.m = -inf: 0
            st.l = __fmul2_rn(st.l, f2(al));
#pragma unroll
            for (int gr = 0; gr < NG; gr++)
#pragma unroll
                for (int j = 0; j < 8; j++)
#pragma unroll
                    for (int c = 0; c < 4; c++) st.o[gr][j][c] *= al;
            st.m = m;
        }
    }
    const float2 mf = f2(st.m == -INFINITY ? 0.0f : -st.m * st.f), ff = f2(st.f);
#pragma unroll
    for (int nt = 0; nt < 8; nt++) {
        s[nt] = __ffma2_rn(s[nt], ff, mf);
        s[nt].x = ex2(s[nt].x);
        s[nt].y = ex2(s[nt].y);
        st.l = __fadd2_rn(st.l, s[nt]);
    }
    const uint8_t* vp = blk + kv4_vcode(HD) + t * ROW + (g ^ ((t & 2) << 1)) * 4 * NG;
#pragma unroll
    for (int kk = 0; kk < 4; kk++) {
        if (MASK && j0 + kk * 16 >= n_max) break;
        // weights times scales of positions 2t, 2t + 1 (nt even), 2t + 8, 2t + 9 (nt odd)
        uint32_t a[NG][4];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int nt = 2 * kk + h;
            float2 sc[NG];
            scale_pairs<NG>(blk + kv4_vscale(HD), nt * 8 + 2 * t, sc);
            if (MASK) {  // rows never written may hold any scale
#pragma unroll
                for (int gr = 0; gr < NG; gr++) {
                    if (j0 + nt * 8 + 2 * t >= st.n) sc[gr].x = 0.0f;
                    if (j0 + nt * 8 + 2 * t + 1 >= st.n) sc[gr].y = 0.0f;
                }
            }
#pragma unroll
            for (int gr = 0; gr < NG; gr++) split2(__fmul2_rn(s[nt], sc[gr]), a[gr][2 * h], a[gr][2 * h + 1]);
        }
        uint32_t vw[4][NG];  // rows 2t, 2t + 1, 2t + 8, 2t + 9 at places t, 4 + t, 8 + t, 12 + t
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const uint8_t* p = vp + (kk * 16 + 4 * r) * ROW;
            if (NG == 2) {
                const uint2 w = *reinterpret_cast<const uint2*>(p);
                vw[r][0] = w.x, vw[r][NG - 1] = w.y;
            } else {
                vw[r][0] = *reinterpret_cast<const uint32_t*>(p);
            }
        }
#pragma unroll
        for (int gr = 0; gr < NG; gr++)
#pragma unroll
            for (int q = 0; q < 2; q++) {  // values 4q .. 4q + 3 of the words
                uint32_t x = __byte_perm(vw[0][gr], vw[1][gr], q ? 0x7632 : 0x5410);
                uint32_t y = __byte_perm(vw[2][gr], vw[3][gr], q ? 0x7632 : 0x5410);
#pragma unroll
                for (int p = 0; p < 2; p++) {
                    mma16816(st.o[gr][4 * q + 2 * p], a[gr][0], a[gr][1], a[gr][2], a[gr][3], code_even(x), code_even(y));
                    mma16816(st.o[gr][4 * q + 2 * p + 1], a[gr][0], a[gr][1], a[gr][2], a[gr][3], code_odd(x), code_odd(y));
                    x >>= 8;
                    y >>= 8;
                }
            }
    }
}

// Bound by HBM for long caches (the codes and scales are read once, 4.25 bits
// per value) and by launch and load latency for short ones. Each warp has a ring
// of two whole blocks, filled by one bulk copy each; no barrier between warps
// but for the sum of a block that is inside one segment.
template <int HD, typename T>
__global__ void __launch_bounds__(kv4_warps(HD) * 32, 1) k_kv4_attn(kv4_dims c, int l, jl_kv4_attn_args a, int R, int whole) {
    extern __shared__ __align__(128) uint8_t smem[];
    constexpr int BLK = kv4_smem<HD>::BLK, NG = HD / 64, NW = kv4_warps(HD);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    uint8_t* ring = smem + warp * kKvRing * BLK;
    uint64_t* bar = reinterpret_cast<uint64_t*>(smem + kv4_smem<HD>::bars) + warp * kKvRing;
    if (lane == 0) {
        for (int i = 0; i < kKvRing; i++) mbar_init(bar + i, 1);
        mbar_fence_init();
    }
    __syncwarp();
    griddep_wait();
    griddep_launch_dependents();
    const int gsz = a.H / c.KH, rows = a.T * gsz, S = R * c.KH;
    const kv4_seqs seqs = {a.slots, a.lens, a.len_add, a.longest, c.slots, whole};
    // sequences without positions: zeros (and the status bit for those outside the cache)
    for (int b = warp * gridDim.x + blockIdx.x; b < a.B; b += NW * gridDim.x) {
        const int n = seqs.len(b);
        if (n > 0) continue;
        if (n < 0 && lane == 0 && a.err) atomicOr(a.err, kErrKvIndex);
        const float z[8] = {};
        const long long r0 = (long long)b * a.T, n8 = (long long)a.T * a.H * HD / 8;
        for (long long i = lane; i < n8; i += 32) put8(static_cast<T*>(a.out) + r0 * a.H * HD + 8 * i, z);
        if (a.outT)
            for (long long i = lane; i < 8 * n8; i += 32)
                a.outT[(size_t)(i % (a.H * HD)) * a.outT_ld + r0 + i / (a.H * HD)] = 0.0f;
    }
    const uint32_t U = warp_total(seqs, a.B) * S;
    if (U == 0) return;
    const kv4_cut cut(U, gridDim.x, NW);
    if (warp >= cut.nw || blockIdx.x >= cut.ctas) return;
    const int wid = blockIdx.x * cut.nw + warp;
    const kv4_split mine = cut.by_warp(blockIdx.x);
    const uint32_t c0 = cut.start(blockIdx.x), c1 = cut.start(blockIdx.x + 1), u0 = c0 + mine.start(warp);
    int units = mine.start(warp + 1) - mine.start(warp);  // blocks of this warp's run
    int b;
    uint32_t off;
    warp_find(seqs, a.B, S, u0, b, off);
    struct cursor {
        int b, s, j, nb;
        const uint8_t* p;
    } pr;
    pr.b = b;
    pr.nb = seqs.blocks(b);
    pr.s = (int)(whole ? off : off / pr.nb);
    pr.j = (int)(whole ? 0 : off % pr.nb);
    if (whole) {  // so many segments, each with its sequence's blocks
        int segs = units, bb = b, ss = pr.s;
        for (units = 0; segs; segs--) {
            units += seqs.blocks(bb);
            if (++ss == S && segs > 1) {
                ss = 0;
                do bb++;
                while (seqs.blocks(bb) == 0);
            }
        }
    }
    pr.p = c.run(a.slots[b], l, pr.s / R) + (size_t)pr.j * BLK;
    auto advance = [&](cursor& x) {  // not past the last unit
        x.j++;
        x.p += BLK;
        if (x.j == x.nb) {
            x.j = 0;
            if (++x.s == S) {
                x.s = 0;
                do x.nb = seqs.blocks(++x.b);
                while (x.nb == 0);
            }
            x.p = c.run(a.slots[x.b], l, x.s / R);
        }
    };
    cursor co = pr;
    // the block's run is inside one segment: its warps' sums meet here
    const uint32_t seg0 = u0 - pr.j;
    const bool joined = !whole && cut.nw > 1 && c0 >= seg0 && c1 <= seg0 + pr.nb;
    int issued = 0;
    auto issue = [&]() {
        if (lane == 0) {
            const int k = issued % kKvRing;
            mbar_expect_tx(bar + k, BLK);
            bulk_g2s(ring + k * BLK, pr.p, BLK, bar + k);
        }
        if (++issued < units) advance(pr);
    };
    while (issued < min(units, kKvRing)) issue();
    kv4_state<HD> st;
    int slot_k = 0, phase = 0, n_min = 0, n_max = 0, row = 0;
    bool began = false;
    for (int i = 0; i < units; i++) {
        if (!began) {  // a new segment: its rows (those past the last repeat it and are not written)
            const int kh = co.s / R, rt = co.s % R, r = min(rt * kKvTile + g, rows - 1);
            const int tok = r / gsz, h = kh * gsz + r % gsz, len = seqs.len(co.b);
            row = rt * kKvTile + g;
            kv4_load_q<HD, T>(st, static_cast<const T*>(a.q) + ((long long)co.b * a.T + tok) * a.q_stride + h * HD,
                              a.scale);
            st.n = max(0, len - a.T + 1 + tok);
            n_min = max(0, len - a.T + 1 + rt * kKvTile / gsz);
            n_max = max(0, len - a.T + 1 + min(rt * kKvTile + kKvTile - 1, rows - 1) / gsz);
            began = true;
        }
        if (!mbar_wait_bounded(bar + slot_k, phase, a.err)) break;  // flagged; the block's sum still meets
        const uint8_t* blk = ring + slot_k * BLK;
        const int j0 = co.j * kKv4Rows;
        if (j0 + kKv4Rows <= n_min) kv4_block<HD, false>(st, blk, j0, n_max);
        else if (j0 < n_max) kv4_block<HD, true>(st, blk, j0, n_max);
        fence_proxy_async_smem();
        __syncwarp();
        if (issued < units) issue();
        if (++slot_k == kKvRing) slot_k = 0, phase ^= 1;
        const bool ends = co.j == co.nb - 1;
        if (ends || i == units - 1) {
            float lsum = st.l.x + st.l.y;
            lsum += __shfl_xor_sync(0xffffffffu, lsum, 1);
            lsum += __shfl_xor_sync(0xffffffffu, lsum, 2);
            const bool from_start = i >= co.j;  // the segment's first block is in this warp's run
            if (ends && from_start) {
                const float inv = lsum == 0.0f ? 0.0f : 1.0f / lsum;
                if (row < rows) {
                    const int tok = row / gsz, h = co.s / R * gsz + row % gsz;
                    const long long orow = (long long)co.b * a.T + tok;
                    T* out = static_cast<T*>(a.out) + (orow * a.H + h) * HD;
#pragma unroll
                    for (int gr = 0; gr < NG; gr++)
#pragma unroll
                        for (int cc = 0; cc < 2; cc++) {
                            float x[8];
#pragma unroll
                            for (int j = 0; j < 8; j++)
                                x[j] = fmaf(st.o[gr][j][2 + cc], 1.0f / kLoScale, st.o[gr][j][cc]) * inv;
                            const int d = gr * 64 + 8 * (2 * t + cc);
                            put8(out + d, x);
                            if (a.outT)
#pragma unroll
                                for (int j = 0; j < 8; j++) a.outT[(size_t)(h * HD + d + j) * a.outT_ld + orow] = x[j];
                        }
                }
            } else {
                float* part = joined ? reinterpret_cast<float*>(ring)
                                     : static_cast<float*>(a.ws) + ((size_t)wid * 2 + from_start) * kv4_part_floats(HD);
                float* ml = joined ? reinterpret_cast<float*>(smem + kv4_smem<HD>::stat) + warp * 2 * kKvTile
                                   : part + kKvTile * HD;
#pragma unroll
                for (int gr = 0; gr < NG; gr++)
#pragma unroll
                    for (int cc = 0; cc < 2; cc++) {
                        float x[8];
#pragma unroll
                        for (int j = 0; j < 8; j++) x[j] = fmaf(st.o[gr][j][2 + cc], 1.0f / kLoScale, st.o[gr][j][cc]);
                        put8(part + g * HD + gr * 64 + 8 * (2 * t + cc), x);
                    }
                if (t == 0) {
                    ml[g] = st.m == -INFINITY ? st.m : st.m * st.f;
                    ml[kKvTile + g] = lsum;
                }
            }
            began = false;
        }
        if (i + 1 < units) advance(co);
    }
    if (!joined) return;
    // all cut.nw warps of the block come here: the warps' sums, in their order
    asm volatile("bar.sync 1, %0;" ::"r"(cut.nw * 32) : "memory");
    const float* ml = reinterpret_cast<const float*>(smem + kv4_smem<HD>::stat);
    float* part = static_cast<float*>(a.ws) +
                  ((size_t)blockIdx.x * cut.nw * 2 + (c0 == seg0)) * kv4_part_floats(HD);
    for (int x = threadIdx.x; x < kKvTile * HD / 4; x += cut.nw * 32) {
        const int r = x / (HD / 4);
        float m = -INFINITY, lsum = 0.0f;
        for (int w = 0; w < (int)cut.nw; w++) m = fmaxf(m, ml[w * 2 * kKvTile + r]);
        const float mu = m == -INFINITY ? 0.0f : m;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int w = 0; w < (int)cut.nw; w++) {
            const float f = ex2(ml[w * 2 * kKvTile + r] - mu);
            const float4 v = reinterpret_cast<const float4*>(smem + w * kKvRing * BLK)[x];
            lsum = fmaf(ml[w * 2 * kKvTile + kKvTile + r], f, lsum);
            o = make_float4(fmaf(v.x, f, o.x), fmaf(v.y, f, o.y), fmaf(v.z, f, o.z), fmaf(v.w, f, o.w));
        }
        reinterpret_cast<float4*>(part)[x] = o;
        if (x % (HD / 4) == 0) {
            part[kKvTile * HD + r] = m;
            part[kKvTile * HD + kKvTile + r] = lsum;
        }
    }
}

// Adds up the parts of segments that several warps shared: block = RB rows of
// one segment, 8 / RB warps per row, each adding every (8 / RB)-th part.
template <int HD, typename T>
__global__ void __launch_bounds__(256) k_kv4_merge(kv4_dims c, jl_kv4_attn_args a, int R, int ctas, int RB) {
    constexpr int V = HD / 32, NW = kv4_warps(HD), PF = kv4_part_floats(HD);  // V values per lane
    __shared__ float sums[8][HD], stat[8][2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int gsz = a.H / c.KH, rows = a.T * gsz, S = R * c.KH;
    const kv4_seqs seqs = {a.slots, a.lens, a.len_add, a.longest, c.slots, 0};
    // The attention's blocks have all passed their own wait when this kernel
    // starts, so lens and slots are there before this kernel's wait.
    const int b = blockIdx.x / S, s = blockIdx.x % S, nb = seqs.blocks(b);
    uint32_t before = 0, U = 0;
    for (int i = lane; i < a.B; i += 32) {
        const int n = seqs.blocks(i);
        U += n;
        if (i < b) before += n;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        U += __shfl_xor_sync(0xffffffffu, U, o);
        before += __shfl_xor_sync(0xffffffffu, before, o);
    }
    const kv4_cut cut(max(1u, U * S), ctas, NW);
    const uint32_t first = before * S + s * nb, last = first + nb;
    const int w0 = nb ? cut.warp_of(first) : 0, w1 = nb ? cut.warp_of(last - 1) : 0, nw = cut.nw;
    griddep_wait();
    griddep_launch_dependents();
    if (w0 == w1) return;  // nothing to add, or one warp had it all
    // Parts: one per warp of the first and last block where these reach out of
    // the segment, one per block in between.
    int b0 = w0 / nw, b1 = w1 / nw + 1;  // joined blocks [b0, b1)
    if (cut.start(b0) < first) b0++;
    if (cut.start(b1) > last) b1--;
    if (nw == 1 || b1 <= b0) b0 = b1 = w1 / nw + 1;
    const int head = min(w1 + 1, b0 * nw) - w0, tail = max(0, w1 + 1 - b1 * nw), n = head + b1 - b0 + tail;
    const int g = blockIdx.y * RB + warp % RB, lanes = 8 / RB, pl = warp / RB;
    const float* ws = static_cast<const float*>(a.ws) + g * HD;
    // warp w0 began the segment: its part 1
    auto part = [&](int i) {
        const int w = i < head ? w0 + i : i < head + b1 - b0 ? (b0 + i - head) * nw : b1 * nw + i - head - (b1 - b0);
        return ws + ((size_t)w * 2 + (w == w0)) * PF;
    };
    const int so = kKvTile * HD + g - g * HD;  // m from the row's values; l is kKvTile further
    float m = -INFINITY, lsum = 0.0f, x[V] = {};
    for (int i0 = pl; i0 < n; i0 += 4 * lanes) {
        float v[4][V], pm[4], pl4[4], mx = m;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int i = i0 + k * lanes;
            pm[k] = -INFINITY, pl4[k] = 0.0f;
#pragma unroll
            for (int e = 0; e < V; e++) v[k][e] = 0.0f;
            if (i < n) {
                const float* p = part(i);
                pm[k] = p[so];
                pl4[k] = p[so + kKvTile];
#pragma unroll
                for (int e = 0; e < V; e++) v[k][e] = p[lane + 32 * e];
            }
        }
#pragma unroll
        for (int k = 0; k < 4; k++) mx = fmaxf(mx, pm[k]);
        const float mu = mx == -INFINITY ? 0.0f : mx, al = ex2(m - mu);
        lsum *= al;
#pragma unroll
        for (int e = 0; e < V; e++) x[e] *= al;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float f = ex2(pm[k] - mu);
            lsum = fmaf(pl4[k], f, lsum);
#pragma unroll
            for (int e = 0; e < V; e++) x[e] = fmaf(v[k][e], f, x[e]);
        }
        m = mx;
    }
    if (lanes > 1) {
#pragma unroll
        for (int e = 0; e < V; e++) sums[warp][lane + 32 * e] = x[e];
        if (lane == 0) stat[warp][0] = m, stat[warp][1] = lsum;
        __syncthreads();
        if (pl) return;
        float mx = m;
        for (int w = 1; w < lanes; w++) mx = fmaxf(mx, stat[warp + w * RB][0]);
        const float mu = mx == -INFINITY ? 0.0f : mx, al = ex2(m - mu);
        lsum *= al;
#pragma unroll
        for (int e = 0; e < V; e++) x[e] *= al;
        for (int w = 1; w < lanes; w++) {
            const float f = ex2(stat[warp + w * RB][0] - mu);
            lsum = fmaf(stat[warp + w * RB][1], f, lsum);
#pragma unroll
            for (int e = 0; e < V; e++) x[e] = fmaf(sums[warp + w * RB][lane + 32 * e], f, x[e]);
        }
    }
    const int row = s % R * kKvTile + g;
    if (row >= rows) return;
    const int h = s / R * gsz + row % gsz;
    const long long orow = (long long)b * a.T + row / gsz;
    const float inv = lsum == 0.0f ? 0.0f : 1.0f / lsum;
#pragma unroll
    for (int e = 0; e < V; e++) {
        const int d = lane + 32 * e;
        put1(static_cast<T*>(a.out) + (orow * a.H + h) * HD + d, x[e] * inv);
        if (a.outT) a.outT[(size_t)(h * HD + d) * a.outT_ld + orow] = x[e] * inv;
    }
}

}  // namespace jl

namespace {

int sm_count() {
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        return 0;
    return n;
}

int row_tiles(const jl::kv4_dims& c, int T, int H) { return (T * (H / c.KH) + jl::kKvTile - 1) / jl::kKvTile; }

constexpr int kMaxSms = 256;  // the workspace is sized without asking the device

template <int HD>
int attn_attrs() {
    using namespace jl;
    JL_CUDA(cudaFuncSetAttribute(k_kv4_attn<HD, float>, cudaFuncAttributeMaxDynamicSharedMemorySize, kv4_smem<HD>::total));
    JL_CUDA(cudaFuncSetAttribute(k_kv4_attn<HD, __half>, cudaFuncAttributeMaxDynamicSharedMemorySize, kv4_smem<HD>::total));
    JL_CUDA(cudaFuncSetAttribute(k_kv4_attn<HD, __nv_bfloat16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 kv4_smem<HD>::total));
    return JL_OK;
}

template <int HD, typename T>
int launch_t(const jl::kv4_dims& c, int l, const jl_kv4_attn_args& a, cudaStream_t s) {
    using namespace jl;
    const int sms = std::min(sm_count(), kMaxSms), R = row_tiles(c, a.T, a.H);
    if (sms < 1) return JL_ERR_CUDA;
    const long long segs = (long long)a.B * R * c.KH;
    if (segs > INT_MAX || segs * c.nb > INT_MAX) return JL_ERR_INVALID;  // the cut counts in 32 bits
    // Segments of at most 4 blocks are not cut: a warp takes that many sooner
    // than a second kernel starts.
    const int whole = a.longest <= 4 * kKv4Rows;
    const int rc = launch(k_kv4_attn<HD, T>, dim3(sms), dim3(kv4_warps(HD) * 32), (size_t)kv4_smem<HD>::total, s, c, l, a, R,
                          whole);
    if (rc || whole) return rc;
    const int RB = segs >= sms ? 8 : segs * 4 >= sms ? 2 : 1;
    return launch(k_kv4_merge<HD, T>, dim3((unsigned)segs, kKvTile / RB), dim3(256), 0, s, c, a, R, sms, RB);
}

template <int HD>
int launch_hd(const jl::kv4_dims& c, int l, const jl_kv4_attn_args& a, cudaStream_t s) {
    if (a.dtype == JL_F32) return launch_t<HD, float>(c, l, a, s);
    if (a.dtype == JL_F16) return launch_t<HD, __half>(c, l, a, s);
    return launch_t<HD, __nv_bfloat16>(c, l, a, s);
}

}  // namespace

// Two parts for each warp that has blocks.
long long jl_kv4_attn_ws_bytes(const jl::kv4_dims& c, int B, int T, int H) {
    const long long segs = (long long)B * row_tiles(c, T, H) * c.KH, warps = (long long)kMaxSms * jl::kv4_warps(c.hd);
    const long long n = segs >= warps ? warps : std::min(warps, segs * c.nb);
    return n * 2 * jl::kv4_part_floats(c.hd) * (long long)sizeof(float);
}

int jl_launch_kv4_attn(const jl::kv4_dims& c, int l, const jl_kv4_attn_args& a, cudaStream_t s) {
    const int rc = jl_device_once(kOnceKv4, [] {
        const int r = attn_attrs<64>();
        return r ? r : attn_attrs<128>();
    });
    if (rc) return rc;
    return c.hd == 64 ? launch_hd<64>(c, l, a, s) : launch_hd<128>(c, l, a, s);
}
