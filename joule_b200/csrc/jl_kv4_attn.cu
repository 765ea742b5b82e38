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

constexpr int kKvWarps = 8;    // warps per block, one block per SM
constexpr int kKvRing = 3;     // cache blocks in a warp's ring
constexpr int kKvTile = 8;     // query rows of a tile
constexpr float kLoScale = 2048.0f;

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

// (x, y) as fp16 pairs: hi = the nearest, lo = 2048 times what hi misses, so
// that hi + lo / 2048 holds 22 bits and lo does not underflow before hi does.
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    hi = h2bits(h);
    lo = h2bits(__floats2half2_rn((x - f.x) * kLoScale, (y - f.y) * kLoScale));
}

// n - 8 of the nibbles at bits 0-3 (even) or 4-7 (odd) of both halves, exactly,
// as fp16: 1024 + n (1024 + 16 n) by its bits, then one packed sum (FMA).
__device__ __forceinline__ uint32_t code_even(uint32_t x) {
    x = (x & 0x000F000Fu) | 0x64006400u;
    return h2bits(__hsub2(*reinterpret_cast<__half2*>(&x), __floats2half2_rn(1032.0f, 1032.0f)));
}
__device__ __forceinline__ uint32_t code_odd(uint32_t x) {
    x = (x & 0x00F000F0u) | 0x64006400u;
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
__device__ __forceinline__ long long warp_total(const kv4_seqs& q, int B) {
    long long n = 0;
    for (int b = threadIdx.x & 31; b < B; b += 32) n += q.weight(b);
#pragma unroll
    for (int o = 16; o; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    return n;
}
__device__ __forceinline__ void warp_find(const kv4_seqs& q, int B, int S, long long u, int& b_out, long long& off) {
    const int lane = threadIdx.x & 31;
    long long base = 0;
    for (int b0 = 0; b0 < B; b0 += 32) {
        const long long n = b0 + lane < B ? (long long)q.weight(b0 + lane) * S : 0;
        long long inc = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long v = __shfl_up_sync(0xffffffffu, inc, o);
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

// Units per warp: the same on every warp and in k_kv4_merge.
__device__ __forceinline__ long long units_per_warp(long long U, int W) { return (U + W - 1) / W; }

// A partial result in the workspace: O [8][HD], m [8], l [8] (fp32, base-2
// exponents). Warp w's part 0 belongs to the segment that began before its run,
// part 1 to the one that goes on past it.
__host__ __device__ constexpr int kv4_part_floats(int hd) { return kKvTile * hd + 2 * kKvTile; }

template <int HD>
struct kv4_smem {
    static constexpr int BLK = 68 * HD;
    static constexpr int bars = kKvWarps * kKvRing * BLK;
    static constexpr int total = bars + kKvWarps * kKvRing * 8;
};

// One warp's running state for the segment it is in. The matrix instruction's
// 16 rows are the tile's 8 query rows twice: rows 0-7 the hi parts of q (and of
// the weights), rows 8-15 the lo parts, so a 22-bit operand costs no further
// instruction. Thread (g, t) = (lane / 4, lane % 4) holds row g.
template <int HD>
struct kv4_state {
    static constexpr int NG = HD / 64;
    uint32_t qf[NG * 4][4];   // q fragments per k step of 16 values
    float f;                  // accumulator -> score in base 2
    float o[NG][8][4];        // o[g][j][c], [2 + c]: hi, lo sums of value 64 g + 8 (2 t + c) + j
    float m, l;
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
            for (int j = 0; j < 8; j++) mx = fmaxf(mx, fabsf(x[g][w][j]));
        }
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    // q by a power of two so that its largest value is in [1, 2): fp16 has room for the rest
    int e = (int)(__float_as_uint(mx) >> 23);
    e = e == 0 ? 127 : min(e, 253);
    const float inv = __uint_as_float((uint32_t)(254 - e) << 23);
    st.f = scale * 1.4426950408889634f * __uint_as_float((uint32_t)e << 23);
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
                split2(v[2 * s], v[2 * s + 4], a[0], a[1]);
                split2(v[2 * s + 1], v[2 * s + 5], a[2], a[3]);
            }
        }
#pragma unroll
        for (int j = 0; j < 8; j++)
#pragma unroll
            for (int c = 0; c < 4; c++) st.o[g][j][c] = 0.0f;
    }
    st.m = -INFINITY;
    st.l = 0.0f;
}

// One block of 64 positions (j0 = its first) against the tile.
//
// Codes become n - 8 exactly, by one AND-OR into 1024's mantissa and one packed
// fp16 sum per two values (the offset's own sum would be far larger than the
// results'). K's scale multiplies the accumulated group, V's the weight, both in
// fp32.
template <int HD, bool MASK>
__device__ __forceinline__ void kv4_block(kv4_state<HD>& st, const uint8_t* blk, int j0) {
    constexpr int NG = HD / 64, ROW = HD / 2;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    float s[8][2];
#pragma unroll
    for (int nt = 0; nt < 8; nt++) {
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
        for (int gr = 0; gr < NG; gr++) {
            acc[gr][0] = acc[gr][1] = acc[gr][2] = acc[gr][3] = 0.0f;
        }
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
        // scales of keys 2t, 2t + 1
        float sc[2][NG];
        const uint8_t* sp = blk + kv4_kscale(HD) + (nt * 8 + 2 * t) * 2 * NG;
        if (NG == 2) {
            const uint2 w = *reinterpret_cast<const uint2*>(sp);
            const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x));
            const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
            sc[0][0] = a.x, sc[0][NG - 1] = a.y, sc[1][0] = b.x, sc[1][NG - 1] = b.y;
        } else {
            const float2 a = __half22float2(*reinterpret_cast<const __half2*>(sp));
            sc[0][0] = a.x, sc[1][0] = a.y;
        }
#pragma unroll
        for (int c = 0; c < 2; c++) {
            float v = sc[c][0] * fmaf(acc[0][2 + c], 1.0f / kLoScale, acc[0][c]);
            if (NG == 2) v = fmaf(sc[c][NG - 1], fmaf(acc[NG - 1][2 + c], 1.0f / kLoScale, acc[NG - 1][c]), v);
            v *= st.f;
            if (MASK && j0 + nt * 8 + 2 * t + c >= st.n) v = -INFINITY;
            s[nt][c] = v;
        }
    }
    float m = s[0][0];
#pragma unroll
    for (int nt = 0; nt < 8; nt++) m = fmaxf(m, fmaxf(s[nt][0], s[nt][1]));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
    m = fmaxf(m, st.m);
    if (__any_sync(0xffffffffu, m > st.m)) {
        const float al = m > st.m ? ex2(st.m - m) : 1.0f;  // st.m = -inf: 0
        st.l *= al;
#pragma unroll
        for (int gr = 0; gr < NG; gr++)
#pragma unroll
            for (int j = 0; j < 8; j++)
#pragma unroll
                for (int c = 0; c < 4; c++) st.o[gr][j][c] *= al;
        st.m = m;
    }
    const float mu = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int nt = 0; nt < 8; nt++)
#pragma unroll
        for (int c = 0; c < 2; c++) {
            s[nt][c] = ex2(s[nt][c] - mu);
            st.l += s[nt][c];
        }
    const uint8_t* vp = blk + kv4_vcode(HD) + t * ROW + (g ^ ((t & 2) << 1)) * 4 * NG;
#pragma unroll
    for (int kk = 0; kk < 4; kk++) {
        // weights times scales of positions 2t, 2t + 1 (nt even), 2t + 8, 2t + 9 (nt odd)
        uint32_t a[NG][4];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int nt = 2 * kk + h;
            float sc[2][NG];
            const uint8_t* sp = blk + kv4_vscale(HD) + (nt * 8 + 2 * t) * 2 * NG;
            if (NG == 2) {
                const uint2 w = *reinterpret_cast<const uint2*>(sp);
                const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w.x));
                const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
                sc[0][0] = x.x, sc[0][NG - 1] = x.y, sc[1][0] = y.x, sc[1][NG - 1] = y.y;
            } else {
                const float2 x = __half22float2(*reinterpret_cast<const __half2*>(sp));
                sc[0][0] = x.x, sc[1][0] = x.y;
            }
            if (MASK) {  // rows never written may hold any scale
#pragma unroll
                for (int c = 0; c < 2; c++)
                    if (j0 + nt * 8 + 2 * t + c >= st.n) {
#pragma unroll
                        for (int gr = 0; gr < NG; gr++) sc[c][gr] = 0.0f;
                    }
            }
#pragma unroll
            for (int gr = 0; gr < NG; gr++)
                split2(s[nt][0] * sc[0][gr], s[nt][1] * sc[1][gr], a[gr][2 * h], a[gr][2 * h + 1]);
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
// per value) and by launch and load latency for short ones. Eight warps per
// SM, each with a ring of three whole blocks filled by one bulk copy each, and
// no barrier between warps.
template <int HD, typename T>
__global__ void __launch_bounds__(kKvWarps * 32, 1) k_kv4_attn(kv4_dims c, int l, jl_kv4_attn_args a, int R, int whole) {
    extern __shared__ __align__(128) uint8_t smem[];
    constexpr int BLK = kv4_smem<HD>::BLK, NG = HD / 64;
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
    const int W = gridDim.x * kKvWarps, wid = warp * gridDim.x + blockIdx.x;
    const int gsz = a.H / c.KH, rows = a.T * gsz, S = R * c.KH;
    const kv4_seqs seqs = {a.slots, a.lens, a.len_add, a.longest, c.slots, whole};
    // sequences without positions: zeros (and the status bit for those outside the cache)
    for (int b = wid; b < a.B; b += W) {
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
    const long long U = warp_total(seqs, a.B) * S, per = units_per_warp(U, W), u0 = wid * per;
    if (u0 >= U) return;
    int units = (int)min(per, U - u0);  // blocks of this warp's run
    int b;
    long long off;
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
        if (!mbar_wait_bounded(bar + slot_k, phase, a.err)) return;
        const uint8_t* blk = ring + slot_k * BLK;
        const int j0 = co.j * kKv4Rows;
        if (j0 + kKv4Rows <= n_min) kv4_block<HD, false>(st, blk, j0);
        else if (j0 < n_max) kv4_block<HD, true>(st, blk, j0);
        fence_proxy_async_smem();
        __syncwarp();
        if (issued < units) issue();
        if (++slot_k == kKvRing) slot_k = 0, phase ^= 1;
        const bool ends = co.j == co.nb - 1;
        if (ends || i == units - 1) {
            float lsum = st.l + __shfl_xor_sync(0xffffffffu, st.l, 1);
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
                float* part = static_cast<float*>(a.ws) + ((size_t)wid * 2 + from_start) * kv4_part_floats(HD);
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
                    part[kKvTile * HD + g] = st.m;
                    part[kKvTile * HD + kKvTile + g] = lsum;
                }
            }
            began = false;
        }
        if (i + 1 < units) advance(co);
    }
}

// Adds up the parts of segments that several warps shared: block = RB rows of
// one segment, 8 / RB warps per row, each adding every (8 / RB)-th part.
template <int HD, typename T>
__global__ void __launch_bounds__(256) k_kv4_merge(kv4_dims c, jl_kv4_attn_args a, int R, int W, int RB) {
    constexpr int V = HD / 32;  // values per lane
    __shared__ float sums[8][HD];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    griddep_wait();
    griddep_launch_dependents();
    const int gsz = a.H / c.KH, rows = a.T * gsz, S = R * c.KH;
    const kv4_seqs seqs = {a.slots, a.lens, a.len_add, a.longest, c.slots, 0};
    const int b = blockIdx.x / S, s = blockIdx.x % S, nb = seqs.blocks(b);
    if (nb == 0) return;
    long long before = 0, U = 0;
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
    const long long per = units_per_warp(U * S, W), first = before * S + (long long)s * nb;
    const int w0 = (int)(first / per), w1 = (int)((first + nb - 1) / per);
    if (w0 == w1) return;  // one warp had it all
    const int g = blockIdx.y * RB + warp % RB, lanes = 8 / RB, pl = warp / RB;
    const float* ws = static_cast<const float*>(a.ws);
    // warp w0 began the segment (its part 1), unless its run begins just there: part 1 all the same
    auto part = [&](int w) { return ws + ((size_t)w * 2 + (w == w0)) * kv4_part_floats(HD); };
    float m = -INFINITY;
    for (int w = w0 + lane; w <= w1; w += 32) m = fmaxf(m, part(w)[kKvTile * HD + g]);
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float mu = m == -INFINITY ? 0.0f : m;
    float lsum = 0.0f;
    for (int w = w0 + lane; w <= w1; w += 32)
        lsum += part(w)[kKvTile * HD + kKvTile + g] * ex2(part(w)[kKvTile * HD + g] - mu);
#pragma unroll
    for (int o = 16; o; o >>= 1) lsum += __shfl_xor_sync(0xffffffffu, lsum, o);
    float x[V] = {};
#pragma unroll 4
    for (int w = w0 + pl; w <= w1; w += lanes) {
        const float* p = part(w);
        const float f = ex2(p[kKvTile * HD + g] - mu);
#pragma unroll
        for (int e = 0; e < V; e++) x[e] = fmaf(p[g * HD + lane + 32 * e], f, x[e]);
    }
    if (lanes > 1) {
#pragma unroll
        for (int e = 0; e < V; e++) sums[warp][lane + 32 * e] = x[e];
        __syncthreads();
        if (pl) return;
        for (int w = 1; w < lanes; w++)
#pragma unroll
            for (int e = 0; e < V; e++) x[e] += sums[warp + w * RB][lane + 32 * e];
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
    if (segs > INT_MAX) return JL_ERR_INVALID;
    // Segments of at most 4 blocks are not cut: a warp takes that many sooner
    // than a second kernel starts.
    const int whole = a.longest <= 4 * kKv4Rows;
    const int rc = launch(k_kv4_attn<HD, T>, dim3(sms), dim3(kKvWarps * 32), (size_t)kv4_smem<HD>::total, s, c, l, a, R,
                          whole);
    if (rc || whole) return rc;
    const int RB = segs >= 2 * sms ? 8 : segs * 4 >= 2 * sms ? 2 : 1;
    return launch(k_kv4_merge<HD, T>, dim3((unsigned)segs, kKvTile / RB), dim3(256), 0, s, c, a, R, sms * kKvWarps,
                  RB);
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
    const long long segs = (long long)B * row_tiles(c, T, H) * c.KH, warps = (long long)kMaxSms * jl::kKvWarps;
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
