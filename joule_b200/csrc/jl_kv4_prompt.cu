// Attention of a prompt's rows over the 4-bit KV cache on tcgen05 (layout:
// jl_kv4.cuh; the form for few rows: jl_kv4_attn.cu).
//
// The query rows (token i, head h of the kv head's group; r = i * group + h) of
// one (sequence, kv head) form tiles of 128, two of them per block. Per cache
// block of 64 positions and tile: S = q K^T, softmax by the thread that owns the
// row (= TMEM lane), O += P V, both products on the tensor cores with fp32 sums
// in TMEM. Codes enter as n - 8, which fp16 holds exactly, as it does a 16-bit q
// (down to 2^-34 of a row's largest value); a fp32 q and the weights are hi and lo
// parts (22 bits), two instructions onto the same sums.
// K's scales multiply the finished sums of a 64-value group (one accumulator per
// group), V's the weights of a group, both in fp32. The exponents' references
// (kv4_ref) move only when a weight times its scale would pass 2^15, and the sums
// are then rescaled in TMEM.
//
// Roles (12 warps, so that the softmax has 168 registers a thread): 0-3 and 4-7
// softmax of tile 0 and 1, 8-10 unpack the cache block into the two operands (K as
// [64 positions][values], V as [values][64 positions]) and copy the next one in, 11
// issues the instructions. The tiles take turns on the tensor cores: one's products
// run beside the other's softmax. Every wait is bounded; a timeout sets the status
// bit and an abort flag on which every role leaves its loop.
//
// A unit is the 256 rows of one block. When there are fewer units than SMs, S blocks
// share a unit's cache blocks; their sums meet in k_kv4_prompt_merge (fp32, 32/4 heads
// of 128: 64 tokens over 2,048 positions 25 us, 256 over 4,096 67, 512 over 16,384 415;
// the form for few rows 30, 150 and 1,102).
//
// Bound by the tensor cores and the softmax's latency alike: in fp32 two passes of each
// product (a product of 64 positions takes 60 to 75 cycles where its arithmetic takes 32,
// q being read from shared memory), in 16 bits one of the scores and two of the values.
// 2,047 rows of 32/4 heads of 128 over 4,100 positions: fp32 338 us, 123 at the measured
// bf16 rate, bf16 332, 92 at that rate.
#include <algorithm>
#include <atomic>
#include <climits>

#include "jl_internal.h"
#include "jl_kv4_dev.cuh"
#include "jl_umma.cuh"

namespace jl {

constexpr int kPrTile = 128, kPrPair = 2 * kPrTile, kPrThreads = 12 * 32, kPrUnpack = 3;  // unpacking warps
// The tensor cores' sums are cut off, not rounded: over n blocks they come out short by
// about 1e-7 n of themselves. The sums therefore move to the rows of `out` (16-bit calls:
// their lower halves; the upper ones to shared memory) every kPrFold blocks, which hold
// them until the end, and TMEM starts anew. fp32, 2,047 rows of 32/4 heads of 128 over
// 4,100 positions: error 1.1e-6 and 338 us (never: 6.8e-6, 299 us; every 12: 1.7e-6, 326 us,
// every 16: 2.2e-6, 319 us); 120 tokens of 96/4 heads over 23,000: 1.2e-6 (never: 1.7e-5).
// In 16-bit calls 32 blocks' 3e-6 are far below a step of the output.
template <bool F32>
constexpr int kPrFold = F32 ? 8 : 32;
constexpr int kPrCore = 144;  // bytes between V's core matrices (128 of data: stores without bank conflicts)

struct pr_bars {
    uint64_t raw_full[2], raw_empty[2], kv_full[2], kv_empty[2], q_full;
    uint64_t s_full[2], p_full[2], pv_done[2], fin;
    uint32_t tmem;
    int abort;
    int* err;         // of waits that ran out
    long long limit;  // of a wait, in cycles
    uint2 range[2][2];  // per buffer, per warp of positions: bits of V's largest and smallest scale
};

struct pr_held {
    void* out;               // the sequence's first token, the kv head's first head
    int H, gsz, row0, rows;
    float ref[kPrPair];      // of what a row's places hold
    template <typename P>    // P: what four values of a row are there
    struct place {
        P* p;
        int left, run, rest, gap;  // pieces left in the run; a run's; of a step past whole runs; between runs
        long long step;
        __device__ P* next() {
            P* at = p;
            p += step;
            if ((left -= rest) <= 0) left += run, p += gap;
            return at;
        }
    };
    __device__ bool mine() const { return row0 + (int)threadIdx.x < rows; }
    template <int HD, typename P>
    __device__ place<P> first() const {
        const int r0 = row0 + (int)(threadIdx.x & ~31u), nv = min(32, rows - r0), run = gsz * (HD / 4), gap = (H - gsz) * (HD / 4);
        const int at = r0 % gsz * (HD / 4) + (int)(threadIdx.x & 31), left = run - at % run;
        P* p = static_cast<P*>(out) + (long long)(r0 / gsz + at / run) * H * (HD / 4) + (run - left);
        return place<P>{p, left, run, nv % run, gap, nv + (long long)(nv / run) * gap};
    }
};

// A thread's places in turn. HALF: 16-bit rows hold the lower halves of the four values,
// shared memory behind pr_held ([piece][thread]) the upper ones.
template <int HD, bool HALF>
struct pr_places;
template <int HD>
struct pr_places<HD, false> {
    pr_held::place<float4> at;
    __device__ pr_places(pr_held* held) : at(held->first<HD, float4>()) {}
    __device__ float4 get() { return *at.next(); }
    __device__ void put(float4 x) { *at.next() = x; }
};
template <int HD>
struct pr_places<HD, true> {
    pr_held::place<uint2> at;
    uint2* upper;
    __device__ pr_places(pr_held* held)
        : at(held->first<HD, uint2>()), upper(reinterpret_cast<uint2*>(held + 1) + threadIdx.x) {}
    __device__ float4 get() {
        const uint2 lo = *at.next(), hi = *upper;
        upper += kPrPair;
        return make_float4(__uint_as_float(__byte_perm(lo.x, hi.x, 0x5410)), __uint_as_float(__byte_perm(lo.x, hi.x, 0x7632)),
                           __uint_as_float(__byte_perm(lo.y, hi.y, 0x5410)), __uint_as_float(__byte_perm(lo.y, hi.y, 0x7632)));
    }
    __device__ void put(float4 x) {
        const uint32_t a = __float_as_uint(x.x), b = __float_as_uint(x.y), c = __float_as_uint(x.z), d = __float_as_uint(x.w);
        *at.next() = make_uint2(__byte_perm(a, b, 0x5410), __byte_perm(c, d, 0x5410));
        *upper = make_uint2(__byte_perm(a, b, 0x7632), __byte_perm(c, d, 0x7632));
        upper += kPrPair;
    }
};

// A split's sums in the workspace: [32 rows' group][pieces of a row][32 rows][4 values],
// then (reference, sum of weights) of each row.
template <int HD>
struct pr_part {
    static constexpr int floats = kPrPair * HD + 2 * kPrPair;
    __device__ static float* of(void* ws, size_t i) { return static_cast<float*>(ws) + i * floats; }
    __device__ static float2* stats(float* part) { return reinterpret_cast<float2*>(part + kPrPair * HD); }
};

template <int HD, bool F32>
struct pr_smem {
    static constexpr int NG = HD / 64, PARTS = F32 ? 2 : 1;  // parts of q
    static constexpr int QCHUNK = kPrTile * 16 + 16;  // bytes of 8 values of all rows (16 more: stores spread over the banks)
    static constexpr int QTILE = HD / 8 * QCHUNK, KTILE = kKv4Rows * HD * 2, VTILE = NG * 64 * kPrCore;
    static constexpr int sc = 512;                       // fp32 scales [2 buffers][K g0, K g1, V g0, V g1][64]
    static constexpr int q = sc + 2 * 4 * kKv4Rows * 4;  // [tile][part][chunk of 8 values][128 rows x 16 B]
    static constexpr int k = q + 2 * PARTS * QTILE;      // [buffer][chunk][64 positions x 16 B]
    static constexpr int v = k + 2 * KTILE;              // [buffer][group][8 positions' chunk][8 values' core]
    static constexpr int raw = v + 2 * VTILE;
    static constexpr int held = raw + 2 * kv4_block_bytes(HD);
    static constexpr int total = held + (int)sizeof(pr_held) + (F32 ? 0 : kPrPair * HD * 2);
    static constexpr int SCOLS = NG * 64, TCOLS = 2 * SCOLS;  // TMEM columns of a tile: S (then P), O
    static_assert(sizeof(pr_bars) <= 512 && sizeof(pr_held) % 8 == 0 && total <= 227 * 1024, "shared memory");
};

// Where waits that ran out are recorded when the call has no status word.
__device__ int g_kv4_status;

// A wait of a whole warp, bounded; false when it ran out or another role gave up.
// (mbarrier.test_wait in place of try_wait, polling without a suspension, was 6 %
// slower: the polls take the softmax's issue slots.)
__device__ __forceinline__ bool pr_wait(uint64_t* bar, uint32_t parity, pr_bars& sh) {
    bool ok = mbar_try_wait(bar, parity);
    if (!ok) {
        const long long t0 = clock64();
        for (int i = 1; !ok; i++) {
            ok = mbar_try_wait(bar, parity);
            if (!ok && (i & 63) == 0) {
                volatile int* abort = &sh.abort;
                if (*abort) break;
                if (clock64() - t0 > sh.limit) {
                    atomicOr(sh.err, kErrTimeout);
                    *abort = 1;
                    break;
                }
            }
        }
    }
    return __all_sync(0xffffffffu, ok);
}

__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
template <typename T>
__device__ __forceinline__ float4 load4(const T* p) {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    const T* h = reinterpret_cast<const T*>(&w);
    return make_float4(to_f32(h[0]), to_f32(h[1]), to_f32(h[2]), to_f32(h[3]));
}

// The warp's 32 q rows, by a power of two each (the largest value in [2^10, 2^11)), into
// the operand from row r0 on: 16-bit values exactly, fp32 ones as hi and lo parts. Returns
// the inverse of the power of row `lane` (what else makes base-2 scores of the sums is in
// K's scales: a factor that is no power of two would round scores that weights are
// differences of). HD / 4 lanes read a row (a row per thread touched 32 lines a load and
// took 13 us a block). src(i): row i.
template <int HD, bool F32, typename T, typename F>
__device__ __forceinline__ float pr_load_q(F src, uint8_t* dst, int r0) {
    constexpr int LPR = HD / 4, RPW = 32 / LPR, ROWS = 8;  // rows of a lane in flight
    using SM = pr_smem<HD, F32>;
    const int lane = threadIdx.x & 31, w = lane % LPR;
    float f = 0.0f;
#pragma unroll 1
    for (int i0 = 0; i0 < 32; i0 += ROWS * RPW) {
        float4 x[ROWS];
#pragma unroll
        for (int i = 0; i < ROWS; i++) x[i] = load4(src(i0 + i * RPW + lane / LPR) + 4 * w);
#pragma unroll
        for (int i = 0; i < ROWS; i++) {
            const int row = i0 + i * RPW + lane / LPR;
            float4 y = x[i];
            float mx = fmaxf(fmaxf(fabsf(y.x), fabsf(y.y)), fmaxf(fabsf(y.z), fabsf(y.w)));
#pragma unroll
            for (int o = LPR / 2; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            int e = (int)(__float_as_uint(mx) >> 23);
            e = min(max(e, 11), 253);
            const float inv = __uint_as_float((uint32_t)(264 - e) << 23), fr = __uint_as_float((uint32_t)(e - 10) << 23);
#pragma unroll
            for (int q = 0; q < RPW; q++) {
                const float fq = __shfl_sync(0xffffffffu, fr, q * LPR);
                if (lane == i0 + i * RPW + q) f = fq;
            }
            y = make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
            // values (0, 4), (1, 5) of a chunk in its even lane, (2, 6), (3, 7) in its odd one: an unpacked word's order
            const bool odd = w & 1;
            const float sa = __shfl_xor_sync(0xffffffffu, odd ? y.x : y.z, 1), sb = __shfl_xor_sync(0xffffffffu, odd ? y.y : y.w, 1);
            uint2 hi, lo;
            split2(odd ? make_float2(sa, y.z) : make_float2(y.x, sa), hi.x, lo.x);
            split2(odd ? make_float2(sb, y.w) : make_float2(y.y, sb), hi.y, lo.y);
            uint8_t* p = dst + w / 2 * SM::QCHUNK + (r0 + row) * 16 + (w & 1) * 8;
            *reinterpret_cast<uint2*>(p) = hi;
            if (F32) *reinterpret_cast<uint2*>(p + SM::QTILE) = lo;
        }
    }
    return f;
}

// 16 bytes of values.
__device__ __forceinline__ void store_piece(float* p, const float* x) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
}
template <typename T>
__device__ __forceinline__ void store_piece(T* p, const float* x) {
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; j++) y[j] = x[j];
    put8(p, y);
}

// Unpacks one cache block (kPrUnpack warps, tid from 0) into operand tiles and fp32
// scales (K's times `factor`); positions from n on (never written) get scales of 0.
template <int HD>
__device__ __forceinline__ void pr_unpack(const uint8_t* raw, uint8_t* kt, uint8_t* vt, float* sc, uint2* range, float factor, int n, int tid) {
    constexpr int NG = HD / 64, ROW = HD / 2;
    const int lane = tid & 31, w = tid >> 5;
    // K: lane (t, position of 8) takes words 2t, 2t + 1 of the groups
#pragma unroll
    for (int o = w; o < 8; o += kPrUnpack) {
        const int t = lane >> 3, r = 8 * o + (lane & 7);
        uint32_t kw[2 * NG];
        if (NG == 2) {
            const uint4 x = *reinterpret_cast<const uint4*>(raw + r * ROW + 16 * t);
            kw[0] = x.x, kw[1] = x.y, kw[NG] = x.z, kw[2 * NG - 1] = x.w;
        } else {
            const uint2 x = *reinterpret_cast<const uint2*>(raw + r * ROW + 8 * t);
            kw[0] = x.x, kw[1] = x.y;
        }
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int g = 0; g < NG; g++) {
                const uint32_t x = kw[u * NG + g], y = x >> 8;
                *reinterpret_cast<uint4*>(kt + (g * 8 + 2 * t + u) * 1024 + o * 128 + (lane & 7) * 16) =
                    make_uint4(code_even(x), code_odd(x), code_even(y), code_odd(y));
            }
    }
    // V: thread (8 positions o, word u of group g) writes the 8 x 8 core matrix of its values
#pragma unroll
    for (int i0 = 0; i0 < 64 * NG; i0 += 32 * kPrUnpack) {
        const int task = i0 + tid;
        if (task >= 64 * NG) break;
        const int u = task & 7, g = NG == 2 ? task >> 3 & 1 : 0, o = task >> (NG == 2 ? 4 : 3);
        uint32_t x[8];
#pragma unroll
        for (int i = 0; i < 8; i++)
            x[i] = *reinterpret_cast<const uint32_t*>(raw + kv4_word_off(HD, 1, 8 * o + i, g, u));
        uint8_t* core = vt + ((g * 8 + o) * 8 + u) * kPrCore;
#pragma unroll
        for (int q = 0; q < 2; q++) {
            uint32_t p[4];
#pragma unroll
            for (int i = 0; i < 4; i++) p[i] = __byte_perm(x[2 * i], x[2 * i + 1], q ? 0x7632 : 0x5410);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                *reinterpret_cast<uint4*>(core + (4 * q + 2 * h) * 16) =
                    make_uint4(code_even(p[0]), code_even(p[1]), code_even(p[2]), code_even(p[3]));
                *reinterpret_cast<uint4*>(core + (4 * q + 2 * h + 1) * 16) =
                    make_uint4(code_odd(p[0]), code_odd(p[1]), code_odd(p[2]), code_odd(p[3]));
#pragma unroll
                for (int i = 0; i < 4; i++) p[i] >>= 8;
            }
        }
    }
    if (tid < kKv4Rows) {
        const uint16_t* ks = reinterpret_cast<const uint16_t*>(raw + kv4_kscale(HD)) + tid * NG;
        const uint16_t* vs = reinterpret_cast<const uint16_t*>(raw + kv4_vscale(HD)) + tid * NG;
        uint32_t most = 0, least = 0xFFFFu;
#pragma unroll
        for (int g = 0; g < NG; g++) {
            const uint32_t b = tid < n ? vs[g] : 0;
            sc[g * kKv4Rows + tid] = tid < n ? half_bits_to_f32(ks[g]) * factor : 0.0f;
            sc[(2 + g) * kKv4Rows + tid] = half_bits_to_f32((uint16_t)b);
            most = max(most, b), least = min(least, b);
        }
        most = __reduce_max_sync(0xffffffffu, most), least = __reduce_min_sync(0xffffffffu, least);
        if (lane == 0) range[w] = make_uint2(most, least);
    }
}

// Moves the finished sums in TMEM (HD columns from `to`; less: what brings the second
// group's to the first's scale) to their places, onto what earlier calls put there,
// rescaled to the reference `ref`. Places: pieces (4 values) of
// the warp's rows in turn over the rows' own part of `out` (runs of the kv head's heads,
// one run a token) or of the workspace. A call of its own that finds its arguments in
// shared memory, out of the softmax's registers.
template <int HD, bool HALF>
__device__ __noinline__ void pr_fold(uint32_t to, float ref, float less, pr_held* held, bool holds) {
    const float href = held->ref[threadIdx.x], al = ex2(href - (ref == -INFINITY ? 0.0f : ref));
    const bool mine = held->mine();
    held->ref[threadIdx.x] = ref;
    pr_places<HD, HALF> st(held), ld(held);
#pragma unroll 1
    for (int q = 0; q < HD; q += 32) {
        float4 y[8];
        if (holds && mine)
#pragma unroll
            for (int i = 0; i < 8; i++) y[i] = ld.get();
#pragma unroll
        for (int p = 0; p < 2; p++) {
            float o[16];
            __syncwarp();
            tc_ld16(to + q + 16 * p, o);
            const float m = q < 64 ? 1.0f : less;
            if (mine)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float4 x = make_float4(o[4 * i] * m, o[4 * i + 1] * m, o[4 * i + 2] * m, o[4 * i + 3] * m);
                    const float4 z = y[4 * p + i];
                    if (holds) x = make_float4(fmaf(z.x, al, x.x), fmaf(z.y, al, x.y), fmaf(z.z, al, x.z), fmaf(z.w, al, x.w));
                    st.put(x);
                }
        }
    }
}

// At the end: what the places hold, back onto the last sums in TMEM (more: the second
// group's factor).
template <int HD, bool HALF>
__device__ __noinline__ void pr_unfold(uint32_t to, float ref, float more, pr_held* held) {
    const float al0 = ex2(held->ref[threadIdx.x] - (ref == -INFINITY ? 0.0f : ref));
    pr_places<HD, HALF> at(held);
#pragma unroll 1
    for (int q = 0; q < HD; q += 16) {
        float4 y[4] = {};
        if (held->mine())
#pragma unroll
            for (int i = 0; i < 4; i++) y[i] = at.get();
        float o[16];
        __syncwarp();
        tc_ld16(to + q, o);
        const float al = q < 64 ? al0 : al0 * more;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            o[4 * i] = fmaf(y[i].x, al, o[4 * i]), o[4 * i + 1] = fmaf(y[i].y, al, o[4 * i + 1]);
            o[4 * i + 2] = fmaf(y[i].z, al, o[4 * i + 2]), o[4 * i + 3] = fmaf(y[i].w, al, o[4 * i + 3]);
        }
        tc_st16(to + q, o);
    }
    tc_wait_st();
}

// Scores (but for the row's power of two) of positions 16 q .. 16 q + 15 from the sums in
// TMEM and K's scales.
template <int HD>
__device__ __forceinline__ void pr_scores(uint32_t ts, const float* sc, int q, float2* x) {
    constexpr int NG = HD / 64;
    float a0[16], a1[16];
    if (NG == 2) tc_ld16x2(ts + 16 * q, ts + 64 + 16 * q, a0, a1);
    else tc_ld16(ts + 16 * q, a0);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float4 k0 = *reinterpret_cast<const float4*>(sc + 16 * q + 4 * i);
        float2 u = __fmul2_rn(make_float2(a0[4 * i], a0[4 * i + 1]), make_float2(k0.x, k0.y));
        float2 v = __fmul2_rn(make_float2(a0[4 * i + 2], a0[4 * i + 3]), make_float2(k0.z, k0.w));
        if (NG == 2) {
            const float4 k1 = *reinterpret_cast<const float4*>(sc + kKv4Rows + 16 * q + 4 * i);
            u = __ffma2_rn(make_float2(a1[4 * i], a1[4 * i + 1]), make_float2(k1.x, k1.y), u);
            v = __ffma2_rn(make_float2(a1[4 * i + 2], a1[4 * i + 3]), make_float2(k1.z, k1.w), v);
        }
        x[2 * i] = u;
        x[2 * i + 1] = v;
    }
}
// Scores of positions from n on: -infinity.
template <int COUNT>
__device__ __forceinline__ void pr_mask(float2* x, int n) {
#pragma unroll
    for (int i = 0; i < COUNT / 2; i++) {
        if (2 * i >= n) x[i].x = -INFINITY;
        if (2 * i + 1 >= n) x[i].y = -INFINITY;
    }
}

// Weights of a block, 16 positions at a time, times V's scales of a group (MORE: and the
// second group's factor), hi and lo, into S's place; returns their sum.
template <int HD, bool MORE>
__device__ __forceinline__ float2 pr_weights(uint32_t ts, const float* sc, const float2 (&x)[32], float f, float minus, float more) {
    constexpr int NG = HD / 64;
    const float2 nr = f2(minus), ff = f2(f);
    float2 sum;
#pragma unroll
    for (int q = 0; q < 4; q++) {
        float4 v0[4], v1[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v0[i] = *reinterpret_cast<const float4*>(sc + 2 * kKv4Rows + 16 * q + 4 * i);
            if (NG == 2) v1[i] = *reinterpret_cast<const float4*>(sc + 3 * kKv4Rows + 16 * q + 4 * i);
        }
        uint32_t hi[NG][8], lo[NG][8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float2 p = __ffma2_rn(x[8 * q + i], ff, nr);
            p.x = ex2(p.x);
            p.y = ex2(p.y);
            sum = q + i ? __fadd2_rn(sum, p) : p;
            const float4 w0 = v0[i / 2], w1 = NG == 2 ? v1[i / 2] : w0;
            const float2 y0 = __fmul2_rn(p, i & 1 ? make_float2(w0.z, w0.w) : make_float2(w0.x, w0.y));
            split2(y0, hi[0][i], lo[0][i]);
            if (NG == 2) {
                float2 y1 = __fmul2_rn(p, i & 1 ? make_float2(w1.z, w1.w) : make_float2(w1.x, w1.y));
                if (MORE) y1 = __fmul2_rn(y1, f2(more));
                split2(y1, hi[NG - 1][i], lo[NG - 1][i]);
            }
        }
#pragma unroll
        for (int g = 0; g < NG; g++) {
            tc_st8(ts + 64 * g + 8 * q, hi[g]);
            tc_st8(ts + 64 * g + 32 + 8 * q, lo[g]);
        }
    }
    return sum;
}

// Exponents above a row's products with the scales of each group in a block (kv4_ref), from
// the sums in TMEM: n positions are seen. 16 at a time, brought to the largest score. A call
// of its own, before the softmax's registers are in use (computed from the softmax's own
// scores it made every block slower, 8 % of a prompt).
template <int HD>
__device__ __noinline__ float2 pr_products(uint32_t ts, float f, const float* sc, int n) {
    constexpr int NG = HD / 64;
    float mx = -INFINITY, b0 = kLeast, b1 = kLeast;
#pragma unroll 1
    for (int q = 0; q < 4; q++) {
        float2 x[8];
        __syncwarp();
        pr_scores<HD>(ts, sc, q, x);
        pr_mask<16>(x, n - 16 * q);
        float m = -INFINITY, m0 = 0.0f, m1 = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) m = fmaxf(m, fmaxf(x[i].x, x[i].y));
        m *= f;
        const float2 nm = f2(m == -INFINITY ? 0.0f : -m);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float2 p = __ffma2_rn(x[i], f2(f), nm);
            p.x = ex2(p.x), p.y = ex2(p.y);
            const float2 y0 = __fmul2_rn(p, *reinterpret_cast<const float2*>(sc + 2 * kKv4Rows + 16 * q + 2 * i));
            m0 = fmaxf(m0, fmaxf(y0.x, y0.y));
            if (NG == 2) {
                const float2 y1 = __fmul2_rn(p, *reinterpret_cast<const float2*>(sc + 3 * kKv4Rows + 16 * q + 2 * i));
                m1 = fmaxf(m1, fmaxf(y1.x, y1.y));
            }
        }
        const float to = fmaxf(mx, m), up = to == -INFINITY ? 0.0f : mx - to, down = to == -INFINITY ? 0.0f : m - to;
        b0 = fmaxf(fmaxf(b0 + up, exponent_of(m0) + down), kLeast);
        b1 = fmaxf(fmaxf(b1 + up, exponent_of(m1) + down), kLeast);
        mx = to;
    }
    return make_float2(b0, b1);
}

// The softmax of a thread's row over blocks from st.j on: ends at nb, at a wait that ran out
// (st.j = -1), or, without MORE, at a block whose weights need a factor in some row of the
// warp (its references are moved then, its sums folded and rescaled).
template <int HD>
struct pr_run {
    kv4_ref<HD == 128> r;
    kv4_sum lsum;
    int j;  // -1: not ok
};
template <int HD, bool F32, bool MORE>
__device__ __forceinline__ pr_run<HD> pr_softmax(uint8_t* smem, int t, uint32_t ts, float f, int nb, int S, int n_row,
                                                 int n_min, pr_run<HD> st) {
    using SM = pr_smem<HD, F32>;
    constexpr int NG = SM::NG, FOLD = kPrFold<F32>;
    pr_bars& sh = *reinterpret_cast<pr_bars*>(smem);
    pr_held* held = reinterpret_cast<pr_held*>(smem + SM::held);
    const uint32_t to = ts + SM::SCOLS;
    const int from = st.j;
    for (; st.j < nb; st.j++) {
        const int j = st.j, s = j & 1, j0 = j * kKv4Rows;
        // the scales (kv_full), then the scores
        if (!pr_wait(&sh.kv_full[s], j >> 1 & 1, sh) || !pr_wait(&sh.s_full[t], j & 1, sh)) {
            st.j = -1;
            return st;
        }
        tc_fence_after();
        const bool starts = j % FOLD == 0;  // TMEM's sums start anew
        if (j > 0 && starts && !(MORE && j == from)) {  // S was issued after the last block's values: the sums are complete
            if (F32 || S > 1) pr_fold<HD, false>(to, st.r.ref, st.r.less(), held, j > FOLD);
            else pr_fold<HD, true>(to, st.r.ref, st.r.less(), held, j > FOLD);
            __syncwarp();
        }
        const float* sc = reinterpret_cast<const float*>(smem + SM::sc) + s * 4 * kKv4Rows;
        const uint32_t most = max(sh.range[s][0].x, sh.range[s][1].x), least = min(sh.range[s][0].y, sh.range[s][1].y);
        float2 bound = f2(kv4_top(most));
        if (j0 + kKv4Rows > n_min || kv4_spread(most, least)) bound = pr_products<HD>(ts, f, sc, n_row - j0);
        float2 x[32];
        float mx = -INFINITY;
#pragma unroll
        for (int q = 0; q < 4; q++) pr_scores<HD>(ts, sc, q, x + 8 * q);
        if (j0 + kKv4Rows > n_min) pr_mask<64>(x, n_row - j0);
#pragma unroll
        for (int i = 0; i < 32; i++) mx = fmaxf(mx, fmaxf(x[i].x, x[i].y));
        mx *= f;
        const bool past = st.r.past(mx, bound.x, bound.y);  // a product past the limit, or the row's first
        if (__any_sync(0xffffffffu, past)) {
            const float2 al = past ? st.r.move(mx, bound.x, bound.y) : f2(1.0f);
            st.lsum.scale(al.x);
            __syncwarp();  // (rows part above; the loads below are the whole warp's)
            if (!starts) {  // the sums of earlier blocks are complete (S was issued after them)
#pragma unroll 1
                for (int q = 0; q < NG * 4; q++) {
                    float o[16];
                    tc_ld16(to + 16 * q, o);
#pragma unroll
                    for (int i = 0; i < 16; i++) o[i] *= q < 4 ? al.x : al.y;
                    tc_st16(to + 16 * q, o);
                }
                tc_wait_st();
            }
            if (NG == 2 && !MORE && __any_sync(0xffffffffu, st.r.lifted())) break;
        }
        st.lsum.add(pr_weights<HD, MORE>(ts, sc, x, f, st.r.minus(), MORE ? st.r.more() : 1.0f));
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(&sh.p_full[t]);
    }
    return st;
}
// With factors: a call of its own (multiplying by them in all blocks took 4 % of a prompt).
template <int HD, bool F32>
__device__ __noinline__ pr_run<HD> pr_softmax_lifted(uint8_t* smem, int t, uint32_t ts, float f, int nb, int S, int n_row,
                                                     int n_min, pr_run<HD> st) {
    return pr_softmax<HD, F32, true>(smem, t, ts, f, nb, S, n_row, n_min, st);
}

template <int HD, typename T>
__global__ void __launch_bounds__(kPrThreads, 1) k_kv4_prompt(kv4_dims c, int l, jl_kv4_attn_args a, int pairs, int S) {
    extern __shared__ __align__(1024) uint8_t smem[];
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int FOLD = kPrFold<F32>;
    using SM = pr_smem<HD, F32>;
    constexpr int NG = SM::NG, PARTS = SM::PARTS, BLK = kv4_block_bytes(HD);
    pr_bars& sh = *reinterpret_cast<pr_bars*>(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    griddep_wait();
    // blocks in the order of falling work: the last rows of a prompt see the most
    const int per = c.KH * a.B, unit = blockIdx.x / S, split = blockIdx.x % S;
    const int pair = pairs - 1 - unit / per, kh = unit % c.KH, b = unit % per / c.KH;
    const int gsz = a.H / c.KH, rows = a.T * gsz, row0 = pair * kPrPair;
    const kv4_seqs seqs = {a.slots, a.lens, a.len_add, a.longest, c.slots, 0};
    const int len = seqs.len(b);
    if (len < 0 && threadIdx.x == 0 && pair == 0 && kh == 0 && split == 0 && a.err) atomicOr(a.err, kErrKvIndex);
    auto sees = [&](int r) { return max(0, len - a.T + 1 + min(r, rows - 1) / gsz); };  // positions that row r sees
    const int all = (sees(row0 + kPrPair - 1) + kKv4Rows - 1) / kKv4Rows;  // the pair's cache blocks, this split's: [jb, jb + nb)
    const int jb = (int)((long long)all * split / S), nb = (int)((long long)all * (split + 1) / S) - jb, off = jb * kKv4Rows;
    const int tiles = rows - row0 > kPrTile ? 2 : 1;
    // softmax threads: the row's place in q and out (rows past the last repeat it and are not written)
    const int row = row0 + (int)threadIdx.x, rc = min(row, rows - 1), tok = rc / gsz, h = kh * gsz + rc % gsz;
    const long long orow = (long long)b * a.T + tok;
    auto write = [&](int d, const float (&x)[8]) {
        put8(static_cast<T*>(a.out) + (orow * a.H + h) * HD + d, x);
        if (a.outT)
#pragma unroll
            for (int j = 0; j < 8; j++) a.outT[(size_t)(h * HD + d + j) * a.outT_ld + orow] = x[j];
    };
    if (nb == 0 && S > 1) {
        if (warp < 8) pr_part<HD>::stats(pr_part<HD>::of(a.ws, blockIdx.x))[threadIdx.x] = make_float2(-INFINITY, 0.0f);
        return;
    }
    if (nb == 0) {  // nothing to see for any row
        const float z[8] = {};
        if (warp < 8 && row < rows)
            for (int d = 0; d < HD; d += 8) write(d, z);
        return;
    }
    pr_held* held = reinterpret_cast<pr_held*>(smem + SM::held);
    if (threadIdx.x == 0) {
        sh.abort = 0, sh.err = a.err ? a.err : &g_kv4_status, sh.limit = a.wait_limit;
        if (S > 1) {
            held->out = pr_part<HD>::of(a.ws, blockIdx.x), held->H = held->gsz = 1, held->row0 = 0, held->rows = kPrPair;
        } else {
            held->out = static_cast<T*>(a.out) + ((long long)b * a.T * a.H + kh * gsz) * HD;
            held->H = a.H, held->gsz = gsz, held->row0 = row0, held->rows = rows;
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&sh.raw_full[i], 1);
            mbar_init(&sh.raw_empty[i], kPrUnpack);
            mbar_init(&sh.kv_full[i], kPrUnpack);
            mbar_init(&sh.kv_empty[i], tiles);
            mbar_init(&sh.s_full[i], 1);
            mbar_init(&sh.p_full[i], 4);
            mbar_init(&sh.pv_done[i], 1);
        }
        mbar_init(&sh.q_full, 4 * tiles);
        mbar_init(&sh.fin, 1);
        mbar_fence_init();
    }
    if (warp == 11) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)),
                     "r"(2 * SM::TCOLS));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    const bool gives_up = a.wait_limit == 0;  // every role leaves at its first wait
    if (gives_up && threadIdx.x == 0) atomicOr(sh.err, kErrTimeout);
    auto starts = [](int j) { return j % FOLD == 0; };  // blocks at which TMEM's sums start anew

    if (warp < 8) {
        // ---------------- softmax: thread = row of tile t = TMEM lane
        const int t = warp >> 2;
        if (t < tiles) {
            uint8_t* qs = smem + SM::q + t * PARTS * SM::QTILE;
            const float f = pr_load_q<HD, F32, T>(
                [&](int i) {
                    const int r = min(row0 + warp * 32 + i, rows - 1);
                    return static_cast<const T*>(a.q) + ((long long)b * a.T + r / gsz) * a.q_stride + (kh * gsz + r % gsz) * HD;
                },
                qs, (warp & 3) * 32);
            fence_proxy_async_smem();  // before the tensor cores read it
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.q_full);
            const int n_row = sees(row) - off, n_min = sees(row0 + t * kPrTile) - off;
            const uint32_t ts = tmem + ((uint32_t)((warp & 3) * 32) << 16) + t * SM::TCOLS, to = ts + SM::SCOLS;
            pr_run<HD> st;
            st.r.clear(), st.lsum.clear(), st.j = 0;
            if (gives_up) st.j = -1;
            else st = pr_softmax<HD, F32, false>(smem, t, ts, f, nb, S, n_row, n_min, st);
            if (st.j >= 0 && st.j < nb) st = pr_softmax_lifted<HD, F32>(smem, t, ts, f, nb, S, n_row, n_min, st);
            const kv4_ref<NG == 2> r = st.r;
            if (st.j == nb && pr_wait(&sh.pv_done[t], (nb - 1) & 1, sh)) {
                tc_fence_after();
                const float ls = st.lsum.total();
                int tx = threadIdx.x;
                asm volatile("" : "+r"(tx));  // the row's place again (kept over the loop it took registers)
                const int row = row0 + tx, rc = min(row, rows - 1), h = kh * gsz + rc % gsz;
                const long long orow = (long long)b * a.T + rc / gsz;
                griddep_launch_dependents();  // not before: the next kernel's blocks, the merge's, would poll beside this one's
                if (S > 1) {
                    pr_fold<HD, false>(to, r.ref, r.less(), held, nb > FOLD);
                    pr_part<HD>::stats(static_cast<float*>(held->out))[threadIdx.x] = make_float2(r.ref, ls);
                } else {
                    if (nb > FOLD) pr_unfold<HD, !F32>(to, r.ref, r.more(), held);
                    const float inv = ls == 0.0f ? 0.0f : 1.0f / ls;
                    // through the tile's q (no longer read), 16 bytes at a time, so that whole rows are written at once
                    constexpr int VPC = 16 / sizeof(T), CPR = HD / VPC;  // values of a piece, pieces of a row
                    T* st = reinterpret_cast<T*>(qs) + (warp & 3) * 32 * HD;
#pragma unroll 1
                    for (int q = 0; q < NG * 4; q++) {
                        float o[16];
                        tc_ld16(to + 16 * q, o);
#pragma unroll
                        for (int i = 0; i < 16; i++) o[i] = ls == 0.0f ? 0.0f : o[i] * (q < 4 ? inv : inv * r.less());
#pragma unroll
                        for (int i = 0; i < 16; i += VPC) {
                            const int p = (16 * q + i) / VPC;
                            store_piece(st + (lane * CPR + (p ^ (lane & 7))) * VPC, o + i);
                        }
                        if (a.outT && row < rows)
#pragma unroll
                            for (int i = 0; i < 16; i++) a.outT[(size_t)(h * HD + 16 * q + i) * a.outT_ld + orow] = o[i];
                    }
                    __syncwarp();  // (and the warp has taken what `out` held)
#pragma unroll 4
                    for (int i = lane; i < 32 * CPR; i += 32) {
                        const int r = i / CPR, p = i % CPR, g = row0 + warp * 32 + r;
                        if (g >= rows) break;
                        const long long to_row = (long long)b * a.T + g / gsz;
                        *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + (to_row * a.H + kh * gsz + g % gsz) * HD + p * VPC) =
                            *reinterpret_cast<const uint4*>(st + (r * CPR + (p ^ (r & 7))) * VPC);
                    }
                }
            }
        }
    } else if (warp < 8 + kPrUnpack) {
        // ---------------- unpack, and the copies of the cache's blocks
        const int tid = threadIdx.x - 256, w = warp - 8;
        const float factor = a.scale * 1.4426950408889634f;
        const uint8_t* src = c.run(a.slots[b], l, kh) + (size_t)jb * BLK;
        uint8_t* raw = smem + SM::raw;
        auto issue = [&](int j) {
            mbar_expect_tx(&sh.raw_full[j & 1], BLK);
            bulk_g2s(raw + (j & 1) * BLK, src + (size_t)j * BLK, BLK, &sh.raw_full[j & 1]);
        };
        int issued = 0, j = 0;
        if (tid == 0)
            while (issued < min(nb, 2)) issue(issued++);
        __syncwarp();
        for (; j < nb; j++) {
            const int s = j & 1;
            if (gives_up || !pr_wait(&sh.raw_full[s], j >> 1 & 1, sh)) break;
            if (j >= 2 && !pr_wait(&sh.kv_empty[s], (j >> 1) + 1 & 1, sh)) break;
            pr_unpack<HD>(raw + s * BLK, smem + SM::k + s * SM::KTILE, smem + SM::v + s * SM::VTILE,
                          reinterpret_cast<float*>(smem + SM::sc) + s * 4 * kKv4Rows, sh.range[s], factor, len - off - j * kKv4Rows, tid);
            fence_proxy_async_smem();  // the operands to the tensor cores, the reads before the next copy
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&sh.kv_full[s]);
                mbar_arrive(&sh.raw_empty[s]);
            }
            if (w == 0 && j + 2 < nb) {
                if (!pr_wait(&sh.raw_empty[s], j >> 1 & 1, sh)) {
                    j++;
                    break;
                }
                if (tid == 0) issue(issued++);
                __syncwarp();
            }
        }
        if (tid == 0)
            for (; j < issued; j++) mbar_wait_bounded(&sh.raw_full[j & 1], j >> 1 & 1, sh.err);  // no copy left in flight
    } else {
        // ---------------- the instructions (a whole warp, one elected lane issues). The
        // tiles take turns: a tile's values and its next scores go out together, and
        // the other tile's softmax runs meanwhile. (With an issuer per tile both were in
        // the same phase and nothing overlapped: 6,760 cycles for a block of both.)
        const uint32_t idesc = umma_idesc_f16(64);
        const uint64_t kd = umma_desc(smem + SM::k, 1024, 128);
        const uint64_t vd = umma_desc(smem + SM::v, 8 * kPrCore, kPrCore);
        auto scores = [&](int t, int j) {
            if (!pr_wait(&sh.kv_full[j & 1], j >> 1 & 1, sh)) return false;
            tc_fence_after();
            if (elect_one()) {
                const uint64_t qd = umma_desc(smem + SM::q + t * PARTS * SM::QTILE, SM::QCHUNK, 128);
                // lo first: half of the cut-off sums are small then (a prompt's error 1.5e-6 -> 1.1e-6)
#pragma unroll
                for (int g = 0; g < NG; g++)
#pragma unroll
                    for (int p = 0; p < PARTS; p++)
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            tc_mma_ss(tmem + t * SM::TCOLS + 64 * g, qd + (((PARTS - 1 - p) * SM::QTILE + (g * 4 + k) * 2 * SM::QCHUNK) >> 4),
                                      kd + (((j & 1) * SM::KTILE + (g * 4 + k) * 2048) >> 4), idesc, p + k > 0);
                tc_commit(&sh.s_full[t]);
            }
            __syncwarp();
            return true;
        };
        bool ok = !gives_up && pr_wait(&sh.q_full, 0, sh);
        for (int t = 0; ok && t < tiles; t++) ok = scores(t, 0);
        for (int j = 0; ok && j < nb; j++)
            for (int t = 0; ok && t < tiles; t++) {
                const int s = j & 1;
                if (!pr_wait(&sh.p_full[t], j & 1, sh)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                if (elect_one()) {
                    const bool fresh = starts(j);
                    const uint32_t ts = tmem + t * SM::TCOLS, to = ts + SM::SCOLS;
#pragma unroll
                    for (int g = 0; g < NG; g++)
#pragma unroll
                        for (int p = 0; p < 2; p++)
#pragma unroll
                            for (int k = 0; k < 4; k++)
                                tc_mma_ts(to + 64 * g, ts + 64 * g + 32 * (1 - p) + 8 * k,
                                          vd + ((s * SM::VTILE + (g * 64 + k * 16) * kPrCore) >> 4), idesc,
                                          p + k > 0 || !fresh);
                    tc_commit(&sh.pv_done[t]);
                    tc_commit(&sh.kv_empty[s]);
                }
                __syncwarp();
                // the next scores go where these weights are: after the product that reads them
                if (j + 1 < nb) ok = pr_wait(&sh.pv_done[t], j & 1, sh) && scores(t, j + 1);
            }
        if (elect_one()) tc_commit(&sh.fin);  // no instruction left in flight
        __syncwarp();
        mbar_wait_bounded(&sh.fin, 0, sh.err);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 11)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * SM::TCOLS));
}

// Adds the splits of 32 rows up: warp w takes splits w, w + 8, ..., lane = row, 32
// values of each (blockIdx.y).
template <int HD, typename T>
__global__ void __launch_bounds__(256) k_kv4_prompt_merge(kv4_dims c, jl_kv4_attn_args a, int pairs, int S) {
    __shared__ float4 sums[8][8][32];
    __shared__ float2 stats[8][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, per = c.KH * a.B, unit = blockIdx.x / 8, grp = blockIdx.x % 8;
    const int pair = pairs - 1 - unit / per, kh = unit % c.KH, b = unit % per / c.KH;
    const int gsz = a.H / c.KH, rows = a.T * gsz, row = pair * kPrPair + grp * 32 + lane;
    griddep_wait();
    griddep_launch_dependents();
    if (row - lane >= rows) return;
    float m = -INFINITY, ls = 0.0f;
    float4 x[8] = {};
    for (int s = warp; s < S; s += 8) {
        float* p = pr_part<HD>::of(a.ws, (size_t)unit * S + s);
        const float4* y = reinterpret_cast<const float4*>(p) + (grp * (HD / 4) + blockIdx.y * 8) * 32 + lane;
        const float2 st = pr_part<HD>::stats(p)[grp * 32 + lane];
        float4 v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = y[i * 32];
        if (st.y == 0.0f) continue;  // (a split of no blocks wrote no sums)
        const float nm = fmaxf(m, st.x), al = ex2(m - nm), f = ex2(st.x - nm);
        m = nm;
        ls = fmaf(ls, al, st.y * f);
#pragma unroll
        for (int i = 0; i < 8; i++)
            x[i] = make_float4(fmaf(x[i].x, al, v[i].x * f), fmaf(x[i].y, al, v[i].y * f), fmaf(x[i].z, al, v[i].z * f),
                               fmaf(x[i].w, al, v[i].w * f));
    }
#pragma unroll
    for (int i = 0; i < 8; i++) sums[warp][i][lane] = x[i];
    stats[warp][lane] = make_float2(m, ls);
    __syncthreads();
    // warp w: piece w of the 32 values
    m = -INFINITY;
#pragma unroll
    for (int w = 0; w < 8; w++) m = fmaxf(m, stats[w][lane].x);
    m = m == -INFINITY ? 0.0f : m;
    ls = 0.0f;
    float o[4] = {};
#pragma unroll
    for (int w = 0; w < 8; w++) {
        const float2 st = stats[w][lane];
        const float f = ex2(st.x - m);
        const float4 v = sums[w][warp][lane];
        ls = fmaf(st.y, f, ls);
        o[0] = fmaf(v.x, f, o[0]), o[1] = fmaf(v.y, f, o[1]), o[2] = fmaf(v.z, f, o[2]), o[3] = fmaf(v.w, f, o[3]);
    }
    if (row >= rows) return;
    const float inv = ls == 0.0f ? 0.0f : 1.0f / ls;
    const int h = kh * gsz + row % gsz, d = blockIdx.y * 32 + warp * 4;
    const long long orow = (long long)b * a.T + row / gsz;
    T* to = static_cast<T*>(a.out) + (orow * a.H + h) * HD + d;
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] *= inv;
    put4(to, o);
    if (a.outT)
#pragma unroll
        for (int i = 0; i < 4; i++) a.outT[(size_t)(h * HD + d + i) * a.outT_ld + orow] = o[i];
}

}  // namespace jl

namespace {

std::atomic<long long> g_wait_limit{jl::kWaitLimitCycles};

template <int HD, typename T>
int launch_t(const jl::kv4_dims& c, int l, const jl_kv4_attn_args& a, int S, cudaStream_t s) {
    using namespace jl;
    const long long units = jl_kv4_prompt_units(c, a.B, a.T, a.H), pairs = units / ((long long)c.KH * a.B);
    if (units > INT_MAX / 8) return JL_ERR_INVALID;
    const int rc = launch(k_kv4_prompt<HD, T>, dim3((unsigned)units * S), dim3(kPrThreads),
                          (size_t)pr_smem<HD, sizeof(T) == 4>::total, s, c, l, a, (int)pairs, S);
    if (rc || S == 1) return rc;
    return launch(k_kv4_prompt_merge<HD, T>, dim3((unsigned)units * 8, HD / 32), dim3(256), 0, s, c, a, (int)pairs, S);
}

template <int HD>
int prompt_attrs() {
    using namespace jl;
    JL_CUDA(cudaFuncSetAttribute(k_kv4_prompt<HD, float>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (pr_smem<HD, true>::total)));
    JL_CUDA(cudaFuncSetAttribute(k_kv4_prompt<HD, __half>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (pr_smem<HD, false>::total)));
    JL_CUDA(cudaFuncSetAttribute(k_kv4_prompt<HD, __nv_bfloat16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (pr_smem<HD, false>::total)));
    return JL_OK;
}

}  // namespace

long long jl_kv4_prompt_units(const jl::kv4_dims& c, int B, int T, int H) {
    return ((long long)T * (H / c.KH) + jl::kPrPair - 1) / jl::kPrPair * c.KH * B;
}

long long jl_kv4_prompt_ws_bytes(const jl::kv4_dims& c, long long units, int S) {
    return S > 1 ? units * S * (c.hd == 64 ? jl::pr_part<64>::floats : jl::pr_part<128>::floats) * (long long)sizeof(float) : 0;
}

int jl_launch_kv4_prompt(const jl::kv4_dims& c, int l, const jl_kv4_attn_args& args, int S, cudaStream_t s) {
    jl_kv4_attn_args a = args;
    a.wait_limit = g_wait_limit.load(std::memory_order_relaxed);
    const int rc = jl_device_once(kOnceKv4Prompt, [] {
        const int r = prompt_attrs<64>();
        return r ? r : prompt_attrs<128>();
    });
    if (rc) return rc;
    if (a.dtype == JL_F32) return c.hd == 64 ? launch_t<64, float>(c, l, a, S, s) : launch_t<128, float>(c, l, a, S, s);
    if (a.dtype == JL_F16) return c.hd == 64 ? launch_t<64, __half>(c, l, a, S, s) : launch_t<128, __half>(c, l, a, S, s);
    return c.hd == 64 ? launch_t<64, __nv_bfloat16>(c, l, a, S, s) : launch_t<128, __nv_bfloat16>(c, l, a, S, s);
}

extern "C" int jl_kv4_set_wait_limit(long long ns) {
    if (ns < 0) return JL_ERR_INVALID;
    // clock64 counts SM cycles; 2 a ns bound a wait by at least `ns` at any SM clock up to 2 GHz
    g_wait_limit.store(ns > (1ll << 61) ? 1ll << 62 : 2 * ns, std::memory_order_relaxed);
    return JL_OK;
}

extern "C" int jl_kv4_check(void* stream) {
    cudaStream_t s = (cudaStream_t)stream;
    int err = 0;
    JL_CUDA(cudaMemcpyFromSymbolAsync(&err, jl::g_kv4_status, sizeof(int), 0, cudaMemcpyDeviceToHost, s));
    JL_CUDA(cudaStreamSynchronize(s));
    if (!err) return JL_OK;
    const int zero = 0;
    JL_CUDA(cudaMemcpyToSymbolAsync(jl::g_kv4_status, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, s));
    JL_CUDA(cudaStreamSynchronize(s));
    return JL_ERR_TIMEOUT;
}
