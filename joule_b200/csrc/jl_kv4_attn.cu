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
#include <algorithm>
#include <climits>
#include <cmath>

#include "jl_internal.h"
#include "jl_kv4_dev.cuh"

namespace jl {

constexpr int kKvRing = 2;     // units in a warp's ring
constexpr int kKvTile = 8;     // query rows of a tile

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same onto zeros.
__device__ __forceinline__ void mma16816_0(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                           uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
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
// spread over all blocks first; a block of fewer units than nw leaves warps idle).
// U >= 1.
struct kv4_cut {
    uint32_t ctas, nw;
    kv4_split by_block;
    __device__ kv4_cut(uint32_t U, uint32_t blocks, uint32_t NW)
        : ctas(min(blocks, U)), nw(min(NW, (U - 1) / min(blocks, U) + 1)), by_block(U, min(blocks, U)) {}
    __device__ uint32_t start(uint32_t c) const { return by_block.start(c); }
    __device__ uint32_t warps(uint32_t c) const { return min(nw, start(c + 1) - start(c)); }  // that have units
    __device__ kv4_split by_warp(uint32_t c) const { return kv4_split(start(c + 1) - start(c), warps(c)); }
    __device__ uint32_t warp_of(uint32_t u) const {  // nw * block + warp
        const uint32_t c = by_block.of(u);
        return c * nw + by_warp(c).of(u - start(c));
    }
};

// A partial result in the workspace: O [8][HD], then per row the reference of its
// exponents (base 2) and its sum of weights. Warp w's part 0 belongs to the segment
// that began before its run, part 1 to the one that begins in it and goes on past
// it. Where all warps of a block are inside one segment, the block's first warp
// holds their sum.
__host__ __device__ constexpr int kv4_part_floats(int hd) { return kKvTile * hd + 2 * kKvTile; }

constexpr int kKvWarps = 12;  // warps per block, one block per SM (168 registers a thread, 209 KB at hd = 128)
template <int HD>
struct kv4_smem {
    static constexpr int UNIT = kv4_block_bytes(HD);
    // the warps' rings, then (reference, sum) [warps][2][8] of the block's sum
    __host__ __device__ static constexpr int stat(int warps) { return warps * kKvRing * UNIT; }
    static constexpr int bytes(int warps) { return stat(warps) + warps * 2 * kKvTile * 4; }
    static constexpr int total = bytes(kKvWarps);
    static_assert(kKvRing * UNIT >= kKvTile * HD * 4, "a warp's ring holds its sums");
};

// One warp's running state for the segment it is in. Both operands that are not
// codes enter as hi and lo parts of 11 bits each. Scores are S = q K^T with q's hi
// parts in the instruction's rows 0-7 and its lo parts in rows 8-15 (one instruction
// for both); values are O^T = V^T P^T with the 8 rows of the tile as the columns (an
// instruction each for hi and lo, onto the same 32 registers of sums). A thread's
// scores are then where the second product wants its weights: thread (g, t) =
// (lane / 4, lane % 4) has row g at positions 2 t, 2 t + 1, 2 t + 8, 2 t + 9, and
// sums of rows 2 t and 2 t + 1.
template <int HD>
struct kv4_state {
    static constexpr int NG = HD / 64;
    uint32_t qf[NG * 4][4];  // q of row g per step of 16 values
    float f;                 // accumulator -> score in base 2 (a power of two)
    kv4_ref<NG == 2> r;      // row g's references
    kv4_sum l;               // this thread's sum of row g's weights
    float o[NG][4][4];       // o[gr][i][c]: value 64 gr + 8 g + 2 i + c / 2 of row 2 t + c % 2
    int n;                   // positions that row g sees
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
    // q by a power of two so that its largest value is in [2^10, 2^11)
    int e = (int)(__float_as_uint(mx) >> 23);
    e = min(max(e, 11), 253);
    const float inv = __uint_as_float((uint32_t)(264 - e) << 23);
    st.f = __uint_as_float((uint32_t)(e - 10) << 23);
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
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int c = 0; c < 4; c++) st.o[g][i][c] = 0.0f;
    }
    st.r.clear();
    st.l.clear();
}

// Scores in base 2 of positions r0 .. r0 + 15 of a block: s[h] = those of
// r0 + 8 h + 2 t and the next. Codes become n - 8 exactly, by one AND-OR into
// 1024's mantissa and one packed fp16 sum per two values (the offset's own sum would
// be far larger than the results'). K's scale multiplies the accumulated group in
// fp32. Four sums take turns, since an instruction's result is there 20 cycles
// later and the next one can start after 8.
template <int HD>
__device__ __forceinline__ void kv4_scores(const kv4_state<HD>& st, const uint8_t* blk, int r0, float2 (&s)[2]) {
    constexpr int NG = HD / 64, ROW = HD / 2;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    float acc[2][NG][4];
    uint32_t kw[2][NG * 2];
    const uint8_t* kp = blk + (r0 + g) * ROW + t * 8 * NG;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        if (NG == 2) {
            const uint4 w = *reinterpret_cast<const uint4*>(kp + 8 * h * ROW);
            kw[h][0] = w.x, kw[h][1] = w.y, kw[h][NG] = w.z, kw[h][2 * NG - 1] = w.w;
        } else {
            const uint2 w = *reinterpret_cast<const uint2*>(kp + 8 * h * ROW);
            kw[h][0] = w.x, kw[h][1] = w.y;
        }
    }
#pragma unroll
    for (int w = 0; w < 2; w++)
#pragma unroll
        for (int sh = 0; sh < 2; sh++)
#pragma unroll
            for (int gr = 0; gr < NG; gr++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint32_t x = sh ? kw[h][w * NG + gr] >> 8 : kw[h][w * NG + gr];
                    const uint32_t (&a)[4] = st.qf[gr * 4 + w * 2 + sh];
                    if (w + sh == 0) mma16816_0(acc[h][gr], a[0], a[1], a[2], a[3], code_even(x), code_odd(x));
                    else mma16816(acc[h][gr], a[0], a[1], a[2], a[3], code_even(x), code_odd(x));
                }
#pragma unroll
    for (int h = 0; h < 2; h++) {
        float2 sc[NG];
        scale_pairs<NG>(blk + kv4_kscale(HD), r0 + 8 * h + 2 * t, sc);
        s[h] = __fmul2_rn(sc[0], __fadd2_rn(make_float2(acc[h][0][0], acc[h][0][1]), make_float2(acc[h][0][2], acc[h][0][3])));
        if (NG == 2)
            s[h] = __ffma2_rn(sc[NG - 1], __fadd2_rn(make_float2(acc[h][NG - 1][0], acc[h][NG - 1][1]),
                                                     make_float2(acc[h][NG - 1][2], acc[h][NG - 1][3])), s[h]);
        s[h] = __fmul2_rn(s[h], f2(st.f));
    }
}

// A product past the limit (or the first of a row): its row takes new references, and
// its sums are brought to them. mx, b0, b1 (kv4_ref): this thread's part of row g.
template <int HD>
__device__ __forceinline__ void kv4_new_reference(kv4_state<HD>& st, float mx, float b0, float b1) {
    const int t = threadIdx.x & 3;
#pragma unroll
    for (int o = 1; o <= 2; o <<= 1) {
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        b0 = fmaxf(b0, __shfl_xor_sync(0xffffffffu, b0, o));
        if (HD == 128) b1 = fmaxf(b1, __shfl_xor_sync(0xffffffffu, b1, o));
    }
    const float2 al = st.r.past(mx, b0, b1) ? st.r.move(mx, b0, b1) : f2(1.0f);
    st.l.scale(al.x);
#pragma unroll
    for (int gr = 0; gr < HD / 64; gr++) {
        const float x = gr ? al.y : al.x;
        const float2 ac = make_float2(__shfl_sync(0xffffffffu, x, 8 * t), __shfl_sync(0xffffffffu, x, 8 * t + 4));
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int c = 0; c < 4; c++) st.o[gr][i][c] *= c & 1 ? ac.y : ac.x;
    }
}

// Weights of positions r0 .. r0 + 15 from their scores, and the weighted values
// onto the sums; adds the weights to l. V's scale multiplies the weight in fp32. MASK: row g does not see
// positions from n on (in the block's numbering); those may hold any scale.
template <int HD, bool MASK>
__device__ __forceinline__ void kv4_values(kv4_state<HD>& st, const uint8_t* blk, int r0, float2 (&s)[2], float2& l, int n) {
    constexpr int NG = HD / 64, ROW = HD / 2;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    uint32_t bh[NG][2], bl[NG][2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        float2 sc[NG];
        scale_pairs<NG>(blk + kv4_vscale(HD), r0 + 8 * h + 2 * t, sc);
        s[h] = __fadd2_rn(s[h], f2(st.r.minus()));
        s[h].x = ex2(s[h].x);
        s[h].y = ex2(s[h].y);
        l = __fadd2_rn(l, s[h]);
#pragma unroll
        for (int gr = 0; gr < NG; gr++) {
            float2 w = __fmul2_rn(s[h], sc[gr]);
            if (gr) w = __fmul2_rn(w, f2(st.r.more()));
            if (MASK) {
                if (r0 + 8 * h + 2 * t >= n) w.x = 0.0f;
                if (r0 + 8 * h + 2 * t + 1 >= n) w.y = 0.0f;
            }
            split2(w, bh[gr][h], bl[gr][h]);
        }
    }
    // thread (g, t) unpacks values 8 g .. 8 g + 7 of each group at positions 2t, 2t + 1, 2t + 8, 2t + 9
    // (places t, 4 + t, 8 + t, 12 + t)
    uint32_t vw[4][NG];
    const uint8_t* vp = blk + kv4_vcode(HD) + (r0 + t) * ROW + (g ^ ((t & 2) << 1)) * 4 * NG;
#pragma unroll
    for (int r = 0; r < 4; r++) {
        if (NG == 2) {
            const uint2 w = *reinterpret_cast<const uint2*>(vp + 4 * r * ROW);
            vw[r][0] = w.x, vw[r][NG - 1] = w.y;
        } else {
            vw[r][0] = *reinterpret_cast<const uint32_t*>(vp + 4 * r * ROW);
        }
    }
#pragma unroll
    for (int q = 0; q < 2; q++) {  // values 4q .. 4q + 3 of the words, 2 per instruction: four sums take turns
        uint32_t f[NG][2][4];
#pragma unroll
        for (int gr = 0; gr < NG; gr++) {
            const uint32_t x = __byte_perm(vw[0][gr], vw[1][gr], q ? 0x7632 : 0x5410);
            const uint32_t y = __byte_perm(vw[2][gr], vw[3][gr], q ? 0x7632 : 0x5410);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                f[gr][i][0] = code_even(i ? x >> 8 : x), f[gr][i][1] = code_odd(i ? x >> 8 : x);
                f[gr][i][2] = code_even(i ? y >> 8 : y), f[gr][i][3] = code_odd(i ? y >> 8 : y);
            }
        }
        // The instruction's sums are cut off, not rounded: 16 positions start from zero and
        // are added here, or a long run's outputs shrink (by 1.3e-6 of themselves after 18
        // blocks, and on with the length).
        float acc[NG][2][4];
#pragma unroll
        for (int gr = 0; gr < NG; gr++)
#pragma unroll
            for (int i = 0; i < 2; i++)
                mma16816_0(acc[gr][i], f[gr][i][0], f[gr][i][1], f[gr][i][2], f[gr][i][3], bl[gr][0], bl[gr][1]);
#pragma unroll
        for (int gr = 0; gr < NG; gr++)
#pragma unroll
            for (int i = 0; i < 2; i++)
                mma16816(acc[gr][i], f[gr][i][0], f[gr][i][1], f[gr][i][2], f[gr][i][3], bh[gr][0], bh[gr][1]);
#pragma unroll
        for (int gr = 0; gr < NG; gr++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                float (&o)[4] = st.o[gr][2 * q + i];
                const float2 x0 = __fadd2_rn(make_float2(o[0], o[1]), make_float2(acc[gr][i][0], acc[gr][i][1]));
                const float2 x1 = __fadd2_rn(make_float2(o[2], o[3]), make_float2(acc[gr][i][2], acc[gr][i][3]));
                o[0] = x0.x, o[1] = x0.y, o[2] = x1.x, o[3] = x1.y;
            }
    }
}

// One block (j0 = its first position's number): rows see all positions below n_min
// and none from n_max on. A block that all rows see whole, with scales of about one
// size, is one stretch of code with one branch; others go by 16 positions.
template <int HD>
__device__ __forceinline__ void kv4_block(kv4_state<HD>& st, const uint8_t* blk, int j0, int n_min, int n_max) {
    constexpr int NG = HD / 64;
    const int lane = threadIdx.x & 31, t = lane & 3;
    if (j0 + kKv4Rows <= n_min) {
        const uint16_t* p = reinterpret_cast<const uint16_t*>(blk + kv4_vscale(HD)) + lane * NG;
        uint32_t most = max(p[0], p[32 * NG]), least = min(p[0], p[32 * NG]);
        if (NG == 2) most = max(most, max(p[1], p[32 * NG + 1])), least = min(least, min(p[1], p[32 * NG + 1]));
        most = __reduce_max_sync(0xffffffffu, most);
        if (!kv4_spread(most, __reduce_min_sync(0xffffffffu, least))) {
            const float top = kv4_top(most);
            float2 s[4][2], l = f2(0.0f);
            float mx = -INFINITY;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                kv4_scores<HD>(st, blk, 16 * k, s[k]);
                mx = fmaxf(mx, fmaxf(fmaxf(s[k][0].x, s[k][0].y), fmaxf(s[k][1].x, s[k][1].y)));
            }
            if (__any_sync(0xffffffffu, st.r.past(mx, top, top))) kv4_new_reference<HD>(st, mx, top, top);
#pragma unroll
            for (int k = 0; k < 4; k++) kv4_values<HD, false>(st, blk, 16 * k, s[k], l, 0);
            st.l.add(l);
            return;
        }
    }
    const int n = st.n - j0;
#pragma unroll 1
    for (int r0 = 0; r0 < min(kKv4Rows, n_max - j0); r0 += 16) {
        float2 s[2], l = f2(0.0f);
        kv4_scores<HD>(st, blk, r0, s);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            if (r0 + 8 * h + 2 * t >= n) s[h].x = -INFINITY;
            if (r0 + 8 * h + 2 * t + 1 >= n) s[h].y = -INFINITY;
        }
        float mx = fmaxf(fmaxf(s[0].x, s[0].y), fmaxf(s[1].x, s[1].y)), b[2] = {kLeast, kLeast};
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
#pragma unroll
        for (int h = 0; h < 2; h++) {  // (an unseen position's score stays -infinity whatever its scale's bits are)
            float2 sc[NG];
            scale_pairs<NG>(blk + kv4_vscale(HD), r0 + 8 * h + 2 * t, sc);
#pragma unroll
            for (int gr = 0; gr < NG; gr++)
                b[gr] = fmaxf(b[gr], fmaxf((s[h].x - mx) + exponent_of(sc[gr].x), (s[h].y - mx) + exponent_of(sc[gr].y)));
        }
        if (__any_sync(0xffffffffu, st.r.past(mx, b[0], b[1]))) kv4_new_reference<HD>(st, mx, b[0], b[1]);
        kv4_values<HD, true>(st, blk, r0, s, l, n);
        st.l.add(l);
    }
}

// Bound by issue slots for long caches (1,545 instructions a cache block and tile, two
// fifths of them taking codes apart; the codes and scales are read once, DRAM at 36 %) and by
// launch and load latency for short ones. Each warp has a ring
// of two whole cache blocks, filled by 16-byte asynchronous copies (17 instructions a
// block; a bulk copy held its issuing warp for hundreds of ns); no barrier between
// warps but for the sum of a block that is inside one segment.
// BLOCK: a segment per block (of 12 warps or, two and three to an SM, of 6 and 4), whose
// warps share it and join here; no cut, no second kernel.
template <int HD, typename T, bool BLOCK>
__global__ void __launch_bounds__(kKvWarps * 32, 1) k_kv4_attn(kv4_dims c, int l, jl_kv4_attn_args a, int R, int whole) {
    extern __shared__ __align__(128) uint8_t smem[];
    using SM = kv4_smem<HD>;
    constexpr int UNIT = SM::UNIT, NG = HD / 64;
    const int NW = BLOCK ? blockDim.x >> 5 : kKvWarps;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    uint8_t* ring = smem + warp * kKvRing * UNIT;
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
    struct cursor {
        int b, s, j, nu;  // sequence, segment, unit of nu
        const uint8_t* p;  // the unit
    } pr;
    int used, nw = 1, units;  // warps of the block that have units, of any block; units of this warp's run
    uint32_t c0, c1, u0;       // the block's units, the warp's first
    if constexpr (BLOCK) {
        pr.b = blockIdx.x / S, pr.s = blockIdx.x % S, pr.nu = seqs.units(pr.b);
        used = min(NW, pr.nu), c0 = 0, c1 = pr.nu;
        const kv4_split mine(max(1, pr.nu), max(1, used));
        pr.j = u0 = warp < used ? mine.start(warp) : 0;
        units = warp < used ? mine.start(warp + 1) - u0 : 0;  // (all warps join the sums)
    } else {
        const uint32_t U = warp_total(seqs, a.B) * S;
        if (U == 0) return;
        const kv4_cut cut(U, gridDim.x, NW);
        if (blockIdx.x >= cut.ctas) return;
        used = cut.warps(blockIdx.x);
        if (warp >= used) return;
        nw = cut.nw;
        const kv4_split mine = cut.by_warp(blockIdx.x);
        c0 = cut.start(blockIdx.x), c1 = cut.start(blockIdx.x + 1), u0 = c0 + mine.start(warp);
        units = mine.start(warp + 1) - mine.start(warp);
        uint32_t off;
        warp_find(seqs, a.B, S, u0, pr.b, off);
        pr.nu = seqs.units(pr.b);
        pr.s = (int)(whole ? off : off / pr.nu);
        pr.j = (int)(whole ? 0 : off % pr.nu);
    }
    if (!BLOCK && whole) {  // so many segments, each with its sequence's units
        int segs = units, bb = pr.b, ss = pr.s;
        for (units = 0; segs; segs--) {
            units += seqs.units(bb);
            if (++ss == S && segs > 1) {
                ss = 0;
                do bb++;
                while (seqs.units(bb) == 0);
            }
        }
    }
    pr.p = c.run(a.slots[pr.b], l, pr.s / R) + (size_t)pr.j * UNIT;
    auto advance = [&](cursor& x) {  // not past the last unit
        x.p += UNIT;
        if (++x.j == x.nu) {
            x.j = 0;
            if (++x.s == S) {
                x.s = 0;
                do x.nu = seqs.units(++x.b);
                while (x.nu == 0);
            }
            x.p = c.run(a.slots[x.b], l, x.s / R);
        }
    };
    cursor co = pr;
    // the block's run is inside one segment: its warps' sums meet here
    const uint32_t seg0 = u0 - pr.j;
    const bool joined = BLOCK ? used > 1 : !whole && nw > 1 && c0 >= seg0 && c1 <= seg0 + pr.nu;
    int issued = 0;
    auto issue = [&]() {  // one group of copies per unit, an empty one past the last
        if (issued < units) {
            uint8_t* dst = ring + issued % kKvRing * UNIT + lane * 16;
#pragma unroll
            for (int i = 0; i < (UNIT / 16 + 31) / 32; i++)
                if (UNIT % 512 == 0 || i * 512 + lane * 16 < UNIT) cp_async16(dst + i * 512, pr.p + i * 512 + lane * 16);
            if (++issued < units) advance(pr);
        }
        cp_async_commit();
    };
    issue();  // all warps' first units before anyone's others
    kv4_state<HD> st;
    int n_min = 0, n_max = 0;
    bool began = false;
    for (int i = 0; i < units; i++) {
        if (!began) {  // a new segment: its rows (those past the last repeat it and are not written)
            const int kh = co.s / R, rt = co.s % R, len = seqs.len(co.b);
            auto row_of = [&](int r) { return min(rt * kKvTile + r, rows - 1); };
            auto sees = [&](int r) { return max(0, len - a.T + 1 + row_of(r) / gsz); };
            const int r = row_of(g), tok = r / gsz, h = kh * gsz + r % gsz;
            kv4_load_q<HD, T>(st, static_cast<const T*>(a.q) + ((long long)co.b * a.T + tok) * a.q_stride + h * HD,
                              a.scale);
            st.n = sees(g);
            n_min = sees(0), n_max = sees(kKvTile - 1);
            began = true;
            if (i == 0) {
#pragma unroll
                for (int k = 1; k < kKvRing; k++) issue();
            }
        }
        cp_async_wait<kKvRing - 1>();  // this unit's copies, by every lane
        __syncwarp();
        const int j0 = co.j * kKvUnit;
        if (j0 < n_max) kv4_block<HD>(st, ring + i % kKvRing * UNIT, j0, n_min, n_max);
        __syncwarp();
        issue();
        const bool ends = co.j == co.nu - 1;
        if (ends || i == units - 1) {
            float lrow = st.l.total();
            lrow += __shfl_xor_sync(0xffffffffu, lrow, 1);
            lrow += __shfl_xor_sync(0xffffffffu, lrow, 2);
            const float2 lsum = make_float2(__shfl_sync(0xffffffffu, lrow, 8 * t), __shfl_sync(0xffffffffu, lrow, 8 * t + 4));
            if (NG == 2) {  // both groups' sums on one scale
                const float x = st.r.less(), x0 = __shfl_sync(0xffffffffu, x, 8 * t), x1 = __shfl_sync(0xffffffffu, x, 8 * t + 4);
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int c = 0; c < 4; c++) st.o[NG - 1][j][c] *= c & 1 ? x1 : x0;
            }
            const bool from_start = i >= co.j;  // the segment's first unit is in this warp's run
            if (ends && from_start) {
#pragma unroll
                for (int cc = 0; cc < 2; cc++) {
                    const int row = co.s % R * kKvTile + 2 * t + cc;
                    if (row >= rows) continue;
                    const float ls = cc ? lsum.y : lsum.x, inv = ls == 0.0f ? 0.0f : 1.0f / ls;
                    const int h = co.s / R * gsz + row % gsz;
                    const long long orow = (long long)co.b * a.T + row / gsz;
                    T* out = static_cast<T*>(a.out) + (orow * a.H + h) * HD;
#pragma unroll
                    for (int gr = 0; gr < NG; gr++) {
                        float x[8];
#pragma unroll
                        for (int j = 0; j < 8; j++) x[j] = st.o[gr][j / 2][j % 2 * 2 + cc] * inv;
                        const int d = gr * 64 + 8 * g;
                        put8(out + d, x);
                        if (a.outT)
#pragma unroll
                            for (int j = 0; j < 8; j++) a.outT[(size_t)(h * HD + d + j) * a.outT_ld + orow] = x[j];
                    }
                }
            } else {
                float* part = joined ? reinterpret_cast<float*>(ring)
                                     : static_cast<float*>(a.ws) + ((size_t)(blockIdx.x * nw + warp) * 2 + from_start) * kv4_part_floats(HD);
                float* ml = joined ? reinterpret_cast<float*>(smem + SM::stat(NW)) + warp * 2 * kKvTile : part + kKvTile * HD;
#pragma unroll
                for (int cc = 0; cc < 2; cc++) {
#pragma unroll
                    for (int gr = 0; gr < NG; gr++) {
                        float x[8];
#pragma unroll
                        for (int j = 0; j < 8; j++) x[j] = st.o[gr][j / 2][j % 2 * 2 + cc];
                        put8(part + (2 * t + cc) * HD + gr * 64 + 8 * g, x);
                    }
                }
                if (t == 0) {
                    ml[g] = st.r.ref;
                    ml[kKvTile + g] = lrow;
                }
            }
            began = false;
        }
        if (i + 1 < units) advance(co);
    }
    if (!joined) return;
    // the warps' sums, in their order
    const int joining = (BLOCK ? NW : used) * 32;
    asm volatile("bar.sync 1, %0;" ::"r"(joining) : "memory");
    const float* ml = reinterpret_cast<const float*>(smem + SM::stat(NW));
    float* part = static_cast<float*>(a.ws) +
                  ((size_t)blockIdx.x * nw * 2 + (c0 == seg0)) * kv4_part_floats(HD);
    for (int x = threadIdx.x; x < kKvTile * HD / 4; x += joining) {
        const int r = x / (HD / 4);
        float m = -INFINITY, lsum = 0.0f;
        for (int w = 0; w < used; w++) m = fmaxf(m, ml[w * 2 * kKvTile + r]);
        const float mu = m == -INFINITY ? 0.0f : m;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int w = 0; w < used; w++) {
            const float f = ex2(ml[w * 2 * kKvTile + r] - mu);
            const float4 v = reinterpret_cast<const float4*>(smem + w * kKvRing * UNIT)[x];
            lsum = fmaf(ml[w * 2 * kKvTile + kKvTile + r], f, lsum);
            o = make_float4(fmaf(v.x, f, o.x), fmaf(v.y, f, o.y), fmaf(v.z, f, o.z), fmaf(v.w, f, o.w));
        }
        if constexpr (BLOCK) {
            const int row = blockIdx.x % S % R * kKvTile + r, h = blockIdx.x % S / R * gsz + row % gsz, d = x % (HD / 4) * 4;
            if (row >= rows) continue;
            const float inv = lsum == 0.0f ? 0.0f : 1.0f / lsum, y[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
            const long long orow = (long long)(blockIdx.x / S) * a.T + row / gsz;
            put4(static_cast<T*>(a.out) + (orow * a.H + h) * HD + d, y);
            if (a.outT)
#pragma unroll
                for (int j = 0; j < 4; j++) a.outT[(size_t)(h * HD + d + j) * a.outT_ld + orow] = y[j];
            continue;
        }
        reinterpret_cast<float4*>(part)[x] = o;
        if (x % (HD / 4) == 0) {
            part[kKvTile * HD + r] = m;
            part[kKvTile * HD + kKvTile + r] = lsum;
        }
    }
}

// Adds up the parts of segments that several warps shared: block = RB rows of a run
// of segments, 8 / RB warps per row, each adding every (8 / RB)-th part.
// RUN: `per` segments a block, where a block each (2 us of latency, four to an SM)
// took longer than the sums (256 sequences of 16/16 heads over 512: 8 us of 98).
template <int HD, typename T, bool RUN>
__global__ void __launch_bounds__(256) k_kv4_merge(kv4_dims c, jl_kv4_attn_args a, int R, int ctas, int RB,
                                                   int per) {
    constexpr int V = HD / 32, NW = kKvWarps, PF = kv4_part_floats(HD);  // V values per lane
    __shared__ float sums[8][HD], stat[8][2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int gsz = a.H / c.KH, rows = a.T * gsz, S = R * c.KH;
    const kv4_seqs seqs = {a.slots, a.lens, a.len_add, a.longest, c.slots, 0};
    // The attention's blocks have all passed their own wait when this kernel
    // starts, so lens and slots are there before this kernel's wait.
    const int i0 = RUN ? blockIdx.x * per : blockIdx.x, i1 = RUN ? min(i0 + per, a.B * S) : i0 + 1;
    int b = i0 / S, s = i0 % S, nu = seqs.units(b);
    uint32_t before = 0, U = 0;
    for (int i = lane; i < a.B; i += 32) {
        const int n = seqs.units(i);
        U += n;
        if (i < b) before += n;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        U += __shfl_xor_sync(0xffffffffu, U, o);
        before += __shfl_xor_sync(0xffffffffu, before, o);
    }
    const kv4_cut cut(max(1u, U * S), ctas, NW);
    auto merge = [&]() {
        const uint32_t first = before * S + s * nu, last = first + nu;
        const int w0 = nu ? cut.warp_of(first) : 0, w1 = nu ? cut.warp_of(last - 1) : 0, nw = cut.nw;
        griddep_wait();  // (the cut before it)
        griddep_launch_dependents();
        if (w0 == w1) return;  // nothing to add, or one warp had it all
        // Parts: one per warp of the first and last block where these reach out of
        // the segment, one per block in between.
        int b0 = w0 / nw, b1 = w1 / nw + 1;  // joined blocks [b0, b1)
        if (cut.start(b0) < first) b0++;
        if (cut.start(b1) > last) b1--;
        if (nw == 1) b0 = b1 = w1 + 1;  // (a unit per block)
        else if (b1 <= b0) b0 = b1 = max(w0 / nw + 1, w1 / nw);
        const int c0 = w0 / nw, first_end = c0 * nw + (int)cut.warps(c0);  // past the first block's warps
        const int head = nw == 1 ? w1 + 1 - w0 : b0 > c0 ? min(w1 + 1, first_end) - w0 : 0, tail = max(0, w1 + 1 - b1 * nw), n = head + b1 - b0 + tail;
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
    };
    merge();
    for (int i = i0 + 1; RUN && i < i1; i++) {  // (RB = 8: no barrier inside)
        if (++s == S) {
            s = 0;
            before += nu;
            nu = seqs.units(++b);
        }
        merge();
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

// How a call is run: kernel, splits of a unit (tcgen05 form) or blocks to an SM (block
// form), workspace.
enum class kv4_form { whole, block, cut, prompt, none };
struct kv4_plan {
    kv4_form form;
    int S;
    long long ws;
};

// Splits of each unit of a call in the tcgen05 form: as many as fill the SMs, of at
// least kMinSplit cache blocks each (with 4, 64 tokens of 32/4 heads of 128 take as long over
// 4,096 positions, and were 4 us slower over 1,024). Calls of at most 256 positions have
// no workspace.
constexpr int kMinSplit = 2;
int splits_of(long long units, int longest, int sms) {
    if (longest <= 256 || units >= sms) return 1;
    return std::max(1, (int)std::min<long long>(sms / units, (longest + jl::kKv4Rows - 1) / jl::kKv4Rows / kMinSplit));
}

kv4_plan plan(const jl::kv4_dims& c, int B, int T, int H, int longest, int sms) {
    using namespace jl;
    const long long nb = (longest + kKv4Rows - 1) / kKv4Rows, rows = (long long)B * T * H, units = jl_kv4_prompt_units(c, B, T, H);
    // The tcgen05 kernel takes the time of its units of 256 rows, however few rows fill
    // them, and some 14 us beside (start, q, joining); this file's a time by the rows.
    // fp32, 32/4 heads of 128, here / there: 8 tokens (64 rows a unit) over 16,384
    // positions 30 / 36 us, 16 of 4 sequences (128 a unit) 149 / 98; 64 tokens (2,048
    // rows) over 512 12 / 22, over 1,024 17 / 23, over 2,048 30 / 26, over 4,096 48 / 31.
    // Over 802 calls of fp32 and bf16, 1 to 16 sequences of 8 to 512 tokens, 3 to 32 heads
    // of 64 and 128, and 200 to 16,384 positions, the rule is within 0.6 % of the better
    // one (geometric mean).
    if (rows >= 76 * units && rows * nb >= 310ll * sms) {
        const int S = splits_of(units, longest, sms);
        return {kv4_form::prompt, S, jl_kv4_prompt_ws_bytes(c, units, S)};
    }
    const long long segs = (long long)B * row_tiles(c, T, H) * c.KH;
    if (segs > INT_MAX || segs * nb > INT_MAX) return {kv4_form::none, 0, 0};  // the cut counts in 32 bits
    // Three ways to share the segments' blocks out, with what they take in fp32 at head
    // dim 128, in units of 0.35 us (a block alone takes a warp 2 us, with all warps busy 4):
    // a warp per segment, a thread block per segment (one to three to an SM), or all blocks
    // cut evenly and a second kernel that adds up. 32/4 heads, 8 / 32 / 64 / 256 sequences,
    // us: over 128 positions 8.7 / 9.0 / 9.4 / 13.1 by warps, 6.0 / 6.3 / 6.8 / 19.2 by
    // blocks, over 512 11.9 / 12.9 / 17.8 / 36 cut, 7.4 / 7.7 / 11.6 / 31 by blocks, over
    // 2,048 13.1 / 21 / 30 / 88 and 15.7 / 16 / 27 / 96 (lengths spread evenly: 11.8 / 17.3 /
    // 24 / 70 and 15.5 / 15.8 / 25 / 65). The cut's work follows the lengths and is counted at
    // 3/4 of the longest; a block of head dim 64 takes half.
    const double per_sm = (double)segs / sms, work = c.hd == 64 ? 0.5 * nb : nb, u = per_sm * work;
    const double whole = 10 + work * (6 + std::min(per_sm, 12.0) / 2) * std::max(1.0, std::ceil(per_sm / kKvWarps));
    const double cut = 24 + std::min(9.0, 6 * u) + 0.75 * u;
    double block = INFINITY;
    int to_sm = 1;  // blocks that share an SM take longer each, and fewer of them wait
    for (int k = 1; k <= 3; k++) {
        const double t = (double)((segs - 1) / ((long long)k * sms) + 1) * (12 + k * work);
        if (t < block) block = t, to_sm = k;
    }
    if (longest <= 256 && whole < block) return {kv4_form::whole, 1, 0};
    if (longest <= 256 || block < cut) return {kv4_form::block, to_sm, 0};
    // two parts for each warp that has blocks (blocks x warps of a cut: below its units + blocks)
    const long long warps = std::min<long long>((long long)sms * kKvWarps, 2 * segs * nb);
    return {kv4_form::cut, 1, warps * 2 * kv4_part_floats(c.hd) * (long long)sizeof(float)};
}

template <int HD, typename T>
int attn_attrs_t() {
    using namespace jl;
    JL_CUDA(cudaFuncSetAttribute(k_kv4_attn<HD, T, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kv4_smem<HD>::total));
    JL_CUDA(cudaFuncSetAttribute(k_kv4_attn<HD, T, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kv4_smem<HD>::total));
    return JL_OK;
}

template <int HD>
int attn_attrs() {
    int rc = attn_attrs_t<HD, float>();
    if (!rc) rc = attn_attrs_t<HD, __half>();
    if (!rc) rc = attn_attrs_t<HD, __nv_bfloat16>();
    return rc;
}

template <int HD, typename T>
int launch_t(const jl::kv4_dims& c, int l, const jl_kv4_attn_args& a, const kv4_plan& p, int sms, cudaStream_t s) {
    using namespace jl;
    const int R = row_tiles(c, a.T, a.H);
    const unsigned segs = (unsigned)((long long)a.B * R * c.KH);
    if (p.form == kv4_form::block) {
        const int warps = kKvWarps / p.S;
        return launch(k_kv4_attn<HD, T, true>, dim3(segs), dim3(warps * 32), (size_t)kv4_smem<HD>::bytes(warps), s, c, l, a, R, 0);
    }
    const int rc = launch(k_kv4_attn<HD, T, false>, dim3(sms), dim3(kKvWarps * 32), (size_t)kv4_smem<HD>::total, s, c, l, a, R,
                          (int)(p.form == kv4_form::whole));
    if (rc || p.form == kv4_form::whole) return rc;
    const int RB = segs >= (unsigned)sms ? 8 : segs * 4 >= (unsigned)sms ? 2 : 1, per = (int)((segs - 1) / (4 * sms) + 1);
    if (per == 1) return launch(k_kv4_merge<HD, T, false>, dim3(segs, kKvTile / RB), dim3(256), 0, s, c, a, R, sms, RB, 1);
    return launch(k_kv4_merge<HD, T, true>, dim3((segs - 1) / per + 1), dim3(256), 0, s, c, a, R, sms, 8, per);
}

template <int HD>
int launch_hd(const jl::kv4_dims& c, int l, const jl_kv4_attn_args& a, const kv4_plan& p, int sms, cudaStream_t s) {
    if (a.dtype == JL_F32) return launch_t<HD, float>(c, l, a, p, sms, s);
    if (a.dtype == JL_F16) return launch_t<HD, __half>(c, l, a, p, sms, s);
    return launch_t<HD, __nv_bfloat16>(c, l, a, p, sms, s);
}

}  // namespace

// (Without a device: a B200's 148 SMs.)
long long jl_kv4_attn_ws_bytes(const jl::kv4_dims& c, int B, int T, int H, int longest) {
    const int sms = sm_count();
    return plan(c, B, T, H, longest, sms > 0 ? sms : 148).ws;
}

long long jl_kv4_attn_ws_most(const jl::kv4_dims& c) {
    const long long sms = sm_count();
    return std::max(sms * jl::kKvWarps * 2 * jl::kv4_part_floats(c.hd) * (long long)sizeof(float),
                    jl_kv4_prompt_ws_bytes(c, 1, (int)sms));
}

int jl_launch_kv4_attn(const jl::kv4_dims& c, int l, const jl_kv4_attn_args& a, cudaStream_t s) {
    const int sms = sm_count();
    if (sms < 1) return JL_ERR_CUDA;
    const kv4_plan p = plan(c, a.B, a.T, a.H, a.longest, sms);
    if (p.form == kv4_form::none) return JL_ERR_INVALID;
    if (p.form == kv4_form::prompt) return jl_launch_kv4_prompt(c, l, a, p.S, s);
    const int rc = jl_device_once(kOnceKv4, [] {
        const int r = attn_attrs<64>();
        return r ? r : attn_attrs<128>();
    });
    if (rc) return rc;
    return c.hd == 64 ? launch_hd<64>(c, l, a, p, sms, s) : launch_hd<128>(c, l, a, p, sms, s);
}
