"""The digits of the 4-bit cache's attention, against its definition in 64 bits
over the values that the cache holds (read back, which is exact).

With e = 2^-24. Scores: as in tests/test_kv4_gpu.py, |ds| <= scale * (16 + 4 (hd + 16)) e
(|q| . |k|) + 8 e |s|. What a weight is off by is measured against the sum that it is
part of: M = sum_t p_t amax_t, p the exact weights and amax_t the largest value of the
position's group of 64, because a product of a weight and a scale is rounded before
the code multiplies it. Weights times scales are held in 22 bits, sums in fp32, so an
output is off by at most (4 |ds| + (2 n + 64) e) M plus half a step of its type. The
roundings being independent, the root mean square of error / M over all outputs is
held to RMS = 64 e max(1, max|s|).

Results in 16 bits are the nearest to a value that is off by that much. One of them
differs from the nearest to the exact value only where that value lies within the
error of the middle of two steps, so of many results at most a share 2 RMS M / step each
does, plus five standard deviations of their count.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
E = 2.0 ** -24


def _i32(x):
    return torch.as_tensor(np.asarray(x, np.int32)).cuda()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _cache(rows, maxT=None):
    """A cache of the sequences' rows [(k, v)] (each [n, kv, hd] fp32), slot b for sequence b."""
    from joule_b200 import kv4
    kv, hd = rows[0][0].shape[1:]
    cache = kv4.kv4_cache(len(rows), 1, kv, hd, maxT or max(max(k.shape[0] for k, _ in rows), 1))
    cache.random_(0, 256)
    for b, (k, v) in enumerate(rows):
        n = k.shape[0]
        if n:
            kv4.kv4_append(cache, 0, k, v, _i32([b] * n), _i32(range(n)))
    return cache


def _held(cache, slot, n):
    from joule_b200 import kv4
    k, v = kv4.kv4_read(cache, 0, _i32([slot] * n), _i32(range(n)))
    return k.double(), v.double()


def _exact(q, k, v, scale, rows=None):
    """q [T, H, hd] over k, v [n, kv, hd] (64 bits): out, M, the bound of |ds| [., H, .]
    of the given rows of T, and the largest |score|."""
    T, H, hd = q.shape
    n, kv = k.shape[:2]
    rows = torch.arange(T, device="cuda") if rows is None else rows
    out, M, ds = (torch.zeros(len(rows), H, hd, dtype=torch.float64, device="cuda") for _ in range(3))
    top = 0.0
    amax = v.unflatten(-1, (-1, 64)).abs().amax(-1, keepdim=True).expand(n, kv, hd // 64, 64).flatten(-2)
    for h in range(H):
        g = h // (H // kv)
        for a in range(0, len(rows), 64):
            r = rows[a:a + 64]
            x = q[r, h].double()
            s = scale * (x @ k[:, g].T)
            seen = torch.arange(n, device="cuda")[None] < (n - T + 1 + r)[:, None]
            some = seen.any(1)
            s = torch.where(seen, s, -math.inf)
            p = torch.where(some[:, None], torch.softmax(torch.where(some[:, None], s, 0.0), -1), 0.0)
            out[a:a + 64, h] = p @ v[:, g]
            M[a:a + 64, h] = p @ amax[:, g]
            big = torch.where(seen, s.abs(), 0.0).amax()
            ab = torch.where(seen, x.abs() @ k[:, g].abs().T, 0.0).amax(1)
            ds[a:a + 64, h] = (abs(scale) * (16 + 4 * (hd + 16)) * E * ab + 8 * E * big)[:, None]
            top = max(top, float(big))
    return out, M, ds, top


def _close(got, want, M, ds, top, n):
    """fp32 results within both bounds."""
    err, some = (got.double() - want).abs(), M > 0
    assert torch.isfinite(got).all() and (err[~some] == 0).all()
    bad = err > (4 * ds + (2 * n + 64) * E) * M + E * want.abs()
    assert not bad.any(), (bad.sum().item(), (err / M.clamp_min(1e-300)).amax().item())
    rms = (err / torch.where(some, M, 1.0)).pow(2).mean().sqrt().item()
    assert rms <= 64 * E * max(1.0, top), rms


def _step_of(x, t):
    """The distance of the type's numbers around x."""
    e = torch.frexp(x.abs().clamp_min(1e-30))[1].double() - 1
    bits, low = {"f16": (10, -14), "bf16": (7, -126)}[t]
    return torch.exp2(e.clamp_min(low) - bits)


def _nearest(got, want, M, ds, top, n, t):
    """16-bit results are the nearest ones but for the share that the bound allows."""
    step = _step_of(want, t)
    err = (got.double() - want).abs()
    assert not (err > step / 2 * (1 + 2.0 ** -20) + (4 * ds + (2 * n + 64) * E) * M).any()
    share = (2 * 64 * E * max(1.0, top) * M / step).clamp_max(1.0)
    off = (got != want.to(DT[t])).double()
    allowed = share.sum().item()
    assert off.sum().item() <= allowed + 5 * math.sqrt(allowed) + 3, (off.sum().item(), allowed, off.numel())


def _sampled(B, T, rows):
    b = torch.tensor([0, B - 1] if B > 1 else [0])
    r = torch.unique(torch.linspace(0, T - 1, min(rows, T)).long()).cuda()
    return b, r


# ---------------------------------------------------------------------------
# 16-bit calls

STEPS16 = [  # B, T, H, kv, hd, lens: a warp per sequence and head, a block, a cut, drafts
    (300, 1, 8, 8, 64, [1 + (31 * b) % 40 for b in range(300)]), (8, 1, 32, 4, 128, [9 + 5 * b for b in range(8)]),
    (40, 1, 16, 4, 128, [(211 * b) % 1501 for b in range(40)]), (5, 5, 10, 2, 64, [40, 5, 7, 30, 21]),
]


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("B,T,H,kv,hd,lens", STEPS16)
def test_16_bit_results_are_the_nearest(B, T, H, kv, hd, lens, t):
    """q, weights and sums of a 16-bit call have as many digits as those of a fp32 one:
    over values of one sign (outputs of the size of M) the results are the exact
    ones rounded once."""
    from joule_b200 import kv4
    g = _gen(B + T)
    rows = [(torch.randn(n, kv, hd, device="cuda", generator=g), torch.rand(n, kv, hd, device="cuda", generator=g) + 0.5)
            for n in lens]
    cache = _cache(rows)
    q = (torch.randn(B, T, H, hd, device="cuda", generator=g) * 0.5).to(DT[t])
    got = kv4.kv4_attention(cache, 0, q, _i32(range(B)), _i32(lens))
    parts = [_exact(q[b], *_held(cache, b, n), hd ** -0.5) for b, n in enumerate(lens) if n]
    at = [b for b, n in enumerate(lens) if n]
    want, M, ds = (torch.cat([p[i] for p in parts]) for i in range(3))
    _nearest(torch.cat([got[b] for b in at]), want, M, ds, max(p[3] for p in parts), max(lens), t)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("T,H,kv,lens,size", [(700, 16, 4, [720, 705], 4.0), (700, 16, 4, [720, 705], 1.5), (40, 32, 2, [3000, 2999], 4.0)])
def test_q_of_a_16_bit_prompt_is_not_rounded(T, H, kv, lens, size, t):
    """A 16-bit q is exact in the product of the scores whatever the scale: its error is
    that of sums of hd products, 16 at a time, each cut off at 2 e of the largest score at
    most: 16 e in all. The norm of the results' errors is that of the exact results rounded
    once and of weights off by so much (and by 64 e as they are in all calls)."""
    from joule_b200 import kv4
    g, hd, B, scale = _gen(T), 128, len(lens), 0.0931
    rows = [tuple(torch.randn(n, kv, hd, device="cuda", generator=g) for _ in range(2)) for n in lens]
    cache = _cache(rows)
    q = (torch.randn(B, T, H, hd, device="cuda", generator=g) * size).to(DT[t])
    got = kv4.kv4_attention(cache, 0, q, _i32(range(B)), _i32(lens), scale=scale)
    parts = [_exact(q[b], *_held(cache, b, n), scale) for b, n in enumerate(lens)]
    want, M = (torch.cat([p[i] for p in parts]) for i in range(2))
    top = max(p[3] for p in parts)
    once = (want.to(DT[t]).double() - want).norm()
    err = (got.flatten(0, 1).double() - want).norm()
    assert err <= once + (64 + 16 * top) * E * M.norm(), (err / want.norm(), once / want.norm(), top)


@pytest.mark.parametrize("T", [1, 9, 720])
@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-42, 3e-39, -1e-30, 1e30])
def test_any_finite_scale(T, t, scale):
    """Scales of either sign, of zero, and of the ends of fp32's range, with q so large
    and so small that the scores are ordinary or vanish."""
    from joule_b200 import kv4
    g, n, kv, hd, H = _gen(T), 900, 2, 64, 32
    k, v = (torch.randn(n, kv, hd, device="cuda", generator=g) for _ in range(2))
    cache = _cache([(k, v)])
    size = min(max(0.3 / abs(scale), 1e-30), 1e30) if scale else 1.0
    size = min(max(size, 2e-4), 2e3) if t == "f16" else size
    q = (torch.randn(1, T, H, hd, device="cuda", generator=g) * size).to(DT[t])
    if t == "f16" and scale == 1e30:
        q.zero_()
    got = kv4.kv4_attention(cache, 0, q, _i32([0]), _i32([n]), scale=scale)
    want, M, ds, top = _exact(q[0], *_held(cache, 0, n), float(np.float32(scale)))
    half = _step_of(want, t) / 2 * (1 + 2.0 ** -20) if t == "f16" else E * want.abs()
    assert not ((got[0].double() - want).abs() > half + (4 * ds + (2 * n + 64) * E) * M).any()


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("B,T,H,kv,hd,lens,maxT", [(2, 700, 16, 4, 128, [700, 700], 720), (3, 900, 6, 2, 64, [900, 905, 1000], 1000),
                                                   (1, 64, 32, 4, 128, [70], 4096), (1, 70, 32, 2, 64, [71], 3000)])
def test_weights_of_a_16_bit_prompt(B, T, H, kv, hd, lens, maxT, t):
    """The first 60 rows of a prompt, over a few positions each, whole and in splits (most
    of them empty)."""
    from joule_b200 import kv4
    g = _gen(B + T)
    rows = [(torch.randn(n, kv, hd, device="cuda", generator=g), torch.rand(n, kv, hd, device="cuda", generator=g) + 0.5)
            for n in lens]
    cache = _cache(rows, maxT)
    q = (torch.randn(B, T, H, hd, device="cuda", generator=g) * 0.1).to(DT[t])
    got = kv4.kv4_attention(cache, 0, q, _i32(range(B)), _i32(lens))[:, :60]
    first = torch.arange(60, device="cuda")
    parts = [_exact(q[b], *_held(cache, b, n), hd ** -0.5, first) for b, n in enumerate(lens)]
    want, M, ds = (torch.cat([p[i] for p in parts]) for i in range(3))
    _nearest(got.flatten(0, 1), want, M, ds, 1.0, 160, t)
    assert max(p[3] for p in parts) < 1.0


@pytest.mark.parametrize("T,H,kv,hd,n", [(1184, 32, 4, 128, 23000), (1, 32, 4, 128, 60000), (300, 8, 1, 64, 23000), (2500, 16, 4, 64, 23000),
                                         (2100, 24, 3, 128, 2900)])
def test_sums_of_16_bit_calls_do_not_shrink(T, H, kv, hd, n):
    """Values of one sign over many positions. The part of the results along the exact ones
    is off by no more than products cut off rather than rounded over at most 32 blocks make
    (1.6e-7 each, half of that on the way), fp32 sums (64 e), and five standard deviations of
    the mean of the results' own roundings."""
    from joule_b200 import kv4
    g = _gen(T)
    k, v = torch.randn(n, kv, hd, device="cuda", generator=g), torch.rand(n, kv, hd, device="cuda", generator=g) + 0.5
    cache = _cache([(k, v)])
    q = torch.randn(1, T, H, hd, device="cuda", generator=g).half()
    got = kv4.kv4_attention(cache, 0, q, _i32([0]), _i32([n]))[0]
    r = torch.unique(torch.linspace(0, T - 1, min(24, T)).long()).cuda()
    want, M, ds, top = _exact(q[0], *_held(cache, 0, n), hd ** -0.5, r)
    err = got[r].double() - want
    assert (err.abs() <= _step_of(want, "f16") / 2 * (1 + 2.0 ** -20) + (4 * ds + (2 * n + 64) * E) * M).all()
    bias = ((err * want).sum() / (want * want).sum()).item()
    assert abs(bias) <= 32 * 0.8e-7 + 64 * E + 5 * 2.0 ** -11 / math.sqrt(3 * err.numel()), bias


@pytest.mark.parametrize("T", [1, 30, 720])
@pytest.mark.parametrize("size", [1e4, 1e6])
def test_scores_past_the_fraction_of_a_float(T, size):
    """One key ahead of all others by thousands at scores of 1e6 to 1e10: its values."""
    from joule_b200 import kv4
    g = _gen(44)
    n, kv, hd, H = 800, 2, 128, 16
    k, v = (torch.randn(n, kv, hd, device="cuda", generator=g) for _ in range(2))
    v *= 0.01
    k[:, :, 0] = 7.0
    k[3, :, 0] = 14.0
    k *= size / 100
    q = torch.zeros(1, T, H, hd, device="cuda")
    q[..., 0] = size
    got = kv4.kv4_attention(_cache([(k, v)]), 0, q, _i32([0]), _i32([n]), scale=1.0)
    c = _cache([(k, v)])
    kk, vv = _held(c, 0, n)
    assert (kk[3, :, 0] > kk[torch.arange(n) != 3][:, :, 0].amax()).all()
    want = vv[3].repeat_interleave(H // kv, 0)
    assert (got[0].double() - want).abs().amax() <= 8 * E * want.abs().amax()


# ---------------------------------------------------------------------------
# V rows of very different size

FORMS = [  # B, T, H, kv, hd, lens
    (2, 1, 8, 2, 128, [333, 90]), (2, 1, 8, 2, 64, [333, 90]), (200, 1, 8, 8, 64, [20 + (31 * b) % 231 for b in range(200)]),
    (40, 1, 16, 4, 128, [20 + (211 * b) % 1481 for b in range(40)]), (3, 24, 8, 2, 128, [500, 90, 30]),
    (2, 90, 32, 2, 128, [1500, 1000]), (1, 90, 32, 2, 64, [1500]), (2, 720, 8, 2, 128, [1333, 730]),
    (3, 1000, 16, 4, 64, [1100, 1000, 1024]),
]


def _spread_case(B, T, H, kv, hd, lens, seed, make):
    """Attention of one row's size of scores over rows that make(v, n) scales; key 5 of every
    sequence (and what make returns as hidden) has a score of some -130 in base 2."""
    from joule_b200 import kv4
    g = _gen(seed)
    rows = []
    for n in lens:
        k = torch.randn(n, kv, hd, device="cuda", generator=g) * 0.5
        v = torch.randn(n, kv, hd, device="cuda", generator=g)
        k[..., 0] = 0.0
        for j, x in make(v, n).items():
            k[j, :, 0] = x
        rows.append((k, v))
    cache = _cache(rows)
    q = torch.randn(B, T, H, hd, device="cuda", generator=g)
    q[..., 0] = 1.0
    got = kv4.kv4_attention(cache, 0, q, _i32(range(B)), _i32(lens), scale=0.1)
    for b, n in enumerate(lens):
        # (the keys with an outlier are exact in element 0 alone; scores are those of the held keys)
        want, M, ds, top = _exact(q[b], *_held(cache, b, n), 0.1)
        yield got[b], want, M, ds, n


def _check_spread(B, T, H, kv, hd, lens, seed, make):
    for got, want, M, ds, n in _spread_case(B, T, H, kv, hd, lens, seed, make):
        # the hidden keys' scores carry no weight: those of the others are below 4
        err, some = (got.double() - want).abs(), M > 0
        assert torch.isfinite(got).all()
        assert not (err > (4 * ds + (2 * n + 64) * E) * M + E * want.abs()).any(), (err / M).amax()
        rms = (err / torch.where(some, M, 1.0)).pow(2).mean().sqrt().item()
        assert rms <= 64 * E * 4.0, rms


@pytest.mark.parametrize("factor", [1e3, 1e5, 1e7, 1e9])
@pytest.mark.parametrize("B,T,H,kv,hd,lens", FORMS)
def test_a_large_row_without_weight(B, T, H, kv, hd, lens, factor):
    """A V row of 1e5 whose weight is nothing beside rows smaller by the factor."""
    def make(v, n):
        v *= 1e5 / factor
        v[5] = v[5].sign() * 1e5
        return {5: -1000.0}
    _check_spread(B, T, H, kv, hd, lens, 40, make)


@pytest.mark.parametrize("B,T,H,kv,hd,lens", FORMS)
def test_groups_of_different_size(B, T, H, kv, hd, lens):
    """The two groups of a head, and the kv heads, differ by 1e8; rows by powers of ten."""
    def make(v, n):
        v *= 10 ** torch.linspace(-1, 1, n, device="cuda")[torch.randperm(n, device="cuda", generator=_gen(n))][:, None, None]
        v[..., 64:] *= 1e-4
        v[..., :64] *= 1e4
        v[:, ::2] *= 0.01
        return {5: -1000.0}
    _check_spread(B, T, H, kv, hd, lens, 41, make)


@pytest.mark.parametrize("B,T,H,kv,hd,lens", FORMS)
def test_a_key_of_all_weight_with_values_of_zero(B, T, H, kv, hd, lens):
    """The first position takes the weight by a factor of e^20 and has no value; what is
    left is that small sum of the others' values."""
    def make(v, n):
        v[0] = 0.0
        return {0: 200.0}
    for got, want, M, ds, n in _spread_case(B, T, H, kv, hd, lens, 42, make):
        err = (got.double() - want).abs()
        assert not (err > (4 * ds + (2 * n + 64) * E) * M + E * want.abs()).any()
        rms = (err / torch.where(M > 0, M, 1.0)).pow(2).mean().sqrt().item()
        assert rms <= 64 * E * 24.0, rms


@pytest.mark.parametrize("T,H,kv,hd,n", [(5, 8, 2, 128, 300), (24, 8, 1, 64, 70), (90, 32, 2, 128, 1500), (720, 32, 4, 128, 1333)])
def test_a_later_row_does_not_change_an_earlier_result(T, H, kv, hd, n):
    """Query i's digits do not depend on the values of positions that it does not see."""
    from joule_b200 import kv4
    g = _gen(43)
    k, v = (torch.randn(n, kv, hd, device="cuda", generator=g) for _ in range(2))
    q = torch.randn(1, T, H, hd, device="cuda", generator=g)
    got = []
    for x in (1.0, 1e5):
        v[n - 3:] *= x
        got.append(kv4.kv4_attention(_cache([(k, v)]), 0, q, _i32([0]), _i32([n])))
    assert torch.equal(got[0][:, :T - 3], got[1][:, :T - 3])
    assert not torch.equal(got[0][:, T - 3:], got[1][:, T - 3:])


@pytest.mark.parametrize("B,T,H,kv,hd,n", [(1, 1, 32, 4, 128, 131072), (1, 64, 32, 4, 128, 50000), (1, 1184, 32, 4, 128, 23000)])
def test_sizes_that_change_from_block_to_block(B, T, H, kv, hd, n):
    """V's size rises and falls by 2^10 from one block to the next, so that references move
    by V's scales alone, across folds and joins."""
    from joule_b200 import kv4
    g = _gen(n)
    k, v = (torch.randn(n, kv, hd, device="cuda", generator=g) for _ in range(2))
    v *= torch.exp2(10.0 * ((torch.arange(n, device="cuda") // 64 * 7919) % 11 % 3 - 1).float())[:, None, None]
    cache = _cache([(k, v)])
    q = torch.randn(B, T, H, hd, device="cuda", generator=g)
    got = kv4.kv4_attention(cache, 0, q, _i32([0] * B), _i32([n] * B))
    _, r = _sampled(B, T, 16)
    want, M, ds, top = _exact(q[0], *_held(cache, 0, n), hd ** -0.5, r)
    _close(got[0][r], want, M, ds, top, n)


# ---------------------------------------------------------------------------
# long histories

LONG = [  # B, T, H, kv, hd, n: a cut (few and many blocks to a warp), a prompt in splits, two whole ones
    (1, 1, 32, 4, 128, 131072), (64, 1, 32, 4, 128, 131072), (8, 1, 8, 8, 64, 50000), (1, 64, 32, 4, 128, 131072),
    (1, 1184, 32, 4, 128, 23000), (1, 2368, 16, 4, 64, 131072),
]


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("B,T,H,kv,hd,n", LONG)
def test_nothing_grows_with_the_length(B, T, H, kv, hd, n, t):
    """One key ahead and all others equal: every weight of the sum rounds the same way.
    The output's part along the exact one is off by no more than a fixed bound: sums of 64
    weights (32 roundings in a row, 16 e), the block's into a total that keeps what it
    rounds off, products cut off rather than rounded over at most 8 blocks (16-bit calls:
    32) of 64 positions, measured at 1.6e-7 a block: 4e-6 in fp32; 16 bits add 6e-6."""
    from joule_b200 import kv4
    g = _gen(n + T)
    k = torch.randn(1, kv, hd, device="cuda", generator=g).expand(n, kv, hd).contiguous()
    k[7] *= 1.5
    v = torch.rand(n, kv, hd, device="cuda", generator=g) + 0.5
    cache = _cache([(k, v)])
    kk, vv = _held(cache, 0, n)
    q = (kk[0].float().repeat_interleave(H // kv, 0) * 0.05 * (1 + torch.rand(B, T, H, 1, device="cuda", generator=g))).to(DT[t])
    got = kv4.kv4_attention(cache, 0, q, _i32([0] * B), _i32([n] * B), scale=1.0)
    bs, r = _sampled(B, T, 24)
    num = den = 0.0
    for b in bs.tolist():
        want = _exact(q[b], kk, vv, 1.0, r)[0]
        num += ((got[b][r].double() - want) * want).sum().item()
        den += (want * want).sum().item()
        if t == "f32":
            assert ((got[b][r].double() - want).abs() <= 2e-5 * want.abs()).all()
    # 16-bit results of equal weights repeat from row to row: kv * hd independent roundings
    assert abs(num / den) <= 4e-6 + (6e-6 + 5 * 2.0 ** -12 / math.sqrt(3 * kv * hd) if t == "f16" else 0.0), num / den


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,T,H,kv,hd,lens", [(4, 640, 15, 3, 128, [2500, 2300, 640, 0]), (6, 500, 14, 2, 64, [2400, 3000, 500, 499, 1, 2111]),
                                              (1, 3, 1030, 1, 128, [4500])])
def test_sums_in_places_of_odd_groups(B, T, H, kv, hd, lens, t):
    """Units whose sums move to their rows of the output and back while they are computed:
    groups of 5 and 7 heads, rows that end inside a warp, sequences shorter than the chunk."""
    from joule_b200 import kv4
    g = _gen(B + T)
    rows = [tuple(torch.randn(n, kv, hd, device="cuda", generator=g) for _ in range(2)) for n in lens]
    cache = _cache(rows)
    q = torch.randn(B, T, H, hd, device="cuda", generator=g).to(DT[t])
    got = kv4.kv4_attention(cache, 0, q, _i32(range(B)), _i32(lens))
    for b, n in enumerate(lens):
        assert (got[b, :max(0, T - n)] == 0).all()
        if n:
            r = torch.unique(torch.cat([torch.arange(3), torch.linspace(0, T - 1, min(T, 40)).long()]).clamp_max(T - 1)).cuda()
            want, M, ds, _ = _exact(q[b], *_held(cache, b, n), hd ** -0.5, r)
            half = E * want.abs() if t == "f32" else _step_of(want, t) / 2 * (1 + 2.0 ** -20)
            assert not ((got[b][r].double() - want).abs() > half + (4 * ds + (2 * n + 64) * E) * M).any()


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("B,T,H,kv,n", [(1, 1, 32, 4, 9000), (1, 90, 32, 2, 9000), (3, 400, 32, 4, 3500), (2, 720, 8, 2, 1333)])
def test_groups_that_change_places(B, T, H, kv, n, t):
    """The two groups of a head differ by 1e6 one way in the first part of a history and the
    other way in the second: factors that come and go across folds, splits and joins."""
    from joule_b200 import kv4
    g, hd = _gen(n + T), 128
    k, v = (torch.randn(n, kv, hd, device="cuda", generator=g) for _ in range(2))
    turn = (torch.arange(n, device="cuda") * 5 // n % 2 == 0)[:, None, None]
    v *= torch.where(turn == (torch.arange(hd, device="cuda") < 64), 1e3, 1e-3)
    k[:, :, :4] += 2.0 * (torch.arange(n, device="cuda") * 5 // n)[:, None, None] / 4
    cache = _cache([(k, v)])
    q = torch.randn(B, T, H, hd, device="cuda", generator=g).to(DT[t])
    got = kv4.kv4_attention(cache, 0, q, _i32([0] * B), _i32([n] * B))
    r = torch.unique(torch.linspace(0, T - 1, min(T, 30)).long()).cuda()
    for b in range(B):
        want, M, ds, top = _exact(q[b], *_held(cache, 0, n), hd ** -0.5, r)
        if t == "f32":
            _close(got[b][r], want, M, ds, top, n)
        else:
            half = _step_of(want, t) / 2 * (1 + 2.0 ** -20)
            assert not ((got[b][r].double() - want).abs() > half + (4 * ds + (2 * n + 64) * E) * M).any()
