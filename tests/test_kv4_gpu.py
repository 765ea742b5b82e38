"""The 4-bit KV cache on the GPU against its 64-bit restatement (oracle/kv4.py).

Tolerances. Appending and reading are exact: the cached values are compared
with `==`, 16-bit results with the oracle's rounding of the exact value.

Attention, with e = 2^-24. A score s is scale * (a sum of hd products). The
kernel holds q in at least 22 bits, sums in fp32 in any order with the codes'
offset of 8 possibly summed along (at most 4 times the magnitude of the
products themselves, |code| <= 15 against |code - 8| <= 8), and forms
exponents in base 2: |ds| <= scale * (4 * 4 + 4 * (hd + 16)) * e * (|q| . |k|) + 8 e |s|.
A weight exp(s - max) is then off by at most the factor exp(2 |ds|) and four
roundings. Weights times scales are held in 22 bits, and the n of them are
summed in fp32. So each output is off by at most
    (2 * (2 |ds|) + (2 * n + 64) * e) * max|v|, plus half a step of its type.
That is a bound for the worst case; the roundings being independent, the norm of
all outputs' errors is held to 64 e * max(1, max|s|) of their norm, plus half a
step of the type.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kv4 as okv4

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
E = 2.0 ** -24


def _i32(x):
    return torch.as_tensor(np.asarray(x, np.int32)).cuda()


def _to(x: np.ndarray, t: str) -> torch.Tensor:
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).cuda().to(DT[t])


def _rows(rng, n, kv, hd):
    """Rows whose groups differ in size by powers of ten, some of them zero."""
    x = rng.standard_normal((n, kv, hd // 64, 64)) * np.exp(rng.uniform(-6, 4, (n, kv, hd // 64, 1)))
    x[rng.random((n, kv, hd // 64)) < 0.05] = 0.0
    return x.reshape(n, kv, hd).astype(np.float32)


def _filled(rng, slots, L, kv, hd, maxT, l, lens, slot_of, ksize=1.0):
    """A cache of random bytes with the first lens[b] rows of slot_of[b] appended; their held values."""
    from joule_b200 import kv4
    cache = kv4.kv4_cache(slots, L, kv, hd, maxT)
    cache.copy_(torch.from_numpy(rng.integers(0, 256, tuple(cache.shape), dtype=np.uint8)))
    ks, vs = [], []
    for b, n in enumerate(lens):
        k = (rng.standard_normal((n, kv, hd)) * ksize).astype(np.float32)
        v = rng.standard_normal((n, kv, hd)).astype(np.float32)
        if n:
            kv4.kv4_append(cache, l, _to(k, "f32"), _to(v, "f32"), _i32([slot_of[b]] * n), _i32(np.arange(n)))
        ks.append(okv4.held(k) if n else k.astype(np.float64))
        vs.append(okv4.held(v) if n else v.astype(np.float64))
    return cache, ks, vs


def _check(got, q, ks, vs, scale, t):
    """got [B, T, H, hd] (torch) against the oracle; q as float64 of the values passed."""
    got = got.double().cpu().numpy()
    half = {"f32": E, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[t]
    num = den = 0.0
    top = 0.0
    for b in range(q.shape[0]):
        n, hd = ks[b].shape[0], q.shape[-1]
        want, absdot, s = okv4.attention(q[b], ks[b], vs[b], scale)
        ds = abs(scale) * (16 + 4 * (hd + 16)) * E * absdot + 8 * E * s
        vmax = np.abs(vs[b]).max() if n else 0.0
        tiny = 2.0 ** -25 if t == "f16" else 0.0  # half of fp16's subnormal step
        tol = ((4 * ds + (2 * n + 64) * E) * vmax)[..., None] + half * np.abs(want) * (1 + 4 * ds[..., None]) + tiny
        bad = np.abs(got[b] - want) > tol
        assert not bad.any(), (b, np.argwhere(bad)[:3].tolist(), np.abs(got[b] - want).max(), tol.min())
        num += float(((got[b] - want) ** 2).sum())
        den += float((want ** 2).sum())
        top = max(top, s)
    assert num ** 0.5 <= (64 * E * max(1.0, top) + half) * den ** 0.5


# ---------------------------------------------------------------------------
# append and read

@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd,kv,n", [(128, 4, 1), (64, 3, 7), (128, 1, 130), (64, 8, 65), (128, 5, 1000)])
def test_append_then_read_is_exact(hd, kv, n, t):
    from joule_b200 import kv4
    rng = np.random.default_rng(n + hd)
    slots, L, maxT, l = 5, 3, 300, 1
    cache = kv4.kv4_cache(slots, L, kv, hd, maxT)
    before = torch.from_numpy(rng.integers(0, 256, tuple(cache.shape), dtype=np.uint8)).cuda()
    cache.copy_(before)
    at = rng.permutation(slots * maxT)[:n]
    s, p = at // maxT, at % maxT
    k, v = _to(_rows(rng, n, kv, hd), t), _to(_rows(rng, n, kv, hd), t)
    kv4.kv4_append(cache, l, k, v, _i32(s), _i32(p))
    wk, wv = (okv4.held(x.float().cpu().numpy()) for x in (k, v))
    for rt in DT:
        gk, gv = kv4.kv4_read(cache, l, _i32(s), _i32(p), dtype=DT[rt])
        for got, want in ((gk, wk), (gv, wv)):
            assert got.dtype == DT[rt] and got.shape == (n, kv, hd)
            assert torch.equal(got.cpu(), torch.from_numpy(want).to(DT[rt]))
    # nothing but those records changed
    mask = torch.zeros(cache.shape, dtype=torch.bool)
    for a, b in zip(s, p):
        r = b % 64
        for is_v in (False, True):
            first = [okv4.byte_of(hd, is_v, r, d) for d in range(0, hd, 2)]
            sc = [okv4.scale_byte(hd, is_v, r, g) + i for g in range(hd // 64) for i in (0, 1)]
            mask[a, l, :, b // 64, torch.tensor(first + sc)] = True
    assert torch.equal(cache.cpu()[~mask], before.cpu()[~mask])


@pytest.mark.parametrize("hd", [64, 128])
def test_block_bytes_match_the_layout(hd):
    from joule_b200 import kv4
    rng = np.random.default_rng(5)
    cache = kv4.kv4_cache(1, 1, 2, hd, 64)
    cache.zero_()
    k, v = _rows(rng, 64, 2, hd), _rows(rng, 64, 2, hd)
    order = rng.permutation(64)
    kv4.kv4_append(cache, 0, _to(k[order], "f32"), _to(v[order], "f32"), _i32(np.zeros(64)), _i32(order))
    for h in range(2):
        assert np.array_equal(cache[0, 0, h, 0].cpu().numpy(), okv4.pack_block(k[:, h], v[:, h]))


def test_values_a_record_cannot_hold():
    """Infinities and values past fp16's scales saturate, NaN becomes 0, tiny
    groups become 0; the cached values are always finite."""
    from joule_b200 import kv4
    rng = np.random.default_rng(6)
    x = np.zeros((6, 1, 64), np.float32)
    x[0] = rng.standard_normal(64) * 1e30
    x[1] = rng.standard_normal(64)
    x[1, 0, 7] = np.inf
    x[1, 0, 8] = -np.inf
    x[2] = rng.standard_normal(64)
    x[2, 0, ::3] = np.nan
    x[3] = np.nan
    x[4] = rng.standard_normal(64) * 1e-9
    x[5] = rng.standard_normal(64) * 3e-7
    cache = kv4.kv4_cache(1, 1, 1, 64, 6)
    kv4.kv4_append(cache, 0, _to(x, "f32"), _to(-x, "f32"), _i32([0] * 6), _i32(range(6)))
    gk, gv = kv4.kv4_read(cache, 0, _i32([0] * 6), _i32(range(6)))
    assert torch.isfinite(gk).all() and torch.isfinite(gv).all()
    assert np.array_equal(gk.double().cpu().numpy(), okv4.held(x))
    assert np.array_equal(gv.double().cpu().numpy(), okv4.held(-x))


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("low,high", [(4, 14), (-9, -4), (-7.5, -6)])
def test_values_around_the_largest_and_smallest_scales(low, high, t):
    """Groups whose largest value passes 7 * 65504 by a little, by 16 steps, by far,
    and groups whose scale is a few of fp16's smallest steps, rounded by up to half
    one: every value is the nearest of -8 .. 7 steps, none wraps."""
    from joule_b200 import kv4
    rng = np.random.default_rng(29)
    n = 300
    x = rng.standard_normal((n, 2, 64)) * 10 ** rng.uniform(low, high, (n, 2, 1))
    x = _to(x, t).float().cpu().numpy()
    cache = kv4.kv4_cache(1, 1, 2, 64, n)
    at = (_i32([0] * n), _i32(range(n)))
    kv4.kv4_append(cache, 0, _to(x, t), _to(-x, t), *at)
    gk, gv = kv4.kv4_read(cache, 0, *at)
    assert np.array_equal(gk.double().cpu().numpy(), okv4.held(x))
    assert np.array_equal(gv.double().cpu().numpy(), okv4.held(-x))


def test_append_takes_strided_rows_and_other_orders():
    """Rows inside a fused projection, every second row, a transposed tensor, an odd offset."""
    from joule_b200 import kv4
    rng = np.random.default_rng(8)
    kv, hd, n = 2, 64, 9
    base = _to(rng.standard_normal((n, 5 * kv * hd)), "f32")
    fused_k = base[:, kv * hd:2 * kv * hd].unflatten(1, (kv, hd))
    second = _to(rng.standard_normal((2 * n, kv, hd)), "f32")[::2]
    turned = _to(rng.standard_normal((kv, n, hd)), "f32").transpose(0, 1)
    odd = _to(rng.standard_normal(n * kv * hd + 1), "f32")[1:].view(n, kv, hd)
    one = _to(rng.standard_normal((1, kv, hd)), "f32").expand(n, kv, hd)
    at = _i32([0] * n), _i32(range(n))
    for k, v in ((fused_k, second), (turned, odd), (odd.half(), fused_k.half()), (one, turned)):
        cache = kv4.kv4_cache(1, 1, kv, hd, n)
        kv4.kv4_append(cache, 0, k, v, *at)
        gk, gv = kv4.kv4_read(cache, 0, *at)
        assert np.array_equal(gk.double().cpu().numpy(), okv4.held(k.float().cpu().numpy()))
        assert np.array_equal(gv.double().cpu().numpy(), okv4.held(v.float().cpu().numpy()))


def test_rows_outside_the_cache_are_skipped_and_flagged():
    from joule_b200 import kv4
    rng = np.random.default_rng(9)
    kv, hd = 2, 128
    cache = kv4.kv4_cache(2, 1, kv, hd, 64)
    cache.copy_(torch.from_numpy(rng.integers(0, 256, tuple(cache.shape), dtype=np.uint8)))
    before = cache.clone()
    k = _to(rng.standard_normal((5, kv, hd)), "f32")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    s, p = _i32([-1, 2, 0, 1, 1]), _i32([0, 0, 64, -1, 5])
    kv4.kv4_append(cache, 0, k[:4], k[:4], s[:4].contiguous(), p[:4].contiguous(), status=status)
    assert status.item() == kv4.KV4_BAD_INDEX and torch.equal(cache, before)
    status.zero_()
    gk, gv = kv4.kv4_read(cache, 0, s, p, status=status)
    assert status.item() == kv4.KV4_BAD_INDEX
    assert (gk[:4] == 0).all() and (gv[:4] == 0).all() and (gk[4] != 0).any()
    status.zero_()
    kv4.kv4_append(cache, 0, k[4:], k[4:], s[4:].contiguous(), p[4:].contiguous(), status=status)
    assert status.item() == 0 and not torch.equal(cache, before)


# ---------------------------------------------------------------------------
# attention

STEP = [  # B, H, kv, hd, lens
    (1, 1, 1, 64, [1]), (1, 32, 4, 128, [1]), (3, 8, 1, 128, [63, 64, 65]), (5, 6, 2, 64, [0, 1, 2, 200, 127]),
    (2, 7, 7, 128, [700, 3]), (4, 10, 2, 64, [129, 0, 640, 511]), (3, 16, 1, 128, [300, 5, 77]),
    (2, 22, 2, 64, [90, 1000]), (1, 16, 16, 128, [2500]), (7, 4, 4, 64, [0, 0, 0, 0, 0, 0, 0]),
    (40, 8, 2, 128, [(37 * b) % 190 for b in range(40)]), (170, 2, 1, 64, [(53 * b) % 301 for b in range(170)]),
]


# more (sequence, kv head) pairs than SMs, with short, middle and long caches: a warp for each, all
# blocks cut over all warps, runs of pairs in the adding up; and one long sequence
STEP += [(200, 8, 8, 64, [(31 * b) % 251 for b in range(200)]), (40, 16, 4, 128, [(211 * b) % 1501 for b in range(40)]),
         (40, 15, 5, 64, [(211 * b) % 1501 for b in range(40)]), (80, 16, 8, 64, [(53 * b) % 701 for b in range(80)]),
         (75, 8, 8, 128, [(53 * b) % 1701 for b in range(75)]), (1, 16, 2, 128, [3000])]


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("B,H,kv,hd,lens", STEP)
def test_step(B, H, kv, hd, lens, t):
    """One query row per sequence, slots in any order, other layers and unwritten rows full of noise."""
    from joule_b200 import kv4
    rng = np.random.default_rng(B * 1000 + H)
    maxT = max(max(lens), 1) + 70
    slot_of = rng.permutation(B + 2)[:B]
    cache, ks, vs = _filled(rng, B + 2, 2, kv, hd, maxT, 1, lens, slot_of)
    q = _to(rng.standard_normal((B, 1, H, hd)) * 1.5, t)
    got = kv4.kv4_attention(cache, 1, q, _i32(slot_of), _i32(lens))
    assert got.dtype == q.dtype and got.shape == q.shape
    _check(got, q.double().cpu().numpy(), ks, vs, hd ** -0.5, t)
    assert torch.equal(kv4.kv4_attention(cache, 1, q[:, 0], _i32(slot_of), _i32(lens)), got[:, 0])
    # a bound of the lengths gives the same values up to the order of sums
    if max(lens):
        _check(kv4.kv4_attention(cache, 1, q, _i32(slot_of), _i32(lens), longest=max(lens)),
               q.double().cpu().numpy(), ks, vs, hd ** -0.5, t)


CHUNK = [  # B, T, H, kv, hd, lens
    (1, 2, 4, 2, 64, [2]), (1, 5, 8, 1, 128, [5]), (2, 3, 5, 5, 64, [100, 2]), (1, 64, 8, 1, 128, [64]),
    (3, 17, 6, 2, 128, [300, 17, 0]), (1, 33, 10, 2, 64, [700]), (2, 130, 4, 2, 128, [190, 131]),
    (1, 200, 3, 1, 64, [200]), (4, 16, 16, 1, 128, [64, 65, 500, 1]), (1, 257, 2, 1, 128, [900]),
    (5, 7, 40, 4, 128, [2000, 6, 1999, 0, 700]),
]


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,T,H,kv,hd,lens", CHUNK)
def test_chunk(B, T, H, kv, hd, lens, t):
    """Several query rows per sequence, each seeing the rows up to its own; rows
    of a sequence shorter than T see nothing and are zero."""
    from joule_b200 import kv4
    rng = np.random.default_rng(T * 100 + H)
    slot_of = rng.permutation(B + 1)[:B]
    cache, ks, vs = _filled(rng, B + 1, 1, kv, hd, max(lens) + 3, 0, lens, slot_of)
    q = _to(rng.standard_normal((B, T, H, hd)), t)
    got = kv4.kv4_attention(cache, 0, q, _i32(slot_of), _i32(lens))
    for b in range(B):
        assert (got[b, :max(0, T - lens[b])] == 0).all()
    _check(got, q.double().cpu().numpy(), ks, vs, hd ** -0.5, t)


MANY = [  # B, T, H, kv, hd, lens: 76 rows and more for each SM of 148 and each block of 256
    (1, 710, 16, 4, 128, [1300]), (3, 260, 15, 3, 64, [1100, 259, 700]), (2, 40, 142, 2, 128, [600, 0]),
    (70, 8, 24, 2, 64, [(37 * b) % 301 for b in range(70)]), (1, 2900, 4, 4, 128, [2900]), (1, 2, 6002, 2, 64, [1290]),
    (1, 1, 11904, 1, 128, [577]), (2, 360, 16, 4, 64, [512, 513]),
]


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,T,H,kv,hd,lens", MANY)
def test_many_rows(B, T, H, kv, hd, lens, t):
    """Calls whose rows fill the tensor cores' tiles: ends inside a tile, blocks of one
    tile, sums of one block to 46, tokens whose heads pass a tile, empty sequences."""
    test_chunk(B, T, H, kv, hd, lens, t)


@pytest.mark.parametrize("T", [1, 24, 720])
@pytest.mark.parametrize("scale,ksize,vsize", [(0.0, 1, 1), (-0.3, 1, 1), (1.0, 8, 1), (0.1, 1e-5, 1e-4), (0.05, 300, 3e4)])
def test_scales_and_magnitudes(T, scale, ksize, vsize):
    """Uniform weights (scale 0), negative scales, one key taking all the weight
    (scores in the hundreds), small and large K and V."""
    from joule_b200 import kv4
    rng = np.random.default_rng(12)
    B, H, kv, hd, lens = 2, 8, 2, 128, [333, 90]
    cache = kv4.kv4_cache(B, 1, kv, hd, 400)
    ks, vs = [], []
    for b, n in enumerate(lens):
        k = (rng.standard_normal((n, kv, hd)) * ksize).astype(np.float32)
        v = (rng.standard_normal((n, kv, hd)) * vsize).astype(np.float32)
        kv4.kv4_append(cache, 0, _to(k, "f32"), _to(v, "f32"), _i32([b] * n), _i32(range(n)))
        ks.append(okv4.held(k)), vs.append(okv4.held(v))
    q = _to(rng.standard_normal((B, T, H, hd)) * np.exp(rng.uniform(-5, 3, (B, T, H, 1))), "f32")
    got = kv4.kv4_attention(cache, 0, q, _i32([0, 1]), _i32(lens), scale=scale)
    _check(got, q.double().cpu().numpy(), ks, vs, scale, "f32")


@pytest.mark.parametrize("T,lens", [(3, [150, 70]), (704, [1500, 690])])
def test_rows_of_q_do_not_mix(T, lens):
    """A NaN or an infinity in one head's q leaves every other head's output as it was."""
    from joule_b200 import kv4
    rng = np.random.default_rng(13)
    B, H, kv, hd = 2, 8, 1, 128
    cache, ks, vs = _filled(rng, B, 1, kv, hd, 1500, 0, lens, [0, 1])
    q = _to(rng.standard_normal((B, T, H, hd)), "f32")
    want = kv4.kv4_attention(cache, 0, q, _i32([0, 1]), _i32(lens))
    q[0, 1, 3, 5], q[1, T - 1, 0, 0] = float("nan"), float("inf")
    got = kv4.kv4_attention(cache, 0, q, _i32([0, 1]), _i32(lens))
    bad = torch.zeros(B, T, H, dtype=torch.bool, device="cuda")
    bad[0, 1, 3] = bad[1, T - 1, 0] = True
    assert torch.equal(got[~bad], want[~bad])
    assert torch.isnan(got[0, 1, 3]).all() and not torch.isfinite(got[1, T - 1, 0]).any()


@pytest.mark.parametrize("T", [1, 20, 1000])
def test_bad_slots_and_lengths_give_zeros_and_a_flag(T):
    from joule_b200 import kv4
    rng = np.random.default_rng(14)
    H, kv, hd = 8, 2, 64
    cache, ks, vs = _filled(rng, 2, 1, kv, hd, 128, 0, [100, 64], [0, 1])
    q = _to(rng.standard_normal((6, T, H, hd)), "f32")
    slots, lens = _i32([0, 2, -1, 0, 1, 1]), _i32([100, 50, 50, 129, -1, 64])
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = kv4.kv4_attention(cache, 0, q, slots, lens, status=status)
    assert status.item() == kv4.KV4_BAD_INDEX and (got[1:5] == 0).all()
    _check(got[[0, 5]], q[[0, 5]].double().cpu().numpy(), ks, vs, hd ** -0.5, "f32")
    status.zero_()
    got = kv4.kv4_attention(cache, 0, q[[0, 5]], slots[[0, 5]], lens[[0, 5]], longest=99, status=status)
    assert status.item() == kv4.KV4_BAD_INDEX and (got[0] == 0).all() and (got[1] != 0).any()


@pytest.mark.parametrize("T", [1, 40, 650])
def test_two_sequences_of_one_slot_and_strided_q(T):
    """Entries of a batch may share a slot; q may be a slice of a fused projection or transposed."""
    from joule_b200 import kv4
    rng = np.random.default_rng(15)
    H, kv, hd = 6, 2, 128
    cache, ks, vs = _filled(rng, 1, 1, kv, hd, 200, 0, [180], [0])
    lens = [180, 44, 180]
    fused = _to(rng.standard_normal((3 * T, (H + 2 * kv) * hd)), "f32")
    q = fused[:, :H * hd].unflatten(0, (3, T)).unflatten(2, (H, hd))
    got = kv4.kv4_attention(cache, 0, q, _i32([0, 0, 0]), _i32(lens))
    _check(got, q.double().cpu().numpy(), [ks[0][:n] for n in lens], [vs[0][:n] for n in lens], hd ** -0.5, "f32")
    turned = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(kv4.kv4_attention(cache, 0, turned, _i32([0, 0, 0]), _i32(lens)), got)


def test_long_cache_offsets_pass_32_bits():
    """A cache of more than 4 GiB: the last slot's records lie past 2^32 bytes."""
    from joule_b200 import kv4
    rng = np.random.default_rng(16)
    kv, hd, maxT = 16, 128, 17000
    slots = 40  # 40 * 3 * 16 * 266 blocks * 8704 B = 4.4 GB
    cache = kv4.kv4_cache(slots, 3, kv, hd, maxT)
    assert int(cache.numel()) > 2 ** 32
    n = 100
    k, v = (rng.standard_normal((n, kv, hd)).astype(np.float32) for _ in range(2))
    at = _i32([slots - 1] * n), _i32(range(n))
    kv4.kv4_append(cache, 2, _to(k, "f32"), _to(v, "f32"), *at)
    gk, gv = kv4.kv4_read(cache, 2, *at)
    assert np.array_equal(gk.double().cpu().numpy(), okv4.held(k))
    q = _to(rng.standard_normal((1, 1, 16, hd)), "f32")
    got = kv4.kv4_attention(cache, 2, q, _i32([slots - 1]), _i32([n]))
    _check(got, q.double().cpu().numpy(), [okv4.held(k)], [okv4.held(v)], hd ** -0.5, "f32")


def test_streams_and_repeated_calls():
    """A call on a stream of its own, ordered by events, gives the same bits."""
    from joule_b200 import kv4
    rng = np.random.default_rng(17)
    cache, ks, vs = _filled(rng, 3, 1, 2, 128, 1500, 0, [1500, 700, 33], [0, 1, 2])
    q = _to(rng.standard_normal((3, 1, 16, 128)), "f32")
    args = (_i32([0, 1, 2]), _i32([1500, 700, 33]))
    want = kv4.kv4_attention(cache, 0, q, *args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = [kv4.kv4_attention(cache, 0, q, *args, stream=side) for _ in range(3)]
    raw = kv4.kv4_attention(cache, 0, q, *args, stream=side.cuda_stream)
    torch.cuda.current_stream().wait_stream(side)
    for g in got + [raw]:
        assert torch.equal(g, want)


def test_a_step_captured_and_replayed():
    """Append then attend, captured once with the lengths on the device, replayed
    as the sequences grow; a second graph runs on another stream meanwhile."""
    from joule_b200 import kv4
    rng = np.random.default_rng(18)
    B, H, kv, hd, maxT, steps = 2, 8, 2, 64, 200, 70
    caches = [kv4.kv4_cache(B, 1, kv, hd, maxT) for _ in range(2)]
    slots = _i32([1, 0])
    k, v = (rng.standard_normal((2, steps, B, kv, hd)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((2, steps, B, H, hd)).astype(np.float32)
    bufs, graphs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for w in range(2):
        buf = dict(k=_to(k[w, 0], "f32"), v=_to(v[w, 0], "f32"), q=_to(q[w, 0], "f32"), pos=_i32([0, 0]), len=_i32([1, 1]))
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[w]):
            kv4.kv4_append(caches[w], 0, buf["k"], buf["v"], slots, buf["pos"])
            buf["out"] = kv4.kv4_attention(caches[w], 0, buf["q"], slots, buf["len"])
            buf["pos"] += 1
            buf["len"] += 1
        bufs.append(buf), graphs.append(g)
    outs = [[], []]
    for i in range(steps):
        for w in range(2):
            with torch.cuda.stream(streams[w]):
                for n, x in (("k", k), ("v", v), ("q", q)):
                    bufs[w][n].copy_(torch.from_numpy(x[w, i]))
                graphs[w].replay()
                outs[w].append(bufs[w]["out"].clone())
    torch.cuda.synchronize()
    for w in range(2):
        for i in (0, 1, 40, 63, 64, steps - 1):
            ks = [okv4.held(k[w, :i + 1, b]) for b in range(B)]
            vs = [okv4.held(v[w, :i + 1, b]) for b in range(B)]
            _check(outs[w][i][:, None], q[w, i][:, None].astype(np.float64), ks, vs, hd ** -0.5, "f32")


def test_graphs_of_all_kinds_of_calls_follow_their_inputs():
    """A warp or a block per sequence, a cut, a chunk in splits and a full one: each
    captured at short lengths, replayed in turns after q, lengths and cache changed."""
    from joule_b200 import kv4
    rng = np.random.default_rng(31)
    calls = [(300, 1, 8, 8, 64, 250), (20, 1, 8, 2, 128, 700), (60, 1, 16, 4, 128, 1900), (1, 90, 32, 2, 128, 1500),
             (3, 900, 8, 2, 64, 1000)]
    made = []
    for B, T, H, kv, hd, maxT in calls:
        cache = kv4.kv4_cache(B, 1, kv, hd, maxT)
        k, v = (_to(rng.standard_normal((B * maxT, kv, hd)), "bf16") for _ in range(2))
        at = np.arange(B * maxT)
        kv4.kv4_append(cache, 0, k, v, _i32(at // maxT), _i32(at % maxT))
        q = _to(rng.standard_normal((B, T, H, hd)), "f32")
        slots, lens = _i32(rng.permutation(B)), _i32(np.minimum(T, maxT) + np.zeros(B))
        kw = dict(longest=maxT)
        kv4.kv4_attention(cache, 0, q, slots, lens, **kw)
        g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=side):
            out = kv4.kv4_attention(cache, 0, q, slots, lens, **kw)
        made.append((g, out, cache, q, slots, lens, kw, maxT))
    for turn in range(3):
        for g, out, cache, q, slots, lens, kw, maxT in made:
            q.copy_(torch.randn_like(q) * (turn + 1))
            lens.copy_(torch.randint(0, maxT + 1, lens.shape, device="cuda").int())
            lens[0] = maxT
        for m in made:
            m[0].replay()
        torch.cuda.synchronize()
        for g, out, cache, q, slots, lens, kw, maxT in made:
            assert torch.equal(out, kv4.kv4_attention(cache, 0, q, slots, lens, **kw))


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_compiled_and_interpreted_calls_agree(t):
    """A call with a status word goes through the Python function, one without
    through its compiled form, when the tensors are regular; misaligned and strided
    ones are copied either way. References to the arguments are as before."""
    import sys
    from joule_b200 import kv4
    rng = np.random.default_rng(23)
    B, H, kv, hd = 3, 6, 2, 64
    caches = [kv4.kv4_cache(B, 2, kv, hd, 700).zero_() for _ in range(2)]
    n = 900
    k, v = (_to(rng.standard_normal((n, kv, hd)), t) for _ in range(2))
    at = rng.permutation(B * 700)[:n]
    slots, pos, status = _i32(at // 700), _i32(at % 700), _i32([0])
    lens, ls = _i32([700, 1, 0]), _i32([2, 0, 1])
    q = _to(rng.standard_normal((B, 4, H, hd)), t)
    args = [caches[0], k, v, slots, pos, q, lens, ls]
    before = [sys.getrefcount(a) for a in args]
    kv4.kv4_append(caches[0], 1, k, v, slots, pos)
    kv4.kv4_append(caches[1], 1, k, v, slots, pos, status=status)
    assert torch.equal(caches[0], caches[1])
    for dt in DT.values():
        a, b = kv4.kv4_read(caches[0], 1, slots, pos, dtype=dt), kv4.kv4_read(caches[0], 1, slots, pos, dtype=dt, status=status)
        assert all(x.dtype is dt and torch.equal(x, y) for x, y in zip(a, b))
    for x in (q, q[:, 0], q.transpose(1, 2).contiguous().transpose(1, 2), torch.cat([q.flatten()[:1], q.flatten()])[1:].view(q.shape)):
        for kw in (dict(), dict(scale=0.3), dict(longest=700), dict(longest=699)):
            a, b = kv4.kv4_attention(caches[0], 1, x, ls, lens, **kw), kv4.kv4_attention(caches[0], 1, x, ls, lens, status=status, **kw)
            assert a.shape == x.shape and a.dtype is x.dtype and a.is_contiguous() and torch.equal(a, b)
    del x, a, b
    assert [sys.getrefcount(a) for a in args] == before


def test_front_end_refusals():
    from joule_b200 import kv4
    cache = kv4.kv4_cache(2, 1, 2, 64, 64)
    x, q, i = torch.zeros(2, 2, 64, device="cuda"), torch.zeros(2, 4, 64, device="cuda"), _i32([0, 1])
    bad = [lambda: kv4.kv4_append(cache, 1, x, x, i, i), lambda: kv4.kv4_append(cache, -1, x, x, i, i),
           lambda: kv4.kv4_append(cache, 0, x[:, :1], x[:, :1], i, i), lambda: kv4.kv4_append(cache, 0, x, x.half(), i, i),
           lambda: kv4.kv4_append(cache, 0, x.double(), x.double(), i, i), lambda: kv4.kv4_append(cache, 0, x, x, i.long(), i),
           lambda: kv4.kv4_append(cache, 0, x, x, i[:1], i), lambda: kv4.kv4_append(cache, 0, x, x, i, i.cpu()),
           lambda: kv4.kv4_append(cache, 0, x.cpu(), x.cpu(), i, i), lambda: kv4.kv4_append(cache[:, :, :1], 0, x, x, i, i),
           lambda: kv4.kv4_append(cache.float(), 0, x, x, i, i), lambda: kv4.kv4_append(cache[..., :100], 0, x, x, i, i),
           lambda: kv4.kv4_append(cache, 0, x, x, i, i, status=i.long()),
           lambda: kv4.kv4_read(cache, 0, i, i, dtype=torch.float64), lambda: kv4.kv4_read(cache, 0, i, i[:1]),
           lambda: kv4.kv4_attention(cache, 0, q[:, :3], i, i), lambda: kv4.kv4_attention(cache, 0, q[..., :32], i, i),
           lambda: kv4.kv4_attention(cache, 0, q.double(), i, i), lambda: kv4.kv4_attention(cache, 0, q, i[:1], i),
           lambda: kv4.kv4_attention(cache, 0, q, i, i, longest=65), lambda: kv4.kv4_attention(cache, 0, q, i, i, longest=0),
           lambda: kv4.kv4_attention(cache, 0, q, i, i, out=torch.empty_like(q, dtype=torch.float16)),
           lambda: kv4.kv4_attention(cache, 0, q.view(2, 1, 4, 64)[:, :0], i, i)]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    from joule_b200.native import JouleError
    with pytest.raises(JouleError):
        kv4.kv4_attention(cache, 0, q, i, i, scale=float("nan"))
    with pytest.raises(JouleError):
        kv4.kv4_attention(cache, 0, q, i, i, out=q)
    # empty batches do nothing
    e = _i32([])
    kv4.kv4_append(cache, 0, x[:0], x[:0], e, e)
    assert kv4.kv4_read(cache, 0, e, e)[0].shape == (0, 2, 64)
    assert kv4.kv4_attention(cache, 0, q[:0], e, e).shape == (0, 4, 64)
