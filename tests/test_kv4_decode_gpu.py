"""The decoder with a 4-bit KV cache (JL_DEC_KV4) on the GPU: prompts, batched
steps and a captured step, against the restatement of the decode step with
attention over the values that the GPU's own cache holds (oracle/kv4.py), and
the cached rows against the rows that should have been written.

Layer 0's rows are those of the fp32 decoder bit for bit, so its records are
held to `==`. Later rows follow attention in another order of sums: a cached
value may be off by half a step of its group (its scale, fp16, is at most
max|x| / 7 * (1 + 2^-11)) plus what the row itself may be off.

Logits: with e = 2^-24, each projection of K values is off by at most K e of the
sum of its products' sizes, and the attention's weights by 64 e max(1, max|s|)
(tests/test_kv4_gpu.py); the bound adds these over all layers for the norm of the
logits, times 4 for what norms and the gated FFN may make of an error, plus
expf_fast's arguments in the router and the FFN (the same function on both sides).
"""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import kv4 as okv4

pytestmark = pytest.mark.gpu
E = 2.0 ** -24


def _shape(name, **kw):
    from oracle.decode import SHAPES, DecodeShape
    return DecodeShape(**(SHAPES[name].__dict__ | kw))


def _decoder(model, max_batch, slots, kv4=True):
    from joule_b200.decoder import Decoder
    from joule_b200.native import PATH_EXACT
    from test_decode_gpu import _structs
    cfg, W, tables = _structs(model)
    dec = Decoder(cfg, W, max_batch, slots, False, kv4=kv4)
    dec._tables = tables
    dec.set_moe_path(PATH_EXACT)
    return dec


def _step(dec, slots, positions, x):
    s, p = (torch.as_tensor(np.asarray(a, np.int32)).cuda() for a in (slots, positions))
    xd = torch.from_numpy(np.ascontiguousarray(x, np.float32)).cuda()
    logits = torch.empty(len(slots), dec.cfg.V, device="cuda")
    tok = torch.empty(len(slots), dtype=torch.int32, device="cuda")
    dec.step(s, p, xd, tok=tok, logits=logits)
    dec.check()
    return logits.double().cpu().numpy(), tok.cpu().numpy()


def _cached(dec, slot, n):
    """(k, v) [L][n, n_kv, hd] of a slot's first n rows, as the cache holds them."""
    from joule_b200 import kv4
    at = (torch.full((n,), slot, dtype=torch.int32, device="cuda"), torch.arange(n, dtype=torch.int32, device="cuda"))
    return [tuple(t.double().cpu().numpy() for t in kv4.kv4_read(dec.kv4_cache(), l, *at)) for l in range(dec.cfg.L)]


def _tol(s, top):
    per = (2 * s.d + s.H * s.hd + s.m) * E + 64 * E * max(1.0, top)
    return 4 * (s.L * per + s.d * E)


def _held_near(got, rows, slack):
    """Cached values against the rows written: half a step of their group, and `slack` of the row's largest value."""
    g = rows.astype(np.float64).reshape(*rows.shape[:-1], -1, 64)
    amax = np.abs(g).max(-1, keepdims=True)
    tol = amax / 14 * (1 + 2.0 ** -10) + slack * np.abs(g).max() + 2.0 ** -24
    assert (np.abs(got.reshape(g.shape) - g) <= tol).all()


MODELS = [("qwen3s", {}), ("olmoes", {}), ("qwen2s", {}), ("qwen3s", dict(H=8, KH=1, hd=128, maxT=300)),
          ("qwen3s", dict(H=10, KH=2, maxT=200))]


@pytest.mark.parametrize("name,kw", MODELS)
def test_prompts_and_steps(name, kw):
    """Prompts of odd lengths in chunks of 5 rows into slots in any order, then
    batched ragged steps: the last position's logits, the cached rows and tokens."""
    from oracle.decode import embed, make_model
    s = _shape(name, **kw)
    model = make_model(s, seed=51)
    rng = np.random.default_rng(4)
    lens, slots = [13, 1, 37], [4, 0, 2]
    prompts = [rng.integers(0, s.V, n).astype(np.int32) for n in lens]
    dec, ref = _decoder(model, 5, 5), _decoder(model, 5, 5, kv4=False)
    kp, vp = ctypes.c_void_p(), ctypes.c_void_p()
    assert dec._L.jl_dec_kv(dec.h, ctypes.byref(kp), ctypes.byref(vp)) == -1
    assert ref._L.jl_dec_kv(ref.h, ctypes.byref(kp), ctypes.byref(vp)) == 0
    from test_decode_batch_gpu import _DevArray
    kc = torch.as_tensor(_DevArray(kp.value, (5, s.L, s.maxT, s.KH, s.hd)), device="cuda")
    vc = torch.as_tensor(_DevArray(vp.value, (5, s.L, s.maxT, s.KH, s.hd)), device="cuda")
    for slot, p in zip(slots, prompts):
        pt = torch.from_numpy(p).cuda()
        logits = torch.empty(s.V, device="cuda")
        dec.prefill(slot, pt, logits=logits)
        ref.prefill(slot, pt)
        dec.check(), ref.check()
        n = len(p)
        rows = _cached(dec, slot, n)
        # layer 0's records are those of the fp32 decoder's rows
        for got, want in zip(rows[0], (kc[slot, 0, :n], vc[slot, 0, :n])):
            assert np.array_equal(got, okv4.held(want.cpu().numpy()))
        want, ks, vs, top = okv4.decode_step(model, embed(model, p[-1:]), [n - 1], lambda l, b: rows[l])
        for l in range(s.L):
            _held_near(rows[l][0][-1], ks[l][0], _tol(s, top))
            _held_near(rows[l][1][-1], vs[l][0], _tol(s, top))
        err = np.linalg.norm(logits.double().cpu().numpy() - want[0]) / np.linalg.norm(want[0])
        assert err <= _tol(s, top), err
    pos = np.array(lens, np.int32)
    cur = rng.integers(0, s.V, 3).astype(np.int32)
    for _ in range(4):
        x = embed(model, cur)
        got, tok = _step(dec, slots, pos, x)
        held = [_cached(dec, slot, p + 1) for slot, p in zip(slots, pos)]
        want, ks, vs, top = okv4.decode_step(model, x, pos, lambda l, b: held[b][l])
        err = np.linalg.norm(got - want) / np.linalg.norm(want)
        assert err <= _tol(s, top), err
        for b in range(3):
            for l in range(s.L):
                _held_near(held[b][l][0][-1], ks[l][b], _tol(s, top))
                _held_near(held[b][l][1][-1], vs[l][b], _tol(s, top))
        assert np.array_equal(tok, got.argmax(1))
        cur, pos = tok, pos + 1
    dec.close(), ref.close()


@pytest.mark.parametrize("hd", [64, 128])
def test_a_prompt_in_one_chunk(hd):
    """A prompt of 713 rows of 16 heads in one call: the last position's logits over
    the values that the cache then holds, and the last cached rows."""
    from oracle.decode import embed, make_model
    s = _shape("qwen3s", H=16, KH=4, hd=hd, maxT=720)
    model = make_model(s, seed=54)
    n = 713
    p = np.random.default_rng(hd).integers(0, s.V, n).astype(np.int32)
    dec = _decoder(model, n, n)
    logits = torch.empty(s.V, device="cuda")
    dec.prefill(1, torch.from_numpy(p).cuda(), logits=logits)
    dec.check()
    rows = _cached(dec, 1, n)
    want, ks, vs, top = okv4.decode_step(model, embed(model, p[-1:]), [n - 1], lambda l, b: rows[l])
    for l in range(s.L):
        _held_near(rows[l][0][-1], ks[l][0], _tol(s, top))
        _held_near(rows[l][1][-1], vs[l][0], _tol(s, top))
    err = np.linalg.norm(logits.double().cpu().numpy() - want[0]) / np.linalg.norm(want[0])
    assert err <= _tol(s, top), err
    dec.close()


@pytest.mark.parametrize("B", [16, 33])
def test_large_batches(B):
    """Batches whose matvecs read the attention's column-major copy; ragged positions over seeded caches."""
    from joule_b200 import kv4
    from oracle.decode import embed, make_model
    s = _shape("qwen3s", H=8, KH=2, hd=128, maxT=500, V=4096)
    model = make_model(s, seed=52)
    rng = np.random.default_rng(B)
    dec = _decoder(model, B, B + 1)
    pos = np.array([(7 + 31 * b) % (s.maxT - 1) for b in range(B)], np.int32)
    pos[1] = 0
    slots = rng.permutation(B + 1)[:B]
    for b in range(B):
        n = int(pos[b])
        if n:
            at = (torch.full((n,), int(slots[b]), dtype=torch.int32, device="cuda"),
                  torch.arange(n, dtype=torch.int32, device="cuda"))
            for l in range(s.L):
                k, v = (torch.from_numpy(rng.standard_normal((n, s.KH, s.hd), np.float32)).cuda() for _ in range(2))
                kv4.kv4_append(dec.kv4_cache(), l, k, v, *at)
    x = embed(model, rng.integers(0, s.V, B))
    got, tok = _step(dec, slots, pos, x)
    held = [_cached(dec, int(slots[b]), int(pos[b]) + 1) for b in range(B)]
    want, ks, vs, top = okv4.decode_step(model, x, pos, lambda l, b: held[b][l])
    err = np.linalg.norm(got - want, axis=1) / np.linalg.norm(want, axis=1)
    assert err.max() <= _tol(s, top), err
    assert np.array_equal(tok, got.argmax(1))
    dec.close()


def test_prefill_equals_steps_up_to_rounding_and_a_graph_replays():
    """One chunk of 24 rows against 24 single steps (the same cached records in
    layer 0), then a captured step replayed with tokens and positions on the device."""
    from oracle.decode import embed, make_model
    s = _shape("qwen3s", maxT=80)
    model = make_model(s, seed=53)
    p = np.random.default_rng(3).integers(0, s.V, 24).astype(np.int32)
    dec = _decoder(model, 24, 24)
    logits = torch.empty(s.V, device="cuda")
    dec.prefill(0, torch.from_numpy(p).cuda(), logits=logits)
    for i, t in enumerate(p):
        one, _ = _step(dec, [1], [i], embed(model, [t]))
    a, b = _cached(dec, 0, 24), _cached(dec, 1, 24)
    assert np.array_equal(a[0][0], b[0][0]) and np.array_equal(a[0][1], b[0][1])
    # eager steps of slot 0, then the same from a graph on slot 1
    eager, x = [], torch.empty(1, s.d, device="cuda")
    tok = torch.tensor([5], dtype=torch.int32, device="cuda")
    pos = torch.tensor([24], dtype=torch.int32, device="cuda")
    slot0, slot1 = (torch.tensor([i], dtype=torch.int32, device="cuda") for i in (0, 1))
    cache = dec.kv4_cache()
    cache[1].copy_(cache[0])
    for _ in range(6):
        dec.embed(tok, x)
        dec.step(slot0, pos, x, tok=tok)
        eager.append(tok.item())
        pos += 1
    tok.fill_(5), pos.fill_(24)
    torch.cuda.synchronize()
    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=side):
        dec.embed(tok, x)
        dec.step(slot1, pos, x, tok=tok)
        pos += 1
    got = []
    for _ in range(6):
        g.replay()
        torch.cuda.synchronize()
        got.append(tok.item())
    dec.check()
    assert got == eager
    dec.close()


def test_positions_outside_are_reported():
    from joule_b200.native import JouleError
    from oracle.decode import embed, make_model
    s = _shape("qwen3s")
    model = make_model(s, seed=54)
    dec = _decoder(model, 2, 2)
    x = embed(model, [1, 2])
    with pytest.raises(JouleError):
        _step(dec, [0, 1], [s.maxT, 0], x)
    with pytest.raises(JouleError):
        _step(dec, [2, 0], [0, 0], x)
    got, _ = _step(dec, [0, 1], [0, 0], x)
    assert np.isfinite(got).all()
    dec.close()


def test_memory_is_a_seventh():
    """48 layers of the Qwen3 shape's cache: 68 bytes per 128 values against 512."""
    from joule_b200.native import Kv4, get_dll
    n = get_dll().jl_kv4_bytes(ctypes.byref(Kv4(None, 64, 48, 4, 128, 4096)))
    assert n * 512 == 64 * 48 * 4096 * 4 * 2 * 512 * 68
