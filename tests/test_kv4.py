"""The 4-bit KV cache without a GPU: argument checks of the C entries and of the
Python front end, sizes, and the oracle's layout and quantiser."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from joule_b200 import kv4, native
from joule_b200.native import Kv4
from oracle import kv4 as okv4


@pytest.fixture(scope="module")
def dll():
    if not native.lib_path().exists():
        from joule_b200 import build
        build.build()
    return native.get_dll()


def test_struct_layout():
    assert ctypes.sizeof(Kv4) == 32 and Kv4.slots.offset == 8 and Kv4.maxT.offset == 24


@pytest.mark.parametrize("hd", [64, 128])
def test_layout_is_a_bijection(hd):
    """Every nibble and scale byte of a block belongs to exactly one value."""
    seen = np.zeros((68 * hd, 2), int)
    for is_v in (False, True):
        for r in range(64):
            for d in range(hd):
                seen[okv4.byte_of(hd, is_v, r, d), d % 2] += 1
            for g in range(hd // 64):
                b = okv4.scale_byte(hd, is_v, r, g)
                seen[b:b + 2] += 1
    assert (seen == 1).all()


def test_quantiser_matches_the_store_format():
    """Finite rows get the Q4 store's own codes and scales (q4_store.py:40-55)."""
    from oracle import q4
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((50, 128)) * np.exp(rng.uniform(-12, 6, (50, 1)))).astype(np.float32)
    codes, s = okv4.quantise(x)
    scales, packed = q4.quantize(x)
    assert np.array_equal(scales, s.reshape(-1).view(np.uint16))
    pk = packed.reshape(50, 64)
    assert np.array_equal(pk & 15, codes[:, 0::2]) and np.array_equal(pk >> 4, codes[:, 1::2])


def test_bytes(dll):
    c = Kv4(None, 3, 2, 4, 128, 100)
    assert dll.jl_kv4_bytes(ctypes.byref(c)) == 3 * 2 * 4 * 2 * 68 * 128
    c.hd = 96
    assert dll.jl_kv4_bytes(ctypes.byref(c)) == -1
    assert dll.jl_kv4_bytes(None) == -1
    big = Kv4(None, 2**31 - 1, 2**31 - 1, 2**31 - 1, 128, 100)
    assert dll.jl_kv4_bytes(ctypes.byref(big)) == -1


def _c(**kw):
    return Kv4(**(dict(base=4096, slots=2, L=2, n_kv=2, hd=128, maxT=128) | kw))


@pytest.mark.parametrize("kw,l", [(dict(base=None), 0), (dict(base=4100), 0), (dict(hd=32), 0), (dict(hd=96), 0),
                                  (dict(slots=0), 0), (dict(maxT=0), 0), (dict(n_kv=0), 0), (dict(), 2), (dict(), -1)])
def test_bad_caches_are_refused(dll, kw, l):
    c = _c(**kw)
    r = ctypes.byref(c)
    assert dll.jl_kv4_append(r, l, 4096, 4096, 0, 256, 256, 4096, 4096, 1, None, None) == -1
    assert dll.jl_kv4_read(r, l, 4096, 4096, 1, 4096, 4096, 0, None, None) == -1
    assert dll.jl_kv4_attn(r, l, 4096, 0, 512, 4096, 4096, 0, 1, 1, 4, 1.0, 1 << 20, 4096, 1 << 40, None, None) == -1


def test_bad_arguments_are_refused(dll):
    c = _c()
    r = ctypes.byref(c)
    ap = lambda k=4096, v=4096, t=0, ks=256, vs=256, s=4096, p=4096, n=2: dll.jl_kv4_append(  # noqa: E731
        r, 0, k, v, t, ks, vs, s, p, n, None, None)
    assert ap(n=0) == 0 and ap(k=None, v=None, s=None, p=None, n=0) == 0
    assert all(x == -1 for x in (ap(n=-1), ap(k=None), ap(v=None), ap(s=None), ap(p=None), ap(t=3), ap(t=-1),
                                 ap(k=4100), ap(v=4104), ap(ks=255), ap(vs=128), ap(t=1, ks=260)))
    rd = lambda t=0, s=4096, p=4096, n=1, k=4096, v=4096: dll.jl_kv4_read(r, 0, s, p, n, k, v, t, None, None)  # noqa: E731
    assert rd(n=0) == 0
    assert all(x == -1 for x in (rd(n=-1), rd(t=3), rd(s=None), rd(p=None), rd(k=None), rd(v=4100)))

    def at(q=4096, t=0, qs=512, s=4096, n=4096, longest=0, B=2, T=1, H=4, scale=1.0, out=1 << 20, ws=4096, wb=1 << 40):
        return dll.jl_kv4_attn(r, 0, q, t, qs, s, n, longest, B, T, H, scale, out, ws, wb, None, None)
    assert at(B=0) == 0
    assert all(x == -1 for x in (at(q=None), at(q=4100), at(t=3), at(qs=511), at(qs=256), at(s=None), at(n=None),
                                 at(longest=-1), at(longest=129), at(B=-1), at(T=0), at(H=3), at(H=0),
                                 at(scale=float("nan")), at(scale=float("inf")), at(out=None), at(out=(1 << 20) + 8),
                                 at(out=4096), at(out=4096 + 2 * 512 * 4 - 16), at(qs=1 << 20, out=1 << 20),
                                 at(B=2**20, T=2**20), at(B=1, H=2**25, out=1 << 40)))
    ws = dll.jl_kv4_attn_ws
    assert all(x == -1 for x in (ws(r, 2, 1, 3, 0), ws(r, 2, 0, 4, 0), ws(r, -1, 1, 4, 0), ws(r, 2, 1, 4, -1),
                                 ws(r, 2, 1, 4, 129), ws(r, 2**20, 2**20, 4, 0)))
    assert ws(r, 0, 1, 4, 0) == 0 and ws(r, 2, 1, 4, 0) == 0


@pytest.mark.parametrize("B,T,longest", [(64, 1, 0), (2, 1, 9000), (1, 64, 3000)])
def test_calls_without_their_workspace_are_refused(dll, B, T, longest):
    """Steps that are cut over all warps, and chunks whose cache is split."""
    c = _c(slots=64, maxT=10000)
    r = ctypes.byref(c)
    need = dll.jl_kv4_attn_ws(r, B, T, 16, longest)
    assert need > 0 and dll.jl_kv4_attn_ws(r, B, T, 16, 256) == 0
    at = lambda ws, wb: dll.jl_kv4_attn(r, 0, 4096, 0, 2048, 4096, 4096, longest, B, T, 16, 1.0, 1 << 30, ws, wb, None,  # noqa: E731
                                        None)
    assert at(None, need) == -1 and at(4096, need - 1) == -1 and at(4100, need) == -1


def test_front_end_refuses_without_a_device():
    """Host tensors and wrong types end with ValueError before any call."""
    cache = torch.zeros(2, 1, 2, 1, 68 * 64, dtype=torch.uint8)
    i = torch.zeros(2, dtype=torch.int32)
    x = torch.zeros(2, 2, 64)
    with pytest.raises(ValueError):
        kv4.kv4_append(cache, 0, x, x, i, i)
    with pytest.raises(ValueError):
        kv4.kv4_read(cache, 0, i, i)
    with pytest.raises(ValueError):
        kv4.kv4_attention(cache, 0, x, i, i)
    for bad in (dict(hd=96), dict(slots=0), dict(maxT=0)):
        with pytest.raises(ValueError):
            kv4.kv4_cache(**(dict(slots=1, L=1, n_kv=1, hd=64, maxT=1, device="cpu") | bad))
    assert kv4.kv4_cache(2, 3, 4, 128, 65, device="cpu").shape == (2, 3, 4, 2, 68 * 128)


def test_decoder_flags_are_checked(dll):
    """jl_dec_create_ex refuses flags it does not know and head dims that the
    4-bit cache does not hold, before any device work."""
    from joule_b200.native import DEC_KV4, KernelCfg, KernelW
    W = KernelW()
    for n in ("embed", "lm_head", "final_norm", "norm1", "norm2", "wq", "wk", "wv", "wo", "gate_w", "cos", "sin"):
        setattr(W, n, 4096)
    h = ctypes.c_void_p()
    cfg = dict(L=1, d=256, n_heads=4, n_kv=2, hd=32, E=8, topk=2, V=64, maxT=16, intermediate=128)
    make = lambda flags, **kw: dll.jl_dec_create_ex(ctypes.byref(KernelCfg(**(cfg | kw))), ctypes.byref(W), 2, 2, 0,  # noqa: E731
                                                    flags, ctypes.byref(h))
    assert make(DEC_KV4) == -1 and make(2, hd=64) == -1 and make(-1, hd=64) == -1
    c = Kv4()
    assert dll.jl_dec_kv4(None, ctypes.byref(c)) == -1


def test_the_compiled_calls_pass_on_what_is_not_regular():
    """joule_b200._kv4_call answers None, and leaves no error set, to arguments
    that the Python function must copy, refuse or raise on."""
    kv4._bind()
    call = kv4._call
    cache = torch.zeros(2, 1, 2, 1, 68 * 64, dtype=torch.uint8)
    i, x, q = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 2, 64), torch.zeros(2, 4, 64)
    for bad in (cache, None, 3, "x", torch.zeros(1, 1, 1, 1, 1, 1)):
        assert call.append(bad, 0, x, x, i, i) is None
        assert call.read(bad, 0, i, i, torch.float32) is None
        assert call.attention(bad, 0, q, i, i, None, None) is None
    assert call.append() is None and call.read(cache) is None and call.attention(cache, 0) is None
    assert call.read(cache, 0, i, i, torch.float64) is None
    with pytest.raises(TypeError):
        call.bind(1)


def test_wait_limits_and_devices_are_checked(dll):
    assert dll.jl_kv4_set_wait_limit(-1) == -1
    with pytest.raises(ValueError):
        kv4.kv4_check("cpu")


def test_the_decoders_cache_is_on_its_own_device(monkeypatch):
    """Decoder.kv4_cache asks for the device that the decoder was created on, whichever is
    current; with the current one it would be a copy there."""
    from joule_b200 import decoder

    class Lib:
        def jl_dec_kv4(self, h, c):
            c._obj.base, c._obj.slots, c._obj.L, c._obj.n_kv, c._obj.hd, c._obj.maxT = 4096, 2, 1, 2, 64, 65
            return 0

        def jl_dec_destroy(self, h):
            return 0
    d = decoder.Decoder.__new__(decoder.Decoder)
    d._L, d.h, d.device = Lib(), ctypes.c_void_p(1), torch.device("cuda", 3)
    seen = {}
    monkeypatch.setattr(decoder.torch, "as_tensor", lambda x, device=None: seen.update(x=x, device=device))
    d.kv4_cache()
    assert torch.device(seen["device"]) == torch.device("cuda", 3)
    assert seen["x"].__cuda_array_interface__["shape"] == (2, 1, 2, 2, 68 * 64)


def test_the_compiled_calls_belong_to_one_python_and_can_be_missing(monkeypatch):
    """The module's file carries the interpreter's tag, so that no other one loads it, and
    without it the Python functions do everything."""
    import sys
    import sysconfig

    import joule_b200
    from joule_b200 import build
    assert build.CALL.name == "_kv4_call" + sysconfig.get_config_var("EXT_SUFFIX")
    monkeypatch.delattr(joule_b200, "_kv4_call", raising=False)
    monkeypatch.setitem(sys.modules, "joule_b200._kv4_call", None)
    monkeypatch.setattr(kv4, "_call", None)
    kv4._bind()
    i, x = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 2, 64)
    assert kv4._call is not None and kv4._call.append(x, 0, x, x, i, i) is None
    for call in (lambda c: kv4.kv4_append(c, 0, x, x, i, i), lambda c: kv4.kv4_read(c, 0, i, i),
                 lambda c: kv4.kv4_attention(c, 0, x, i, i)):
        with pytest.raises(ValueError):
            call(torch.zeros(2, 1, 2, 1, 68 * 64, dtype=torch.uint8))
