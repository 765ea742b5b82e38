"""Waits inside the tcgen05 attention that run out: every role of the kernel leaves,
nothing stays in flight, and the failure is reported, by the status word of a call or,
without one, by kv4_check. The limit is set to nothing, so that each wait gives up at
once, or to a nanosecond, so that some may in the middle of the work; the kernel waits
for nothing but its own copies and products."""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEFAULT_NS = 2_000_000_000


def _i32(x):
    return torch.as_tensor(np.asarray(x, np.int32)).cuda()


@pytest.fixture
def limit():
    from joule_b200.native import check, get_dll
    yield lambda ns: check(get_dll().jl_kv4_set_wait_limit(ns), "jl_kv4_set_wait_limit")
    check(get_dll().jl_kv4_set_wait_limit(DEFAULT_NS), "jl_kv4_set_wait_limit")


def _case(T, H, kv, hd, n, t):
    from joule_b200 import kv4
    g = torch.Generator(device="cuda").manual_seed(T)
    k, v = (torch.randn(n, kv, hd, device="cuda", generator=g) for _ in range(2))
    cache = kv4.kv4_cache(1, 1, kv, hd, n)
    kv4.kv4_append(cache, 0, k, v, _i32([0] * n), _i32(range(n)))
    q = torch.randn(1, T, H, hd, device="cuda", generator=g).to(t)
    at = (_i32([0]), _i32([n]))
    return lambda **kw: kv4.kv4_attention(cache, 0, q, *at, **kw)


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,H,kv,hd,n", [(720, 32, 4, 128, 1333), (64, 32, 4, 128, 3000), (1200, 32, 4, 64, 5000)])
def test_a_wait_that_runs_out_is_reported(T, H, kv, hd, n, t, limit):
    from joule_b200 import kv4
    from joule_b200.native import JouleError
    call = _case(T, H, kv, hd, n, t)
    want = call()
    kv4.kv4_check()
    status = _i32([0])
    limit(0)
    call(status=status)
    assert status.item() == kv4.KV4_TIMEOUT
    kv4.kv4_check()  # the call had a word of its own
    call()
    with pytest.raises(JouleError) as e:
        kv4.kv4_check()
    assert e.value.code == -4
    kv4.kv4_check()  # reported once
    limit(1)
    for _ in range(20):
        status.zero_()
        got = call(status=status)
        assert status.item() in (0, kv4.KV4_TIMEOUT)
        if status.item() == 0:
            assert torch.equal(got, want)
    limit(DEFAULT_NS)
    assert torch.equal(call(), want)
    kv4.kv4_check()


def test_a_captured_call_is_reported():
    """The limit is the one of the launch that was captured; each replay reports."""
    from joule_b200 import kv4
    from joule_b200.native import JouleError, check, get_dll
    call = _case(64, 32, 4, 128, 3000, torch.float32)
    want = call()
    torch.cuda.synchronize()
    graphs = []
    try:
        for ns in (0, DEFAULT_NS):
            check(get_dll().jl_kv4_set_wait_limit(ns), "jl_kv4_set_wait_limit")
            g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
            with torch.cuda.graph(g, stream=side):
                out = call()
            graphs.append((g, out))
    finally:
        check(get_dll().jl_kv4_set_wait_limit(DEFAULT_NS), "jl_kv4_set_wait_limit")
    for _ in range(2):
        graphs[0][0].replay()
        with pytest.raises(JouleError):
            kv4.kv4_check()
        graphs[1][0].replay()
        kv4.kv4_check()
        assert torch.equal(graphs[1][1], want)
