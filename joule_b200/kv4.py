"""Python front end of the 4-bit KV cache (jl_kv4_* in joule_moe.h).

A cache is one uint8 CUDA tensor [slots, L, n_kv, blocks, 68 * hd] (``kv4_cache``):
a block holds the K and V records (Q4, groups of 64 along the head, fp16
scales) of 64 positions of one kv head, 4.25 bits per value. ``kv4_append``
quantises K/V rows as it writes them, ``kv4_read`` gives cached values back and
``kv4_attention`` attends over the cache: one query row per sequence in a
decode step, several in a piece of a prompt. The decoder keeps its cache in
this form when it is created with ``kv4=True`` (joule_b200.decoder). The
reference's caches are fp32; this one has no counterpart there.

Calls run on the cache's device, on the current stream there or the one given;
all of them can be captured into CUDA graphs. Nothing is checked on the
device's side of a call but what would leave the cache: a slot, position or
length outside it skips the row (append) or reads as zeros, and sets bit 8 of
``status`` (an int32 CUDA tensor of one element) when one is given.
"""
from __future__ import annotations

import ctypes
import math

import torch

from joule_b200.native import BF16, F16, F32, Kv4, check, get_dll

__all__ = ["KV4_BLOCK", "KV4_BAD_INDEX", "kv4_cache", "kv4_append", "kv4_read", "kv4_attention"]

KV4_BLOCK = 64      # positions per block
KV4_BAD_INDEX = 8   # status bit: a slot, position or length outside the cache
_TYPES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}


def kv4_cache(slots: int, L: int, n_kv: int, hd: int, maxT: int, device=None) -> torch.Tensor:
    """An uninitialised cache of `slots` sequences x L layers x maxT positions
    (rounded up to whole blocks) on `device` (the current CUDA device)."""
    if hd not in (64, 128) or min(slots, L, n_kv, maxT) < 1:
        raise ValueError(f"kv4_cache: hd 64 or 128 and sizes >= 1, got slots {slots}, L {L}, n_kv {n_kv}, "
                         f"hd {hd}, maxT {maxT}")
    if device is None:
        device = torch.device("cuda", torch.cuda.current_device())
    return torch.empty(slots, L, n_kv, -(-maxT // KV4_BLOCK), 68 * hd, dtype=torch.uint8, device=device)


def _view(cache: torch.Tensor, l: int) -> Kv4:
    if cache.dtype != torch.uint8 or cache.dim() != 5 or not cache.is_cuda or not cache.is_contiguous():
        raise ValueError("kv4: the cache is a contiguous uint8 CUDA tensor [slots, L, n_kv, blocks, 68 * hd]")
    slots, L, kh, nb, size = cache.shape
    if size not in (68 * 64, 68 * 128) or cache.numel() == 0:
        raise ValueError(f"kv4: block size {size} is not 68 * hd with hd 64 or 128, or the cache is empty")
    if not 0 <= l < L:
        raise ValueError(f"kv4: layer {l} outside [0, {L})")
    return Kv4(cache.data_ptr(), slots, L, kh, size // 68, nb * KV4_BLOCK)


def _index(t: torch.Tensor, n: int, dev, name: str) -> int:
    if t.dtype != torch.int32 or t.device != dev or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise ValueError(f"kv4: {name} is a contiguous int32 tensor [{n}] on {dev}")
    return t.data_ptr()


def _status(t, dev) -> int | None:
    if t is None:
        return None
    if t.dtype != torch.int32 or t.device != dev or t.numel() < 1:
        raise ValueError(f"kv4: status is an int32 tensor on {dev}")
    return t.data_ptr()


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t [rows, heads, hd] with whole rows at a 16-byte aligned stride; others are copied."""
    _, h, d = t.shape
    es = t.element_size()
    s = t.stride()
    if s[2] != 1 or (h > 1 and s[1] != d) or (t.shape[0] > 1 and (s[0] < h * d or s[0] * es % 16)) \
            or t.data_ptr() % 16:
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
    return t


class _on:
    """The device and stream of a call: tensors it allocates belong to that
    stream, and the current device is the cache's."""

    __slots__ = ("guard", "handle")

    def __init__(self, dev, stream):
        if stream is None and torch.cuda.current_device() == dev.index:
            self.guard = None
            self.handle = torch.cuda.current_stream(dev.index).cuda_stream
            return
        if stream is None:
            stream = torch.cuda.current_stream(dev)
        elif not isinstance(stream, torch.cuda.Stream):
            stream = torch.cuda.ExternalStream(int(stream), device=dev)
        if stream.device != dev:
            raise ValueError(f"kv4: the stream is on {stream.device}, the cache on {dev}")
        self.guard = torch.cuda.stream(stream)
        self.handle = stream.cuda_stream

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        return self.handle

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def kv4_append(cache: torch.Tensor, l: int, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor,
               positions: torch.Tensor, status: torch.Tensor | None = None, stream=None) -> None:
    """Quantise k, v [N, n_kv, hd] (fp32, fp16 or bf16; rows of any stride)
    into positions[n] of slot slots[n] (int32 [N], distinct pairs) of layer l."""
    c = _view(cache, l)
    dev = cache.device
    if k.shape != v.shape or k.dim() != 3 or k.shape[1:] != (c.n_kv, c.hd):
        raise ValueError(f"kv4_append: k and v are [N, {c.n_kv}, {c.hd}], got {tuple(k.shape)} and {tuple(v.shape)}")
    if k.dtype not in _TYPES or v.dtype != k.dtype or k.device != dev or v.device != dev:
        raise ValueError(f"kv4_append: k and v are fp32, fp16 or bf16, of one type, on {dev}")
    n = k.shape[0]
    ps, pp, st = _index(slots, n, dev, "slots"), _index(positions, n, dev, "positions"), _status(status, dev)
    with _on(dev, stream) as s:
        k, v = _rows(k), _rows(v)
        check(get_dll().jl_kv4_append(ctypes.byref(c), l, k.data_ptr(), v.data_ptr(), _TYPES[k.dtype], k.stride(0),
                                      v.stride(0), ps, pp, n, st, s), "jl_kv4_append")


def kv4_read(cache: torch.Tensor, l: int, slots: torch.Tensor, positions: torch.Tensor,
             dtype: torch.dtype = torch.float32, status: torch.Tensor | None = None,
             stream=None) -> tuple[torch.Tensor, torch.Tensor]:
    """The cached keys and values [N, n_kv, hd] of (slots[n], positions[n])."""
    c = _view(cache, l)
    dev = cache.device
    if dtype not in _TYPES:
        raise ValueError(f"kv4_read: dtype is fp32, fp16 or bf16, got {dtype}")
    n = slots.numel()
    ps, pp, st = _index(slots, n, dev, "slots"), _index(positions, n, dev, "positions"), _status(status, dev)
    with _on(dev, stream) as s:
        k = torch.empty(n, c.n_kv, c.hd, dtype=dtype, device=dev)
        v = torch.empty_like(k)
        check(get_dll().jl_kv4_read(ctypes.byref(c), l, ps, pp, n, k.data_ptr(), v.data_ptr(), _TYPES[dtype], st, s),
              "jl_kv4_read")
    return k, v


def kv4_attention(cache: torch.Tensor, l: int, q: torch.Tensor, slots: torch.Tensor, lens: torch.Tensor,
                  scale: float | None = None, longest: int | None = None, out: torch.Tensor | None = None,
                  status: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Attention of q [B, T, H, hd] (or [B, H, hd]: T = 1; fp32, fp16 or bf16)
    over layer l: query i of sequence b sees the first lens[b] - T + 1 + i
    positions of slot slots[b] (int32 [B] each), its own being the last of
    them. H is a multiple of the cache's n_kv. scale: 1 / sqrt(hd) by default.
    longest: a bound of the lens that the caller knows (by default the cache's
    length); a longer entry counts as outside the cache. Rows that see nothing
    are zero. Returns out, of q's shape and type."""
    c = _view(cache, l)
    dev = cache.device
    if q.dim() not in (3, 4) or q.shape[-1] != c.hd or q.shape[-2] < 1 or q.shape[-2] % c.n_kv:
        raise ValueError(f"kv4_attention: q is [B, T, H, {c.hd}] or [B, H, {c.hd}] with H a multiple of {c.n_kv}, "
                         f"got {tuple(q.shape)}")
    if q.dtype not in _TYPES or q.device != dev:
        raise ValueError(f"kv4_attention: q is fp32, fp16 or bf16 on {dev}")
    B, T, H = q.shape[0], 1 if q.dim() == 3 else q.shape[1], q.shape[-2]
    if T < 1:
        raise ValueError("kv4_attention: T is 1 or more")
    if longest is None:
        longest = 0
    elif not 1 <= longest <= c.maxT:
        raise ValueError(f"kv4_attention: longest {longest} outside [1, {c.maxT}]")
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.device != dev
                            or not out.is_contiguous() or out.data_ptr() % 16):
        raise ValueError("kv4_attention: out is contiguous, 16-byte aligned, of q's shape, type and device")
    ps, pl, st = _index(slots, B, dev, "slots"), _index(lens, B, dev, "lens"), _status(status, dev)
    if scale is None:
        scale = 1.0 / math.sqrt(c.hd)
    L = get_dll()
    with _on(dev, stream) as s:
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        rows = _rows(q if q.dim() == 3 else q.flatten(0, 1))
        n = L.jl_kv4_attn_ws(ctypes.byref(c), B, T, H)
        ws = torch.empty(n, dtype=torch.uint8, device=dev) if n > 0 else None
        check(L.jl_kv4_attn(ctypes.byref(c), l, rows.data_ptr(), _TYPES[q.dtype], rows.stride(0), ps, pl, longest,
                            B, T, H, scale, out.data_ptr(), ws.data_ptr() if ws is not None else None, max(n, 0),
                            st, s), "jl_kv4_attn")
    return out
