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
``status`` (an int32 CUDA tensor of one element) when one is given. A wait inside
an attention kernel that runs out (about 2 s, where microseconds are due) leaves
the output undefined: it sets bit 1 of ``status``, and without one the next
``kv4_check`` raises.
"""
from __future__ import annotations

import ctypes
import math

import torch

from joule_b200.native import BF16, F16, F32, Kv4, check, get_dll

__all__ = ["KV4_BLOCK", "KV4_TIMEOUT", "KV4_BAD_INDEX", "kv4_cache", "kv4_append", "kv4_read", "kv4_attention",
           "kv4_check"]

KV4_BLOCK = 64      # positions per block
KV4_TIMEOUT = 1     # status bit: a wait inside a kernel ran out, the output is not valid
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


_raw_stream = torch._C._cuda_getCurrentRawStream  # the current stream's handle without a Stream object
_current_device = torch._C._cuda_getDevice


class _Interpreted:
    """In place of the compiled calls where this interpreter has none: nothing is regular."""
    bind = append = read = attention = staticmethod(lambda *a: None)


_call = None  # the compiled form of regular calls (csrc/kv4_call.c), bound at the first one
_dll = None


def _bind() -> None:
    global _call, _dll
    dll = get_dll()
    try:
        from joule_b200 import _kv4_call
    except ImportError:  # built for another Python: the functions below do all of it, some microseconds slower
        _kv4_call = _Interpreted
    entries = [ctypes.cast(f, ctypes.c_void_p).value
               for f in (dll.jl_kv4_append, dll.jl_kv4_read, dll.jl_kv4_attn, dll.jl_kv4_attn_ws)]
    _kv4_call.bind(torch.uint8, torch.int32, torch.float32, torch.float16, torch.bfloat16, torch.empty_like,
                   _current_device, _raw_stream, *entries)
    _dll, _call = dll, _kv4_call


def _view(cache: torch.Tensor, l: int) -> tuple[Kv4, int]:
    """The cache as the library takes it, and its device's index."""
    shape = cache.shape
    dev = cache.get_device()
    if len(shape) != 5 or cache.dtype is not torch.uint8 or dev < 0 or not cache.is_contiguous():
        raise ValueError("kv4: the cache is a contiguous uint8 CUDA tensor [slots, L, n_kv, blocks, 68 * hd]")
    slots, L, kh, nb, size = shape
    if size != 68 * 64 and size != 68 * 128 or not slots or not kh or not nb:
        raise ValueError(f"kv4: block size {size} is not 68 * hd with hd 64 or 128, or the cache is empty")
    if not 0 <= l < L:
        raise ValueError(f"kv4: layer {l} outside [0, {L})")
    return Kv4(cache.data_ptr(), slots, L, kh, size // 68, nb * KV4_BLOCK), dev


def _indices(slots: torch.Tensor, t: torch.Tensor, n: int, dev: int, name: str) -> tuple[int, int]:
    """Addresses of slots and of t (positions or lens)."""
    if slots.dtype is not torch.int32 or slots.get_device() != dev or slots.shape != (n,) or not slots.is_contiguous():
        raise ValueError(f"kv4: slots is a contiguous int32 tensor [{n}] on cuda:{dev}")
    if t.dtype is not torch.int32 or t.get_device() != dev or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"kv4: {name} is a contiguous int32 tensor [{n}] on cuda:{dev}")
    return slots.data_ptr(), t.data_ptr()


def _status(t: torch.Tensor, dev: int) -> int:
    if t.dtype is not torch.int32 or t.get_device() != dev or t.numel() < 1:
        raise ValueError(f"kv4: status is an int32 tensor on cuda:{dev}")
    return t.data_ptr()


def _aligned(t: torch.Tensor) -> torch.Tensor:
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _rows(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """t [rows, heads, hd] with its row stride, when whole rows lie at a 16-byte aligned stride; else a copy."""
    n, h, d = t.shape
    sn, sh, sd = t.stride()
    if sd == 1 and (sh == d or h == 1) and (n <= 1 or sn >= h * d and sn * t.element_size() % 16 == 0) \
            and t.data_ptr() % 16 == 0:
        return t, sn if n > 1 else h * d
    return _aligned(t), h * d


def _other(dev: int, stream) -> torch.cuda.Stream:
    """A stream given by the caller, or the current one of a device that is not
    current: to be made current for the call, so that what the call allocates
    belongs to it."""
    device = torch.device("cuda", dev)
    if stream is None:
        return torch.cuda.current_stream(device)
    if not isinstance(stream, torch.cuda.Stream):
        return torch.cuda.ExternalStream(int(stream), device=device)
    if stream.device != device:
        raise ValueError(f"kv4: the stream is on {stream.device}, the cache on {device}")
    return stream


def kv4_append(cache: torch.Tensor, l: int, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor,
               positions: torch.Tensor, status: torch.Tensor | None = None, stream=None) -> None:
    """Quantise k, v [N, n_kv, hd] (fp32, fp16 or bf16; rows of any stride)
    into positions[n] of slot slots[n] (int32 [N], distinct pairs) of layer l."""
    if _call is None:
        _bind()
    if status is None and stream is None:
        code = _call.append(cache, l, k, v, slots, positions)
        if code is not None:
            return check(code, "jl_kv4_append") if code else None
    c, dev = _view(cache, l)
    shape = k.shape
    if shape != v.shape or len(shape) != 3 or shape[1] != c.n_kv or shape[2] != c.hd:
        raise ValueError(f"kv4_append: k and v are [N, {c.n_kv}, {c.hd}], got {tuple(k.shape)} and {tuple(v.shape)}")
    kind = _TYPES.get(k.dtype)
    if kind is None or v.dtype is not k.dtype or k.get_device() != dev or v.get_device() != dev:
        raise ValueError(f"kv4_append: k and v are fp32, fp16 or bf16, of one type, on cuda:{dev}")
    n = shape[0]
    ps, pp = _indices(slots, positions, n, dev, "positions")
    st = None if status is None else _status(status, dev)
    if stream is not None or _current_device() != dev:
        with torch.cuda.stream(_other(dev, stream)):
            return kv4_append(cache, l, k, v, slots, positions, status)
    k, sk = _rows(k)
    v, sv = _rows(v)
    check(_dll.jl_kv4_append(c, l, k.data_ptr(), v.data_ptr(), kind, sk, sv, ps, pp, n, st, _raw_stream(dev)), "jl_kv4_append")


def kv4_read(cache: torch.Tensor, l: int, slots: torch.Tensor, positions: torch.Tensor,
             dtype: torch.dtype = torch.float32, status: torch.Tensor | None = None,
             stream=None) -> tuple[torch.Tensor, torch.Tensor]:
    """The cached keys and values [N, n_kv, hd] of (slots[n], positions[n])."""
    if _call is None:
        _bind()
    if status is None and stream is None:
        done = _call.read(cache, l, slots, positions, dtype)
        if done is not None:
            code, k, v = done
            if code:
                check(code, "jl_kv4_read")
            return k, v
    c, dev = _view(cache, l)
    kind = _TYPES.get(dtype)
    if kind is None:
        raise ValueError(f"kv4_read: dtype is fp32, fp16 or bf16, got {dtype}")
    n = slots.numel()
    ps, pp = _indices(slots, positions, n, dev, "positions")
    st = None if status is None else _status(status, dev)
    if stream is not None or _current_device() != dev:
        with torch.cuda.stream(_other(dev, stream)):
            return kv4_read(cache, l, slots, positions, dtype, status)
    k = torch.empty(n, c.n_kv, c.hd, dtype=dtype, device=cache.device)
    v = torch.empty_like(k)
    check(_dll.jl_kv4_read(c, l, ps, pp, n, k.data_ptr(), v.data_ptr(), kind, st, _raw_stream(dev)), "jl_kv4_read")
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
    are zero. Returns out, of q's shape and type; one that is given does not
    overlap q (JouleError)."""
    if _call is None:
        _bind()
    if out is None and status is None and stream is None:
        done = _call.attention(cache, l, q, slots, lens, scale, longest)
        if done is not None:
            code, out = done
            if code:
                check(code, "jl_kv4_attn")
            return out
    c, dev = _view(cache, l)
    shape = q.shape
    hd, dims = c.hd, len(shape)
    B, T, H, d = shape if dims == 4 else (shape[0], 1, *shape[1:]) if dims == 3 else (0, 1, 0, 0)
    if d != hd or H < 1 or H % c.n_kv:
        raise ValueError(f"kv4_attention: q is [B, T, H, {hd}] or [B, H, {hd}] with H a multiple of {c.n_kv}, "
                         f"got {tuple(q.shape)}")
    kind = _TYPES.get(q.dtype)
    if kind is None or q.get_device() != dev:
        raise ValueError(f"kv4_attention: q is fp32, fp16 or bf16 on cuda:{dev}")
    if T < 1:
        raise ValueError("kv4_attention: T is 1 or more")
    if longest is None:
        longest = 0
    elif not 1 <= longest <= c.maxT:
        raise ValueError(f"kv4_attention: longest {longest} outside [1, {c.maxT}]")
    if out is not None and (out.shape != shape or out.dtype is not q.dtype or out.get_device() != dev
                            or not out.is_contiguous() or out.data_ptr() % 16):
        raise ValueError("kv4_attention: out is contiguous, 16-byte aligned, of q's shape, type and device")
    ps, pl = _indices(slots, lens, B, dev, "lens")
    st = None if status is None else _status(status, dev)
    if stream is not None or _current_device() != dev:
        with torch.cuda.stream(_other(dev, stream)):
            return kv4_attention(cache, l, q, slots, lens, scale, longest or None, out, status)
    row, rows, pq = H * hd, q, q.data_ptr()
    if q.is_contiguous() and pq % 16 == 0:
        if out is None:
            out = torch.empty_like(q)
    elif dims == 3:
        rows, row = _rows(q)
    else:  # one stride between all rows, or a copy
        s = q.stride()
        if B == 1 or T == 1 or s[0] == T * s[1]:
            rows, row = _rows(q.as_strided((B * T, H, hd), (s[1] if T > 1 else s[0], s[2], s[3])))
        else:
            rows = _aligned(q)
    if rows is not q:
        pq = rows.data_ptr()
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    n = max(0, _dll.jl_kv4_attn_ws(c, B, T, H, longest))
    ws = torch.empty(n, dtype=torch.uint8, device=cache.device) if n else None
    check(_dll.jl_kv4_attn(c, l, pq, kind, row, ps, pl, longest, B, T, H, 1.0 / math.sqrt(hd) if scale is None else scale,
                           out.data_ptr(), ws.data_ptr() if n else None, n, st, _raw_stream(dev)), "jl_kv4_attn")
    return out


def kv4_check(device=None, stream=None) -> None:
    """Wait for the stream (the current one of `device`, the current CUDA device by
    default) and raise JouleError when a wait inside a kv4_attention call without
    `status` on the device has run out since the last check."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    if device.type != "cuda":
        raise ValueError(f"kv4_check: a CUDA device, got {device}")
    with torch.cuda.device(device):
        s = torch.cuda.current_stream() if stream is None else _other(torch.cuda.current_device(), stream)
        check(get_dll().jl_kv4_check(s.cuda_stream), "jl_kv4_check")
