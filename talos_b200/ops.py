"""Device operators for many sequences that start from one prompt, on torch CUDA
tensors: attention over a prefix that they share (``attention_shared_dev``), the
choice of tokens (``sample_dev``) and moves of rows between cache slots
(``kv_move_dev``).

Each call checks its tensors, enqueues the work on the tensors' device (on the
current stream there unless ``stream`` gives a cudaStream_t) and returns without
waiting. The compute runs in libtalos_cuda.so through the C ABI of
include/talos_cuda.h; torch only holds the memory, and is imported by the first
call, not by the package.
"""
from __future__ import annotations

import ctypes as C
import struct
from array import array
from numbers import Integral, Real

import numpy as np

from . import _lib

_state = None

# The argument structs of the C ABI (native layout), packed at once: a ctypes Structure of
# 27 fields takes 3 us to fill, a tenth of the smallest call.
_ATTENTION = struct.Struct("@3i7IP2N2P2N2P3N2PP2Nf0P")
_SLOTS = struct.Struct("@2iP3I4N0P")
_SAMPLE = struct.Struct("@2i2IPN5Pfiff2P")
assert _ATTENTION.size == C.sizeof(_lib.AttentionSharedArgs) and _SAMPLE.size == C.sizeof(_lib.SampleArgs)


class _Torch:
    """What the calls need of torch, looked up once."""

    def __init__(self):
        import torch

        self.torch = torch
        self.tag = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
        self.f32, self.i32, self.u8 = torch.float32, torch.int32, torch.uint8
        self.lib = _lib.load()
        # the handle of the current stream; through the Stream object it takes 2 us
        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        self.stream = raw or (lambda dev: torch.cuda.current_stream(dev).cuda_stream)


def _torch() -> _Torch:
    global _state
    if _state is None:
        _state = _Torch()
    return _state


def _device(t, name: str) -> int:
    dev = t.get_device()
    if dev < 0:
        raise ValueError(f"{name} is on {t.device}, not on a CUDA device")
    return dev


def _stream(T: _Torch, dev: int, stream) -> int:
    return T.stream(dev) if stream is None else int(stream)


def _empty(T: _Torch, dev: int, stream, like, shape, dtype):
    """A new tensor on like's device for work on ``stream``. With another stream than the
    current one it comes from torch's memory for that stream, so that what is released while
    the work is in flight goes to later work behind it, and its release waits for what the
    current stream has done with it."""
    if stream is None or int(stream) == T.stream(dev):
        return like.new_empty(shape, dtype=dtype)
    cuda = T.torch.cuda
    current = cuda.current_stream(dev)
    handle = int(stream)
    with cuda.stream(cuda.ExternalStream(0 if handle == 1 else handle, device=dev)):  # (1: cudaStreamLegacy)
        new = like.new_empty(shape, dtype=dtype)
    new.record_stream(current)
    return new


def _pack(s: struct.Struct, *values) -> bytes:
    try:
        return s.pack(*values)
    except (struct.error, OverflowError) as e:
        raise ValueError(f"a number that its argument cannot hold: {e}") from None


def _vector(T: _Torch, t, name: str, n: int, dtype, dev: int) -> int:
    """The pointer of a contiguous [n] tensor of dtype on device dev."""
    if t.dtype is not dtype or t.shape != (n,) or t.get_device() != dev or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous [{n}] {dtype} tensor on cuda:{dev}, got "
                         f"{tuple(t.shape)} {t.dtype} on {t.device}")
    return t.data_ptr()


def _setting(T: _Torch, x, name: str, n: int, dtype, dev: int, kind):
    """(pointer, number) of a setting that is no plain Python number: a tensor with a value per
    row, or a number of another kind (numpy's, say)."""
    if isinstance(x, T.torch.Tensor):
        return _vector(T, x, name, n, dtype, dev), 0
    if isinstance(x, kind):
        return 0, x
    raise ValueError(f"{name} must be a number or a [{n}] {dtype} tensor, got {x!r}")


_work_bytes: dict[tuple[int, int, int, int], int] = {}  # of talos_attention_shared_work


def attention_shared_dev(q, k_prefix, v_prefix, k, v, slots, lens, out=None, scale=None, stream=None):
    """talos_attention_shared_dev: attention of n sequences over a prefix they share
    and a suffix of each one's own. ``q`` [n, n_head, head_dim]; ``k_prefix`` /
    ``v_prefix`` [prefix, n_head_kv, head_dim] (prefix 0: an empty tensor); ``k`` /
    ``v`` [n_slots, rows, n_head_kv, head_dim], of which sequence i attends to rows
    0 .. lens[i] - 1 of slot slots[i] (``slots`` None: slot i); ``slots`` and
    ``lens`` int32 on the device. f32 queries go with f32 or f16 caches, f16 and
    bf16 with their own; the last dimension is contiguous. ``scale`` None is
    1 / sqrt(head_dim). Returns ``out`` ([n, n_head, head_dim], q's type): zeros for
    a sequence without keys. An infinite or NaN value in an attended row makes its
    dimension of the output infinite or NaN; keys are finite; an element of an f32
    cache keeps 22 bits, or 2^-39 of the largest among the 64 rows of its tile. With
    another ``stream`` than the current one, the workspace and a new ``out`` belong
    to that stream, and the caller orders the inputs before it and what reads
    ``out`` behind it."""
    T = _torch()
    dev = _device(q, "q")
    if q.dim() != 3 or k.dim() != 4 or k_prefix.dim() != 3:
        raise ValueError("q is [n, n_head, head_dim], a prefix [prefix, n_head_kv, head_dim], a cache [n_slots, rows, "
                         f"n_head_kv, head_dim], got {tuple(q.shape)}, {tuple(k_prefix.shape)}, {tuple(k.shape)}")
    n, n_head, hd = q.shape
    prefix, (n_slots, rows, n_kv, _) = k_prefix.shape[0], k.shape
    if k.shape[3] != hd or k_prefix.shape[1] != n_kv or k_prefix.shape[2] != hd:
        raise ValueError(f"q {tuple(q.shape)}, prefix {tuple(k_prefix.shape)} and cache {tuple(k.shape)} do not match")
    kt, qs, ps, cs = k.dtype, q.stride(), k_prefix.stride(), k.stride()
    if not (v.shape == k.shape and v_prefix.shape == k_prefix.shape and v.dtype is kt and k_prefix.dtype is kt
            and v_prefix.dtype is kt and v.get_device() == dev == k_prefix.get_device() == v_prefix.get_device()
            and (v.stride() == cs or not v.numel()) and (v_prefix.stride() == ps or not prefix)):
        for name, t, like in (("v_prefix", v_prefix, k_prefix), ("v", v, k), ("k_prefix", k_prefix, k_prefix)):
            if (t.shape != like.shape or t.dtype != kt or t.get_device() != dev
                    or (t.stride() != like.stride() and t.numel())):
                raise ValueError(f"{name} must be {kt} on cuda:{dev} with the shape and strides of its keys, got "
                                 f"{tuple(t.shape)} {t.dtype} {t.stride()} on {t.device}")
    if k.get_device() != dev or (hd > 1 and (qs[2] != 1 or cs[3] != 1 or (prefix and ps[2] != 1))):
        raise ValueError("q and the caches must be on one device with a contiguous last dimension")
    if q.dtype not in T.tag or kt not in T.tag:
        raise ValueError(f"queries of {q.dtype} with a cache of {kt}")
    if out is None:
        out = _empty(T, dev, stream, q, (n, n_head, hd), q.dtype)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or (hd > 1 and out.stride(2) != 1):
        raise ValueError(f"out must be {tuple(q.shape)} {q.dtype} on {q.device} with a contiguous last dimension")
    if n == 0:
        return out
    key = (dev, n, n_head, n_kv)
    size = _work_bytes.get(key)
    if size is None:
        need = C.c_size_t()
        _lib.check(T.lib.talos_attention_shared_work(dev, n, n_head, n_kv, C.byref(need)))
        size = _work_bytes[key] = need.value
    work = _empty(T, dev, stream, q, size, T.u8)
    os_ = out.stride()
    a = _pack(
        _ATTENTION, dev, T.tag[q.dtype], T.tag[kt], n, n_head, n_kv, hd, prefix, n_slots, rows, q.data_ptr(), qs[0], qs[1],
        k_prefix.data_ptr(), v_prefix.data_ptr(), ps[0], ps[1], k.data_ptr(), v.data_ptr(), cs[0], cs[1], cs[2],
        0 if slots is None else _vector(T, slots, "slots", n, T.i32, dev), _vector(T, lens, "lens", n, T.i32, dev),
        out.data_ptr(), os_[0], os_[1], hd ** -0.5 if scale is None else scale)
    _lib.check(T.lib.talos_attention_shared_dev(a, work.data_ptr(), size, _stream(T, dev, stream)))
    return out


def sample_dev(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, tokens=None, probs=None, stream=None):
    """talos_sample_dev: the token of each row of ``logits`` ([n, vocab] or [vocab],
    f32 / f16 / bf16, rows any stride of at least vocab apart) for the random numbers ``u`` ([n] f32 in
    [0, 1)). The settings are numbers, or [n] tensors (f32; top_k int32) with one
    value per row; ``temperature`` 0 is the greedy choice (the lowest index of
    equal logits), ``top_k`` 0, ``top_p`` 1 and ``min_p`` 0 keep everything.
    Returns (tokens int32, probs f32), written into ``tokens`` / ``probs`` if given;
    a row with nothing above -inf gives -1. With another ``stream`` than the current
    one, new ones belong to that stream, and the caller orders the inputs before it
    and what reads them behind it."""
    T = _torch()
    dev = _device(logits, "logits")
    tag = T.tag.get(logits.dtype)
    if tag is None:
        raise ValueError(f"logits of {logits.dtype} (f32, f16 or bf16)")
    if logits.dim() == 1:
        logits = logits[None]
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError(f"logits must be [n, vocab] with neighbouring logits of a row adjacent, got "
                         f"{tuple(logits.shape)} with strides {logits.stride()}")
    n, vocab = logits.shape
    if tokens is None:
        tokens = _empty(T, dev, stream, logits, n, T.i32)
    if probs is None:
        probs = _empty(T, dev, stream, logits, n, T.f32)
    td = kd = pd = md = 0
    if not isinstance(temperature, (int, float)):
        td, temperature = _setting(T, temperature, "temperature", n, T.f32, dev, Real)
    if not isinstance(top_k, int):
        kd, top_k = _setting(T, top_k, "top_k", n, T.i32, dev, Integral)
    if not isinstance(top_p, (int, float)):
        pd, top_p = _setting(T, top_p, "top_p", n, T.f32, dev, Real)
    if not isinstance(min_p, (int, float)):
        md, min_p = _setting(T, min_p, "min_p", n, T.f32, dev, Real)
    a = _pack(_SAMPLE, dev, tag, n, vocab, logits.data_ptr(), logits.stride(0), _vector(T, u, "u", n, T.f32, dev), td,
              kd, pd, md, temperature, top_k, top_p, min_p, _vector(T, tokens, "tokens", n, T.i32, dev),
              _vector(T, probs, "probs", n, T.f32, dev))
    _lib.check(T.lib.talos_sample_dev(a, _stream(T, dev, stream)))
    return tokens, probs


def sample(logits, u: float, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0,
           min_p: float = 0.0) -> int:
    """talos_sample: the token of one row of host logits for the random number
    ``u`` in [0, 1) (src/sample.rs:19-76 with min-p besides)."""
    v = np.ascontiguousarray(logits, np.float32)
    out = C.c_uint32()
    _lib.check(_lib.load().talos_sample(v.ctypes.data, v.size, u, temperature, top_k, top_p, min_p, C.byref(out),
                                        None))
    return int(out.value)


def kv_move_dev(caches, src, dst, lens, starts=None, stream=None) -> None:
    """talos_kv_move_dev: for every i, rows starts[i] .. starts[i] + lens[i] - 1
    (starts: 0) of slot src[i] become those rows of slot dst[i], in each tensor of
    ``caches`` (one or several of one shape, dtype and strides: [slots, layers,
    rows, ...], the dimensions of a row contiguous). All moves read what was there
    before the call; src, dst, lens and starts are host integers."""
    T = _torch()
    first = caches[0]
    dev = _device(first, "caches[0]")
    shape, strides, dtype = first.shape, first.stride(), first.dtype
    if len(shape) < 4:
        raise ValueError(f"a cache is [slots, layers, rows, ...], got {tuple(shape)}")
    width = 1
    for size, step in zip(reversed(shape[3:]), reversed(strides[3:])):
        if size > 1 and step != width:
            raise ValueError(f"the dimensions of a row must be contiguous, got {tuple(shape)} with strides {strides}")
        width *= size
    base = array("Q")
    i = 0
    for c in caches:
        if c.shape != shape or c.stride() != strides or c.dtype is not dtype or c.get_device() != dev:
            raise ValueError(f"caches[{i}] differs from caches[0] in shape, strides, dtype or device")
        base.append(c.data_ptr())
        i += 1
    n = len(src)
    if len(dst) != n or len(lens) != n or (starts is not None and len(starts) != n):
        raise ValueError("src, dst, lens and starts differ in length")
    try:
        m = array("I", [x for move in zip(src, dst, (0,) * n if starts is None else starts, lens) for x in move])
    except OverflowError:
        raise ValueError("negative slot, start or length") from None
    es = first.element_size()
    g = _pack(_SLOTS, dev, len(base), base.buffer_info()[0], shape[0], shape[1], shape[2], strides[0] * es,
              strides[1] * es, strides[2] * es, width * es)
    _lib.check(T.lib.talos_kv_move_dev(g, m.buffer_info()[0], n, _stream(T, dev, stream)))
