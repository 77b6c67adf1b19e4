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

import numpy as np

from . import _lib

_state = None


class _Torch:
    """What the calls need of torch, looked up once."""

    def __init__(self):
        import torch

        self.torch = torch
        self.tag = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
        self.f32, self.i32, self.u8 = torch.float32, torch.int32, torch.uint8
        self.lib = _lib.load()


def _torch() -> _Torch:
    global _state
    if _state is None:
        _state = _Torch()
    return _state


def _device(t, name: str) -> int:
    if not t.is_cuda:
        raise ValueError(f"{name} is on {t.device}, not on a CUDA device")
    return t.device.index


def _stream(T: _Torch, dev: int, stream) -> int:
    return T.torch.cuda.current_stream(dev).cuda_stream if stream is None else int(stream)


def _vector(T: _Torch, t, name: str, n: int, dtype, dev: int) -> int:
    """The pointer of a contiguous [n] tensor of dtype on device dev."""
    if t.dtype != dtype or t.dim() != 1 or t.shape[0] != n or t.device.index != dev or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous [{n}] {dtype} tensor on cuda:{dev}, got "
                         f"{tuple(t.shape)} {t.dtype} on {t.device}")
    return t.data_ptr()


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
    a sequence without keys. The workspace comes from torch's allocator on the
    current stream; with another ``stream`` the caller orders the two."""
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
    for name, t, like, st in (("v_prefix", v_prefix, k_prefix, ps), ("v", v, k, cs), ("k_prefix", k_prefix, k_prefix, ps)):
        if t.shape != like.shape or t.dtype != kt or t.device.index != dev or (t.stride() != st and t.numel()):
            raise ValueError(f"{name} must be {kt} on cuda:{dev} with the shape and strides of its keys, got "
                             f"{tuple(t.shape)} {t.dtype} {t.stride()} on {t.device}")
    if k.device.index != dev or (hd > 1 and (qs[2] != 1 or cs[3] != 1 or (prefix and ps[2] != 1))):
        raise ValueError("q and the caches must be on one device with a contiguous last dimension")
    if q.dtype not in T.tag or kt not in T.tag:
        raise ValueError(f"queries of {q.dtype} with a cache of {kt}")
    if out is None:
        out = T.torch.empty((n, n_head, hd), dtype=q.dtype, device=q.device)
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
    work = T.torch.empty(size, dtype=T.u8, device=q.device)
    os_ = out.stride()
    a = _lib.AttentionSharedArgs(
        dev, T.tag[q.dtype], T.tag[kt], n, n_head, n_kv, hd, prefix, n_slots, rows, q.data_ptr(), qs[0], qs[1],
        k_prefix.data_ptr(), v_prefix.data_ptr(), ps[0], ps[1], k.data_ptr(), v.data_ptr(), cs[0], cs[1], cs[2],
        None if slots is None else _vector(T, slots, "slots", n, T.i32, dev), _vector(T, lens, "lens", n, T.i32, dev),
        out.data_ptr(), os_[0], os_[1], hd ** -0.5 if scale is None else scale)
    _lib.check(T.lib.talos_attention_shared_dev(C.byref(a), work.data_ptr(), size, _stream(T, dev, stream)))
    return out


def sample_dev(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, tokens=None, probs=None, stream=None):
    """talos_sample_dev: the token of each row of ``logits`` ([n, vocab] or [vocab],
    f32 / f16 / bf16, any row stride) for the random numbers ``u`` ([n] f32 in
    [0, 1)). The settings are numbers, or [n] tensors (f32; top_k int32) with one
    value per row; ``temperature`` 0 is the greedy choice (the lowest index of
    equal logits), ``top_k`` 0, ``top_p`` 1 and ``min_p`` 0 keep everything.
    Returns (tokens int32, probs f32), written into ``tokens`` / ``probs`` if given;
    a row with nothing above -inf gives -1."""
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
    a = _lib.SampleArgs(dev, tag, n, vocab, logits.data_ptr(), logits.stride(0), _vector(T, u, "u", n, T.f32, dev))
    if isinstance(temperature, (int, float)):
        a.temperature = temperature
    else:
        a.temperature_dev = _vector(T, temperature, "temperature", n, T.f32, dev)
    if isinstance(top_k, int):
        a.top_k = top_k
    else:
        a.top_k_dev = _vector(T, top_k, "top_k", n, T.i32, dev)
    if isinstance(top_p, (int, float)):
        a.top_p = top_p
    else:
        a.top_p_dev = _vector(T, top_p, "top_p", n, T.f32, dev)
    if isinstance(min_p, (int, float)):
        a.min_p = min_p
    else:
        a.min_p_dev = _vector(T, min_p, "min_p", n, T.f32, dev)
    if tokens is None:
        tokens = T.torch.empty(n, dtype=T.i32, device=logits.device)
    if probs is None:
        probs = T.torch.empty(n, dtype=T.f32, device=logits.device)
    a.tokens = _vector(T, tokens, "tokens", n, T.i32, dev)
    a.probs = _vector(T, probs, "probs", n, T.f32, dev)
    _lib.check(T.lib.talos_sample_dev(C.byref(a), _stream(T, dev, stream)))
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
    base = (C.c_void_p * len(caches))()
    for i, c in enumerate(caches):
        if c.shape != shape or c.stride() != strides or c.dtype != dtype or not c.is_cuda or c.device.index != dev:
            raise ValueError(f"caches[{i}] differs from caches[0] in shape, strides, dtype or device")
        base[i] = c.data_ptr()
    n = len(src)
    if len(dst) != n or len(lens) != n or (starts is not None and len(starts) != n):
        raise ValueError("src, dst, lens and starts differ in length")
    m = (C.c_uint32 * (4 * n))()
    m[0::4], m[1::4], m[3::4] = src, dst, lens
    if starts is not None:
        m[2::4] = starts
    if n and (min(src) < 0 or min(dst) < 0 or min(lens) < 0 or (starts is not None and min(starts) < 0)):
        raise ValueError("negative slot, start or length")
    es = first.element_size()
    g = _lib.KvSlots(dev, len(caches), C.addressof(base), shape[0], shape[1], shape[2], strides[0] * es,
                     strides[1] * es, strides[2] * es, width * es)
    _lib.check(T.lib.talos_kv_move_dev(C.byref(g), m, n, _stream(T, dev, stream)))
