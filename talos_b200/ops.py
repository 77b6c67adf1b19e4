"""Device operators for many sequences that start from one prompt, on torch CUDA
tensors: the choice of tokens (``sample_dev``) and moves of rows between cache
slots (``kv_move_dev``).

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
        self.f32, self.i32 = torch.float32, torch.int32
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
