"""Arguments of the batch operators that are refused before any GPU work, and
the plan of a call's moves (no GPU needed)."""
import ctypes as C

import numpy as np
import pytest

import talos_b200
from talos_b200 import _lib, build


@pytest.fixture(scope="module")
def lib():
    build.build_cuda()
    return _lib.load()


def sample_args(**kw):
    a = _lib.SampleArgs(0, 0, 2, 100, 256, 100, 256)
    a.tokens = 256
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_sample_refusals(lib):
    assert lib.talos_sample_dev(None, None) == _lib.INVALID_ARG
    assert lib.talos_sample_dev(C.byref(sample_args(n=0)), None) == _lib.OK
    assert lib.talos_sample_dev(C.byref(sample_args(type=2)), None) == _lib.UNSUPPORTED
    for kw in (dict(logits=None), dict(u=None), dict(tokens=None), dict(vocab=0), dict(vocab=(1 << 20) + 1),
               dict(row_stride=99), dict(top_k=-1), dict(logits=258), dict(probs=1), dict(top_k_dev=2),
               dict(n=(1 << 24) + 1)):
        assert lib.talos_sample_dev(C.byref(sample_args(**kw)), None) == _lib.INVALID_ARG, kw
    out, v = C.c_uint32(), np.zeros(4, np.float32)
    assert lib.talos_sample(None, 4, 0.5, 1.0, 0, 1.0, 0.0, C.byref(out), None) == _lib.INVALID_ARG
    assert lib.talos_sample(v.ctypes.data, 0, 0.5, 1.0, 0, 1.0, 0.0, C.byref(out), None) == _lib.INVALID_ARG
    assert lib.talos_sample(v.ctypes.data, 4, 0.5, 1.0, -1, 1.0, 0.0, C.byref(out), None) == _lib.INVALID_ARG
    assert lib.talos_sample(v.ctypes.data, 4, 0.5, 1.0, 0, 1.0, 0.0, None, None) == _lib.INVALID_ARG


def attention(lib, work=4096, work_bytes=1 << 30, **kw):
    """A call of 3 sequences, 4 heads over 2 of 64, a prefix of 8, 5 slots of 16 rows."""
    a = _lib.AttentionSharedArgs(
        0, 0, 0, 3, 4, 2, 64, 8, 5, 16, 4096, 256, 64, 4096, 4096, 128, 64, 4096, 4096, 2048, 128, 64, None, 4096, 4096,
        256, 64, 0.125)
    for k, v in kw.items():
        setattr(a, k, v)
    return lib.talos_attention_shared_dev(C.byref(a), work, work_bytes, None)


def test_attention_refusals(lib):
    n = C.c_size_t()
    assert lib.talos_attention_shared_work(0, 3, 4, 2, None) == _lib.INVALID_ARG
    for args in ((0, 4, 2), (1025, 4, 2), (3, 4, 0), (3, 0, 2), (3, 5, 2), (3, 258, 2)):
        assert lib.talos_attention_shared_work(0, *args, C.byref(n)) == _lib.INVALID_ARG, args
    assert lib.talos_attention_shared_work(0, 3, 4, 2, C.byref(n)) == _lib.OK and n.value > 0
    assert attention(lib, work_bytes=n.value - 1) == _lib.INVALID_ARG
    assert lib.talos_attention_shared_dev(None, 4096, 1 << 30, None) == _lib.INVALID_ARG
    assert attention(lib, n=0) == _lib.OK
    for kw in (dict(q_type=30), dict(q_type=1), dict(kv_type=30), dict(kv_type=2), dict(q_type=1, kv_type=30),
               dict(head_dim=0), dict(head_dim=132), dict(head_dim=62), dict(head_dim=60, kv_type=1),
               dict(prefix_len=0x40000000), dict(slot_len=0x40000000)):
        assert attention(lib, **kw) == _lib.UNSUPPORTED, kw
    for kw in (dict(work=None), dict(work=4100), dict(q=None), dict(out=None), dict(lens=None), dict(k_prefix=None),
               dict(v_prefix=None), dict(k=None), dict(v=None), dict(n_slots=0), dict(scale=0.0), dict(scale=float("nan")),
               dict(scale=1e31), dict(scale=-1.0), dict(q=4100), dict(k=4104), dict(v_prefix=4100), dict(out=4100),
               dict(lens=4097), dict(slots=4098), dict(q_stride_h=65), dict(prefix_stride_t=126), dict(slot_stride=2046),
               dict(out_stride_n=257), dict(n_head=5), dict(n_head_kv=0), dict(n=1025),
               dict(out_stride_h=0), dict(out_stride_n=0), dict(out_stride_h=32), dict(out_stride_n=128),
               dict(out_stride_n=64, out_stride_h=128), dict(out_stride_n=64, out_stride_h=64)):
        assert attention(lib, **kw) == _lib.INVALID_ARG, kw


def move(lib, moves, n_slots=4, n_rows=8, bases=(256, 4096), **kw):
    base = (C.c_void_p * max(len(bases), 1))(*bases)
    g = _lib.KvSlots(0, len(bases), C.addressof(base), n_slots, 1, n_rows, 64 * n_rows, 64 * n_rows * n_slots, 64, 64)
    for k, v in kw.items():
        setattr(g, k, v)
    m = (C.c_uint32 * (4 * len(moves)))(*[x for y in moves for x in y])
    return lib.talos_kv_move_dev(C.byref(g), m, len(moves), None)


def test_move_refusals(lib):
    assert lib.talos_kv_move_dev(None, None, 0, None) == _lib.INVALID_ARG
    assert move(lib, []) == _lib.OK
    assert move(lib, [(1, 1, 0, 8), (0, 2, 3, 0)]) == _lib.OK  # nothing to do
    for moves in ([(4, 0, 0, 1)], [(0, 4, 0, 1)], [(0, 1, 0, 9)], [(0, 1, 8, 1)], [(0, 1, 0xffffffff, 2)],
                  [(0, 2, 0, 1), (1, 2, 4, 1)], [(0, 1, 0, 1)] * 513):
        assert move(lib, moves) == _lib.INVALID_ARG, moves[:2]
    one = [(0, 1, 0, 1)]
    for kw in (dict(bases=()), dict(bases=(256, 256)), dict(bases=(256, 0)), dict(bases=tuple(range(256, 256 * 10, 256))),
               dict(row_stride=63), dict(slot_stride=63 * 8), dict(row_bytes=0), dict(n_outer=0),
               dict(n_outer=2, outer_stride=64), dict(base=None)):
        assert move(lib, one, **kw) == _lib.INVALID_ARG, kw
    m = (C.c_uint32 * 4)(0, 1, 0, 1)
    base = (C.c_void_p * 1)(256)
    g = _lib.KvSlots(0, 1, C.addressof(base), 4, 1, 8, 512, 2048, 64, 64)
    assert lib.talos_kv_move_dev(C.byref(g), None, 1, None) == _lib.INVALID_ARG
    assert lib.talos_kv_move_dev(C.byref(g), m, 0, None) == _lib.OK


def test_python_checks_without_a_gpu():
    torch = pytest.importorskip("torch")
    x = torch.zeros(2, 5)
    with pytest.raises(ValueError, match="CUDA"):
        talos_b200.sample_dev(x, torch.zeros(2))
    with pytest.raises(ValueError, match="CUDA"):
        talos_b200.kv_move_dev([torch.zeros(2, 1, 4, 4)], [0], [1], [1])
    with pytest.raises(ValueError, match="CUDA"):
        talos_b200.attention_shared_dev(torch.zeros(2, 2, 8), *[torch.zeros(4, 1, 8)] * 2, *[torch.zeros(2, 4, 1, 8)] * 2,
                                        None, torch.zeros(2, dtype=torch.int32))


def test_packed_arguments_have_the_structs_layout():
    from talos_b200 import ops

    for packed, struct_ in ((ops._ATTENTION, _lib.AttentionSharedArgs), (ops._SAMPLE, _lib.SampleArgs),
                            (ops._SLOTS, _lib.KvSlots)):
        fields = [name for name, _ in struct_._fields_]
        got = struct_.from_buffer_copy(packed.pack(*range(1, len(fields) + 1)))
        assert [int(getattr(got, name)) for name in fields] == list(range(1, len(fields) + 1))


def test_attention_sizes_beyond_the_kernels_counts(lib):
    """Row tiles times key tiles, and heads, that 32-bit counts do not hold."""
    wide = dict(n=1024, n_head=128, n_head_kv=1, out_stride_n=128 * 64)
    assert attention(lib, prefix_len=1 << 27, **wide) == _lib.UNSUPPORTED
    assert attention(lib, slot_len=1 << 27, **wide) == _lib.UNSUPPORTED
    for n, heads in ((128, 1 << 17), (1, 1 << 24)):
        kw = dict(n=n, n_head=heads, n_head_kv=heads, prefix_len=0, out_stride_n=heads * 64)
        assert attention(lib, **kw) == _lib.UNSUPPORTED


def test_move_arrays_that_overlap(lib):
    """Two arrays whose rows coincide in part are refused, interleaved ones are not: compared
    with the rows' bytes one by one."""
    def geometry(dims, row_bytes, off):
        (n_rows, row_stride), (n_outer, outer_stride), (n_slots, slot_stride) = dims
        base = (C.c_void_p * 2)(1 << 20, (1 << 20) + off)
        g = _lib.KvSlots(0, 2, C.addressof(base), n_slots, n_outer, n_rows, slot_stride, outer_stride, row_stride,
                         row_bytes)
        return lib.talos_kv_move_dev(C.byref(g), None, 0, None)

    dims = ((8, 64), (2, 512), (4, 1024))
    for off in (64, -64, 32, 512, 1024, 1024 + 64, -3 * 1024 - 512, 4096 - 64):
        assert geometry(dims, 64, off) == _lib.INVALID_ARG, off
    assert geometry(dims, 64, 4096) == geometry(dims, 64, -4096) == _lib.OK
    wide = ((8, 128), (2, 1024), (4, 2048))  # K and V rows in turn
    assert geometry(wide, 64, 64) == geometry(wide, 64, -64) == _lib.OK
    assert geometry(wide, 64, 63) == geometry(wide, 64, 65) == _lib.INVALID_ARG

    rng = np.random.default_rng(0)
    seen = set()
    for _ in range(2000):
        row_bytes = int(rng.integers(1, 5))
        span, dims = row_bytes, []
        for _ in range(3):
            count = int(rng.integers(1, 4))
            stride = span + int(rng.integers(0, 12))
            dims.append((count, stride))
            span += stride * (count - 1)
        dims = [dims[i] for i in rng.permutation(3)]
        at = {a * dims[0][1] + b * dims[1][1] + c * dims[2][1] + x for a in range(dims[0][0]) for b in range(dims[1][0])
              for c in range(dims[2][0]) for x in range(row_bytes)}
        off = int(rng.integers(1, span + 5)) * (1 if rng.random() < 0.5 else -1)
        want = _lib.INVALID_ARG if any(x + off in at for x in at) else _lib.OK
        assert geometry(dims, row_bytes, off) == want, (dims, row_bytes, off)
        seen.add(want)
    assert len(seen) == 2
