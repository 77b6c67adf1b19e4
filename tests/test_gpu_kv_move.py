"""talos_kv_move_dev: rows moved between cache slots, compared exactly with
copies made one after the other from a snapshot (every move reads what the
slots held before the call). A slot's bytes carry their own address, so a row in
a wrong place shows."""
import numpy as np
import pytest

import talos_b200
from talos_b200._lib import TalosError

pytestmark = pytest.mark.gpu


def caches(shape, dtype, n=2, layout="slots"):
    import torch

    size = int(np.prod(shape))
    out = []
    for i in range(n):
        x = (torch.arange(size, device="cuda", dtype=torch.int64) * (2 * i + 1)) % 65521
        x = x.to(torch.int16).view(torch.float16) if dtype == "float16" else x.to(getattr(torch, dtype))
        x = x.view(shape)
        if layout == "layers":  # [layers, slots, rows, ...] seen as [slots, layers, rows, ...]
            x = x.transpose(0, 1).contiguous().transpose(0, 1)
        out.append(x)
    return out


def bits(t):
    import torch

    return t.view(torch.int16) if t.dtype == torch.float16 else t


def run(cs, src, dst, lens, starts=None):
    import torch

    before = [c.clone() for c in cs]
    want = [c.clone() for c in cs]
    for i, (a, b, n) in enumerate(zip(src, dst, lens)):
        s = starts[i] if starts else 0
        for w, o in zip(want, before):
            w[b, :, s:s + n] = o[a, :, s:s + n]
    talos_b200.kv_move_dev(cs, src, dst, lens, starts)
    for c, w in zip(cs, want):
        assert torch.equal(bits(c), bits(w))


@pytest.mark.parametrize("layout", ["slots", "layers"])
@pytest.mark.parametrize("dtype,width", [("float32", 96), ("float16", 48), ("float16", 33), ("int32", 1),
                                         ("uint8", 7), ("float32", 1024)])
def test_fork_compact_permute(dtype, width, layout):
    for src, dst, lens, starts in [
        ([0], [3], [17], None),
        ([2, 2, 2, 2], [0, 1, 3, 5], [40, 40, 1, 23], None),         # one to many, ragged
        ([1, 3, 4, 7], [0, 1, 2, 3], [40, 5, 39, 11], None),         # compaction
        ([0, 1], [1, 0], [40, 40], None),                            # swap
        ([0, 1, 2, 3, 4, 5, 6, 7], [1, 2, 3, 4, 5, 6, 7, 0], [40] * 8, None),  # one cycle
        ([0, 1, 2, 2, 3, 3], [1, 2, 0, 4, 5, 6], [9, 40, 30, 13, 40, 7], None),  # a cycle with branches
        ([5, 5, 1, 4], [5, 4, 1, 6], [40, 12, 40, 0], None),         # onto itself; no rows
        ([0, 1, 2], [1, 2, 0], [10, 20, 30], [30, 15, 3]),           # ranges that start later
        ([6, 6], [0, 7], [1, 1], [39, 0]),
    ]:
        run(caches((8, 3, 40, width), dtype, layout=layout), src, dst, lens, starts)


def test_random_moves():
    rng = np.random.default_rng(4)
    for _ in range(30):
        n = int(rng.integers(1, 65))
        m = int(rng.integers(1, n + 1))
        src, dst = rng.integers(0, n, m).tolist(), rng.permutation(n)[:m].tolist()
        starts = rng.integers(0, 9, m).tolist()
        lens = [int(rng.integers(0, 10 - s)) for s in starts]
        run(caches((n, 2, 9, 20), "float32"), src, dst, lens, starts)


def test_many_moves_and_arrays():
    """More moves than the small parameter block, a cycle over 500 slots, eight arrays."""
    rng = np.random.default_rng(6)
    run(caches((500, 1, 5, 6), "float32"), list(range(500)), [(i + 1) % 500 for i in range(500)], [5] * 500)
    run(caches((600, 2, 3, 4), "float16", n=8), rng.integers(0, 600, 512).tolist(),
        rng.permutation(600)[:512].tolist(), rng.integers(0, 4, 512).tolist())
    run(caches((512, 1, 4, 4), "float32"), [i ^ 1 for i in range(512)], list(range(512)), [4] * 512)  # 256 swaps


def test_misaligned_rows():
    """Bases and strides off the 16-byte grid take narrower accesses."""
    import torch

    for off in (1, 2, 4, 8, 16):
        flat = [torch.randint(0, 255, (3 * 2 * 11 * 48 + off,), dtype=torch.uint8, device="cuda") for _ in range(2)]
        run([f[off:].view(3, 2, 11, 48) for f in flat], [0, 2], [1, 0], [11, 7])


def test_offsets_beyond_32_bits():
    """A cache of more than 4 GB: the last slot's rows, both ways."""
    import torch

    c = torch.zeros(5, 2, 4096, 1 << 17, dtype=torch.uint8, device="cuda")  # 5.4 GB
    c[4, 1, 4000:] = torch.randint(1, 255, (96, 1 << 17), dtype=torch.uint8, device="cuda")
    talos_b200.kv_move_dev([c], [4], [0], [96], [4000])
    assert torch.equal(c[0, 1, 4000:], c[4, 1, 4000:]) and not c[0, 1, :4000].any() and not c[1:4].any()
    c[0, 0, 17] = 9
    talos_b200.kv_move_dev([c], [0, 4], [4, 0], [4096, 1])
    assert (c[4, 0, 17] == 9).all() and torch.equal(c[0, 1, 4000:], c[4, 1, 4000:])


def test_stream_capture_and_replay():
    import torch

    cs = caches((4, 2, 8, 16), "float32")
    g = torch.cuda.CUDAGraph()
    want = [c.clone() for c in cs]
    with torch.cuda.graph(g):
        talos_b200.kv_move_dev(cs, [0, 1, 2], [1, 2, 0], [8, 8, 8])
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    for c, w in zip(cs, want):
        assert torch.equal(c, w)  # three turns of a cycle of three


def test_refusals():
    cs = caches((4, 2, 8, 16), "float32")
    keep = [c.clone() for c in cs]
    for bad in [([4], [0], [1]), ([0], [4], [1]), ([0], [1], [9]), ([0, 1], [2, 2], [1, 1]), ([0, 1], [2, 2], [1, 0])]:
        with pytest.raises(TalosError, match="INVALID_ARG"):
            talos_b200.kv_move_dev(cs, *bad)
    with pytest.raises(TalosError, match="INVALID_ARG"):
        talos_b200.kv_move_dev(cs, [0], [1], [4], [5])
    with pytest.raises(TalosError, match="INVALID_ARG"):
        talos_b200.kv_move_dev([cs[0], cs[0]], [0], [1], [4])
    with pytest.raises(TalosError, match="INVALID_ARG"):
        talos_b200.kv_move_dev([cs[0][:1].expand(4, 2, 8, 16)], [0], [1], [4])  # slots that overlap
    with pytest.raises(TalosError, match="INVALID_ARG"):
        talos_b200.kv_move_dev(cs, [0] * 513, list(range(513)), [1] * 513)
    for bad in [([0], [1, 2], [1]), ([-1], [0], [1])]:
        with pytest.raises(ValueError):
            talos_b200.kv_move_dev(cs, *bad)
    for c in ([cs[0], cs[1].half()], [cs[0].cpu()], [cs[0][0]], [cs[0].transpose(2, 3)], [cs[0], cs[1][:2]]):
        if c[0].dim() == 4 and c[0].is_cuda and len(c) == 1:
            c = [c[0].reshape(4, 2, 16, 2, 4).transpose(3, 4)]
        with pytest.raises(ValueError):
            talos_b200.kv_move_dev(c, [0], [1], [1])
    import torch

    for c, w in zip(cs, keep):
        assert torch.equal(c, w)


def test_no_moves():
    cs = caches((2, 1, 4, 4), "float32")
    talos_b200.kv_move_dev(cs, [], [], [])
    talos_b200.kv_move_dev(cs, [1], [1], [4])


def test_long_runs_of_several_chains():
    """Chains long enough that a thread takes several offsets, with rows that end inside a
    block's run; then the same arrays with an exchange and a fork."""
    cs = caches((9, 8, 1024, 1024), "float32")
    run(cs, [1, 2, 3, 6, 7], [0, 1, 2, 5, 6], [1024, 1003, 700, 1021, 977])
    run(cs, [3, 4, 8, 7], [2, 3, 6, 5], [1000, 1024, 1, 513], [24, 0, 1023, 11])
    run(cs, [0, 1, 4, 4], [1, 0, 7, 8], [1024, 1024, 301, 1024])


def test_arrays_within_one_tensor():
    """Keys and values side by side in one tensor's rows, planes or slots are moved; views that
    share rows are refused and stay as they are."""
    import torch

    for dim in range(4):
        shape = [4, 3, 10, 8]
        shape.insert(dim, 2)
        x = torch.randn(shape, device="cuda")
        run(list(x.unbind(dim)), [0, 1, 3], [1, 0, 2], [10, 10, 7], [0, 0, 3])
    x = torch.randn(4, 3, 10, 8, device="cuda")
    keep = x.clone()
    for a, b in ((x[:, :, :9], x[:, :, 1:]), (x[:, :2], x[:, 1:]), (x[:3], x[1:]), (x[..., :5], x[..., 3:])):
        with pytest.raises(TalosError, match="INVALID_ARG"):
            talos_b200.kv_move_dev([a, b], [0, 1], [1, 0], [5, 5])
    assert torch.equal(x, keep)
