"""Attention of many sequences over a shared prefix and their own suffixes
(talos_attention_shared_dev) against the definition in 64 bits, one sequence at
a time.

Bounds, per output element, for V values up to Vmax and scores whose terms add
up to A = max scale * sum_d |q_d k_d| (all in f32 steps of 2^-23):
 * a score: hd / 16 truncating accumulations and the 22-bit splits of q and k,
   (hd / 16 + 5) A; the exponential and the splits of P and V, 6; the products of a
   tile, 24; the sums of weights and of tiles, 32 + tiles: relative error of a weight
   d = 2^-23 ((hd / 16 + 5) A + 64 + tiles);
 * an error d of every weight moves a weighted mean by at most 2 d Vmax;
 * 16-bit types: half a step (eps / 2) of every weight, eps / 2 * Vmax, and of the
   result, eps / 2 * |out|."""
import numpy as np
import pytest

import talos_b200
from talos_b200 import _lib
from talos_b200._lib import TalosError

pytestmark = pytest.mark.gpu

TYPES = [("float32", "float32"), ("float32", "float16"), ("float16", "float16"), ("bfloat16", "bfloat16")]


def make(n, heads, kvh, hd, prefix, rows, types, seed=0, lens=None, n_slots=None):
    import torch

    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    qt, kt = (getattr(torch, t) for t in types)
    n_slots = n if n_slots is None else n_slots

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    q = (normal(n, heads, hd) * 2).to(qt)
    kp, vp = normal(prefix, kvh, hd).to(kt), normal(prefix, kvh, hd).to(kt)
    k, v = normal(n_slots, rows, kvh, hd).to(kt), normal(n_slots, rows, kvh, hd).to(kt)
    rng = np.random.default_rng(seed)
    slots = rng.permutation(n_slots)[:n] if n_slots >= n else rng.integers(0, n_slots, n)
    lens = rng.integers(0, rows + 1, n) if lens is None else np.asarray(lens)
    dev = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")  # noqa: E731
    return q, kp, vp, k, v, dev(slots), dev(lens)


def oracle(q, kp, vp, k, v, slots, lens, scale=None):
    """(out, bound's A, Vmax per head) in f64."""
    import torch

    n, heads, hd = q.shape
    kvh = k.shape[2]
    group = heads // kvh
    scale = hd ** -0.5 if scale is None else scale
    q = q.double()
    out = torch.zeros(n, heads, hd, dtype=torch.float64, device="cuda")
    vmax = torch.zeros(n, heads, 1, dtype=torch.float64, device="cuda")
    slots = torch.arange(n) if slots is None else slots
    top, keys = 0.0, 0
    for i in range(n):
        s, m = int(slots[i]), int(min(max(int(lens[i]), 0), k.shape[1]))
        m = m if 0 <= s < k.shape[0] else 0
        s = s if 0 <= s < k.shape[0] else 0
        kk = torch.cat([kp, k[s, :m]]).double().transpose(0, 1)  # [kvh, keys, hd]
        vv = torch.cat([vp, v[s, :m]]).double().transpose(0, 1)
        keys = max(keys, kk.shape[1])
        if kk.shape[1] == 0:
            continue
        qi = q[i].view(kvh, group, hd)
        a = torch.softmax(torch.matmul(qi, kk.transpose(1, 2)) * scale, -1)
        out[i] = torch.matmul(a, vv).reshape(heads, hd)
        top = max(top, float((torch.matmul(qi.abs(), kk.abs().transpose(1, 2)) * scale).max()))
        vmax[i] = vv.abs().amax((1, 2)).repeat_interleave(group)[:, None]
    return out, top, vmax, keys


def check(args, scale=None, out=None, want_rel=None):
    import torch

    q, k = args[0], args[3]
    got = talos_b200.attention_shared_dev(*args, out=out, scale=scale)
    ref, top, vmax, keys = oracle(*args, scale=scale)
    assert got.dtype == q.dtype and got.shape == q.shape
    bound = 2 * 2.0**-23 * ((q.shape[2] / 16 + 5) * top + 64 + keys / 64) * vmax
    if q.dtype != torch.float32:
        h = torch.finfo(q.dtype).eps / 2
        bound = bound + h * (vmax + ref.abs())
    err = (got.double() - ref).abs()
    worst = float((err / (bound + 1e-300)).max())
    assert torch.isfinite(got).all() and bool((err <= bound).all()), f"error {worst:.3g} of the bound"
    return got


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("n,heads,kvh,hd,prefix,rows", [
    (1, 1, 1, 64, 5, 3), (2, 6, 2, 48, 40, 16), (3, 4, 4, 128, 0, 130), (1, 8, 1, 128, 64, 0), (5, 8, 2, 64, 129, 7),
])
def test_small(types, n, heads, kvh, hd, prefix, rows):
    check(make(n, heads, kvh, hd, prefix, rows, types))


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("n,heads,kvh,hd,prefix,rows", [
    (1, 32, 8, 128, 0, 1), (1, 32, 8, 128, 1, 1), (32, 32, 8, 128, 1000, 200), (33, 32, 8, 128, 127, 65),
    (64, 64, 8, 128, 2049, 300), (17, 12, 4, 80, 777, 333), (64, 32, 8, 128, 63, 64), (7, 28, 4, 96, 500, 20),
    (130, 8, 8, 64, 256, 33), (9, 128, 1, 16, 321, 50), (200, 2, 1, 8, 70, 9), (40, 7, 1, 24, 3000, 128),
    (2, 16, 16, 112, 20000, 5), (300, 64, 4, 40, 10, 3),
])
def test_matches_definition(types, n, heads, kvh, hd, prefix, rows):
    check(make(n, heads, kvh, hd, prefix, rows, types, seed=n))


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("prefix", [0, 1, 63, 64, 65, 127, 128, 129, 192, 1024])
def test_prefix_ends_around_tiles(types, prefix):
    check(make(6, 8, 2, 128, prefix, 130, types, seed=prefix, lens=[0, 1, 63, 64, 128, 130]))


@pytest.mark.parametrize("hd", [4, 12, 20, 68, 100, 124])
def test_f32_heads_of_any_four(hd):
    check(make(5, 6, 3, hd, 200, 70, ("float32", "float32"), seed=hd))


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("prefix,lens", [(0, [0] * 9), (0, [0, 5, 0, 0, 300, 0, 1, 0, 0]), (3, [0] * 9)])
def test_sequences_without_keys(types, prefix, lens):
    """No prefix and no suffix: zeros, not NaN, beside sequences that have some."""
    import torch

    for heads in (8, 128):
        args = make(9, heads, 2, 64, prefix, 300, types, lens=lens)
        out = torch.full_like(args[0], float("nan"))
        check(args, out=out)


@pytest.mark.parametrize("types", TYPES)
def test_rows_that_are_not_attended_to(types):
    """NaN and infinities behind a sequence's last row, in slots that nobody names,
    and around the prefix change nothing."""
    import torch

    args = make(11, 16, 4, 128, 300, 200, types, seed=3, n_slots=20)
    clean = talos_b200.attention_shared_dev(*args)
    q, kp, vp, k, v, slots, lens = args
    dead = torch.ones(20, 200, dtype=torch.bool, device="cuda")
    for s, m in zip(slots.tolist(), lens.tolist()):
        dead[s, :m] = False
    for t, x in ((k, float("nan")), (v, float("inf"))):
        t[dead] = x
    v[dead.nonzero()[::2, 0], dead.nonzero()[::2, 1]] = float("nan")
    wide = [torch.full((320, 4, 128), float("nan"), dtype=kp.dtype, device="cuda") for _ in range(2)]
    for w, p in zip(wide, (kp, vp)):
        w[10:310] = p
    got = talos_b200.attention_shared_dev(q, wide[0][10:310], wide[1][10:310], k, v, slots, lens)
    assert torch.equal(got, clean)


@pytest.mark.parametrize("types", TYPES)
def test_one_sequences_nan_stays_its_own(types):
    import torch

    args = make(20, 8, 2, 64, 90, 40, types, seed=8, lens=[40] * 20)
    clean = talos_b200.attention_shared_dev(*args)
    bad = [3, 11]
    for i in bad:
        args[3][int(args[5][i]), 7] = float("nan")
        args[4][int(args[5][i]), 9] = float("inf")
    args[0][15] = float("nan")
    got = talos_b200.attention_shared_dev(*args)
    keep = [i for i in range(20) if i not in bad + [15]]
    assert torch.equal(got[keep], clean[keep])
    assert torch.isnan(got[bad]).all() and torch.isnan(got[15]).all()


@pytest.mark.parametrize("types", TYPES)
def test_slots_and_lengths_out_of_range(types):
    """Clamped: nothing outside the caches is read."""
    import torch

    args = list(make(6, 8, 2, 64, 70, 30, types, n_slots=4))
    args[5] = torch.tensor([0, -1, 4, 3, 2000000000, 1], dtype=torch.int32, device="cuda")
    args[6] = torch.tensor([31, 5, 5, -3, 5, 2000000000], dtype=torch.int32, device="cuda")
    check(args)


def test_same_slot_for_several_sequences_and_no_slots():
    import torch

    args = list(make(12, 8, 2, 128, 100, 150, ("float32", "float16"), n_slots=12))
    args[5] = torch.tensor([3, 3, 3, 0, 0, 1, 11, 11, 3, 2, 2, 2], dtype=torch.int32, device="cuda")
    check(args)
    args[5] = None
    check(args)


@pytest.mark.parametrize("types", TYPES)
def test_strided_tensors(types):
    """Queries inside a fused projection, a cache with layers, heads before
    positions, an output inside a wider one."""
    import torch

    q, kp, vp, k, v, slots, lens = make(9, 8, 4, 64, 150, 70, types, seed=5)
    fused = torch.full((9, 16, 64), 7.0, dtype=q.dtype, device="cuda")
    fused[:, 4:12] = q
    layered = [torch.full((9, 3, 4, 70, 64), 7.0, dtype=k.dtype, device="cuda") for _ in range(2)]
    for t, x in zip(layered, (k, v)):
        t[:, 1] = x.transpose(1, 2)
    pre = [torch.stack([p, p * 0 + 7]).permute(2, 1, 0, 3).contiguous() for p in (kp, vp)]  # [kvh, prefix, 2, hd]
    out = torch.full((9, 10, 64), -3.0, dtype=q.dtype, device="cuda")
    args = (fused[:, 4:12], *(p[:, :, 0].transpose(0, 1) for p in pre), *(t[:, 1].transpose(1, 2) for t in layered),
            slots, lens)
    check(args, out=out[:, 1:9])
    assert (out[:, 0] == -3).all() and (out[:, 9] == -3).all()
    assert torch.equal(out[:, 1:9], talos_b200.attention_shared_dev(q, kp, vp, k, v, slots, lens))


@pytest.mark.parametrize("scale", [1e-6, 1.0, 40.0])
@pytest.mark.parametrize("types", TYPES)
def test_scales(types, scale):
    """From almost uniform to one key taking all."""
    check(make(8, 8, 2, 64, 600, 40, types, seed=2), scale=scale)


def test_f32_magnitudes():
    """f32 inputs far outside f16's range and of mixed size: every row and key has
    its own power of two."""
    import torch

    types = ("float32", "float32")
    for qm, km, vm in [(1e6, 1e-6, 1e-20), (1e-12, 1e12, 1e20), (1.0, 1.0, 1e30), (1e-30, 1e25, 1e-30)]:
        q, kp, vp, k, v, slots, lens = make(6, 8, 2, 128, 200, 70, types, seed=4)
        check((q * qm, kp * km, vp * vm, k * km, v * vm, slots, lens), scale=0.05 / (qm * km) ** 0.5 if qm * km > 100 else
              0.1)
    q, kp, vp, k, v, slots, lens = make(6, 8, 2, 128, 300, 70, types, seed=6)
    spread = lambda *s: 10 ** (torch.rand(*s, device="cuda") * 8 - 4)  # noqa: E731
    check((q * spread(6, 8, 1), kp * spread(300, 2, 1) * 0.01, vp * spread(300, 2, 1), k * spread(6, 70, 2, 1) * 0.01,
           v * spread(6, 70, 2, 1), slots, lens), scale=0.01)
    vp[::3] = 0
    kp[5::7] = 0
    q[2] = 0
    check((q, kp, vp, k * 0, v * 0, slots, lens))
    check((q, kp, vp * 0, k, v * 0, slots, lens))


def test_f16_cache_at_its_limits():
    import torch

    q, kp, vp, k, v, slots, lens = make(6, 8, 2, 128, 200, 70, ("float32", "float16"), seed=4)
    check((q, kp * 1000, (vp * 15000).clamp(-65504, 65504), k * 1000, v * 15000, slots, lens), scale=1e-4)
    check((q * 1e5, kp * 6e-8, vp * 6e-8, k * 6e-8, v * 6e-8, slots, lens), scale=1.0)  # subnormals


@pytest.mark.parametrize("types", TYPES)
def test_a_key_far_above_the_rest(types):
    """The running maximum jumps late, early, and in the suffix."""
    for at in (0, 511, 1023):
        q, kp, vp, k, v, slots, lens = make(5, 8, 2, 64, 1024, 80, types, seed=at, lens=[80, 0, 1, 40, 64])
        kp[at] *= 12
        k[:, 39] *= 14
        check((q, kp, vp, k, v, slots, lens))


@pytest.mark.parametrize("types", TYPES)
def test_rerun_bit_identical(types):
    import torch

    args = make(50, 32, 8, 128, 3000, 500, types, seed=1)
    first = talos_b200.attention_shared_dev(*args)
    for _ in range(3):
        assert torch.equal(first, talos_b200.attention_shared_dev(*args))


def test_stream_capture_and_replay():
    """Two graphs with workspaces of their own, replayed with other inputs in
    the same buffers (lengths too), interleaved on two streams."""
    import torch

    sets = [make(20, 16, 4, 128, 700, 100, t, seed=s) for s, t in ((1, TYPES[0]), (2, TYPES[3]))]
    graphs, outs = [], []
    for a in sets:
        talos_b200.attention_shared_dev(*a)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(talos_b200.attention_shared_dev(*a))
        graphs.append(g)
    for seed in (5, 6):
        fresh = [make(20, 16, 4, 128, 700, 100, t, seed=seed + s) for s, t in ((1, TYPES[0]), (2, TYPES[3]))]
        for a, f in zip(sets, fresh):
            for x, y in zip(a, f):
                x.copy_(y)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for _ in range(3):
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        for a, o in zip(sets, outs):
            assert torch.equal(o, talos_b200.attention_shared_dev(*a))
            check(a)


def test_side_stream():
    import torch

    args = make(8, 8, 2, 64, 500, 50, TYPES[1])
    want = talos_b200.attention_shared_dev(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = talos_b200.attention_shared_dev(*args)
    side.synchronize()
    assert torch.equal(got, want)


def test_offsets_beyond_32_bits():
    """The last slots of a cache of more than 2^32 elements."""
    import torch

    n_slots, rows, kvh, hd = 70, 60000, 8, 128  # 4.3e9 elements, 8.6 GB each
    k = torch.zeros(n_slots, rows, kvh, hd, dtype=torch.float16, device="cuda")
    v = torch.zeros(n_slots, rows, kvh, hd, dtype=torch.float16, device="cuda")
    tail = slice(0, 300)
    for s in (0, 68, 69):
        k[s, tail] = torch.randn(300, kvh, hd, device="cuda").half()
        v[s, tail] = torch.randn(300, kvh, hd, device="cuda").half()
    q = torch.randn(3, 16, hd, device="cuda")
    kp, vp = torch.randn(2, 100, kvh, hd, device="cuda").half()
    slots = torch.tensor([69, 0, 68], dtype=torch.int32, device="cuda")
    lens = torch.tensor([300, 17, 129], dtype=torch.int32, device="cuda")
    check((q, kp, vp, k, v, slots, lens))


def test_no_sequences():
    import torch

    args = list(make(2, 4, 2, 64, 9, 5, TYPES[0]))
    args[0], args[5], args[6] = args[0][:0], args[5][:0], args[6][:0]
    assert talos_b200.attention_shared_dev(*args).shape == (0, 4, 64)


def test_refusals():
    import torch

    good = dict(zip(("q", "k_prefix", "v_prefix", "k", "v", "slots", "lens"), make(3, 8, 2, 64, 20, 10, TYPES[0])))
    bad = [dict(q=good["q"].double()), dict(q=good["q"].cpu()), dict(q=good["q"][0]), dict(q=good["q"].transpose(1, 2)),
           dict(v=good["v"].half()), dict(v=good["v"][:, :5]), dict(v_prefix=good["v_prefix"][:5]),
           dict(k_prefix=good["k_prefix"].half()), dict(k_prefix=good["k_prefix"][:, :1], v_prefix=good["v_prefix"][:, :1]),
           dict(lens=good["lens"].long()), dict(lens=good["lens"][:2]), dict(lens=good["lens"].cpu()),
           dict(slots=good["slots"].float()), dict(out=torch.empty(3, 8, 64, device="cuda", dtype=torch.half)),
           dict(out=torch.empty(2, 8, 64, device="cuda")), dict(v=good["v"].transpose(1, 2).contiguous().transpose(1, 2))]
    for b in bad:
        with pytest.raises(ValueError):
            talos_b200.attention_shared_dev(**{**good, **b})
    for b in (dict(q=good["q"].half()), dict(q=good["q"].bfloat16())):  # 16-bit queries with an f32 cache
        with pytest.raises(TalosError, match="UNSUPPORTED"):
            talos_b200.attention_shared_dev(**{**good, **b})
    with pytest.raises(TalosError, match="INVALID_ARG"):
        talos_b200.attention_shared_dev(**{**good, "q": good["q"][:, :7]})  # 7 heads over 2
    for s in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(TalosError, match="INVALID_ARG"):
            talos_b200.attention_shared_dev(**good, scale=s)
    with pytest.raises(TalosError, match="UNSUPPORTED"):
        talos_b200.attention_shared_dev(*make(2, 2, 1, 136, 5, 5, TYPES[0]))
    with pytest.raises(TalosError, match="UNSUPPORTED"):
        talos_b200.attention_shared_dev(*make(2, 2, 1, 60, 5, 5, TYPES[1]))
    with pytest.raises(TalosError, match="INVALID_ARG"):
        talos_b200.attention_shared_dev(*make(2, 129, 1, 64, 5, 5, TYPES[1]))
    with pytest.raises(TalosError, match="INVALID_ARG"):
        talos_b200.attention_shared_dev(*make(1025, 1, 1, 64, 5, 5, TYPES[1]))
    odd = torch.zeros(3, 8, 66, device="cuda", dtype=torch.half)[:, :, :64]  # rows of 132 bytes
    a = make(3, 8, 2, 64, 20, 10, TYPES[2])
    with pytest.raises(TalosError, match="INVALID_ARG"):
        talos_b200.attention_shared_dev(odd, *a[1:])
    assert _lib.load().talos_attention_shared_dev(None, None, 0, None) == _lib.INVALID_ARG


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("n,heads,kvh,hd,prefix,rows", [(1024, 32, 1, 64, 100, 5), (160, 128, 1, 16, 300, 3),
                                                        (1024, 2, 2, 128, 65, 9), (152, 200, 2, 32, 0, 70)])
def test_more_row_tiles_than_sms(types, n, heads, kvh, hd, prefix, rows):
    check(make(n, heads, kvh, hd, prefix, rows, types, seed=n + hd))


def test_two_calls_at_once():
    """Calls on two streams, each with its own workspace, give what each gives alone."""
    import torch

    a = make(32, 32, 8, 128, 1500, 200, ("float32", "float32"), seed=1)
    b = make(48, 32, 8, 128, 900, 300, ("bfloat16", "bfloat16"), seed=2)
    wa, wb = check(a), check(b)
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for _ in range(5):
        with torch.cuda.stream(sa):
            outs.append((talos_b200.attention_shared_dev(*a), wa))
        with torch.cuda.stream(sb):
            outs.append((talos_b200.attention_shared_dev(*b), wb))
    torch.cuda.synchronize()
    for got, want in outs:
        assert torch.equal(got, want)


@pytest.mark.parametrize("types", TYPES[2:])
def test_long_prefix_of_one_cta(types):
    """Row tiles enough that one CTA walks a head's whole prefix of 2,048 tiles. Every V is 1,
    and so is the output: the weights are summed as rounded. Of the f32 sums behind it, the
    row's adds one rounding a tile (2,048 of 2^-24); O's, with a run of 16 tiles that adds 16
    keys 128 times, loses at most 17 / 4 of 2^-23 each time (17 terms cut two bits below the
    sum's last place) and one rounding a run; the rest is below 2^-18. Together 2.0e-4, where
    f16 has its half step below 1 at 2.4e-4 (bf16 further)."""
    import torch

    n, prefix = 1024, 2048 * 128
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    t = getattr(torch, types[0])
    q = (torch.randn(n, 16, 64, device="cuda", generator=g) * 2).to(t)
    kp = torch.randn(prefix, 1, 64, device="cuda", generator=g).to(t)
    k = torch.randn(4, 3, 1, 64, device="cuda", generator=g).to(t)
    lens = torch.arange(n, dtype=torch.int32, device="cuda") % 4
    slots = torch.arange(n, dtype=torch.int32, device="cuda") % 5  # 4: no suffix
    got = talos_b200.attention_shared_dev(q, kp, torch.ones_like(kp), k, torch.ones_like(k), slots, lens)
    assert bool((got == 1).all()), f"off by up to {float((got.double() - 1).abs().max()):.3g}"


@pytest.mark.parametrize("types", TYPES[2:])
@pytest.mark.parametrize("prefix,rows", [(64 * 128, 130), (3 * 64 * 128 + 77, 5), (65 * 128, 0), (16 * 128, 40)])
def test_prefix_runs_and_late_maxima(types, prefix, rows):
    """Runs of 16 prefix tiles that end with the prefix or behind it, with maxima that grow
    around a run's end."""
    q, kp, vp, k, v, slots, lens = make(140, 128, 1, 64, prefix, rows, types, seed=prefix)
    for at in (16 * 128 - 1, 16 * 128 + 1, 64 * 128, prefix - 3):
        if at < prefix:
            kp[at] *= 1 + at / prefix
    check((q, kp, vp, k, v, slots, lens))


@pytest.mark.parametrize("kvh,hd", [(1, 64), (2, 128)])
def test_f32_tiles_of_changing_magnitude(kvh, hd):
    """Every tile of 64 keys has values of its own magnitude (and so its own power of two),
    over many prefix tiles and many suffix tiles, most of which end early."""
    import torch

    types = ("float32", "float32")
    for n, prefix, rows in ((40, 5000, 300), (128, 0, 140), (16, 64 * 70, 64 * 9)):
        q, kp, vp, k, v, slots, lens = make(n, 4 * kvh, kvh, hd, prefix, rows, types, seed=n)
        f = 2.0 ** torch.randint(-8, 9, (prefix // 64 + 1,), device="cuda")
        g = 2.0 ** torch.randint(-8, 9, (n, rows // 64 + 1), device="cuda")
        vp *= f.repeat_interleave(64)[:prefix, None, None]
        v *= g.repeat_interleave(64, 1)[:, :rows, None, None]
        for _ in range(3):
            check((q, kp, vp, k, v, slots, lens))


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("n,kvh,group,hd,prefix", [(256, 64, 1, 64, 40), (130, 40, 16, 48, 64), (1024, 6, 16, 64, 1),
                                                   (64, 300, 2, 32, 20), (64, 64, 2, 128, 33)])
def test_one_tile_per_kv_head(types, n, kvh, group, hd, prefix):
    """CTAs that take one tile of one kv head after another: the queries change with every
    tile (room for long suffixes, of which there are none or few)."""
    lens = np.zeros(n, np.int64)
    check(make(n, kvh * group, kvh, hd, prefix, 300, types, seed=n, lens=lens, n_slots=4))
    lens[n // 2] = 3
    check(make(n, kvh * group, kvh, hd, prefix, 300, types, seed=n, lens=lens, n_slots=4))


@pytest.mark.parametrize("scale", [1e-10, 1e-30])
def test_zero_queries_with_small_scales(scale):
    """A row of zeros has equal weights, whatever the scale: the mean of its values."""
    for types in TYPES[:2]:
        q, kp, vp, k, v, slots, lens = make(6, 8, 2, 64, 200, 70, types, seed=9)
        q[2] = 0
        q[4, 3] = 0
        check((q, kp, vp, k, v, slots, lens), scale=scale)


def test_scores_that_overflow():
    """Keys whose score is -inf in f32 have no weight: they fill the first tiles of the
    prefix, all of some suffixes and some rows alone."""
    import torch

    types = ("bfloat16", "bfloat16")
    q, kp, vp, k, v, slots, lens = make(6, 8, 2, 64, 400, 150, types, seed=12, lens=[150, 0, 1, 130, 64, 129])
    q[:, :, 5] = 3e38
    q[1, 2, 5] = 0.0
    kp[:, :, 5], k[..., 5] = 0, 0
    clean = oracle(q, torch.cat([kp[300:], kp[:0]]), torch.cat([vp[300:], vp[:0]]), k, v, slots, lens * 0)
    kp[:300, :, 5] = -10
    k[..., 5] = -10
    got = talos_b200.attention_shared_dev(q, kp, vp, k, v, slots, lens)
    ref, top, vmax, keys = clean
    # the bound of check() over the keys that count (q's huge element meets zeros there)
    bound = 2 * 2.0**-23 * ((64 / 16 + 5) * top + 64 + 6) * vmax + 2.0**-8 * (vmax + ref.abs())
    rows = torch.ones(6, 8, dtype=torch.bool, device="cuda")
    rows[1, 2] = False  # (this row attends to every key)
    assert torch.isfinite(got).all()
    assert bool(((got.double() - ref).abs() <= bound)[rows].all())
    whole = oracle(q[1:2, 2:3], kp[:, :1], vp[:, :1], k[:, :, :1], v[:, :, :1], slots[1:2], lens[1:2])[0]
    assert bool(((got[1, 2].double() - whole[0, 0]).abs() <= bound[1, 2]).all())


def test_a_sequence_whose_scores_all_overflow():
    """No key with a weight: zeros, in one CTA's tile and in partials."""
    import torch

    for prefix, rows in ((0, 40), (700, 600)):
        q, kp, vp, k, v, slots, lens = make(5, 8, 2, 64, prefix, rows, ("bfloat16", "bfloat16"), seed=3,
                                            lens=[rows] * 5)
        q[:, :, 5] = 0
        kp[:, :, 5], k[..., 5] = -10, -10
        want = talos_b200.attention_shared_dev(q, kp, vp, k, v, slots, lens)
        q[3, :, 5] = 3e38
        got = talos_b200.attention_shared_dev(q, kp, vp, k, v, slots, lens)
        assert not got[3].any()
        keep = [0, 1, 2, 4]
        assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_infinite_values_keep_to_their_dimension(types, bad):
    """An attended value that is infinite or NaN leaves no finite output in its own dimension
    and the others as they are."""
    import torch

    q, kp, vp, k, v, slots, lens = make(7, 8, 2, 128, 150, 90, types, seed=15, lens=[90, 80, 0, 64, 65, 1, 90])
    args = (q, kp, vp, k, v, slots, lens)
    vp[20, 0, 3] = bad
    v[int(slots[3]), 40, 1, 70] = bad
    hit = torch.zeros(7, 8, 128, dtype=torch.bool, device="cuda")
    hit[:, :4, 3] = True
    hit[3, 4:, 70] = True
    got = talos_b200.attention_shared_dev(*args)
    assert not torch.isfinite(got[hit]).any()
    vp[20, 0, 3] = 0
    v[int(slots[3]), 40, 1, 70] = 0
    ref, top, vmax, keys = oracle(*args)
    bound = 2 * 2.0**-23 * ((128 / 16 + 5) * top + 64 + keys / 64) * vmax
    if q.dtype != torch.float32:
        bound = bound + torch.finfo(q.dtype).eps / 2 * (vmax + ref.abs())
    assert bool(((got.double() - ref).abs() <= bound)[~hit].all())


def test_stream_argument_has_memory_of_its_own(monkeypatch):
    """Calls for two streams, made one after the other on a third, do not share a workspace or
    an output that was released in between (the launches are left out here)."""
    import torch

    from talos_b200 import ops

    args = make(8, 8, 2, 64, 500, 50, TYPES[1])
    talos_b200.attention_shared_dev(*args)
    torch.cuda.synchronize()
    works = []

    def launch(a, work, size, stream):
        works.append((work, stream))
        return 0

    monkeypatch.setattr(ops._torch().lib, "talos_attention_shared_dev", launch)
    sides = [torch.cuda.Stream() for _ in range(2)]
    seen = set()
    for s in (*sides, None):
        out = talos_b200.attention_shared_dev(*args, stream=None if s is None else s.cuda_stream)
        assert out.data_ptr() not in seen
        seen.add(out.data_ptr())
        del out
    assert [s for _, s in works] == [*(s.cuda_stream for s in sides), torch.cuda.current_stream().cuda_stream]
    assert len({w for w, _ in works}) == 3 and not seen & {w for w, _ in works}


def test_stream_argument():
    """The work of different calls on several given streams at once, while the current stream
    goes on allocating and writing."""
    import torch

    sets = [make(n, 32, 8, 128, prefix, 200, t, seed=n) for n, prefix, t in
            ((40, 3000, TYPES[0]), (33, 9000, TYPES[3]), (64, 700, TYPES[1]))]
    want = [check(a) for a in sets]
    sides = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = []
    for _ in range(6):
        for a, s in zip(sets, sides):
            got.append(talos_b200.attention_shared_dev(*a, stream=s.cuda_stream))
            junk = [torch.full((1 << k,), float("nan"), device="cuda") for k in range(8, 23)]
            del junk
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert torch.equal(g, want[i % len(sets)])
    default = talos_b200.attention_shared_dev(*sets[0], stream=0)
    with torch.cuda.stream(sides[0]):
        other = talos_b200.attention_shared_dev(*sets[0], stream=0)
    torch.cuda.synchronize()
    assert torch.equal(default, want[0]) and torch.equal(other, want[0])
