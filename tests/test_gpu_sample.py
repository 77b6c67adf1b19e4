"""The choice of tokens on the GPU (talos_sample_dev, talos_sample) against the
definition in 64 bits with numpy, row by row: temperature, top-k, top-p, min-p
and one random number per row (src/sample.rs:19-76 with min-p besides).

Tokens must be equal: the kernel sums weights to 2^-42 of the largest one, the
oracle to f64 rounding, so both sides of a border agree unless a random number
lies within about 1e-11 of it. Probabilities are within 4 half-steps of f32
(the rounding of the result and of the sums behind it: 4 * 2^-24)."""
import numpy as np
import pytest

import talos_b200
from talos_b200 import _lib
from talos_b200._lib import TalosError

pytestmark = pytest.mark.gpu


def choose(logits, u, temperature, top_k, top_p, min_p):
    """(token, probability) of one row by the definition, in f64."""
    l = np.asarray(logits, np.float64).copy()
    l[np.isnan(l)] = -np.inf
    l += 0.0
    top = l.max()
    if top == -np.inf:
        return -1, 0.0
    if not temperature > 0:
        temperature, top_k = 1.0, 1
    order = np.argsort(-l, kind="stable")
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(l[order] == top, 1.0, np.exp((l[order] - top) / np.float64(np.float32(temperature))))
    w[l[order] == -np.inf] = 0.0
    order, w = order[w > 0], w[w > 0]
    if top_k > 0:
        order, w = order[:top_k], w[:top_k]
    p = np.float64(np.float32(top_p))
    if p < 1:
        c = np.cumsum(w)
        keep = int(np.searchsorted(c, p * c[-1], side="left")) + 1
        order, w = order[:keep], w[:keep]
    m = min(np.float64(np.float32(min_p)), 1.0)
    if m > 0:
        order, w = order[w >= m], w[w >= m]
    c = np.cumsum(w)
    j = min(int(np.searchsorted(c, np.float64(np.float32(u)) * c[-1], side="right")), len(w) - 1)
    return int(order[j]), w[j] / c[-1]


def rows(n, vocab, seed, dtype, pad=0):
    import torch

    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((n, vocab + pad)) * rng.uniform(1.0, 5.0, (n, 1))).astype(np.float32)
    return torch.from_numpy(x).cuda().to(dtype)[:, :vocab], rng


def check(logits, u, t=1.0, k=0, p=1.0, m=0.0):
    """Run sample_dev with these settings (numbers or per-row arrays) and compare every row."""
    import torch

    n = logits.shape[0]

    def dev(x, dt):
        return x if isinstance(x, (int, float)) else torch.tensor(np.asarray(x), dtype=dt, device="cuda")

    ud = torch.tensor(np.asarray(u, np.float32), device="cuda")
    tok, prob = talos_b200.sample_dev(logits, ud, temperature=dev(t, torch.float32), top_k=dev(k, torch.int32),
                                      top_p=dev(p, torch.float32), min_p=dev(m, torch.float32))
    again, prob2 = talos_b200.sample_dev(logits, ud, temperature=dev(t, torch.float32), top_k=dev(k, torch.int32),
                                         top_p=dev(p, torch.float32), min_p=dev(m, torch.float32))
    tok, prob, lg = tok.cpu().numpy(), prob.cpu().numpy(), logits.float().cpu().numpy()
    assert np.array_equal(tok, again.cpu().numpy()) and np.array_equal(prob, prob2.cpu().numpy())
    at = lambda x, i: x if isinstance(x, (int, float)) else x[i]  # noqa: E731
    for i in range(n):
        want, wp = choose(lg[i], u[i], at(t, i), at(k, i), at(p, i), at(m, i))
        assert tok[i] == want, f"row {i}: {tok[i]} != {want} (settings {at(t, i)}, {at(k, i)}, {at(p, i)}, {at(m, i)})"
        assert abs(prob[i] - wp) <= 4 * 2.0**-24 * max(wp, 1e-30) + 1e-37
    return tok


SETTINGS = [
    (1.0, 0, 1.0, 0.0), (0.7, 40, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (0.8, 200, 0.95, 0.02), (1.3, 0, 1.0, 0.05),
    (0.0, 0, 1.0, 0.0), (1.0, 1, 0.5, 0.5), (2.0, 5000, 0.999, 0.0), (1.0, 0, 0.99999, 1e-6), (1.0, 0, 1e-6, 0.0),
    (0.05, 700, 0.5, 1.0), (1.5, 600, 0.97, 0.001),
]


@pytest.mark.parametrize("settings", SETTINGS)
@pytest.mark.parametrize("dtype,vocab,pad,n", [("float32", 1, 0, 3), ("float32", 37, 3, 5), ("float32", 4096, 0, 4),
                                               ("bfloat16", 32003, 61, 5), ("float16", 32000, 8, 3),
                                               ("float32", 128256, 0, 3), ("float32", 30001, 1, 70),
                                               ("bfloat16", 150001, 7, 2), ("float32", 262144, 0, 2)])
def test_matches_definition(settings, dtype, vocab, pad, n):
    import torch

    lg, rng = rows(n, vocab, vocab + n, getattr(torch, dtype), pad)
    check(lg, rng.random(n).astype(np.float32), *settings)


def test_settings_per_row():
    import torch

    n, vocab = 64, 20000
    lg, rng = rows(n, vocab, 5, torch.float32)
    s = [SETTINGS[i % len(SETTINGS)] for i in range(n)]
    check(lg, rng.random(n).astype(np.float32), *(list(x) for x in zip(*s)))


@pytest.mark.parametrize("settings", SETTINGS)
@pytest.mark.parametrize("vocab", [2000, 50000, 200000])
def test_equal_and_nearly_equal_logits(vocab, settings):
    """Rows whose logits are all equal, two values, or within one bin of each
    other: the order is by index among equals, and the borders lie inside a bin of
    more elements than the ranked list holds."""
    import torch

    rng = np.random.default_rng(vocab)
    a = np.full((4, vocab), 2.5, np.float32)
    a[1, ::3] = 2.25
    a[2] += rng.uniform(0, 1e-3, vocab).astype(np.float32)
    a[3] = np.where(rng.random(vocab) < 0.5, 0.0, -0.0)  # equal too
    check(torch.from_numpy(a).cuda(), [0.0, 0.37, 0.73, 0.99999994], *settings)


@pytest.mark.parametrize("settings", SETTINGS)
def test_masked_and_special_values(settings):
    """-inf, the lowest finite value, NaN and +inf among the logits."""
    import torch

    rng = np.random.default_rng(3)
    a = rng.standard_normal((8, 5000)).astype(np.float32)
    a[0, 100:] = -np.inf
    a[1, 7:] = np.finfo(np.float32).min
    a[2, ::2] = np.nan
    a[3, [5, 9, 4999]] = np.inf
    a[4, :] = -np.inf  # nothing to choose
    a[5, :] = np.nan
    a[6, :] = np.finfo(np.float32).min  # all equal
    a[7, 1:] = -np.inf
    tok = check(torch.from_numpy(a).cuda(), rng.random(8).astype(np.float32), *settings)
    assert tok[4] == tok[5] == -1 and tok[7] == 0


def test_random_number_at_the_ends():
    import torch

    lg, _ = rows(4, 3000, 9, torch.float32)
    tok = check(lg, [0.0, 0.99999994, 0.5, 0.25], 1.0, 0, 0.9, 0.0)
    order = np.argsort(-lg.cpu().numpy(), kind="stable")
    assert tok[0] == order[0, 0]
    u = torch.tensor([-1.0, 1.0, 7.0, float("nan")], device="cuda")
    t, p = talos_b200.sample_dev(lg, u, top_k=3)
    assert t.tolist() == [order[0, 0], order[1, 2], order[2, 2], order[3, 0]]
    assert torch.all(p > 0)


def test_settings_out_of_range():
    """temperature < 0 or NaN is greedy, min_p above 1 keeps the largest, top_p
    <= 0 keeps the first, top_p NaN and min_p NaN keep all, a negative top_k on the
    device keeps all, an infinite temperature weighs all alike."""
    import torch

    lg, rng = rows(4, 900, 11, torch.float32)
    u = torch.tensor([0.9, 0.5, 0.99, 0.7], device="cuda")
    best = lg.argmax(-1).int()
    nan = float("nan")
    for kw in (dict(temperature=-1.0), dict(temperature=nan), dict(min_p=7.0), dict(top_p=0.0), dict(top_p=-3.0)):
        assert torch.equal(talos_b200.sample_dev(lg, u, **kw)[0], best), kw
    full = talos_b200.sample_dev(lg, u)[0]
    for kw in (dict(top_p=nan), dict(min_p=nan), dict(min_p=-1.0), dict(top_p=2.0),
               dict(top_k=torch.full((4,), -5, dtype=torch.int32, device="cuda"))):
        assert torch.equal(talos_b200.sample_dev(lg, u, **kw)[0], full), kw
    order = np.argsort(-lg.cpu().numpy(), kind="stable")
    t, p = talos_b200.sample_dev(lg, u, temperature=float("inf"))
    want = [order[i, int(np.float64(np.float32(x)) * 900)] for i, x in enumerate([0.9, 0.5, 0.99, 0.7])]
    assert t.tolist() == want and np.allclose(p.cpu().numpy(), 1 / 900, rtol=1e-6)
    tiny = talos_b200.sample_dev(lg, u, temperature=1e-42)[0]  # a denormal temperature
    assert torch.equal(tiny, best)


def test_greedy_agrees_with_argmax_without_ties():
    import torch

    lg, rng = rows(3, 32000, 21, torch.float32)
    t, p = talos_b200.sample_dev(lg, torch.rand(3, device="cuda"), temperature=0.0)
    assert t.tolist() == [talos_b200.argmax(lg[i].cpu().numpy()) for i in range(3)] and p.tolist() == [1.0] * 3


def test_host_call():
    rng = np.random.default_rng(8)
    l = rng.standard_normal(5000).astype(np.float32) * 3
    for u, s in zip(rng.random(6).astype(np.float32), SETTINGS):
        assert talos_b200.sample(l, float(u), *s) == choose(l, u, *s)[0]
    assert talos_b200.sample(l, 0.3, temperature=0.0) == talos_b200.argmax(l)
    with pytest.raises(TalosError, match="INVALID_ARG"):
        talos_b200.sample(np.full(5, -np.inf), 0.3)


def test_distribution():
    """Evenly spread random numbers visit each token in proportion to its weight
    (each count is off by at most one: the cumulative weights are borders)."""
    import torch

    n = 4096
    row = torch.tensor([0.3, -1.0, 2.0, 1.9, -9.0, 0.5], device="cuda")
    u = (torch.arange(n, device="cuda", dtype=torch.float32) + 0.5) / n
    t, _ = talos_b200.sample_dev(row[None].expand(n, 6).contiguous(), u, temperature=0.9)
    w = torch.softmax(row.double() / np.float64(np.float32(0.9)), 0).cpu().numpy()
    assert np.all(np.abs(np.bincount(t.cpu().numpy(), minlength=6) - w * n) <= 1)


def test_stream_capture_and_replay():
    """Captured once, replayed with other logits and numbers in the same buffers,
    on a stream of its own."""
    import torch

    lg, rng = rows(9, 32000, 31, torch.float32)
    buf, u = lg.clone(), torch.rand(9, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        talos_b200.sample_dev(buf, u, temperature=0.9, top_p=0.8)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        tok, prob = talos_b200.sample_dev(buf, u, temperature=0.9, top_p=0.8)
    for seed in (1, 2):
        buf.copy_(rows(9, 32000, seed, torch.float32)[0])
        u.copy_(torch.from_numpy(np.random.default_rng(seed).random(9).astype(np.float32)))
        g.replay()
        torch.cuda.synchronize()
        lg = buf.cpu().numpy()
        assert tok.tolist() == [choose(lg[i], u[i].item(), 0.9, 0, 0.8, 0.0)[0] for i in range(9)]


def test_given_outputs_and_neighbours():
    """tokens / probs given by the caller are the ones written, and nothing beside them."""
    import torch

    lg, _ = rows(5, 700, 41, torch.float32)
    t = torch.full((9,), -77, dtype=torch.int32, device="cuda")
    p = torch.full((9,), -77.0, device="cuda")
    u = torch.rand(5, device="cuda")
    talos_b200.sample_dev(lg, u, tokens=t[2:7], probs=p[2:7], top_k=5)
    want, wp = talos_b200.sample_dev(lg, u, top_k=5)
    assert torch.equal(t[2:7], want) and torch.equal(p[2:7], wp)
    assert (t[[0, 1, 7, 8]] == -77).all() and (p[[0, 1, 7, 8]] == -77).all()


def test_no_rows():
    import torch

    t, p = talos_b200.sample_dev(torch.empty(0, 100, device="cuda"), torch.empty(0, device="cuda"))
    assert t.shape == p.shape == (0,)


def test_refusals():
    import torch

    lg, u = torch.zeros(3, 50, device="cuda"), torch.zeros(3, device="cuda")
    for bad in (dict(logits=lg.double()), dict(logits=lg.cpu()), dict(logits=lg.t()), dict(u=u[:2]), dict(u=u.double()),
                dict(u=u.cpu()), dict(temperature=u[:1]), dict(top_k=u), dict(tokens=u),
                dict(top_p=torch.zeros(3, 2, device="cuda")[:, 0]), dict(logits=lg[None])):
        kw = dict(logits=lg, u=u)
        kw.update(bad)
        with pytest.raises(ValueError):
            talos_b200.sample_dev(**kw)
    with pytest.raises(TalosError, match="INVALID_ARG"):
        talos_b200.sample_dev(lg, u, top_k=-1)
    with pytest.raises(TalosError, match="INVALID_ARG"):
        talos_b200.sample_dev(torch.zeros(1, (1 << 20) + 1, device="cuda"), u[:1])
    with pytest.raises(TalosError, match="INVALID_ARG"):
        talos_b200.sample_dev(torch.zeros(1, 50, device="cuda").expand(3, 50), u)  # rows that overlap
    assert _lib.load().talos_sample_dev(None, None) == _lib.INVALID_ARG


@pytest.mark.parametrize("spread", [1e-45, 1e-40, 3e-37, 1e-30, 1e-20])
@pytest.mark.parametrize("vocab", [2, 5, 1500, 40000])
def test_logits_closer_than_any_bin(spread, vocab):
    """Logits that differ by (almost) nothing share the weight evenly, whatever the bins.
    (At a temperature of 1 every weight is 1 to 1e-20: the oracle's choice is exact.)"""
    import torch

    rng = np.random.default_rng(3)
    x = (rng.integers(0, 9, (3, vocab)) * np.float64(spread)).astype(np.float32)
    x[:, -1] = -np.inf
    u = rng.random(3).astype(np.float32)
    check(torch.from_numpy(x).cuda(), u)
    check(torch.from_numpy(x).cuda(), u, p=0.4, m=0.5)
    check(torch.from_numpy(x).cuda(), u, t=float("inf"))


@pytest.mark.parametrize("t", [1e-3, 1e4, 1e30])
def test_extreme_temperatures_and_ranges(t):
    import torch

    rng = np.random.default_rng(4)
    x = rng.standard_normal((4, 3000)).astype(np.float32)
    x[1] *= 1e30
    x[2, ::3] = -3.4028234663852886e38
    x[3] = np.linspace(-3e38, 3e38, 3000)
    u = rng.random(4).astype(np.float32)
    check(torch.from_numpy(x).cuda(), u, t=t)
    check(torch.from_numpy(x).cuda(), u, t=t, k=700, p=0.7)
    check(torch.from_numpy(x).cuda(), u, t=t, m=0.2)


@pytest.mark.parametrize("settings", [SETTINGS[0], SETTINGS[2], SETTINGS[3], SETTINGS[8], SETTINGS[11]])
@pytest.mark.parametrize("dtype,vocab,pad", [("float32", 100003, 1), ("float32", 100000, 0), ("float16", 100003, 5),
                                             ("bfloat16", 90005, 0)])
def test_slices_that_are_read_again(settings, dtype, vocab, pad):
    """Rows enough that each takes fewer CTAs than would keep it in shared memory, with and
    without 16-byte loads, and slices that end inside a load."""
    import torch

    lg, rng = rows(44, vocab, 7, getattr(torch, dtype), pad)
    check(lg, rng.random(44).astype(np.float32), *settings)


def test_stream_argument():
    """Results for a given stream are not handed out again while its work may be in flight."""
    import torch

    lg, rng = rows(40, 50000, 61, torch.float32)
    u = torch.from_numpy(rng.random(40).astype(np.float32)).cuda()
    want = talos_b200.sample_dev(lg, u, top_p=0.9)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    first = talos_b200.sample_dev(lg, u, top_p=0.9, stream=side.cuda_stream)
    at = {x.data_ptr() for x in first}
    del first
    fresh = [torch.full((40,), -5, dtype=torch.int32, device="cuda") for _ in range(4)]
    assert not at & {x.data_ptr() for x in fresh}
    got = talos_b200.sample_dev(lg, u, top_p=0.9, stream=side.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and all((x == -5).all() for x in fresh)


def test_numpy_numbers_as_settings():
    import torch

    lg, rng = rows(4, 900, 12, torch.float32)
    u = torch.from_numpy(rng.random(4).astype(np.float32)).cuda()
    for kind, whole in ((np.float32, np.int64), (np.float64, np.int32), (np.float16, np.uint8)):
        got = talos_b200.sample_dev(lg, u, temperature=kind(0.5), top_k=whole(50), top_p=kind(0.75), min_p=kind(0.25))
        want = talos_b200.sample_dev(lg, u, temperature=0.5, top_k=50, top_p=0.75, min_p=0.25)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(TalosError, match="INVALID_ARG"):
        talos_b200.sample_dev(lg, u, top_k=np.int64(-1))
    for bad in (dict(top_k=1.5), dict(top_k=np.float32(2)), dict(temperature="1"), dict(min_p=None)):
        with pytest.raises(ValueError):
            talos_b200.sample_dev(lg, u, **bad)


@pytest.mark.parametrize("t", [1e37, 1e38, 3e38, float("inf")])
def test_ranges_beyond_the_largest_float(t):
    """Logits further apart than the largest f32, at temperatures that leave them weights."""
    import torch

    rng = np.random.default_rng(6)
    x = np.stack([np.linspace(-3.4e38, 3.4e38, 3000), rng.uniform(-3e38, 3e38, 3000), rng.uniform(-3e38, 1e31, 3000),
                  np.where(np.arange(3000) % 3, 3.0e38, -3.4028234663852886e38)]).astype(np.float32)
    x[1, ::7] = -np.inf
    u = np.array([0.93, 0.41, 0.77, 0.999], np.float32)
    for kw in (dict(), dict(k=700, p=0.7), dict(p=0.999), dict(m=0.2), dict(k=3), dict(k=900, m=0.3)):
        check(torch.from_numpy(x).cuda(), u, t=t, **kw)
