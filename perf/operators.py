"""The device operators of batched generation, as measured calls and in plain torch.

Three operators serve many sequences that start from one prompt: attention over
a prefix that all sequences share and a suffix of each one's own (`attn`), the
choice of the next token from the logits (`sample`), and moving rows between
the sequences' cache slots (`move`). `run` computes them with elementary torch
operations in 32 bits (64 for the choice of a token, where a rounding error next
to a border changes the answer), or, where `own` is true, with the package.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # the tiny Llama (6/2 heads of 48), two sequences just after a short
        # common prompt: launch latency
        dict(name="attn_tiny_f32", op="attn", n=2, heads=6, kv_heads=2, hd=48, prefix=40, slot_len=16, q="f32",
             kv="f32"),
        # the 7B shape, 32 sequences behind a 1024-token system prompt, the
        # f32 cache that batched steps keep
        dict(name="attn_7b_f32", op="attn", n=32, heads=32, kv_heads=8, hd=128, prefix=1024, slot_len=256, q="f32",
             kv="f32"),
        # the 70B shape, 32 sequences behind a long document, f16 cache
        dict(name="attn_70b_f16", op="attn", n=32, heads=64, kv_heads=8, hd=128, prefix=8192, slot_len=512, q="f32",
             kv="f16"),
        # 64 sequences (the largest batch) behind a very long document, bf16 throughout
        dict(name="attn_70b_bf16_long", op="attn", n=64, heads=64, kv_heads=8, hd=128, prefix=32768, slot_len=1024,
             q="bf16", kv="bf16"),
        # odd sizes: 17 sequences, 12 heads in groups of 3, heads of 80, a
        # prefix that ends inside a tile
        dict(name="attn_odd_f16", op="attn", n=17, heads=12, kv_heads=4, hd=80, prefix=777, slot_len=333, q="f16",
             kv="f16"),
        # one sequence's next token, the 7B vocabulary, all three truncations
        dict(name="sample_one", op="sample", n=1, vocab=32000, pad=0, type="f32", kind="k_p_min"),
        # a batch of 32 with nucleus sampling
        dict(name="sample_7b_p", op="sample", n=32, vocab=32000, pad=0, type="f32", kind="p"),
        # the largest batch and vocabulary, every request with its own settings
        dict(name="sample_70b_mixed", op="sample", n=64, vocab=128256, pad=0, type="f32", kind="mixed"),
        # bf16 logits (many exact ties) with an odd vocabulary in padded rows
        dict(name="sample_odd_bf16", op="sample", n=7, vocab=32003, pad=61, type="bf16", kind="k_p"),
        # one short prompt of the tiny Llama into a second slot: launch latency
        dict(name="move_tiny", op="move", slots=4, layers=6, rows=256, width=96, type="f32", kind="fork", live=2,
             most=30),
        # one 512-token prompt forked into 31 more slots (8 layers of the 7B shape)
        dict(name="move_fork", op="move", slots=32, layers=8, rows=1024, width=1024, type="f32", kind="fork", live=32,
             most=512),
        # 64 slots, 40 of them still generating, moved to the front (f16 cache)
        dict(name="move_compact_f16", op="move", slots=64, layers=8, rows=1024, width=1024, type="f16",
             kind="compact", live=40, most=1000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "sample", "move"])
    if op == "attn":
        heads, kv_heads, hd = rng.choice([(6, 2, 48), (32, 8, 128), (64, 8, 128), (12, 4, 80), (8, 8, 64),
                                          (16, 2, 96), (28, 4, 128)])
        q, kv = rng.choice([("f32", "f32"), ("f32", "f16"), ("f16", "f16"), ("bf16", "bf16")])
        return dict(op="attn", n=_log(rng, 1, 64), heads=heads, kv_heads=kv_heads, hd=hd,
                    prefix=rng.choice([0, 1]) * rng.randint(1, 100) if rng.random() < 0.2 else _log(rng, 16, 20000),
                    slot_len=_log(rng, 1, 1024), q=q, kv=kv)
    if op == "sample":
        return dict(op="sample", n=_log(rng, 1, 64), vocab=_log(rng, 500, 128256), pad=rng.choice([0, 0, 1, 24, 61]),
                    type=rng.choice(["f32", "f32", "f16", "bf16"]), kind=rng.choice(["k_p_min", "p", "k_p", "t", "mixed"]))
    slots = rng.randint(2, 48)
    rows = _log(rng, 16, 1000)
    return dict(op="move", slots=slots, layers=rng.randint(1, 8), rows=rows, width=rng.choice([96, 128, 512, 1024]),
                type=rng.choice(["f32", "f16"]), kind=rng.choice(["fork", "compact"]), live=rng.randint(2, slots),
                most=rng.randint(1, rows))


def _rng(case, seed):
    return np.random.default_rng(seed)


def _lens(case, seed):
    """Rows of each sequence (attn) or of each move (move), on the host."""
    r = _rng(case, seed)
    if case["op"] == "attn":
        return r.integers(0, case["slot_len"] + 1, case["n"])
    if case["kind"] == "fork":
        return np.full(case["live"] - 1, case["most"])
    return r.integers(max(1, case["most"] // 4), case["most"] + 1, case["live"])


def _moves(case, seed):
    """(source slot, destination slot) of each move: one prompt to other slots,
    or the live slots to the front in their order."""
    r = np.random.default_rng(seed + 1)
    if case["kind"] == "fork":
        p = r.permutation(case["slots"])[: case["live"]]
        return [int(p[0])] * (len(p) - 1), [int(x) for x in p[1:]]
    return sorted(int(x) for x in r.permutation(case["slots"])[: case["live"]]), list(range(case["live"]))


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, dtype=torch.float32, scale=1.0):
        x = torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=g)
        return x.mul_(scale) if scale != 1.0 else x

    s = dict(op=case["op"])
    if case["op"] == "attn":
        n, kvh, hd, qt, kt = case["n"], case["kv_heads"], case["hd"], TYPES[case["q"]], TYPES[case["kv"]]
        s["q"] = normal(n, case["heads"], hd, dtype=qt, scale=2.0)
        s["kp"], s["vp"] = normal(case["prefix"], kvh, hd, dtype=kt), normal(case["prefix"], kvh, hd, dtype=kt)
        s["k"], s["v"] = (normal(n, case["slot_len"], kvh, hd, dtype=kt) for _ in range(2))
        s["slots"] = torch.from_numpy(np.random.default_rng(seed + 1).permutation(n).astype(np.int32)).cuda()
        s["lens"] = torch.from_numpy(_lens(case, seed).astype(np.int32)).cuda()
    elif case["op"] == "sample":
        n, v = case["n"], case["vocab"]
        spread = torch.empty(n, 1, device="cuda").uniform_(1.5, 4.0, generator=g)
        full = (normal(n, v + case["pad"]) * spread).to(TYPES[case["type"]])
        s["logits"] = full[:, :v]
        s["u"] = torch.rand(n, device="cuda", generator=g)
        kind = case["kind"]
        s["temperature"], s["top_k"], s["top_p"], s["min_p"] = dict(
            k_p_min=(0.8, 200, 0.95, 0.02), p=(1.0, 0, 0.9, 0.0), k_p=(0.7, 50, 0.9, 0.0), t=(1.1, 0, 1.0, 0.0),
            mixed=(1.0, 0, 1.0, 0.0))[kind]
        if kind == "mixed":  # greedy, plain temperature, top-k, nucleus and min-p requests side by side
            r = np.random.default_rng(seed + 1)
            kinds = r.integers(0, 5, n)
            t = np.where(kinds == 0, 0.0, r.uniform(0.3, 1.5, n))
            k = np.where(kinds == 2, np.exp(r.uniform(0, math.log(2000), n)).astype(np.int64), 0)
            p = np.where(kinds == 3, r.uniform(0.3, 0.99, n), 1.0)
            m = np.where(kinds == 4, r.uniform(0.005, 0.3, n), 0.0)
            s["temperature"], s["top_p"], s["min_p"] = (torch.tensor(x, dtype=torch.float32, device="cuda")
                                                        for x in (t, p, m))
            s["top_k"] = torch.tensor(k, dtype=torch.int32, device="cuda")
    else:
        shape = (case["slots"], case["layers"], case["rows"], case["width"])
        s["caches"] = [normal(*shape, dtype=TYPES[case["type"]]) for _ in range(2)]
        s["src"], s["dst"] = _moves(case, seed)
        s["lens"] = [int(x) for x in _lens(case, seed)]
    return s


def _attn(s):
    q, kp, vp = s["q"].float(), s["kp"].float(), s["vp"].float()
    slots, lens = s["slots"].long(), s["lens"].long()
    k, v = s["k"][slots].float(), s["v"][slots].float()  # [n, T, kv_heads, hd]
    n, h, hd = q.shape
    kvh, t = k.shape[2], k.shape[1]
    q = q.view(n, kvh, h // kvh, hd) * (1.0 / math.sqrt(hd))
    live = (torch.arange(t, device=q.device)[None, :] < lens[:, None])[:, :, None, None]
    sp = torch.einsum("nkgd,pkd->nkgp", q, kp)
    ss = torch.einsum("nkgd,ntkd->nkgt", q, k)
    ss = torch.where(live.permute(0, 2, 3, 1), ss, torch.full_like(ss, -math.inf))
    top = torch.maximum(sp.amax(-1) if sp.shape[-1] else torch.full_like(ss[..., 0], -math.inf), ss.amax(-1))
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)[..., None]
    ep, es = torch.exp(sp - top), torch.exp(ss - top)
    z = ep.sum(-1) + es.sum(-1)
    o = torch.einsum("nkgp,pkd->nkgd", ep, vp) + torch.einsum("nkgt,ntkd->nkgd", es, torch.where(live, v, torch.zeros_like(v)))
    o = torch.where(z[..., None] > 0, o / z[..., None], torch.zeros_like(o))  # no key at all: zeros
    return o.view(n, h, hd).to(s["q"].dtype)


def _column(x, like, dtype):
    return (x if torch.is_tensor(x) else torch.full((like.shape[0],), x, dtype=torch.float32, device=like.device)).to(dtype)[:, None]


def _sample(s):
    lg = s["logits"].double()
    t, p, m = (_column(s[k], lg, torch.float32).double() for k in ("temperature", "top_p", "min_p"))
    k = _column(s["top_k"], lg, torch.long)
    lg, order = torch.sort(lg, dim=-1, descending=True, stable=True)  # equal logits: the lowest index first
    rank = torch.arange(lg.shape[1], device=lg.device)[None, :]
    d = lg - lg[:, :1]
    w = torch.where(t > 0, torch.exp(d / torch.where(t > 0, t, torch.ones_like(t))), (rank == 0).double())
    w = torch.where((k > 0) & (rank >= k), torch.zeros_like(w), w)
    cum = torch.cumsum(w, -1)
    w = torch.where((p < 1) & (rank > 0) & (cum - w >= p * cum[:, -1:]), torch.zeros_like(w), w)
    w = torch.where(w < m, torch.zeros_like(w), w)
    cum = torch.cumsum(w, -1)
    at = ((cum <= s["u"].double()[:, None] * cum[:, -1:]).sum(-1, keepdim=True)).clamp_(max=lg.shape[1] - 1)
    prob = torch.gather(w, 1, at) / cum[:, -1:]
    return torch.gather(order, 1, at)[:, 0].int(), prob[:, 0].float()


def _move(s):
    lens = torch.tensor(s["lens"], device="cuda")
    total = sum(s["lens"])
    which = torch.repeat_interleave(torch.arange(len(s["lens"]), device="cuda"), lens, output_size=total)
    row = torch.arange(total, device="cuda") - (torch.cumsum(lens, 0) - lens)[which]
    src, dst = torch.tensor(s["src"], device="cuda")[which], torch.tensor(s["dst"], device="cuda")[which]
    for c in s["caches"]:  # K and V; the right-hand side is read before anything is written
        c[dst, :, row] = c[src, :, row]
    return s["caches"]


def run(state):
    if own:
        import talos_b200 as talos

        if state["op"] == "attn":
            return talos.attention_shared_dev(state["q"], state["kp"], state["vp"], state["k"], state["v"],
                                              state["slots"], state["lens"])
        if state["op"] == "sample":
            return talos.sample_dev(state["logits"], state["u"], temperature=state["temperature"],
                                    top_k=state["top_k"], top_p=state["top_p"], min_p=state["min_p"])
        talos.kv_move_dev(state["caches"], state["src"], state["dst"], state["lens"])
        return state["caches"]
    return dict(attn=_attn, sample=_sample, move=_move)[state["op"]](state)


def work(case):
    if case["op"] == "attn":
        size = dict(f32=4, f16=2, bf16=2)
        h, kvh, hd, n = case["heads"], case["kv_heads"], case["hd"], case["n"]
        keys = n * case["slot_len"] / 2  # on average
        return dict(bytes=2 * (case["prefix"] + keys) * kvh * hd * size[case["kv"]] + 2 * n * h * hd * size[case["q"]],
                    flops=4 * h * hd * (n * case["prefix"] + keys))
    if case["op"] == "sample":
        size = dict(f32=4, f16=2, bf16=2)[case["type"]]
        return dict(bytes=case["n"] * case["vocab"] * size, flops=4 * case["n"] * case["vocab"])
    row = case["layers"] * case["width"] * 2 * dict(f32=4, f16=2)[case["type"]]  # K and V of one position
    if case["kind"] == "fork":
        return dict(bytes=row * case["most"] * case["live"], flops=0)
    return dict(bytes=2 * row * (max(1, case["most"] // 4) + case["most"]) / 2 * case["live"], flops=0)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attn":  # one sequence at a time, its keys in one list
        q, kp, vp = s["q"].double(), s["kp"].double(), s["vp"].double()
        n, h, hd = q.shape
        out = torch.zeros(n, h, hd, dtype=torch.float64, device="cuda")
        group = h // kp.shape[1]
        for i, (slot, keep) in enumerate(zip(s["slots"].tolist(), s["lens"].tolist())):
            k = torch.cat([kp, s["k"][slot, :keep].double()])
            v = torch.cat([vp, s["v"][slot, :keep].double()])
            if not len(k):
                continue
            for j in range(k.shape[1]):
                a = torch.softmax(q[i, j * group:(j + 1) * group] @ k[:, j].T / hd ** 0.5, -1)
                out[i, j * group:(j + 1) * group] = a @ v[:, j]
        return out
    if case["op"] == "sample":
        lg, u = s["logits"].double().cpu().numpy(), s["u"].double().cpu().numpy()
        n, vocab = lg.shape

        def each(x):
            return (x.double().cpu().numpy() if torch.is_tensor(x) else np.full(n, np.float32(x))).astype(np.float64)

        t, k, p, m = (each(s[x]) for x in ("temperature", "top_k", "top_p", "min_p"))
        tokens, probs = np.zeros(n, np.int32), np.zeros(n)
        for i in range(n):
            order = np.argsort(-lg[i], kind="stable")
            if t[i] == 0:
                tokens[i], probs[i] = order[0], 1.0
                continue
            order = order[: int(k[i])] if k[i] > 0 else order
            w = np.exp((lg[i][order] - lg[i][order[0]]) / t[i])
            if p[i] < 1:
                w = w[: int(np.searchsorted(np.cumsum(w), p[i] * w.sum())) + 1]
            w = w[w >= m[i]]
            c = np.cumsum(w)
            j = min(int(np.searchsorted(c, u[i] * c[-1], side="right")), len(w) - 1)
            tokens[i], probs[i] = order[j], w[j] / c[-1]
        return tokens, probs
    new = [c.clone() for c in s["caches"]]
    for a, b, keep in zip(s["src"], s["dst"], s["lens"]):
        for c, to in zip(s["caches"], new):
            to[b, :, :keep] = c[a, :, :keep]
    return new
