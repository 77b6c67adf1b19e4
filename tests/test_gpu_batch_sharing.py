"""A batch that starts from one prompt: the prefix kept and read once
(talos_batch_share), rows moved between cache slots (talos_batch_move), drawn
tokens (talos_generate_batch_sample). Bars as for batched decode without them:
logits within 1e-3 max-abs of one oracle model per sequence, greedy tokens
identical, reruns bit-identical."""
import numpy as np
import pytest

import oracle
from talos_b200 import Model, gguf, synth
from talos_b200._lib import TalosError

from .helpers import prompt, tiny_model
from .test_gpu_sample import choose

pytestmark = pytest.mark.gpu

SHAPE_GQA = synth.Shape(n_embd=512, n_layer=2, n_head=4, n_head_kv=2, n_ff=768, vocab=512, ctx=128)


def oracle_logits(data, toks):
    """Logits after each token of one sequence."""
    cpu = oracle.Model(data=data)
    return [cpu.forward(int(t), p).copy() for p, t in enumerate(toks)]


def load(data, n):
    m = Model.load_bytes(data)
    m.set_batch(n)
    return m


@pytest.mark.parametrize("n_prefix", [1, 37, 64, 150])
def test_shared_prefix_matches_one_oracle_per_sequence(n_prefix):
    """Suffixes of 1 .. 7 tokens behind one prefix, one of them prefilled in one call."""
    data = tiny_model(gguf.Q8_0)
    head = prompt(n_prefix, 4096, 3)
    tails = [prompt(7, 4096, 50 + i) for i in range(5)]
    want = [oracle_logits(data, list(head) + list(t))[n_prefix:] for t in tails]
    m = load(data, 5)
    m.prefill_slot(2, head)  # any slot
    m.batch_share(2, n_prefix)
    last = m.prefill_slot(4, tails[4][:6], n_prefix)
    assert np.max(np.abs(last - want[4][5])) <= 1e-3
    for k in range(6):
        lg = m.forward_batch([t[k] for t in tails[:4]], [n_prefix + k] * 4)
        for i in range(4):
            assert np.max(np.abs(lg[i] - want[i][k])) <= 1e-3, f"sequence {i}, position {k}"
    lg = m.forward_batch([t[6] for t in tails], [n_prefix + 6] * 5)
    assert max(np.max(np.abs(lg[i] - want[i][6])) for i in range(5)) <= 1e-3
    again = m.forward_batch([t[6] for t in tails], [n_prefix + 6] * 5)
    assert np.array_equal(lg, again)
    m.close()


def test_shared_prefix_gqa_long_chunks():
    """Heads that share a kv head, head_dim 128; a suffix of more positions than a
    cache tile, in one prefill, and a batch of 40 sequences (two token tiles)."""
    data = synth.llama_bytes(SHAPE_GQA, 8, wtype=gguf.Q8_0, out_type=gguf.Q6_K)
    head, tail = prompt(20, 512, 5), prompt(90, 512, 6)
    want = oracle_logits(data, list(head) + list(tail))
    m = load(data, 40)
    m.prefill_slot(0, head)
    m.batch_share(0, 20)
    last = m.prefill_slot(39, tail, 20)
    assert np.max(np.abs(last - want[-1])) <= 1e-3
    lg = m.forward_batch([tail[0]] * 39, [20] * 39)
    assert np.max(np.abs(lg - want[20])) <= 1e-3
    lg = m.forward_batch([tail[1]] * 39 + [tail[89]], [21] * 39 + [109])
    assert np.max(np.abs(lg[:39] - want[21])) <= 1e-3 and np.max(np.abs(lg[39] - want[-1])) <= 1e-3
    m.close()


def test_prefix_extended_cut_and_dropped():
    data = tiny_model(gguf.Q4_0)
    toks, other = prompt(60, 4096, 8), prompt(12, 4096, 9)
    want = oracle_logits(data, toks)
    m = load(data, 3)
    m.prefill_slot(1, toks[:20])
    m.batch_share(1, 20)
    last = m.prefill_slot(0, toks[20:50], 20)  # slot 0 goes on behind the prefix
    assert np.max(np.abs(last - want[49])) <= 1e-3
    m.batch_share(0, 50)  # and its rows extend it
    lg = m.forward_batch([toks[50]] * 3, [50] * 3)
    assert np.max(np.abs(lg - want[50])) <= 1e-3
    m.batch_share(0, 10)  # cut: the rows behind are read from the slots; slot 1 has its own 10 .. 19
    cut = oracle_logits(data, list(toks[:20]) + [other[0]])[-1]
    lg = m.forward_batch([5, other[0], 5], [10, 20, 10])
    assert np.max(np.abs(lg[1] - cut)) <= 1e-3
    m.batch_share(0, 0)  # no sharing: slot 1 holds all of its rows
    lg = m.forward_batch([5, other[0], 5], [0, 20, 0])
    assert np.max(np.abs(lg[1] - cut)) <= 1e-3
    m.close()


def test_shared_prefix_greedy_generation():
    data = tiny_model(gguf.Q8_0)
    head = prompt(45, 4096, 11)
    m = load(data, 4)
    m.prefill_slot(0, head)
    m.batch_share(0, 45)
    first = [7, 900, 31, 4000]
    gen = m.generate_batch_greedy(first, [45] * 4, 10)
    for i in range(4):
        cpu = oracle.Model(data=data)
        for p, t in enumerate(head):
            cpu.forward(int(t), p)
        t = first[i]
        for k in range(10):
            t = oracle.argmax(cpu.forward(int(t), 45 + k))
            assert int(gen[k, i]) == t, f"sequence {i}, step {k}"
    m.close()


SETTINGS = dict(temperature=[0.0, 1.0, 0.7, 1.3], top_k=[0, 0, 40, 0], top_p=[1.0, 1.0, 0.9, 0.95],
                min_p=[0.0, 0.0, 0.0, 0.05])


def drawn(lg, u):
    return [choose(lg[i], u[i], *(SETTINGS[k][i] for k in ("temperature", "top_k", "top_p", "min_p")))[0]
            for i in range(4)]


@pytest.mark.parametrize("n_prefix", [0, 33])
def test_sampled_generation_draws_from_the_steps_logits(n_prefix):
    """Each token is the definition's choice from the logits that stepping by hand gives
    (the same steps, bit for bit)."""
    data = tiny_model(gguf.Q4_0)
    rng = np.random.default_rng(12)
    u = rng.random((9, 4)).astype(np.float32)
    tok, pos = [3, 500, 77, 4095], [n_prefix] * 4
    runs = []
    for _ in range(2):
        m = load(data, 4)
        if n_prefix:
            m.prefill_slot(3, prompt(n_prefix, 4096, 13))
            m.batch_share(3, n_prefix)
        runs.append(m)
    got = runs[0].generate_batch_sample(tok, pos, u, **SETTINGS)
    for k in range(9):
        lg = runs[1].forward_batch(tok, pos)
        tok, pos = drawn(lg, u[k]), [p + 1 for p in pos]
        assert [int(x) for x in got[k]] == tok, f"step {k}"
    assert np.array_equal(runs[1].generate_batch_sample([3, 500, 77, 4095], [n_prefix] * 4, u, **SETTINGS), got)
    # one setting for all, no steps
    assert runs[0].generate_batch_sample(tok, pos, np.zeros((0, 4), np.float32)).shape == (0, 4)
    one = runs[0].generate_batch_sample(tok, pos, u[:3], temperature=0.0)
    assert np.array_equal(one, runs[1].generate_batch_greedy(tok, pos, 3))
    for m in runs:
        m.close()


def test_moved_slots_go_on_where_they_were():
    data = tiny_model(gguf.Q8_0)
    a, b = list(prompt(30, 4096, 14)), list(prompt(18, 4096, 15))
    nxt = [9, 10, 11]
    wa = [oracle_logits(data, a + [t])[-1] for t in nxt]
    wb = oracle_logits(data, b + [nxt[1]])[-1]
    m = load(data, 5)
    m.prefill_slot(0, a)
    m.prefill_slot(1, b)
    m.batch_move([(0, 2, 0, 30), (0, 3, 0, 30)])  # fork
    lg = m.forward_batch([nxt[0], nxt[1], nxt[1], nxt[2]], [30, 18, 30, 30])
    for got, want in zip(lg, [wa[0], wb, wa[1], wa[2]]):
        assert np.max(np.abs(got - want)) <= 1e-3
    m.batch_move([(0, 1, 0, 30), (1, 0, 0, 30)])  # exchange
    lg = m.forward_batch([nxt[1], nxt[0]], [18, 30])
    assert np.max(np.abs(lg[0] - wb)) <= 1e-3 and np.max(np.abs(lg[1] - wa[0])) <= 1e-3
    m.batch_move([])
    m.batch_move([(4, 4, 0, 10), (2, 1, 5, 0)])  # nothing to copy
    assert np.array_equal(m.forward_batch([nxt[1], nxt[0]], [18, 30]), lg)
    m.close()


def test_prefix_fork_sampling_and_compaction_together():
    """One prompt for six sequences, one of them forked after some tokens, two ended and
    the rest moved to the front: every logit of the live ones matches its own oracle."""
    data = tiny_model(gguf.Q4_0)
    head = list(prompt(70, 4096, 16))
    rng = np.random.default_rng(17)
    m = load(data, 6)
    m.prefill_slot(0, head[:69])
    m.batch_share(0, 69)
    n = 5
    seq = [[head[69]] for _ in range(n)]
    u = rng.random((6, n)).astype(np.float32)
    gen = m.generate_batch_sample([s[-1] for s in seq], [69] * n, u, temperature=1.1, top_k=300)
    for i in range(n):
        seq[i] += [int(x) for x in gen[:, i]]
    # the cache holds positions 69 .. 74 of each; the last token is not fed yet
    m.batch_move([(1, 5, 69, 6)])  # fork sequence 1
    seq.append(list(seq[1]))
    live = [5, 1, 4]  # 0, 2 and 3 have ended
    m.batch_move([(s, d, 69, 6) for d, s in enumerate(live)])
    seq = [seq[s] for s in live]
    seq[0][-1] = 123  # the fork takes another turn
    lg = m.forward_batch([s[-1] for s in seq], [75] * 3)
    for i in range(3):
        want = oracle_logits(data, head[:69] + seq[i])[-1]
        assert np.max(np.abs(lg[i] - want)) <= 1e-3, f"sequence {i}"
    gen = m.generate_batch_sample([s[-1] for s in seq], [75] * 3, rng.random((4, 3)), top_p=0.9)
    seq = [s + [int(x) for x in gen[:, i]] for i, s in enumerate(seq)]
    lg = m.forward_batch([s[-1] for s in seq], [79] * 3)
    for i in range(3):
        want = oracle_logits(data, head[:69] + seq[i])[-1]
        assert np.max(np.abs(lg[i] - want)) <= 1e-3, f"sequence {i}"
    m.close()


def test_refusals_leave_the_batch_as_it_was():
    data = tiny_model(gguf.Q4_0)
    m = Model.load_bytes(data)
    u = np.zeros((2, 1), np.float32)
    for call in (lambda: m.batch_share(0, 1), lambda: m.batch_move([(0, 0, 0, 1)]),
                 lambda: m.generate_batch_sample([1], [0], u)):
        with pytest.raises(TalosError):  # no slots
            call()
    m.set_batch(2)
    before = m.ctx.device_bytes()
    head = prompt(12, 4096, 18)
    m.prefill_slot(0, head)
    for call in (lambda: m.batch_share(2, 1), lambda: m.batch_share(-1, 1), lambda: m.batch_share(0, 257),
                 lambda: m.batch_move([(0, 2, 0, 1)]), lambda: m.batch_move([(0, 1, 0, 257)]),
                 lambda: m.batch_move([(0, 1, 256, 1)]), lambda: m.batch_move([(0, 1, 0, 1), (1, 1, 0, 1)]),
                 lambda: m.generate_batch_sample([1, 2, 3], [0, 0, 0], np.zeros((2, 3))),
                 lambda: m.generate_batch_sample([1], [255], u), lambda: m.generate_batch_sample([4096], [0], u),
                 lambda: m.generate_batch_sample([1], [0], u, top_k=-1)):
        with pytest.raises(TalosError):
            call()
    for call in (lambda: m.batch_move([(0, 1, 0)]), lambda: m.batch_move([(0, -1, 0, 1)]), lambda: m.batch_share(0, -1),
                 lambda: m.generate_batch_sample([1], [0], np.zeros(2)),
                 lambda: m.generate_batch_sample([1, 2], [0], np.zeros((2, 2)))):
        with pytest.raises(ValueError):
            call()
    m.batch_share(0, 12)
    assert m.ctx.device_bytes() > before
    for call in (lambda: m.forward_batch([1, 2], [12, 11]), lambda: m.prefill_slot(1, [1, 2], 11),
                 lambda: m.generate_batch_greedy([1], [0], 2), lambda: m.generate_batch_sample([1], [11], u)):
        with pytest.raises(TalosError):  # positions of the prefix
            call()
    want = oracle_logits(data, list(head) + [77])[-1]
    assert np.max(np.abs(m.forward_batch([77, 77], [12, 12]) - want)) <= 1e-3
    m.cap_context(64)  # releases the slots and the prefix with them
    m.set_batch(2)
    first = oracle_logits(data, [77])[-1]
    assert np.max(np.abs(m.forward_batch([77, 77], [0, 0]) - first)) <= 1e-3
    m.close()


def test_a_row_without_a_choice_ends_the_call():
    """NaN scales in the output matrix make every logit NaN."""
    data = tiny_model(gguf.Q8_0)
    m = load(data, 2)
    rows, cols = 4096, m.cfg.n_embd
    raw = np.zeros((rows * cols // 32, 34), np.uint8)
    raw[:, 1] = 0x7E  # f16 NaN
    m.ctx.upload("output.weight", raw.tobytes(), gguf.Q8_0, rows, cols)
    with pytest.raises(TalosError, match="device check"):
        m.generate_batch_sample([1, 2], [0, 0], np.full((3, 2), 0.5))
    m.close()


def test_sharing_another_prompt_is_refused_while_one_is_shared():
    """A slot filled with a prompt of its own before the sharing is not taken for a
    continuation of the shared one: naming it is refused, at equal, smaller and larger
    lengths, and the prefix stays; after the sharing ended it can be shared."""
    data = tiny_model(gguf.Q8_0)
    a, b = list(prompt(20, 4096, 21)), list(prompt(30, 4096, 22))
    m = load(data, 3)
    m.prefill_slot(0, a)
    m.prefill_slot(1, b)
    m.batch_share(0, 20)
    want = oracle_logits(data, a + [77])[-1]
    for n in (20, 30, 7):
        with pytest.raises(TalosError, match="INVALID_ARG"):
            m.batch_share(1, n)
        assert np.max(np.abs(m.forward_batch([77] * 3, [20] * 3) - want)) <= 1e-3
        m.batch_share(0, 0)  # slot 1's row 20 is the step's now: fill it again
        m.prefill_slot(1, b)
        m.batch_share(0, 20)
    m.batch_share(0, 0)
    m.batch_share(1, 30)
    want = oracle_logits(data, b + [78])[-1]
    assert np.max(np.abs(m.forward_batch([78] * 3, [30] * 3) - want)) <= 1e-3
    m.close()


def test_slots_that_may_be_named_while_a_prefix_is_shared():
    """The slot that it came from (to extend it, and back after another extended it), a reused
    slot that went on behind it, a fork of either; not a slot whose rows behind it are older."""
    data = tiny_model(gguf.Q4_0)
    a, b, tail = list(prompt(40, 4096, 23)), list(prompt(60, 4096, 24)), list(prompt(12, 4096, 25))

    def after(toks):
        return oracle_logits(data, toks + [99])[-1]

    def shares(want, n):
        assert np.max(np.abs(m.forward_batch([99] * 4, [n] * 4) - want)) <= 1e-3

    m = load(data, 6)
    m.prefill_slot(0, a)
    for s in (1, 2, 5):
        m.prefill_slot(s, b)
    m.batch_share(0, 25)
    m.prefill_slot(4, tail, 25)
    m.batch_share(0, 40)  # extended by its own rows
    shares(after(a), 40)
    m.batch_share(0, 25)  # cut
    m.prefill_slot(1, tail, 25)  # a reused slot goes on: rows 25 .. 36
    with pytest.raises(TalosError, match="INVALID_ARG"):
        m.batch_share(1, 38)  # its row 37 is an older prompt's
    m.batch_move([(1, 3, 25, 12), (1, 2, 0, 60)])
    with pytest.raises(TalosError, match="INVALID_ARG"):
        m.batch_share(2, 38)  # as the slot it was copied from
    m.batch_share(3, 37)  # a fork behind the prefix extends it
    shares(after(a[:25] + tail), 37)
    m.batch_share(1, 30)  # a slot that went on behind it cuts it
    shares(after(a[:25] + tail[:5]), 30)
    m.batch_share(0, 25)
    shares(after(a[:25]), 25)
    m.batch_move([(5, 0, 0, 60)])  # the first slot holds another prompt now
    with pytest.raises(TalosError, match="INVALID_ARG"):
        m.batch_share(0, 10)
    m.close()


def test_rows_behind_a_newly_written_position_are_older():
    """The slot that the prefix came from goes on with other tokens in the middle of its rows:
    the older rows behind them do not extend the prefix, the new ones do."""
    data = tiny_model(gguf.Q8_0)
    a = list(prompt(40, 4096, 26))
    m = load(data, 2)
    m.prefill_slot(0, a)
    m.batch_share(0, 25)
    m.generate_batch_greedy([7, 8], [25, 25], 1)
    with pytest.raises(TalosError, match="INVALID_ARG"):
        m.batch_share(0, 40)
    m.batch_share(0, 26)
    want = oracle_logits(data, a[:25] + [7, 9])[-1]
    assert np.max(np.abs(m.forward_batch([9, 9], [26, 26]) - want)) <= 1e-3
    # fed once more as it was, a position leaves nothing behind it in doubt
    m.batch_share(0, 0)
    m.prefill_slot(0, a)
    m.batch_share(0, 25)
    m.prefill_slot(0, a[39:], 39)
    m.batch_share(0, 40)
    want = oracle_logits(data, a + [9])[-1]
    assert np.max(np.abs(m.forward_batch([9, 9], [40, 40]) - want)) <= 1e-3
    m.close()
