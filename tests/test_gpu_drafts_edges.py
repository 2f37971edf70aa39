"""Acceptance of drafted tokens where logits are no ordinary numbers, on rows that the way through the tree is shown to reach; outputs next to inputs."""
import numpy as np
import pytest
import torch

import avelang_amd as ave
from tests import attention_helpers as A
from tests import draft_helpers as D
from tests.test_gpu_drafts import _draft, _parents, _verify

pytestmark = pytest.mark.gpu


def _visited(d, want):
    """Rows of the nodes that are kept."""
    return {int(d["cu"][b] + j) for b, n in enumerate(want[0]) for j in want[1][d["cu"][b]:d["cu"][b] + n]}


def _likeliest(d, nodes):
    """Every node is the first child of the one before and has the token that its parent's row prefers, so that small random numbers accept all of them."""
    for b in range(len(d["cu"]) - 1):
        for j in range(1, nodes):
            x = d["logits"][d["cu"][b] + j - 1]
            d["tokens"][d["cu"][b] + j] = int(np.argmax(np.where(np.isnan(x), -np.inf, x)))
            d["parents"][d["cu"][b] + j] = j - 1


#: what a row of at least 7 tokens holds beside ordinary logits: (where, what)
ODD = [[(3, np.nan)], [(0, np.nan)], [(-1, np.nan)], [(5, np.inf)], [(5, np.inf), (-3, np.inf)], [(2, np.nan), (6, np.inf)], [(1, np.nan), (4, -np.inf)],
       [(slice(0, None, 2), np.nan)], [(slice(1, None, 2), -np.inf), (0, np.nan)], [(slice(0, -2), np.nan)]]


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("vocab", [7, 700, 20011])
@pytest.mark.parametrize("chain", [1, 4])
def test_nan_and_infinity_among_numbers(gpu, chain, vocab, f32, probs):
    """A NaN counts as -inf, +inf as the largest number, in rows that are only drawn from (one node) and in rows whose children are accepted (four)."""
    seen = set()
    for shift in range(0, len(ODD), chain):
        d = _draft(41 + shift, [chain] * 8, vocab, chain=True, f32=f32, probs=probs)
        for row in range(8 * chain):
            for at, value in ODD[(row + shift) % len(ODD)]:
                d["logits"][row, at] = value
        _likeliest(d, chain)
        first = np.arange(0, 8 * chain, chain)
        numbers = d["uniform"][first].copy()
        d["uniform"] *= np.float32(2.0 ** -14)      # accepted
        d["uniform"][first] = numbers               # drawn
        want = _verify(gpu, d, [1.0, 0.6, 1.4, 1.0, 0.3, 1.0, 1.0, 2.0])
        seen |= {(row + shift) % len(ODD) for row in _visited(d, want)}
        assert chain == 1 or (want[0] > 2).sum() >= 6
    assert seen == set(range(len(ODD)))


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("f32", [False, True])
def test_children_without_a_number(gpu, f32, probs):
    """A child whose token has a NaN for a logit is never accepted, whatever its random number, and its elder or younger sibling is."""
    d = _draft(51, [4] * 8, 900, f32=f32, probs=probs)
    for b in range(8):
        r = slice(4 * b, 4 * b + 4)
        d["parents"][r] = [-1, 0, 0, 2 - b % 2]
        order = np.argsort(-d["logits"][4 * b], kind="stable")
        d["tokens"][r] = [0, order[0], order[1], order[2]]
        d["logits"][4 * b, order[b % 2]] = np.nan
        d["logits"][4 * b + 2 - b % 2, order[2]] = np.nan
        if probs:
            d["probs"][4 * b, order[:2]] = 2.0 ** -10
        d["uniform"][r] = [d["uniform"][4 * b], 0.0, 0.0, 0.0] if b < 4 else [d["uniform"][4 * b], 1e-6, 1e-6, 1e-6]
    want = _verify(gpu, d, [1.0, 0.7] * 4)
    assert (want[0] == 2).all() and {int(want[1][4 * b + 1]) for b in range(8)} == {1, 2}


@pytest.mark.parametrize("mask", ["lowest", -1.0e30, -4096.0])
@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("vocab", [12, 3001, 20011])
def test_finite_masks(gpu, vocab, f32, probs, mask):
    """Logits so low that in 64 bits nothing is left of them (e^-745 and less) are neither drawn nor accepted: not by a random number of 0, and not where
    all other tokens have been rejected, which leaves nothing, so that the token comes from the whole row."""
    low = float(np.finfo(np.float32).min if f32 else -np.float32(2 - 2 ** -7) * 2.0 ** 127) if mask == "lowest" else mask
    allowed = [3, vocab - 4]
    d = _draft(61, [3] * 6, vocab, f32=f32, probs=probs)
    d["logits"][:, :3] = d["logits"][:, -3:] = low
    for b in range(6):
        r = slice(3 * b, 3 * b + 3)
        d["parents"][r] = [-1, 0, 0]
        if b < 2:                            # children whose tokens are masked, drawn by 0
            d["tokens"][r], d["uniform"][r] = [0, 1, vocab - 1], 0.0
            if probs:
                d["probs"][r, [0, 1, vocab - 1]] = 0.125
        else:                                # two tokens of a half each, both rejected
            d["logits"][r] = low
            d["logits"][r, allowed] = -1.5
            d["tokens"][r], d["uniform"][r] = [0, *allowed], [(0.0, 0.25, 0.5, 0.75)[b - 2], 1.0, 1.0]
            if probs:
                d["probs"][r] = 0.0
                d["probs"][r, allowed] = 0.5
    want = _verify(gpu, d, [1.0, 0.7, 1.0, 1.0, 0.5, 2.0])
    assert (want[0] == 1).all() and want[2][6::3].tolist() == [3, 3, vocab - 4, vocab - 4]


@pytest.mark.parametrize("number", [1.0, 3.0, np.inf])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("allowed", [2, 3, 9])
def test_a_number_of_one_accepts_nothing(gpu, allowed, f32, number):
    """No probability is above 1, not that of the last token that is left either, and a masked token behind it has none."""
    batch, nodes, vocab = 512, allowed + 2, 40
    d = _draft(62, [nodes] * batch, vocab, f32=f32)
    d["logits"][:, allowed:] = -np.inf
    d["parents"] = np.tile(np.array([-1] + [0] * (nodes - 1), np.int32), batch)
    d["tokens"] = np.tile(np.array([0, *range(allowed), vocab - 1], np.int32), batch)
    numbers = d["uniform"][::nodes].copy()
    d["uniform"][:] = number
    d["uniform"][::nodes] = numbers
    want = _verify(gpu, d, [1.0] * batch)
    assert (want[0] == 1).all()


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("vocab", [101, 2047, 9001, 140001])
def test_numbers_from_one_on_draw_the_last_token(gpu, vocab, probs):
    """No running sum is above the whole, however the two are rounded: the last token that has a weight."""
    batch = 64 if vocab > 1 << 16 else 512
    d = _draft(63, [1] * batch, vocab, f32=True, probs=probs, sharp=1.0)
    d["logits"][:, vocab - 7:] = -np.inf
    d["logits"][:, vocab - 8] = -60.0
    call = lambda uniform: ave.verify_draft(*(D.tensor(d[k], gpu) for k in ("logits", "tokens", "parents", "cu")), D.tensor(uniform, gpu), None,   # noqa: E731
                                            D.tensor(d["probs"], gpu) if probs else None)[2]
    for number in (1.0, 7.0, np.inf):
        assert call(np.full(batch, number, np.float32)).eq(vocab - 8).all()


def test_outputs_between_rows_of_logits(gpu):
    """What lies between rows belongs to nobody: outputs may be there, in rows of an input they may not."""
    d = _draft(71, [5, 4], 100, f32=True)
    rest = [D.tensor(d[k], gpu) for k in ("tokens", "parents", "cu", "uniform")]
    buffer = torch.zeros(9, 140, device=gpu)
    logits, between = buffer[:, :100], buffer.view(torch.int32)
    logits.copy_(D.tensor(d["logits"], gpu))
    want = ave.verify_draft(logits.contiguous(), *rest)
    outs = between[0, 100:102], between[3, 101:110], between[7, 131:140]
    got = ave.verify_draft(logits, *rest, accepted=outs[0], path=outs[1], emitted=outs[2])
    assert all(g.data_ptr() == o.data_ptr() and torch.equal(g, w) for g, o, w in zip(got, outs, want))
    for name, out in (("path", between[8, 99:108]), ("emitted", between.view(-1)[132:141]), ("path", between[2, :9])):
        with pytest.raises(ValueError, match="must not overlap"):
            ave.verify_draft(logits, *rest, **{name: out})


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("border", [False, True])
def test_sampled_with_much_to_read(gpu, border, f32):
    """Rows of more than 64 MB, sampled from: sums of node 0's rows and of those behind the accepted child decide, at several temperatures, in sequences of fewer
    and of more than 64 nodes.  `border`: numbers of children are the fp32 ones nearest to the probabilities that they are compared with."""
    rng = np.random.default_rng(81)
    counts, temps = [80, 9, 14, 1, 12, 20], [1.0, 0.7, 1.3, 1.0, 0.5, 0.9]
    d = _draft(81, counts, 300007, chain=True, f32=f32)
    assert len(d["tokens"]) * 300007 * (4 if f32 else 2) > 64 << 20 and len(d["tokens"]) >= 3 * len(counts)
    exact = {}
    for b, n in enumerate(counts):
        first = d["cu"][b]
        for j in range(1, n):
            # nodes 1 and 2 hang at node 0, 3 and 4 at 2, 5 and 6 at 4: the first has its parent's second token, the other one the first
            d["parents"][first + j] = j - 1 if j % 2 else j - 2
            x = d["logits"][first + d["parents"][first + j]]
            order = np.argpartition(-x, 3)[:4]
            order = order[np.argsort(-x[order], kind="stable")]
            d["tokens"][first + j] = order[j % 2]
            if j % 2 and (not border or b % 2):
                d["uniform"][first + j] = 0.9
            elif not border or j > 6:
                d["uniform"][first + j] *= np.float32(2.0 ** -10)
            else:
                p = D.softmax(x, temps[b])[order]
                exact[first + j] = p[1] if j % 2 else p[0] / (1 - p[1])
                d["uniform"][first + j] = exact[first + j]
    assert all(abs(float(d["uniform"][i]) - e) <= 2.0 ** -24 * e for i, e in exact.items()) and len(exact) == (24 if border else 0)
    want = _verify(gpu, d, temps, extra=2)
    if border:
        assert 2 in want[0] and want[0].max() > 4, want[0]
    else:
        assert want[0][0] > 33 and (want[0][[1, 2, 4, 5]] > 3).all(), want[0]   # (the 64 first nodes and more)


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("vocab", [140001, 600011])
def test_pieces_without_a_number(gpu, vocab, probs):
    """Rows most of whose vocabulary is -inf or NaN, in front, in the middle or behind, more pieces than are looked at together: drawn from, and accepted from."""
    rng = np.random.default_rng(91)
    seen = set()
    for chain in (1, 3):
        d = _draft(91 + chain, [chain] * 6, vocab, chain=True, f32=True)
        for row, x in enumerate(d["logits"]):
            what = np.nan if row % 2 else -np.inf
            if row % 3 == 0:
                x[:8192 * 16] = what
            elif row % 3 == 1:
                x[8192:] = what
            else:
                x[100:vocab - 100] = what
        _likeliest(d, chain)
        if probs:
            d["probs"] = np.stack([D.softmax(x + rng.standard_normal(vocab), 1.0) for x in d["logits"]]).astype(np.float32)
        first = np.arange(0, 6 * chain, chain)
        numbers = d["uniform"][first].copy()
        d["uniform"] *= np.float32(2.0 ** -14)
        d["uniform"][first] = numbers
        want = _verify(gpu, d, [1.0, 0.6, 2.0, 1.0, 0.8, 0.0], extra=1)
        assert (want[0] == chain).all()
        seen |= {row % 6 for row in _visited(d, want)}
    assert seen == set(range(6))


# ---- attention ------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("nodes", [1, 8, 20, 70])
@pytest.mark.parametrize("window", [0, 200])
def test_tables_wide_enough_for_units_beyond_32_bits(gpu, d, nodes, window):
    """The width of the page table alone decides how units are numbered, so that short sequences reach the 64-bit forms: of few rows, of blocks of 64 rows
    and of 128.  (With a window units are few, and 32 bits do.)"""
    hq, hkv, page = 16, 8, 4096
    rows = [(nodes, nodes + 290 - 17 * i) for i in range(14)] + [(nodes, 1500), (0, 9), (nodes, nodes), (min(nodes, 3), 64)]
    pages = (1 << 31) // page - 1
    tokens = sum(n for n, _ in rows)
    assert min(2 * tokens // 128 + len(rows), 2 * tokens) * hkv * (pages * page // 64) > 1 << 32
    batch = A.Batch(rows, hq, hkv, d, page, seed=nodes)
    t = batch.tensors(gpu)
    wide = torch.full((len(rows), pages), 1 << 30, dtype=torch.int32, device=gpu)
    wide[:, :t["page_table"].shape[1]] = t["page_table"]
    above = [D.ancestors(p) for p in _parents(batch, 7)]
    seen = D.tensor(np.concatenate([D.words_of(a, 2) for a in above]), gpu)
    want, want_lse, tol, lse_tol = D.masked_reference(batch, [D.visible(a, k, window) for a, (_, k) in zip(above, batch.rows)], sinks=batch.sinks)
    lse = torch.full(batch.q.shape[:2], float("nan"), device=gpu)
    out = torch.full(batch.q.shape, float("nan"), dtype=torch.bfloat16, device=gpu)
    ave.tree_attention_mxfp4(t["q"], t["cache"], wide, t["seq_lens"], t["cu_q"], seen, out, lse, max_q=nodes, window=window, sinks=D.tensor(batch.sinks, gpu))
    err = np.abs(out.float().cpu().numpy() - want)
    assert (err <= tol).all(), float((err / tol).max())
    assert (np.abs(lse.cpu().numpy() - want_lse) <= lse_tol).all()
