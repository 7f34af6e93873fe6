"""Model.verify: a drafted tree through the model in one pass (rotation and append of its rows, tree attention, log
probabilities, acceptance), against decoding the same tokens one by one.

Tolerances. The projections of verify sum in another order than those of the decode step; rows of logits, and of the cache,
may differ by REL of their largest value, as for a prefilled prompt. A pick is right if no logit of the decode step passes it
by more than REL of the largest: each of the two moves by half of that at most. A log probability is a logit less the
log-sum-exp, and each moves by REL of the largest logit at most; the fp32 sum of V terms adds far less."""
import pytest
import torch

from helpers import DEV, gen

pytestmark = pytest.mark.gpu
REL = 2e-2


@pytest.fixture(scope="module")
def K():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from runtime import ext
    return ext.load()


def model(D=64, max_ctx=256, **cfg):
    from runtime.model import DecodeConfig, Model
    from runtime.synth import LlamaShape, SyntheticLlama
    shape = LlamaShape(256, 2, 4, 2, 512, 1000) if D == 64 else LlamaShape(512, 2, 4, 2, 1024, 1000)
    m = Model(SyntheticLlama(shape, seed=4, device=DEV, std=0.05), shape, DecodeConfig(max_ctx=max_ctx, device=DEV, **cfg))
    m.prepare(max_ctx)
    return m


def prompt(n, seed=1):
    return torch.randint(0, 1000, (n,), generator=gen(seed))


def rel(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    return ((a - b).abs().max() / b.abs().max()).item()


def rows(m, n):
    """K / V of the tokens 0 .. n - 1, [L, 2, n_kv, n, D]."""
    P = m.cfg.page
    return torch.cat([m.kv[:, :, int(m.bt[t // P]), :, t % P:t % P + 1] for t in range(n)], 3)


def checked_verify(m, draft, parents=None):
    """verify, and the same tokens decoded one by one from the same state; returns verify's. Leaves verify's state."""
    start, pending, kv = m.host_pos, int(m.tok), m.kv.clone()
    toks, logp = m.verify(draft, parents)
    n = len(toks)
    assert 1 <= n == len(logp) and m.host_pos == int(m.pos) == start + n and int(m.tok) == toks[-1]
    # the accepted drafts are a path of the tree that nothing in the tree continues
    up = [-1] + (list(range(len(draft))) if parents is None else list(parents))
    ids, node = [pending] + list(draft), 0
    for t in toks[:-1]:
        node = next(c for c in range(1, len(ids)) if up[c] == node and ids[c] == t)
    assert not any(up[c] == node and ids[c] == toks[-1] for c in range(1, len(ids)))
    got = (m.kv.clone(), m.logits.clone())
    m.kv.copy_(kv)
    m.reset(start)
    lf = m.teacher_force([pending] + toks[:-1], collect_logits=True).double()
    big = lf.abs().max(1).values
    for i, t in enumerate(toks):
        assert lf[i].max() - lf[i, t] <= REL * big[i], (i, t)
        want = torch.log_softmax(lf[i], 0)[t]
        assert abs(logp[i] - want.item()) <= 2 * REL * big[i].item(), i
    assert rel(got[1], lf[-1]) <= REL
    want = rows(m, start + n)
    m.kv.copy_(got[0])
    assert rel(rows(m, start + n), want) <= REL
    assert torch.equal(rows(m, start), rows_before(kv, m, start))
    m.tok.fill_(toks[-1])
    m.logits.copy_(got[1])
    return toks, logp


def rows_before(kv, m, n):
    keep, m.kv = m.kv, kv
    out = rows(m, n)
    m.kv = keep
    return out


def greedy(m, n):
    """The next n tokens of greedy decoding and their margins over the second in units of the largest logit, the state kept."""
    start, tok, kv = m.host_pos, m.tok.clone(), m.kv.clone()
    out, margin = [], []
    for _ in range(n):
        m.run_step()
        out.append(int(m.tok))
        top = m.logits.double().topk(2).values
        margin.append(((top[0] - top[1]) / m.logits.double().abs().max()).item())
    m.kv.copy_(kv)
    m.tok.copy_(tok)
    m.reset(start)
    return out, margin


def branching(path, extra, seed):
    """A tree with `path` in it, among `extra` wrong tokens hung on its nodes and on one another; (draft, parents)."""
    g = gen(seed)
    draft, parents, at = [], [], 0
    for i, t in enumerate(path):
        for _ in range(extra // max(1, len(path))):
            draft.append((t + 1 + int(torch.randint(0, 900, (1,), generator=g))) % 1000)
            parents.append(at if torch.rand(1, generator=g) < 0.5 else int(torch.randint(0, len(draft), (1,), generator=g)))
        draft.append(t)
        parents.append(at)
        at = len(draft)
    return draft, parents


@pytest.mark.parametrize("D", (64, 128))
@pytest.mark.parametrize("start,accept,extra", ((1, 1, 0), (45, 4, 12), (130, 5, 75), (16, 3, 60)))
def test_verify_tree(K, D, start, accept, extra):
    m = model(D)
    m.reset(0)
    m.prefill(prompt(start))
    path, margin = greedy(m, accept)
    sure = next((i for i, x in enumerate(margin) if x <= 2 * REL), accept)
    toks, _ = checked_verify(m, *branching(path, extra, seed=start))
    assert len(toks) >= sure + (sure == accept) and toks[:sure] == path[:sure]
    # decoding goes on from there, by the captured step
    ref, _ = greedy(m, 1)
    m.run_step()
    assert int(m.tok) == ref[0] and m.host_pos == start + len(toks) + 1


@pytest.mark.parametrize("weights,head", (("int4", "int4"), ("int4", "fp16"), ("fp16", "fp16")))
def test_verify_chain(K, weights, head):
    m = model(64, weights=weights, lm_head=head)
    m.reset(0)
    m.prefill(prompt(21, seed=3))
    checked_verify(m, [])                                  # the pending token alone: one step
    path, margin = greedy(m, 4)
    toks, _ = checked_verify(m, path)
    sure = next((i for i, x in enumerate(margin) if x <= 2 * REL), 4)
    assert toks[:sure] == path[:sure]
    wrong = [(t + 1) % 1000 for t in greedy(m, 1)[0]]
    n = len(checked_verify(m, wrong * 3)[0])
    assert n >= 1


def test_verify_generates_as_greedy_decoding(K):
    """A whole generation: drafts from a lookup of the last token among those so far, in trees and chains by turns, over page
    and word boundaries; every emitted token is checked against decoding in checked_verify."""
    m = model(128)
    m.reset(0)
    seq = prompt(40, seed=8).tolist()
    m.prefill(seq)
    seq.append(int(m.tok))
    turn = 0
    while len(seq) < 120:
        after = [i + 1 for i in range(len(seq) - 1) if seq[i] == seq[-1]][-3:]
        runs = [seq[i:i + 4] for i in after] + [greedy(m, 3)[0]]
        if turn % 2:
            draft, parents = runs[-1], None
        else:
            draft, parents = [], []
            for r in runs:
                for j, t in enumerate(r):
                    parents.append(len(draft) if j else 0)
                    draft.append(t)
        seq += checked_verify(m, draft, parents)[0]
        turn += 1
    assert m.host_pos == int(m.pos) == len(seq) - 1


def test_captured_verify_replays(K):
    """Two recorded sizes in turn, with eager work (a larger tree, whose buffers grow; decoding; prefill) between the
    replays; capturing leaves the state, and each replay is checked against decoding."""
    m = model(64)
    m.reset(0)
    m.prefill(prompt(20, seed=2))
    before = (m.kv.clone(), int(m.tok), int(m.pos))
    for n in (4, 25):
        m.capture_verify(n)
    assert torch.equal(m.kv, before[0]) and (int(m.tok), int(m.pos)) == before[1:] and m.host_pos == 20
    for turn in range(3):
        path, margin = greedy(m, 4)
        sure = next((i for i, x in enumerate(margin) if x <= 2 * REL), 4)
        toks, _ = checked_verify(m, path)                                         # 4: a recorded chain
        assert toks[:sure] == path[:sure]
        checked_verify(m, *branching(greedy(m, 2)[0], 24 - turn, seed=turn))      # not a recorded size
        path, margin = greedy(m, 5)
        sure = next((i for i, x in enumerate(margin) if x <= 2 * REL), 5)
        draft, parents = branching(path, 20, seed=turn + 9)
        assert len(draft) == 25
        toks, _ = checked_verify(m, draft, parents)                               # 25: a recorded tree
        assert toks[:sure] == path[:sure]
        m.run_step()
        m.prefill([7, 8, 9])
    assert m.host_pos == int(m.pos)


def test_capture_verify_refusals(K):
    with pytest.raises(NotImplementedError, match="INT4"):
        model(64, weights="fp16").capture_verify(4)
    with pytest.raises(NotImplementedError, match="INT4"):
        model(64, lm_head="fp16").capture_verify(4)
    for n in (-1, 1024):
        with pytest.raises(ValueError, match="drafted tokens"):
            model(64).capture_verify(n)


def test_verify_on_a_side_stream(K):
    m = model(64)
    out = []
    side = torch.cuda.Stream()
    for s in (torch.cuda.current_stream(), side):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            m.kv.zero_()
            m.reset(0)
            m.prefill(prompt(30, seed=6))
            out.append((m.verify([3, 4, 5, 6], [0, 1, 0, 3]), m.kv.clone(), m.logits.clone()))
        torch.cuda.synchronize()
    assert out[0][0] == out[1][0] and torch.equal(out[0][1], out[1][1]) and torch.equal(out[0][2], out[1][2])


def test_verify_refusals(K):
    m = model(64)
    m.reset(0)
    m.prefill(prompt(12))
    before = (m.kv.clone(), int(m.tok), int(m.pos))
    for draft, parents, msg in (([5, 1000], None, "token ids"), ([-1], None, "token ids"), ([1, 2], [0], "parents"),
                                ([1, 2], [0, 2], "parent of node"), ([1] * 1024, [0] * 1024, "at most")):
        with pytest.raises(ValueError, match=msg):
            m.verify(draft, parents)
    with pytest.raises(RuntimeError, match="exceeds max_ctx"):
        m.verify([1] * 244)
    assert torch.equal(m.kv, before[0]) and (int(m.tok), int(m.pos)) == before[1:] and m.host_pos == 12
    checked_verify(m, [1] * 243)                           # to the cache's last token
