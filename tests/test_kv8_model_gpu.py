"""Model with a cache in 8-bit codes and with a sliding window: decoding (eager and replayed) and prefill append what the
definition says and attend it. The operators' calls inside the model are recorded and checked against the 64-bit reference;
layer 0's rows, which no attention precedes, are compared with the ones that a model with an fp16 cache keeps."""
import pytest
import torch

import kv8_ref as R
from helpers import DEV, gen

pytestmark = pytest.mark.gpu


def model(D=64, max_ctx=256, seed=4, **cfg):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from runtime.model import DecodeConfig, Model
    from runtime.synth import LlamaShape, SyntheticLlama
    shape = LlamaShape(256, 2, 4, 2, 512, 1000) if D == 64 else LlamaShape(512, 2, 4, 2, 1024, 1000)
    m = Model(SyntheticLlama(shape, seed=seed, device=DEV, std=0.05), shape, DecodeConfig(max_ctx=max_ctx, device=DEV, **cfg))
    m.prepare(max_ctx)
    return m


def tokens(n, seed=1):
    return torch.randint(0, 1000, (n,), generator=gen(seed))


class Recorder:
    """Stands in for the op module and keeps what each attention call was given and gave back."""

    def __init__(self, ops):
        self.ops, self.calls = ops, []

    def __getattr__(self, name):
        fn = getattr(self.ops, name)
        if name == "attention_kv8_decode":
            return self.decode
        if name not in ("attention_kv8", "attention_window"):
            return fn

        def call(q, pos, bt, kc, vc, *rest):
            scales, rest = (rest[:2], rest[2:]) if name == "attention_kv8" else ((None, None), rest)
            before = [q.clone().cpu(), int(pos), *(R.values(c.cpu(), None if s is None else s.cpu())
                                                   for c, s in zip((kc, vc), scales))]
            fn(q, pos, bt, kc, vc, *(s for s in scales if s is not None), *rest)
            self.calls.append((*before, rest[1].clone().cpu()))

        return call

    def decode(self, qkv, cos, sin, pos, bt, kc, vc, ks, vs, n_q, n_kv, max_ctx, out, *rest):
        """One token appended and attended: the cache as it is afterwards, which is the reference's append."""
        was = [t.cpu() for t in (kc, vc, ks, vs)]
        q, want = R.append(qkv.cpu().view(1, -1), cos.cpu(), sin.cpu(), int(pos), bt.cpu(), *was, n_q)
        self.ops.attention_kv8_decode(qkv, cos, sin, pos, bt, kc, vc, ks, vs, n_q, n_kv, max_ctx, out, *rest)
        raw = lambda t: t.cpu().contiguous().view(torch.uint8)
        assert all(torch.equal(raw(t), raw(w)) for t, w in zip((kc, vc, ks, vs), want))
        self.calls.append((q.view(1, -1), int(pos), R.values(kc.cpu(), ks.cpu()), R.values(vc.cpu(), vs.cpu()),
                           out.view(1, -1).clone().cpu()))


CASES = [dict(kv="int8"), dict(kv="e4m3"), dict(kv="e4m3", window=20, sinks=3), dict(window=25, sinks=2), dict(window=9)]
ids = lambda c: "-".join(f"{k}{v}" for k, v in c.items())


@pytest.mark.parametrize("cfg", CASES, ids=ids)
@pytest.mark.parametrize("D,page,fused", [(64, 16, True), (128, 32, True), (64, 16, False)])
@pytest.mark.parametrize("one", [True, False])
def test_decode_and_prefill_attend_their_cache(cfg, D, page, fused, one):
    """Every attention call of a prefill and of steps behind it, against the reference over the cache as it is."""
    m = model(D, page=page, fused_gemv=fused, fused_attention=one, **cfg)
    m.K = rec = Recorder(m.K)
    m.reset(0)
    m.prefill(tokens(37))
    for _ in range(6):
        m.run_step(use_graph=False)
    assert len(rec.calls) == 2 * 7
    for i, (q, pos, kc, vc, out) in enumerate(rec.calls):
        M = q.size(0)
        assert (M, pos) == ((37, 0) if i < 2 else (1, 37 + (i - 2) // 2))
        want, bound = R.attention(q.reshape(M, m.n_q, D), pos, m.bt.cpu(), kc, vc, 256, m.cfg.window, m.cfg.sinks)
        R.within(out, want, bound)


@pytest.mark.parametrize("kv", ["int8", "e4m3"])
def test_first_layer_rows_are_the_fp16_rows_in_codes(kv):
    """A prompt at once, then tokens one by one through the captured graph, blocks growing on the way."""
    a, b = model(), model(kv=kv)
    p, n = tokens(21), 30
    for m in (a, b):
        m.reset(0)
        m.prefill(p)
        m.teacher_force(tokens(n, 2))
    L = 21 + n
    k, v = (t.cpu() for t in a.read_cache(0, 0, L))
    P = b.cfg.page
    kc, vc = (torch.zeros(b.n_pages, b.n_kv, P, b.D, dtype=b.kv.dtype) for _ in "kv")
    ks, vs = (torch.zeros(b.n_pages, b.n_kv, P // 16) for _ in "kv")
    ref, bt = [kc, vc, ks, vs], b.bt.cpu()
    for lo, hi in [(0, 21)] + [(t, t + 1) for t in range(21, L)]:
        rows = torch.cat([torch.zeros(hi - lo, b.D).half(), k[lo:hi].reshape(hi - lo, -1), v[lo:hi].reshape(hi - lo, -1)], 1)
        _, ref = R.append(rows, None, None, lo, bt, *ref, 1)
    got = [t.cpu() for t in b.read_cache(0, 0, L)]
    for g, code, scale in ((got[0], ref[0], ref[2]), (got[1], ref[1], ref[3])):
        val = R.values(code, scale)
        want = torch.stack([val[c[0], :, c[1]] for c in (R.token_row(bt.tolist(), t, P, b.n_pages) for t in range(L))])
        assert torch.equal(g.double(), want)
    back = a.read_cache(1, 5, 9)
    assert torch.equal(back[0], a.kv[1, 0][a.bt[torch.arange(5, 14) // P].long(), :, torch.arange(5, 14) % P])


@pytest.mark.parametrize("cfg", CASES, ids=ids)
def test_replayed_steps_are_the_eager_ones(cfg):
    """The captured step at every position, beside the eager one: the same tokens and the same logits."""
    a, b = model(**cfg), model(**cfg)
    got = []
    for m, graph in ((a, True), (b, False)):
        m.reset(0)
        rows = [m.teacher_force(tokens(40), graph, collect_logits=True)]
        for _ in range(5):
            m.run_step(graph)
            rows.append(m.logits.clone()[None])
        got.append(torch.cat(rows))
    assert torch.equal(*got) and a.host_pos == int(a.pos) == 45


@pytest.mark.parametrize("kv", ["int8", "e4m3"])
def test_preparing_again_keeps_a_sequence_in_codes(kv):
    """The captured step is recorded anew in the middle of a sequence: what follows is what follows without it."""
    a, b = model(kv=kv), model(kv=kv)
    got = []
    for m in (a, b):
        m.reset(0)
        m.prefill(tokens(30))
        if m is b:
            before = [t.clone() for t in (m.kv.view(torch.uint8), m.kv_scale)]
            m.prepare(256)
            assert all(torch.equal(x, y) for x, y in zip(before, (m.kv.view(torch.uint8), m.kv_scale)))
        got.append(m.teacher_force(tokens(10, 5), collect_logits=True))
    assert torch.equal(*got)


def test_window_wider_than_the_sequence_changes_only_the_kernel():
    """The same attention by other kernels: logits within the 2e-2 of the largest that two summation orders of one model are
    given elsewhere."""
    a, b = model(), model(window=256)
    got = []
    for m in (a, b):
        m.reset(0)
        m.prefill(tokens(50))
        got.append(m.logits.clone())
        got.append(m.teacher_force(tokens(20, 3), collect_logits=True))
    for x, y in zip(got[:2], got[2:]):
        assert float((x - y).abs().max()) <= 2e-2 * float(x.abs().max())


def test_a_window_forgets():
    """Two prompts that differ in a token that no window on the way to the last row holds: the same logits to the bit."""
    m = model(kv="e4m3", window=8, sinks=2)
    out = []
    for edit in (3, 700):
        ids = tokens(60)
        ids[20] = edit
        m.reset(0)
        m.prefill(ids)
        out.append(m.logits.clone())
    assert torch.equal(*out)      # two layers of windows of 8 reach 14 tokens back from position 59


def test_config_refusals():
    for cfg, msg in ((dict(kv="fp8"), "kv 'fp8'"), (dict(window=-1), "window -1"), (dict(sinks=3), "belong to a window"),
                     (dict(kv="int8", page=8), "multiple of 16")):
        with pytest.raises(ValueError, match=msg):
            model(**cfg)
    m = model(kv="int8")
    with pytest.raises(NotImplementedError, match="fp16 cache and no window"):
        m.verify([1, 2])
    with pytest.raises(NotImplementedError, match="fp16 cache and no window"):
        model(window=5).capture_verify(3)
    with pytest.raises(ValueError, match="read_cache"):
        m.read_cache(0, 250, 10)
    assert m.kv.element_size() == 1 and m.kv_bytes_per_token(100) == 2 * 2 * 101 * (2 * 64 + 2 * 4 // 16)


@pytest.mark.parametrize("cfg", [dict(), dict(window=25), dict(window=25, sinks=2), dict(page=1), dict(page=1, window=9, sinks=2),
                                 dict(kv="int8", window=25, sinks=2)], ids=ids)
@pytest.mark.parametrize("fails", [False, True])
def test_preparing_again_keeps_a_sequence(cfg, fails):
    """The captured step is recorded anew, or its recording fails, in the middle of a sequence: the cache, token and position
    are as they were, and what follows is what follows without it."""
    a, b = model(**cfg), model(**cfg)
    got = []
    for m in (a, b):
        m.reset(0)
        m.prefill(tokens(30))
        if m is b:
            held = [t for t in (m.kv.view(torch.uint8), m.kv_scale, m.tok, m.pos) if t is not None]
            before, step = [t.clone() for t in held], m.step

            def broken():
                step()
                raise RuntimeError("a step that fails")

            if fails:
                m.step = broken
                with pytest.raises(RuntimeError, match="a step that fails"):
                    m.prepare(256)
                del m.step
            else:
                m.prepare(256)
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(before, held))
            m.prepare(256)
        got.append(m.teacher_force(tokens(10, 5), collect_logits=True))
    assert torch.equal(*got)


@pytest.mark.parametrize("kv", ["fp16", "int8", "e4m3"])
def test_read_cache_of_pages_taken_out(kv):
    """Tokens whose page is no longer in the block table read as zeros, from a cache of any kind; the others as before."""
    m = model(kv=kv)
    m.reset(0)
    m.prefill(tokens(70))
    before = m.read_cache(1, 3, 60)
    P = m.cfg.page
    m.bt[1] = -1
    for t, was in zip(m.read_cache(1, 3, 60), before):
        gone = (torch.arange(3, 63, device=DEV) // P == 1)[:, None, None]
        assert bool((was != 0).any()) and torch.equal(t, torch.where(gone, 0.0, was).half())


def test_bytes_of_a_step_under_a_window():
    """A token reads the cached rows that it attends, window - 1 ahead of it and the sinks, and writes its own."""
    m = model(window=20, sinks=3)
    row = 2 * 2 * 2 * 64 * 2                       # K and V, layers, kv heads, head dim, fp16
    for ctx, rows in ((0, 1), (10, 11), (22, 23), (23, 23), (200, 23)):
        assert m.kv_bytes_per_token(ctx) == row * rows
