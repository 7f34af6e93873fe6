"""GPU tests of the operators of one verification step of speculative decoding, each against its 64-bit reference
(tree_ref) within the error bounds that its roundings allow."""
import pytest
import torch

import tree_ref as T
from helpers import DEV, gen, make_cache
from runtime.model import rope_tables

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from runtime import ext
    return ext.load()


def dev(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------------------------------------ norm + RoPE + append
def qk_inputs(M, n_q, n_kv, D, page, start, norm, tree, seed=0):
    g = gen(seed + M + 7 * D + start)
    qkv = torch.randn(M, (n_q + 2 * n_kv) * D, generator=g).half()
    qw, kw = ((1 + 0.2 * torch.randn(D, generator=g)).half() for _ in "qk") if norm else (None, None)
    kc, vc, bt = make_cache(start + M, n_kv, page, D=D, seed=seed + 1)
    cos, sin = rope_tables(start + M + 1, D, 500000.0)
    depth = None
    if tree:
        p = T.random_parents(M, 3, g)
        depth = torch.zeros(M, dtype=torch.int32)
        for i in range(1, M):
            depth[i] = depth[p[i]] + 1
    return qkv, qw, kw, kc, vc, bt, cos, sin, depth


@pytest.mark.parametrize("M,n_q,n_kv,D,page,start,norm,tree", [
    (1, 32, 8, 128, 16, 40, True, False), (1, 32, 4, 64, 16, 0, False, False), (5, 3, 1, 64, 16, 33, True, True),
    (61, 32, 4, 64, 16, 100, False, True), (26, 32, 8, 128, 32, 70, True, True), (130, 16, 2, 128, 16, 0, True, False),
    (300, 8, 8, 64, 64, 5, True, False), (7, 40, 8, 128, 1, 3, True, True), (2, 1, 1, 128, 4, 1, False, False)])
def test_qk_norm_rope_append_rows(K, M, n_q, n_kv, D, page, start, norm, tree):
    qkv, qw, kw, kc, vc, bt, cos, sin, depth = qk_inputs(M, n_q, n_kv, D, page, start, norm, tree)
    q, qb, k64, kb, v64, _ = T.qk_norm_rope(qkv, qw, kw, 1e-6, cos, sin, start, depth, bt, kc, vc, n_q, n_kv)
    a = dev(qkv, qw, kw, cos, sin, depth, bt, kc, vc)
    x, qw, kw, cos, sin, depth, bt, kcd, vcd = a
    wide = torch.full((M, n_q * D + 24), 7.0, dtype=torch.half, device=DEV)
    K.qk_norm_rope_append_rows(x, qw, kw, 1e-6, cos, sin, i32(start), depth, bt, kcd, vcd, n_q, n_kv, wide[:, :n_q * D])
    T.within(wide[:, :n_q * D].reshape(M, n_q, D), q, qb)
    T.within(kcd, k64, kb)
    assert torch.equal(vcd.cpu().double(), v64)          # v is copied, every other row is as it was
    assert torch.equal(x.cpu(), qkv) and bool((wide[:, n_q * D:] == 7).all())
    # in place: the same q over qkv's own, k and v of qkv untouched
    K.qk_norm_rope_append_rows(x, qw, kw, 1e-6, cos, sin, i32(start), depth, bt, kcd, vcd, n_q, n_kv)
    assert torch.equal(x[:, :n_q * D], wide[:, :n_q * D]) and torch.equal(x[:, n_q * D:].cpu(), qkv[:, n_q * D:])


def test_qk_norm_without_weights_is_rope_append_rows(K):
    qkv, _, _, kc, vc, bt, cos, sin, _ = qk_inputs(37, 32, 8, 128, 16, 21, False, False)
    x, cos, sin, bt, k1, v1 = dev(qkv, cos, sin, bt, kc, vc)
    y, k2, v2 = x.clone(), k1.clone(), v1.clone()
    K.rope_append_rows(x, cos, sin, i32(21), bt, k1, v1, 32, 8)
    K.qk_norm_rope_append_rows(y, None, None, 0.0, cos, sin, i32(21), None, bt, k2, v2, 32, 8)
    assert torch.equal(x, y) and torch.equal(k1, k2) and torch.equal(v1, v2)


@pytest.mark.parametrize("start,rows,edit", [
    (-3, 6, None),               # rows of tokens before 0 touch nothing
    (40, 12, "short table"),     # rotations past the tables touch nothing
    (40, 12, "short bt"),        # tokens past the block table: rotated, not appended
    (40, 12, "unmapped"),        # a page that is no page of the cache: rotated, not appended
    (40, 12, "far depth")])      # depths that leave the tables on both sides
def test_qk_norm_rows_out_of_range(K, start, rows, edit):
    n_q, n_kv, D, page = 8, 2, 64, 4
    qkv, qw, kw, kc, vc, bt, cos, sin, depth = qk_inputs(rows, n_q, n_kv, D, page, max(start, 0), True, True)
    if edit == "short table":
        cos, sin = cos[:start + 2].contiguous(), sin[:start + 2].contiguous()
    if edit == "short bt":
        bt = bt[:(start + 5) // page].contiguous()
    if edit == "unmapped":
        bt[(start + 3) // page], bt[(start + 7) // page] = -1, kc.size(0)
    if edit == "far depth":
        depth[3], depth[5], depth[6] = -start - 1, 2 ** 31 - 1, -2 ** 31
    q, qb, k64, kb, v64, touched = T.qk_norm_rope(qkv, qw, kw, 1e-6, cos, sin, start, depth, bt, kc, vc, n_q, n_kv)
    x, qw, kw, cos, sin, depth, bt, kcd, vcd = dev(qkv, qw, kw, cos, sin, depth, bt, kc, vc)
    out = torch.full((rows, n_q * D), float("nan"), dtype=torch.half, device=DEV)
    K.qk_norm_rope_append_rows(x, qw, kw, 1e-6, cos, sin, i32(start), depth, bt, kcd, vcd, n_q, n_kv, out)
    assert any(touched) and (edit in ("short bt", "unmapped") or not all(touched))
    T.within(out.view(rows, n_q, D), q, qb)
    T.within(kcd, k64, kb)
    assert torch.equal(vcd.cpu().double(), v64)


# ------------------------------------------------------------------------------------------------ tree attention
def tree_inputs(M, n_q, n_kv, D, page, ctx, branch, seed=0, peaky=1.0):
    g = gen(seed + 3 * M + ctx)
    kc, vc, bt = make_cache(ctx + M, n_kv, page, D=D, peaky=peaky, seed=seed + ctx)
    q = torch.randn(M, n_q, D, generator=g).half()
    rows = T.mask_rows(T.random_parents(M, branch, g))
    return q, rows, kc, vc, bt


def run_tree(K, q, words, pos, bt, kc, vc, max_ctx, workspace="full"):
    M, n_q, D = q.shape
    out = torch.full((M, n_q * D), float("nan"), dtype=torch.half, device=DEV)
    need = K.attention_tree_workspace_bytes(M, n_q, kc.size(1), D, max_ctx)
    ws = None
    if need and workspace != "none":
        ws = torch.full((need if workspace == "full" else need // 2 + 7,), 255, dtype=torch.uint8, device=DEV)
    K.attention_tree(q, words, pos, bt, kc, vc, max_ctx, out, ws)
    return out


@pytest.mark.parametrize("M,n_q,n_kv,D,page,ctx,branch", [
    (1, 32, 8, 128, 16, 0, 1), (1, 32, 4, 64, 16, 300, 1), (2, 8, 8, 64, 16, 1, 1), (5, 32, 4, 64, 16, 301, 2),
    (26, 32, 8, 128, 16, 777, 4), (33, 8, 4, 128, 32, 64, 1), (64, 32, 8, 128, 16, 1000, 8), (65, 16, 2, 64, 16, 63, 4),
    (100, 4, 4, 128, 16, 129, 2), (130, 8, 1, 64, 64, 500, 5), (250, 8, 2, 128, 16, 200, 8), (7, 16, 8, 64, 1, 90, 3),
    (9, 4, 2, 128, 2, 131, 2), (64, 64, 8, 64, 8, 257, 4), (3, 16, 2, 128, 4, 2000, 2), (17, 2, 1, 64, 16, 4000, 3)])
def test_attention_tree(K, M, n_q, n_kv, D, page, ctx, branch):
    q, rows, kc, vc, bt = tree_inputs(M, n_q, n_kv, D, page, ctx, branch)
    want, bound = T.attention_tree(q, rows, ctx, bt, kc, vc)
    qd, words, btd, kd, vd = dev(q, T.mask_words(rows), bt, kc, vc)
    for ws in ("full", "half", "none"):
        T.within(run_tree(K, qd, words, i32(ctx), btd, kd, vd, ctx + M, ws), want, bound)
    # a larger cap attends no more, a strided q gives the same
    wide = torch.zeros(M, (n_q + 2 * n_kv) * D, dtype=torch.half, device=DEV)
    wide[:, :n_q * D] = qd.view(M, -1)
    out = torch.empty(M, n_q * D, dtype=torch.half, device=DEV)
    need = K.attention_tree_workspace_bytes(M, n_q, n_kv, D, 2 * (ctx + M))
    K.attention_tree(wide[:, :n_q * D], words, i32(ctx), btd, kd, vd, 2 * (ctx + M), out,
                     torch.empty(need, dtype=torch.uint8, device=DEV) if need else None)
    T.within(out, want, bound)


def test_attention_tree_all_nodes(K):
    """The largest tree, and masks that are no tree: random bits, full rows, rows of nothing."""
    M, n_q, n_kv, D, ctx = 1024, 2, 1, 64, 0
    q, _, kc, vc, bt = tree_inputs(M, n_q, n_kv, D, 16, ctx, 4)
    rows = torch.rand(M, M, generator=gen(5)) < 0.05
    rows[10], rows[500], rows[1023] = False, True, False
    want, bound = T.attention_tree(q, rows, ctx, bt, kc, vc)
    qd, words, btd, kd, vd = dev(q, T.mask_words(rows), bt, kc, vc)
    out = run_tree(K, qd, words, i32(ctx), btd, kd, vd, M)
    T.within(out, want, bound)
    assert bool((out[10] == 0).all()) and bool((out[1023] == 0).all())


@pytest.mark.parametrize("M,D,hpg,ctx", [(13, 64, 8, 200), (40, 128, 4, 37), (70, 128, 1, 0), (64, 64, 2, 1500)])
def test_attention_tree_chain_without_mask(K, M, D, hpg, ctx):
    q, _, kc, vc, bt = tree_inputs(M, 2 * hpg, 2, D, 16, ctx, 1)
    want, bound = T.attention_tree(q, torch.ones(M, M).tril().bool(), ctx, bt, kc, vc)
    qd, btd, kd, vd = dev(q, bt, kc, vc)
    T.within(run_tree(K, qd, None, i32(ctx), btd, kd, vd, ctx + M), want, bound)


def test_attention_tree_mask_bits_past_the_last_node(K):
    """Bits at and past M name no node: the tokens behind the tree (NaN here) are not attended."""
    M, ctx = 21, 75
    q, rows, kc, vc, bt = tree_inputs(M, 8, 2, 64, 16, ctx, 3)
    cells = [T.token_row(bt.tolist(), t, 16, kc.size(0)) for t in range(ctx + M, bt.numel() * 16)]
    for c in cells:
        kc[c[0], :, c[1]] = float("nan")
        vc[c[0], :, c[1]] = float("inf")
    want, bound = T.attention_tree(q, rows, ctx, bt, kc, vc)
    qd, words, btd, kd, vd = dev(q, T.mask_words(rows) | (-1 << M), bt, kc, vc)
    T.within(run_tree(K, qd, words, i32(ctx), btd, kd, vd, bt.numel() * 16), want, bound)


@pytest.mark.parametrize("D,ctx,bad", [(64, 100, float("nan")), (128, 61, float("nan")), (128, 200, float("inf")),
                                       (64, 0, float("-inf"))])
def test_attention_tree_keeps_unattended_values_out(K, D, ctx, bad):
    """Node 5 (and a padding node that none attends) holds NaN or infinities in K and V: its descendants see them, no
    other node does."""
    M, n_q, n_kv, page = 40, 8, 2, 16
    q, rows, kc, vc, bt = tree_inputs(M, n_q, n_kv, D, page, ctx, 3)
    rows[:, 39] = False
    rows[39] = False
    for node, dim in ((5, 3), (39, slice(None))):
        c = T.token_row(bt.tolist(), ctx + node, page, kc.size(0))
        kc[c[0], 0, c[1], dim] = bad
        vc[c[0], :, c[1], dim] = bad
    kept = [i for i in range(M) if not rows[i, 5]]
    want, bound = T.attention_tree(q, rows, ctx, bt, kc, vc)
    qd, words, btd, kd, vd = dev(q, T.mask_words(rows), bt, kc, vc)
    out = run_tree(K, qd, words, i32(ctx), btd, kd, vd, ctx + M)
    T.within(out[kept], want[kept], bound[kept])
    assert 39 in kept
    seen = [i for i in range(M) if rows[i, 5]]
    hit = out.view(M, n_q, D)[seen][:, n_q // n_kv:, 3]      # the kv head whose K is finite: the V value alone
    assert len(kept) > 1 and seen and not bool(torch.isfinite(hit).any())


@pytest.mark.parametrize("page", [16, 2])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("M", [20, 60, 80])
@pytest.mark.parametrize("ctx,cap", [(90, 256), (290, 384), (700, 1500), (700, 5000), (700, 20000)])
def test_attention_tree_every_workgroup_shape(K, page, D, M, ctx, cap):
    """The sizes and the cap choose the shape; each against values that must not spread (NaN in K and V of one node, an
    infinity in V of another, a page that is not mapped) and splits without a token."""
    n_q, n_kv = 8, 2
    ctx = min(ctx, cap - M)
    q, rows, kc, vc, bt = tree_inputs(M, n_q, n_kv, D, page, ctx, 3, seed=7)
    for node, bad in ((5, float("nan")), (11, float("inf"))):
        c = T.token_row(bt.tolist(), ctx + node, page, kc.size(0))
        if bad != bad:
            kc[c[0], 0, c[1], 3] = bad
        vc[c[0], :, c[1], 9] = bad
    bt[40 // page] = -1
    kept = [i for i in range(M) if not rows[i, 5] and not rows[i, 11]]
    assert 4 < len(kept) < M - 1
    want, bound = T.attention_tree(q, rows, ctx, bt, kc, vc)
    qd, words, btd, kd, vd = dev(q, T.mask_words(rows), bt, kc, vc)
    for ws in ("full", "none"):
        out = run_tree(K, qd, words, i32(ctx), btd, kd, vd, cap, ws)
        T.within(out[kept], want[kept], bound[kept])
        seen = [i for i in range(M) if rows[i, 5] or rows[i, 11]]
        hit = out.view(M, n_q, D)[seen][:, n_q // n_kv:]         # the kv head whose K is finite
        assert not bool(torch.isfinite(hit[..., 9]).any()) and bool(torch.isfinite(hit[..., :8]).all())


@pytest.mark.parametrize("page", [16, 2])
def test_attention_tree_unmapped_pages_and_cap(K, page):
    """Tokens without a mapped page, past the block table or past max_ctx are not attended, nodes among them too; with
    *pos < 0 nothing is."""
    M, n_q, n_kv, D, ctx = 20, 8, 2, 128, 150
    q, rows, kc, vc, bt = tree_inputs(M, n_q, n_kv, D, page, ctx, 2)
    bt[3], bt[(ctx + 6) // page] = -1, kc.size(0)
    for max_ctx, n_bt in ((ctx + M, bt.numel()), (ctx + 3, bt.numel()), (100, bt.numel()), (ctx + M, 60 // page), (1, 1)):
        b = bt[:n_bt].contiguous()
        want, bound = T.attention_tree(q, rows, ctx, b, kc, vc, max_ctx)
        qd, words, btd, kd, vd = dev(q, T.mask_words(rows), b, kc, vc)
        T.within(run_tree(K, qd, words, i32(ctx), btd, kd, vd, max_ctx), want, bound)
    out = run_tree(K, qd, words, i32(-1), btd, kd, vd, ctx + M)
    assert bool((out == 0).all())


def test_attention_tree_large_scores(K):
    """Scores of hundreds: the running maximum moves by large steps, weights fall to zero."""
    M, ctx = 30, 700
    q, rows, kc, vc, bt = tree_inputs(M, 8, 2, 128, 16, ctx, 3, peaky=30.0)
    want, bound = T.attention_tree(q, rows, ctx, bt, kc, vc)
    qd, words, btd, kd, vd = dev(q, T.mask_words(rows), bt, kc, vc)
    T.within(run_tree(K, qd, words, i32(ctx), btd, kd, vd, ctx + M), want, bound)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("slope,cap", [(0.004, 384), (0.004, 1500), (0.05, 1500), (0.05, 20000), (-0.02, 5000)])
def test_attention_tree_rising_scores(K, D, slope, cap):
    """Scores that rise (or fall) steadily with the position: the reference of the weights moves again and again, by small
    steps and by large ones, and each column's sum and output with it."""
    M, n_q, n_kv = 70, 8, 2
    ctx = min(900, cap - M)
    q, rows, kc, vc, bt = tree_inputs(M, n_q, n_kv, D, 16, ctx, 3, seed=21)
    q = (q * 0.1 + 0.5).half()
    kc = kc * 0.2
    for t in range(ctx + M):
        c = T.token_row(bt.tolist(), t, 16, kc.size(0))
        kc[c[0], :, c[1]] += slope * t
    want, bound = T.attention_tree(q, rows, ctx, bt, kc, vc)
    qd, words, btd, kd, vd = dev(q, T.mask_words(rows), bt, kc, vc)
    for ws in ("full", "none"):
        T.within(run_tree(K, qd, words, i32(ctx), btd, kd, vd, cap, ws), want, bound)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("M,ctx,cap", [(1, 0, 100), (20, 300, 384), (20, 700, 1500), (20, 700, 5000), (80, 700, 1500),
                                       (80, 900, 20000)])
@pytest.mark.parametrize("size", [30.0, 1000.0, 16384.0, 60000.0, -2000.0, -60000.0])
def test_attention_tree_far_scores(K, D, M, ctx, cap, size):
    """Scores as large as finite q and K make them, up to 2^36 in units of log2. Equal ones weigh alike, whatever their
    size: the output is the mean of V over the tokens that a node sees, V itself where it sees one. A token whose score lies
    as far above them has all the weight, wherever it stands.

    Tolerance: fp16's half step of the output and of the weight (the same one for every token), and the fp32 sums, a chain of
    at most n + 64 terms of |v| / n."""
    n_q, n_kv = 8, 2
    q, rows, kc, vc, bt = tree_inputs(M, n_q, n_kv, D, 16, ctx, 3, seed=31)
    g = gen(6)
    q = (abs(size) * (0.5 + 0.5 * torch.rand(q.shape, generator=g))).half()
    kc = (size * (0.5 + 0.5 * torch.rand(n_kv, 1, D, generator=g))).half().expand_as(kc).contiguous()
    if M > 1:
        rows[7] = False
        rows[7, 7] = True                                      # one node and no other
    cells = [T.token_row(bt.tolist(), t, 16, kc.size(0)) for t in range(ctx + M)]
    v = torch.stack([vc[c[0], :, c[1]] for c in cells]).double()                # [tokens, n_kv, D]
    qd, words, btd = dev(q, T.mask_words(rows), bt)

    def expect(see):                                                            # bool [M, tokens]
        n = see.sum(1).clamp(min=1)[:, None, None]
        mean = torch.einsum("mt,thd->mhd", see.double(), v) / n
        size_ = torch.einsum("mt,thd->mhd", see.double(), v.abs()) / n
        bound = 2.0 ** -11 * mean.abs() + (2.0 ** -11 + 2.0 ** -24 * (n + 64)) * size_ + 2.0 ** -25
        wide = lambda x: x.repeat_interleave(n_q // n_kv, 1).reshape(M, -1)
        return wide(mean), wide(bound)

    see = torch.cat([torch.ones(M, ctx, dtype=torch.bool), rows], 1)
    for ws in ("full", "none"):
        T.within(run_tree(K, qd, words, i32(ctx), btd, *dev(kc, vc), cap, ws), *expect(see))
    for t in ([5, ctx // 2, ctx - 1] if ctx else []):
        above = kc.clone()
        above[cells[t][0], :, cells[t][1]] = 65504.0 if size > 0 else 0.0       # the score of one token lies above the others
        only = torch.zeros_like(see)
        only[:, t] = True
        T.within(run_tree(K, qd, words, i32(ctx), btd, *dev(above, vc), cap), *expect(only))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cap", [384, 1500, 20000])
@pytest.mark.parametrize("size", [3.0, 30000.0, -30000.0])
def test_attention_tree_far_scores_beside_nan(K, D, cap, size):
    """Equal scores, large ones among them, and a NaN in V of one node and an infinity in V of another: only their element is
    lost to the nodes that see them, the others are the mean. Tolerance as for far scores."""
    M, n_q, n_kv, ctx = 20, 8, 2, 77
    q, rows, kc, vc, bt = tree_inputs(M, n_q, n_kv, D, 16, ctx, 3, seed=31)
    g = gen(7)
    q = (abs(size) * (0.5 + 0.5 * torch.rand(q.shape, generator=g))).half()
    kc = (size * (0.5 + 0.5 * torch.rand(n_kv, 1, D, generator=g))).half().expand_as(kc).contiguous()
    cells = [T.token_row(bt.tolist(), t, 16, kc.size(0)) for t in range(ctx + M)]
    v = torch.stack([vc[c[0], :, c[1]] for c in cells]).double()
    for node, bad in ((2, float("nan")), (5, float("inf"))):
        c = cells[ctx + node]
        vc[c[0], :, c[1], 9] = bad
    see = torch.cat([torch.ones(M, ctx, dtype=torch.bool), rows], 1).double()
    n = see.sum(1)[:, None, None]
    mean, size_ = (torch.einsum("mt,thd->mhd", see, x).repeat_interleave(n_q // n_kv, 1) / n for x in (v, v.abs()))
    bound = 2.0 ** -11 * mean.abs() + (2.0 ** -11 + 2.0 ** -24 * (n + 64)) * size_ + 2.0 ** -25
    mean[rows[:, 5], :, 9] = float("inf")
    mean[rows[:, 2], :, 9] = float("nan")
    assert 0 < int(rows[:, 2].sum()) < M and 0 < int(rows[:, 5].sum()) < M
    for ws in ("full", "none"):
        out = run_tree(K, *dev(q, T.mask_words(rows)), i32(ctx), *dev(bt, kc, vc), cap, ws)
        T.within(out, mean.view(M, -1), bound.reshape(M, -1))


def test_attention_tree_infinite_scores(K):
    """A score of +infinity, or NaN, leaves no distribution: NaN for the nodes that see it, and for no other."""
    M, n_q, n_kv, D, ctx = 40, 8, 2, 64, 200
    q, rows, kc, vc, bt = tree_inputs(M, n_q, n_kv, D, 16, ctx, 3, seed=5)
    q = q.abs() + 0.5
    want, bound = T.attention_tree(q, rows, ctx, bt, kc, vc)
    for bad in (float("inf"), float("nan")):
        k = kc.clone()
        c = T.token_row(bt.tolist(), ctx + 5, 16, kc.size(0))
        k[c[0], :, c[1], 1] = bad
        qd, words, btd, kd, vd = dev(q, T.mask_words(rows), bt, k, vc)
        out = run_tree(K, qd, words, i32(ctx), btd, kd, vd, ctx + M)
        seen = rows[:, 5]
        assert 0 < int(seen.sum()) < M and bool(torch.isnan(out[seen.to(DEV)]).all())
        T.within(out.cpu()[~seen], want[~seen], bound[~seen])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cap", [384, 1500, 20000])
def test_attention_tree_node_beside_others(K, D, cap):
    """A node's output does not depend, not in a bit, on what the nodes hold that it does not attend: their queries, keys and
    values change (scores that rise much faster than its own), the tokens that it sees do not."""
    M, n_q, n_kv = 24, 8, 2
    ctx = min(900, cap - M)
    q, rows, kc, vc, bt = tree_inputs(M, n_q, n_kv, D, 16, ctx, 3, seed=23)
    q = (q * 0.1 + 0.5).half()
    for t in range(ctx + M):
        c = T.token_row(bt.tolist(), t, 16, kc.size(0))
        kc[c[0], :, c[1]] = kc[c[0], :, c[1]] * 0.2 + 0.01 * t
    words, btd = dev(T.mask_words(rows), bt)
    first = run_tree(K, q.to(DEV), words, i32(ctx), btd, *dev(kc, vc), cap)
    node = 5
    other = [j for j in range(M) if not rows[node, j]]
    for j in other:
        c = T.token_row(bt.tolist(), ctx + j, 16, kc.size(0))
        kc[c[0], :, c[1]] *= 3
        vc[c[0], :, c[1]] += 1
        q[j] *= 0.05 * (j + 1)
    second = run_tree(K, q.to(DEV), words, i32(ctx), btd, *dev(kc, vc), cap)
    same = [i for i in range(M) if not bool(rows[i, other].any())]
    assert node in same and len(other) > 8
    assert torch.equal(first[same], second[same]) and not torch.equal(first, second)


def test_attention_tree_replays_at_other_positions(K):
    """One captured call serves every position up to max_ctx, on a side stream's capture, with eager work between."""
    M, n_q, n_kv, D, cap = 24, 32, 8, 128, 3000
    q, rows, kc, vc, bt = tree_inputs(M, n_q, n_kv, D, 16, cap - M, 3)
    qd, words, btd, kd, vd = dev(q, T.mask_words(rows), bt, kc, vc)
    pos = i32(10)
    out = torch.empty(M, n_q * D, dtype=torch.half, device=DEV)
    ws = torch.empty(K.attention_tree_workspace_bytes(M, n_q, n_kv, D, cap), dtype=torch.uint8, device=DEV)
    K.attention_tree(qd, words, pos, btd, kd, vd, cap, out, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.attention_tree(qd, words, pos, btd, kd, vd, cap, out, ws)
    for p in (0, 10, 64, 999, cap - M, 3):
        pos.fill_(p)
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        eager = torch.empty_like(out)
        K.attention_tree(qd, words, pos, btd, kd, vd, cap, eager, torch.full_like(ws, 255))
        assert torch.equal(got, eager), p
        want, bound = T.attention_tree(q[:, :4], rows, p, bt, kc[:, :1], vc[:, :1])
        T.within(got[:, :4 * D], want, bound)


# ------------------------------------------------------------------------------------------------ log probabilities
def run_logprobs(K, x, tokens, k, workspace=True):
    M, V = x.shape
    lp, ent = (torch.full((M,), 9.0, device=DEV) for _ in range(2))
    ids = torch.full((M, k), -7, dtype=torch.int64, device=DEV) if k else None
    top = torch.full((M, k), 9.0, device=DEV) if k else None
    need = K.token_logprobs_workspace_bytes(M, V, k, x.dtype)
    ws = torch.full((need,), 255, dtype=torch.uint8, device=DEV) if need and workspace else None
    K.token_logprobs(x, tokens, lp, ent, ids, top, ws)
    return lp, ent, ids, top


def check_logprobs(K, x, tokens, k):
    given, gb, ent, eb, order, tops, tb = T.token_logprobs(x.cpu(), tokens.cpu(), k)
    for ws in (True, False):
        lp, e, ids, top = run_logprobs(K, x, tokens, k, ws)
        T.within(lp, given, gb)
        T.within(e, ent, eb)
        if k:
            assert torch.equal(ids.cpu(), order)
            T.within(top, tops, tb)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,V,k", [(1, 1, 1), (1, 32000, 5), (3, 7, 7), (2, 1000, 0), (5, 32001, 32), (17, 4099, 20),
                                   (61, 9000, 1), (2, 128256, 32), (300, 513, 3), (1, 160000, 20)])
def test_token_logprobs(K, dtype, M, V, k):
    g = gen(M + V + k)
    x = torch.randn(M, V, generator=g) * 3
    x[:, torch.randint(0, V, (4,), generator=g)] += 9
    x = x.to(dtype).to(DEV)
    tokens = torch.randint(0, V, (M,), generator=g).to(DEV)
    check_logprobs(K, x, tokens, k)


@pytest.mark.parametrize("M,V,k", [(3, 16376, 4), (3, 16384, 4), (2, 32760, 1), (2, 32768, 1), (2, 32768, 0), (300, 20000, 1),
                                   (300, 20000, 3)])
def test_token_logprobs_last_unsplit_sizes(K, M, V, k):
    """Both sides of the row lengths that one launch takes, with a workspace for as many slices as there are and without."""
    g = gen(M + V + k)
    x = (torch.randn(M, V, generator=g) * 2).half()
    x[0] = 1.0                                            # a row of equal values
    tokens = torch.randint(0, V, (M,), generator=g).to(DEV)
    check_logprobs(K, x.to(DEV), tokens, k)
    assert (K.token_logprobs_workspace_bytes(M, V, k) > 0) == (V in (16384, 32768))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_token_logprobs_strided_rows(K, dtype, offset):
    """Rows of a padded matrix, their starts at every alignment; the padding holds NaN."""
    M, V, k = 9, 3001, 6
    wide = torch.full((M, V + 14), float("nan"), dtype=dtype, device=DEV)
    wide[:, offset:offset + V] = (torch.randn(M, V, generator=gen(offset)) * 4).to(dtype).to(DEV)
    check_logprobs(K, wide[:, offset:offset + V], torch.randint(0, V, (M,), generator=gen(1)).to(DEV), k)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_token_logprobs_special_rows(K, dtype):
    """Ties, equal rows, masked ids, the type's lowest value, infinities, NaN, zeros of both signs, ids out of range."""
    V, k = 5000, 12
    low = torch.finfo(dtype).min
    x = torch.randn(14, V, generator=gen(3)) * 2
    x[0] = 1.5                                     # all equal: the first k ids
    x[1] = float("-inf")                           # nothing left
    x[2, 1:] = float("-inf")                       # one id left
    x[3] = low                                     # a row of the lowest value: uniform
    x[4, ::2] = low                                # half of it masked with the lowest value
    x[5, 4000:] = float("-inf")
    x[6, 77] = float("inf")
    x[7, 4999], x[7, 3] = float("nan"), float("nan")
    x[8] = 0.0
    x[8, 1::2] = -0.0                              # the zeros tie
    x[9] = torch.randint(0, 3, (V,), generator=gen(4)).float()      # thousands of ties
    x[10, 5:] = float("-inf")                      # fewer finite ids than alternatives
    x[11] = torch.linspace(-8, 8, V)               # ascending: the last ids
    x[12] = torch.linspace(8, -8, V)
    x[13] = 60000.0 if dtype == torch.float16 else 3e38              # the largest values
    x = x.to(dtype).to(DEV)
    tokens = torch.randint(0, V, (14,), generator=gen(5)).to(DEV)
    tokens[2], tokens[5], tokens[9], tokens[11], tokens[12], tokens[4] = 0, 4500, -1, V, -100, 2
    check_logprobs(K, x, tokens, k)
    for r in range(14):                            # a row alone is split over workgroups
        check_logprobs(K, x[r:r + 1], tokens[r:r + 1], k)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_token_logprobs_raised_regions(K, dtype):
    """Rows of several blocks (8192 values each, 1024 or 2048 where they are split) whose candidates come in crowds: some
    dozens of equal values in the first block, 250 to 520 larger ones in the second, the winners behind them. Whether the
    second crowd fits the list beside the first or not, none of the winners is lost and none comes twice."""
    V, counts = 4 * 8192 + 5, list(range(250, 521, 3))
    g = gen(11)
    x = torch.randn(len(counts), V, generator=g) * 0.1 - 5
    for r, c in enumerate(counts):
        x[r, torch.randperm(8192, generator=g)[:33 + 37 * r % 200]] = 1.0
        x[r, 8192 + torch.randperm(8192, generator=g)[:c]] = 2.0
        x[r, 24576 + 80 * r + torch.arange(5)] = torch.arange(20, 25).float()
        x[r, 16384 + r] = 18.0
    x = x.to(dtype)
    tokens = 24576 + 80 * torch.arange(len(counts))
    given, gb, ent, eb, order, tops, tb = T.token_logprobs(x, tokens, 32)
    x, tokens = x.to(DEV), tokens.to(DEV)
    for k in (2, 5, 20, 32):
        for ws in (True, False):
            lp, e, ids, top = run_logprobs(K, x, tokens, k, ws)
            assert torch.equal(ids.cpu(), order[:, :k]), (k, ws)
            T.within(top, tops[:, :k], tb[:, :k])
            T.within(lp, given, gb)
            T.within(e, ent, eb)


def test_token_logprobs_rows_whose_level_shifts(K):
    """Normal rows whose mean moves from region to region, as where a mask or a language favours a range of ids."""
    V, k = 5 * 8192, 20
    g = gen(12)
    shift = (torch.rand(200, V // 4096, generator=g) * 4).repeat_interleave(4096, 1)
    x = (torch.randn(200, V, generator=g) + shift).to(DEV)
    tokens = torch.randint(0, V, (200,), generator=g).to(DEV)
    check_logprobs(K, x, tokens, k)


@pytest.mark.parametrize("dtype,low", [(t, l) for t in (torch.float16, torch.bfloat16, torch.float32)
                                       for l in (torch.finfo(t).min, -3e4 if t is torch.float16 else -1e38)])
def test_token_logprobs_masked_regions(K, dtype, low):
    """Whole regions at the type's lowest value, or near it, as a mask leaves them: a lane, a wave, a block, a slice or all
    values but one see nothing else, ahead of the finite values or behind them. Each weighs nothing beside a finite value
    and adds nothing to the entropy."""
    V = 3 * 8192 + 100
    x = torch.randn(8, V, generator=gen(9)) * 2
    x[0, :8192] = low                              # the first block
    x[1, 8192:] = low                              # all but the first
    x[2, 1:] = low                                 # all but the first value
    x[3, :-1] = low                                # all but the last
    x[4, 9000:20000] = low                         # blocks in part
    x[5, (torch.arange(V) // 16) % 3 != 0] = low   # by runs of 16
    x[6, :20000] = low
    x[6, 7000] = 1.0
    x[7] = low
    x[7, 100], x[7, 20000] = 3.0, 2.0
    x = x.to(dtype).to(DEV)
    tokens = torch.tensor([8192, 3, 0, V - 1, 10000, 0, 7000, 20000], device=DEV)
    for k in (0, 1, 5):
        check_logprobs(K, x, tokens, k)


def test_token_logprobs_outputs_alone(K):
    """Any output may be left out."""
    x = (torch.randn(4, 2000, generator=gen(0)) * 3).half().to(DEV)
    tokens = torch.tensor([1, 5, 1999, 0], device=DEV)
    lp, ent, ids, top = run_logprobs(K, x, tokens, 3)
    a, b = torch.empty(4, device=DEV), torch.empty(4, device=DEV)
    K.token_logprobs(x, tokens, a)
    K.token_logprobs(x, None, None, b)
    i, t = torch.empty_like(ids), torch.empty_like(top)
    K.token_logprobs(x, None, None, None, i, t)
    assert torch.equal(a, lp) and torch.equal(b, ent) and torch.equal(i, ids) and torch.equal(t, top)


def test_token_logprobs_top1_is_argmax_advance(K):
    x = (torch.randn(32, 32000, generator=gen(2)) * 2).half().to(DEV)
    _, _, ids, _ = run_logprobs(K, x, torch.zeros(32, dtype=torch.int64, device=DEV), 1)
    tok = torch.empty(1, dtype=torch.int64, device=DEV)
    for r in range(32):
        K.argmax_advance(x[r], tok)
        assert int(tok) == int(ids[r, 0])


def test_token_logprobs_replays(K):
    x = (torch.randn(3, 128256, generator=gen(7)) * 2).half().to(DEV)
    tokens = torch.tensor([5, 9, 100], device=DEV)
    lp, ent = torch.empty(3, device=DEV), torch.empty(3, device=DEV)
    ids, top = torch.empty(3, 4, dtype=torch.int64, device=DEV), torch.empty(3, 4, device=DEV)
    ws = torch.empty(max(1, K.token_logprobs_workspace_bytes(3, 128256, 4)), dtype=torch.uint8, device=DEV)
    K.token_logprobs(x, tokens, lp, ent, ids, top, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.token_logprobs(x, tokens, lp, ent, ids, top, ws)
    for i in range(5):
        x.copy_(torch.randn(3, 128256, generator=gen(20 + i)) * 2)
        ws.fill_(255 if i % 2 else 0)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (lp, ent, ids, top)]
        for a, b in zip(got, run_logprobs(K, x, tokens, 4)):
            assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------------ acceptance
def accept_inputs(M, branch, lead, n_kv, page, D, pos, seed, depth=6, edit=None):
    g = gen(seed)
    parents = T.random_parents(M, branch, g)
    tokens = torch.randint(0, 5, (M,), generator=g) if edit == "few ids" else torch.randperm(50000, generator=g)[:M]
    picks = torch.randint(0, 5, (M,), generator=g) if edit == "few ids" else 60000 + torch.arange(M)
    if edit != "few ids":
        cur = 0
        for _ in range(depth):                     # a path of accepted nodes, the last child of each
            kids = [c for c in range(M) if parents[c] == cur]
            if not kids:
                break
            picks[cur] = tokens[kids[-1]]
            cur = kids[-1]
    n_pages = -(-(pos + M) // page) + 2 if pos >= 0 else 4
    kv = torch.randn(*lead, n_pages, n_kv, page, D, generator=g).half()
    bt = torch.randperm(n_pages, generator=g).int()
    return tokens, torch.tensor(parents, dtype=torch.int32), picks, kv, bt


def check_accept(K, tokens, parents, picks, pos, bt, kv, stride=1):
    want = T.tree_accept(tokens.tolist(), parents.tolist(), picks.tolist(), pos, bt, kv)
    M = tokens.numel()
    tok_d, par_d, bt_d, kv_d = dev(tokens, parents, bt, kv)
    pk = torch.full((M, stride), -5, dtype=torch.int64, device=DEV)
    pk[:, 0] = picks.to(DEV)
    path = torch.full((M,), 99, dtype=torch.int32, device=DEV)
    count, tok = i32(77), torch.tensor([-1], device=DEV)
    K.tree_accept(tok_d, par_d, pk[:, 0], i32(pos), bt_d, kv_d, path, count, tok)
    assert path.tolist() == want[0] and int(count) == want[1] and int(tok) == want[2]
    if kv is not None:
        assert torch.equal(kv_d.cpu(), want[3])
    return want[1]


@pytest.mark.parametrize("M,branch,lead,n_kv,page,D,pos", [
    (1, 1, (2, 2), 2, 16, 64, 0), (5, 1, (3, 2), 4, 16, 64, 30), (26, 4, (2, 2), 8, 16, 128, 100),
    (64, 2, (22, 2), 4, 16, 64, 511), (65, 3, (1, 2), 1, 4, 128, 7), (250, 2, (2, 2), 2, 32, 64, 1),
    (1024, 3, (1, 1), 1, 16, 64, 5), (130, 1, (2,), 3, 1, 64, 0), (40, 2, (), 2, 8, 128, 63)])
def test_tree_accept(K, M, branch, lead, n_kv, page, D, pos):
    n = check_accept(K, *(lambda t, p, k, kv, bt: (t, p, k, pos, bt, kv))(
        *accept_inputs(M, branch, lead, n_kv, page, D, pos, M)), stride=1 + M % 3)
    assert M == 1 or n > 1


@pytest.mark.parametrize("depth", [1, 40, 129])
def test_tree_accept_long_paths(K, depth):
    """Paths longer than a wave, every row moving over rows that are still to be read."""
    M = 300
    parents = torch.tensor([-1, -1] + [0] + list(range(2, M - 1)), dtype=torch.int32)   # a chain shifted by one
    tokens = torch.arange(M) + 10
    picks = torch.full((M,), -1)
    cur = 0
    for _ in range(depth):
        kid = 2 if cur == 0 else cur + 1
        picks[cur] = tokens[kid]
        cur = kid
    g = gen(depth)
    kv = torch.randn(2, 2, 12, 2, 32, 64, generator=g).half()
    assert check_accept(K, tokens, parents, picks, 20, torch.randperm(12, generator=g).int(), kv) == depth + 1


def test_tree_accept_duplicate_ids_and_bad_parents(K):
    """The lowest of several matching children; parents that are no earlier node are never walked."""
    for seed in range(6):
        tokens, parents, picks, kv, bt = accept_inputs(200, 4, (1, 2), 1, 16, 64, 3, seed, edit="few ids")
        check_accept(K, tokens, parents, picks, 3, bt, kv)
        parents[5], parents[9], parents[20], parents[30] = 5, 150, -7, 2 ** 31 - 1
        check_accept(K, tokens, parents, picks, 3, bt, kv)


def test_tree_accept_unmapped_rows(K):
    """Rows whose source or target has no page stay; before token 0 there are none; without a cache only the walk."""
    for pos, edit in ((30, "unmapped"), (30, "short"), (-3, None)):
        tokens, parents, picks, kv, bt = accept_inputs(40, 3, (2, 2), 2, 4, 64, max(pos, 0), 11)
        if edit == "unmapped":
            bt[pos // 4], bt[(pos + 5) // 4], bt[(pos + 20) // 4] = -1, kv.size(2), -9
        if edit == "short":
            bt = bt[:(pos + 9) // 4].contiguous()
        check_accept(K, tokens, parents, picks, pos, bt, kv)
    check_accept(K, tokens, parents, picks, 0, bt, None)


# ------------------------------------------------------------------------------------------------ far offsets
def test_caches_past_32_bit_offsets(K):
    """Pages whose values lie past 2^32 values of the cache: append, attention and the move of accepted rows."""
    n_q, n_kv, D, page, M, ctx = 8, 2, 128, 64, 20, 100
    n_pages = (1 << 32) // (n_kv * page * D) + 8
    q, rows, _, _, _ = tree_inputs(M, n_q, n_kv, D, page, ctx, 3)
    kv = torch.empty(2, n_pages, n_kv, page, D, dtype=torch.half, device=DEV)
    kv[:, -3:] = 0
    bt = torch.tensor([n_pages - 1, n_pages - 3], dtype=torch.int32)
    for b in bt.tolist():
        kv[:, b] = torch.randn(2, n_kv, page, D, generator=gen(b % 97)).half().to(DEV)
    kc, vc, btd = kv[0], kv[1], bt.to(DEV)
    qkv = torch.randn(M, (n_q + 2 * n_kv) * D, generator=gen(1)).half()
    cos, sin = rope_tables(ctx + M, D)
    lo = n_pages - 3
    small = (kc[lo:].cpu(), vc[lo:].cpu(), bt - lo)
    q64, qb, k64, kb, v64, _ = T.qk_norm_rope(qkv, None, None, 0.0, cos, sin, ctx, None, small[2], *small[:2], n_q, n_kv)
    out = torch.empty(M, n_q * D, dtype=torch.half, device=DEV)
    K.qk_norm_rope_append_rows(qkv.to(DEV), None, None, 0.0, *dev(cos, sin), i32(ctx), None, btd, kc, vc, n_q, n_kv, out)
    T.within(out.view(M, n_q, D), q64, qb)
    T.within(kc[lo:], k64, kb)
    assert torch.equal(vc[lo:].cpu().double(), v64)
    want, bound = T.attention_tree(out.view(M, n_q, D).cpu(), rows, ctx, small[2], kc[lo:].cpu(), vc[lo:].cpu())
    T.within(run_tree(K, out.view(M, n_q, D), T.mask_words(rows).to(DEV), i32(ctx), btd, kc, vc, ctx + M), want, bound)
    tokens, parents, picks, _, _ = accept_inputs(M, 2, (), 1, 16, 64, 0, 4)
    want = T.tree_accept(tokens.tolist(), parents.tolist(), picks.tolist(), ctx, bt - lo, kv[:, lo:].cpu())
    path, count, tok = torch.empty(M, dtype=torch.int32, device=DEV), i32(0), torch.tensor([0], device=DEV)
    K.tree_accept(*dev(tokens, parents, picks), i32(ctx), btd, kv, path, count, tok)
    assert path.tolist() == want[0] and int(count) > 1 and torch.equal(kv[:, lo:].cpu(), want[3])


@pytest.mark.parametrize("D", [64, 128])
def test_attention_tree_pages_past_32_bit_offsets(K, D):
    """A page of more than 2^32 bytes per head: K is 0 but for a few tokens on both sides of that offset, so that the exact
    output is known. Tolerance: fp16's half step of the output and of a weight, the scores' fp32 roundings, and sums whose
    chains are as long as a split has tiles (2^31 / D tokens in 64 splits and tiles of 32)."""
    log2P = 33 - (7 if D == 64 else 8)
    tokens, M = (1 << 32) // (2 * D) + 5000, 3
    k, v = (torch.zeros(1, 1, 1 << log2P, D, dtype=torch.half, device=DEV) for _ in "kv")
    at = torch.tensor([7, tokens - 5000 - 1, tokens - 5000 + 7, tokens - 2, tokens + 1])
    g = gen(D)
    q = torch.randn(M, 1, D, generator=g).half()
    kx = ((q[:, 0].float().mean(0) + 0.1 * torch.randn(5, D, generator=g)) * 60 * D ** -0.5).half()   # scores about 20
    vx = torch.randn(5, D, generator=g).half()
    k[0, 0, at.to(DEV)], v[0, 0, at.to(DEV)] = kx.to(DEV), vx.to(DEV)
    rows = torch.eye(M, dtype=torch.bool)
    rows[:, 1] = True                                          # (node 1 is the last of them)
    kc, vc = kx.double(), vx.double()
    sc = q[:, 0].double() @ kc.t() * D ** -0.5
    n = tokens + rows.sum(1, keepdim=True) - torch.tensor([5.0])[None]
    w = torch.exp(sc)
    total = w.sum(1, keepdim=True) + n
    want = (w @ vc) / total
    size = (w @ vc.abs()) / total
    ds = 2.0 ** -24 * ((D + 4) * (q[:, 0].double().abs() @ kc.abs().t()) * D ** -0.5 + 4 * sc.abs()).amax(1, keepdim=True)
    rel = 2.0 ** -11 + 2 * (ds + 2.0 ** -21) + 2.0 ** -24 * (2.0 ** 31 / D / 32 / 64 + 128)
    bound = 2.0 ** -11 * want.abs() + rel * size + 2.0 ** -25
    bt = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = run_tree(K, q.to(DEV), T.mask_words(rows).to(DEV), i32(tokens), bt, k, v, tokens + M)
    assert float(want.abs().max()) > 0.05                      # the few weigh against all the others
    T.within(out, want, bound)


# ------------------------------------------------------------------------------------------------ the op module, streams
def test_op_module_refusals(K):
    """Wrong types, shapes and layouts raise before anything is launched."""
    z = lambda *s, t=torch.half: torch.zeros(*s, dtype=t, device=DEV)
    i64 = torch.int64
    kc, bt, pos, cos = z(4, 2, 16, 64), z(4, t=torch.int32), z(1, t=torch.int32), z(64, 32, t=torch.float32)
    qkv, dep = z(3, 6 * 64), z(3, t=torch.int32)
    qk = dict(qkv=qkv, q_w=None, k_w=None, eps=0.0, cos_t=cos, sin_t=cos, pos=pos, depth=dep, bt=bt, kc=kc, vc=kc.clone(),
              n_q=2, n_kv=2)
    for kw, msg in ((dict(qkv=qkv.float()), "qkv must be"), (dict(qkv=z(6 * 64, 3).t()), "contiguous CUDA"),
                    (dict(qkv=z(3, 320)), "qkv must be"), (dict(q_w=z(64)), "both be"), (dict(depth=dep.long()), "depth must"),
                    (dict(depth=dep[:2].contiguous()), "depth must"), (dict(kc=z(4, 2, 16, 96)), "cache must be"),
                    (dict(vc=z(4, 2, 16, 64).cpu()), "vc must be"), (dict(pos=pos.long()), "pos must be"),
                    (dict(sin_t=z(64, 16, t=torch.float32)), "cos and sin"), (dict(q_out=z(3, 120)), "q_out must"),
                    (dict(q_out=z(128, 3).t()), "q_out must"), (dict(n_kv=1), "cache must be")):
        with pytest.raises(RuntimeError, match=msg):
            K.qk_norm_rope_append_rows(**dict(qk, **kw))
    at = dict(q=z(3, 4, 64), mask=z(3, 1, t=i64), pos=pos, bt=bt, kc=kc, vc=kc, max_ctx=30, out=z(3, 256))
    for kw, msg in ((dict(q=z(3, 4, 128)), "q must be"), (dict(q=z(3, 4, 64).bfloat16()), "q must be"),
                    (dict(q=z(3, 64, 4).transpose(1, 2)), "q must be"), (dict(q=z(3, 250)), "must hold"),
                    (dict(out=z(3, 128)), "must hold"), (dict(mask=z(3, 2, t=i64)), "mask must"),
                    (dict(mask=z(3, 1, t=torch.int32)), "mask must be"), (dict(max_ctx=0), "max_ctx"),
                    (dict(workspace=z(64, 2).t()), "contiguous CUDA"), (dict(q=z(3, 6, 64), out=z(3, 384)), "heads-per-group"),
                    (dict(q=z(1, 256).expand(3, 256)), "q_stride")):
        with pytest.raises(RuntimeError, match=msg):
            K.attention_tree(**dict(at, **kw))
    f = lambda *s: z(*s, t=torch.float32)
    lp = dict(logits=z(3, 100), tokens=z(3, t=i64), logprobs=f(3), entropy=f(3), top_ids=z(3, 4, t=i64), top_logprobs=f(3, 4))
    for kw, msg in ((dict(logits=z(3, 100).double()), "fp16, bf16 or fp32"), (dict(logits=z(100, 3).t()), "contiguous rows"),
                    (dict(tokens=z(3, t=torch.int32)), "tokens must be"), (dict(logprobs=f(2)), "M values"),
                    (dict(top_logprobs=None), "both be"), (dict(top_ids=z(3, 0, t=i64), top_logprobs=f(3, 0)), "both be"),
                    (dict(top_ids=z(3, 40, t=i64), top_logprobs=f(3, 40)), "k must"), (dict(tokens=None), "tokens and logprobs")):
        with pytest.raises(RuntimeError, match=msg):
            K.token_logprobs(**dict(lp, **kw))
    ac = dict(tokens=z(3, t=i64), parents=z(3, t=torch.int32), picks=z(3, t=i64), pos=pos, bt=bt, kv=kc,
              path=z(3, t=torch.int32), count=z(1, t=torch.int32), tok=z(1, t=i64))
    for kw, msg in ((dict(picks=z(3, t=torch.int32)), "picks must"), (dict(picks=z(2, t=i64)), "picks must"),
                    (dict(parents=z(3, t=i64)), "parents must be"), (dict(path=z(2, t=torch.int32)), "M values"),
                    (dict(count=z(2, t=torch.int32)), "count and tok"), (dict(kv=z(4, 2, 16, 96)), "cache must be"),
                    (dict(kv=z(2, 16, 64)), "cache must be"), (dict(bt=None), "null pointer")):
        with pytest.raises(RuntimeError, match=msg):
            K.tree_accept(**dict(ac, **kw))
    torch.cuda.synchronize()


def test_sizes_past_32_bits_are_refused(K):
    """Not taken for what their low 32 bits say."""
    z = lambda *s, t=torch.half: torch.zeros(*s, dtype=t, device=DEV)
    kc, bt, pos, out = z(4, 2, 16, 64), z(4, t=torch.int32), z(1, t=torch.int32), z(3, 256)
    for max_ctx in ((1 << 32) + 30, (1 << 60) + 30, 30 - (1 << 32)):
        with pytest.raises(RuntimeError, match="32 bits"):
            K.attention_tree(z(3, 4, 64), None, pos, bt, kc, kc, max_ctx, out)
    logits = torch.empty(1, (1 << 32) + 100, dtype=torch.half, device=DEV)
    with pytest.raises(RuntimeError, match="32 bits"):
        K.token_logprobs(logits, None, None, z(1, t=torch.float32))
    with pytest.raises(RuntimeError, match="32 bits"):
        K.token_logprobs(logits.view(-1, 1), None, None, z((1 << 32) + 100, t=torch.float32))
    del logits
    torch.cuda.empty_cache()


def test_graphs_share_a_workspace_and_streams(K):
    """Two captured calls of different sizes with one workspace, replayed in turn with eager work (torch's and the ops' own,
    on another stream with a workspace of its own) between; every replay against the eager result."""
    cases = []
    for M, ctx, V in ((30, 900, 40000), (7, 2500, 128256)):
        q, rows, kc, vc, bt = tree_inputs(M, 16, 4, 128, 16, ctx, 3)
        x = torch.randn(M, V, generator=gen(V)).half()
        qd, words, btd, kd, vd, xd = dev(q, T.mask_words(rows), bt, kc, vc, x)
        cases.append(dict(a=(qd, words, i32(ctx), btd, kd, vd, ctx + M), x=xd, tok=torch.arange(M, device=DEV),
                          out=torch.empty(M, 16 * 128, dtype=torch.half, device=DEV), lp=torch.empty(M, device=DEV),
                          ent=torch.empty(M, device=DEV), ids=torch.empty(M, 3, dtype=torch.int64, device=DEV),
                          top=torch.empty(M, 3, device=DEV)))
    need = max([K.attention_tree_workspace_bytes(c["x"].size(0), 16, 4, 128, c["a"][6]) for c in cases] +
               [K.token_logprobs_workspace_bytes(*c["x"].shape, 3) for c in cases])
    assert need > 0
    ws = [torch.full((need,), 255, dtype=torch.uint8, device=DEV) for _ in range(2)]

    def go(c, w):
        K.attention_tree(*c["a"], c["out"], w)
        K.token_logprobs(c["x"], c["tok"], c["lp"], c["ent"], c["ids"], c["top"], w)

    results = lambda c: [c[k].clone() for k in ("out", "lp", "ent", "ids", "top")]
    side = torch.cuda.Stream()
    graphs, want = [], []
    for c in cases:
        go(c, ws[0])
        want.append(results(c))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            go(c, ws[0])
        graphs.append(g)
    for turn in range(3):
        for i, (c, g) in enumerate(zip(cases, graphs)):
            for k in ("out", "lp", "ent", "ids", "top"):
                c[k].zero_()
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(results(c), want[i])), (turn, i)
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                go(cases[1 - i], ws[1])
            torch.cuda.current_stream().wait_stream(side)
            assert all(torch.equal(a, b) for a, b in zip(results(cases[1 - i]), want[1 - i])), (turn, i)
