"""GPU tests of the 8-bit cache and of attention under a sliding window, each against its 64-bit reference (kv8_ref): codes,
scales and q bit for bit, attention within the error bounds that its roundings allow."""
import pytest
import torch

import kv8_ref as R
from helpers import DEV, gen
from runtime.model import rope_tables

pytestmark = pytest.mark.gpu

CODES = [torch.int8, torch.float8_e4m3fn]
CACHES = [torch.half, *CODES]
name = lambda d: str(d).split(".")[-1]


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


def same(a, b):
    """Bit for bit (8-bit types have no torch.equal of their own)."""
    a, b = a.detach().cpu(), b.detach().cpu()
    raw = lambda t: t.contiguous().view(torch.uint8)
    return a.dtype == b.dtype and a.shape == b.shape and torch.equal(raw(a), raw(b))


def empty_cache(n_pages, n_kv, P, D, dtype, g, scale=float("nan")):
    """Two caches of arbitrary bytes, as memory comes, and scales of NaN; with a scale: arbitrary values at that scale."""
    raw = lambda *s: torch.randint(0, 256, s, generator=g, dtype=torch.uint8)
    kc, vc = (raw(n_pages, n_kv, P, D) for _ in "kv")
    if scale == scale:
        kc, vc = (torch.where(c & 0x7F == 0x7F, c & 0xBF, c) for c in (kc, vc))
    ks, vs = (torch.full((n_pages, n_kv, P // R.BLOCK), scale) for _ in "kv")
    return kc.view(dtype), vc.view(dtype), ks, vs


def qkv_rows(M, n_q, n_kv, D, g, spread=1.0):
    return (torch.randn(M, (n_q + 2 * n_kv) * D, generator=g) * torch.exp(spread * torch.randn(M, 1, generator=g))).half()


# ------------------------------------------------------------------------------------------------ append
@pytest.mark.parametrize("dtype", CODES, ids=name)
@pytest.mark.parametrize("M,n_q,n_kv,D,page,start", [
    (1, 32, 8, 128, 16, 0), (1, 8, 4, 64, 16, 15), (2, 3, 1, 64, 32, 15), (3, 32, 8, 128, 16, 5), (16, 4, 2, 128, 64, 16),
    (17, 8, 8, 64, 16, 31), (100, 40, 8, 128, 16, 3), (61, 32, 4, 64, 128, 777),
    (130, 1, 1, 128, 32, 0), (33, 5, 5, 64, 16, 1)])
def test_append_rows(K, dtype, M, n_q, n_kv, D, page, start):
    g = gen(M + start + D)
    n_pages = (start + M) // page + 3
    kc, vc, ks, vs = empty_cache(n_pages, n_kv, page, D, dtype, g)
    bt = torch.randperm(n_pages, generator=g).int()
    cos, sin = rope_tables(start + M + 1, D, 500000.0)
    first = start // 16 * 16
    if first < start:                                 # the tokens that share the first block
        _, (kc, vc, ks, vs) = R.append(qkv_rows(start - first, n_q, n_kv, D, g), cos, sin, first, bt, kc, vc, ks, vs, n_q)
    qkv = qkv_rows(M, n_q, n_kv, D, g)
    q, want = R.append(qkv, cos, sin, start, bt, kc, vc, ks, vs, n_q)
    x, cosd, sind, btd, *c = dev(qkv, cos, sin, bt, kc, vc, ks, vs)
    wide = torch.full((M, n_q * D + 24), 7.0, dtype=torch.half, device=DEV)
    K.kv8_append_rows(x, cosd, sind, i32(start), btd, *c, n_q, n_kv, wide[:, :n_q * D])
    assert torch.equal(wide[:, :n_q * D].cpu().view(M, n_q, D), q)
    for a, b in zip(c, want):
        assert same(a, b)                             # every other byte and scale is as it was
    assert torch.equal(x.cpu(), qkv) and bool((wide[:, n_q * D:] == 7).all())
    # in place and once more: q over qkv's own, the same codes (the first block keeps its scale)
    K.kv8_append_rows(x, cosd, sind, i32(start), btd, *c, n_q, n_kv)
    assert torch.equal(x[:, :n_q * D], wide[:, :n_q * D]) and torch.equal(x[:, n_q * D:].cpu(), qkv[:, n_q * D:])
    assert all(same(a, b) for a, b in zip(c, want))


@pytest.mark.parametrize("dtype", CODES, ids=name)
@pytest.mark.parametrize("D", [64, 128])
def test_append_without_rotation(K, dtype, D):
    M, n_q, n_kv, page, start = 21, 4, 2, 16, 7
    g = gen(D)
    kc, vc, ks, vs = empty_cache(4, n_kv, page, D, dtype, g, 2.0 ** -6)
    vs /= 2
    bt = torch.tensor([2, 0, 3], dtype=torch.int32)
    qkv = qkv_rows(M, n_q, n_kv, D, g)
    q, want = R.append(qkv, None, None, start, bt, kc, vc, ks, vs, n_q)
    x, btd, *c = dev(qkv, bt, kc, vc, ks, vs)
    out = torch.empty(M, n_q * D, dtype=torch.half, device=DEV)
    K.kv8_append_rows(x, None, None, i32(start), btd, *c, n_q, n_kv, out)
    assert torch.equal(out.cpu().view(M, n_q, D), q) and all(same(a, b) for a, b in zip(c, want))
    K.kv8_append_rows(x, None, None, i32(start), btd, *c, n_q, n_kv)
    assert torch.equal(x.cpu(), qkv)


@pytest.mark.parametrize("dtype", CODES, ids=name)
def test_append_token_by_token_is_the_reference(K, dtype):
    """A sequence of 50 tokens whose size wanders over six orders, through blocks that grow; eager calls and replays of a
    captured one."""
    n_q, n_kv, D, page, n = 4, 2, 128, 32, 50
    g = gen(9)
    kc, vc, ks, vs = empty_cache(3, n_kv, page, D, dtype, g)
    bt = torch.tensor([1, 2], dtype=torch.int32)
    rows = qkv_rows(n, n_q, n_kv, D, g, spread=2.5)
    cos, sin = rope_tables(n, D)
    a = dev(kc, vc, ks, vs)
    b = dev(kc, vc, ks, vs)
    cosd, sind, btd, rd = dev(cos, sin, bt, rows)
    x, pos, q = torch.empty_like(rd[:1]), i32(0), torch.empty(1, n_q * D, dtype=torch.half, device=DEV)
    spare = dev(kc, vc, ks, vs)
    K.kv8_append_rows(rd[:1], cosd, sind, pos, btd, *spare, n_q, n_kv, q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.kv8_append_rows(x, cosd, sind, pos, btd, *b, n_q, n_kv, q)
    want = [kc, vc, ks, vs]
    for t in range(n):
        qr, want = R.append(rows[t:t + 1], cos, sin, t, bt, *want, n_q)
        pos.fill_(t)
        K.kv8_append_rows(rd[t:t + 1], cosd, sind, pos, btd, *a, n_q, n_kv, q)
        assert torch.equal(q.cpu().view(1, n_q, D), qr)
        x.copy_(rd[t:t + 1])
        q.zero_()
        graph.replay()
        assert torch.equal(q.cpu().view(1, n_q, D), qr)
    for got in (a, b):
        assert all(same(u, v) for u, v in zip(got, want))


@pytest.mark.parametrize("dtype", CODES, ids=name)
@pytest.mark.parametrize("order", ["sorted", "mixed"])
def test_append_every_fp16_value(K, dtype, order):
    """All 65536 patterns, NaN and infinities among them: sorted by size, so that a block's scale fits its values, and mixed,
    so that almost every block meets the largest scale."""
    D, M = 128, 512
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.half)
    key = torch.nan_to_num(x.float().abs(), nan=1e9, posinf=1e8) if order == "sorted" else torch.rand(65536, generator=gen(1))
    v = x[torch.sort(key, stable=True).indices].view(M, D)
    v = torch.where(torch.isnan(v), torch.full_like(v, float("nan")), v)      # one NaN: its payload is no part of a value
    qkv = torch.cat([torch.zeros(M, D).half(), v, v], 1)
    kc, vc, ks, vs = empty_cache(32, 1, 16, D, dtype, gen(2))
    bt = torch.arange(32).int()
    _, want = R.append(qkv, None, None, 0, bt, kc, vc, ks, vs, 1)
    x, btd, *c = dev(qkv, bt, kc, vc, ks, vs)
    K.kv8_append_rows(x, None, None, i32(0), btd, *c, 1, 1)
    for got, ref in zip(c[2:], want[2:]):
        assert torch.equal(got.cpu(), ref)
    ref = R.values(want[0], want[2])
    for code in c[:2]:
        R.within(R.values(code.cpu(), want[2]), ref, torch.zeros(()))
    back = [torch.empty(M, D, dtype=torch.half, device=DEV) for _ in "kv"]
    K.kv8_read(btd, *c, 0, *back)
    for b in back:
        R.within(b, ref.view(M, D), torch.zeros(()))


@pytest.mark.parametrize("dtype", CODES, ids=name)
@pytest.mark.parametrize("start,rows,edit", [
    (-3, 20, None),              # rows of tokens before 0 touch nothing
    (-40, 20, None),             # none of them exists
    (40, 12, "short table"),     # rows past the tables touch nothing
    (40, 30, "short bt"),        # tokens past the block table: rotated, not appended
    (40, 30, "unmapped"),        # a page that is no page of the cache: rotated, not appended
    (2 ** 31 - 5, 10, "far")])   # positions at the end of 32 bits
def test_append_rows_out_of_range(K, dtype, start, rows, edit):
    n_q, n_kv, D, page = 4, 2, 64, 16
    g = gen(rows)
    kc, vc, ks, vs = empty_cache(6, n_kv, page, D, dtype, g, 2.0 ** -8)
    bt = torch.tensor([5, 2, 1, 0, 4], dtype=torch.int32)
    cos, sin = rope_tables(80, D)
    if edit == "short table":
        cos, sin = cos[:45].contiguous(), sin[:45].contiguous()
    if edit == "short bt":
        bt = bt[:3].contiguous()
    if edit == "unmapped":
        bt[2], bt[3] = -1, 6
    qkv = qkv_rows(rows, n_q, n_kv, D, g)
    q, want = R.append(qkv, cos, sin, start, bt, kc, vc, ks, vs, n_q)
    x, cosd, sind, btd, *c = dev(qkv, cos, sin, bt, kc, vc, ks, vs)
    out = torch.full((rows, n_q * D), float("nan"), dtype=torch.half, device=DEV)
    K.kv8_append_rows(x, cosd, sind, i32(start), btd, *c, n_q, n_kv, out)
    R.within(out.view(rows, n_q, D), q, torch.zeros(()))
    assert all(same(a, b) for a, b in zip(c, want))


# ------------------------------------------------------------------------------------------------ read back
@pytest.mark.parametrize("dtype", CODES, ids=name)
@pytest.mark.parametrize("n_kv,D,page,start,n", [(8, 128, 16, 0, 100), (1, 64, 16, 15, 1), (3, 64, 32, 5, 61),
                                                 (4, 128, 64, 63, 66)])
def test_read(K, dtype, n_kv, D, page, start, n):
    g = gen(n)
    n_pages = (start + n) // page + 2
    kc, vc, ks, vs = empty_cache(n_pages, n_kv, page, D, dtype, g)
    for s in (ks, vs):
        s.copy_(2.0 ** torch.randint(-24, 8, s.shape, generator=g).float())
    bt = torch.randperm(n_pages, generator=g).int()
    if n > 60:
        bt[(start + 40) // page] = -1                 # its tokens read as zeros
    k, v = (torch.full((n + 1, n_kv, D), 7.0, dtype=torch.half, device=DEV) for _ in "kv")
    btd, *c = dev(bt, kc, vc, ks, vs)
    K.kv8_read(btd, *c, start, k[:n], v[:n])
    for got, code, scale in ((k, kc, ks), (v, vc, vs)):
        val, want = R.values(code, scale), torch.zeros(n, n_kv, D, dtype=torch.float64)
        for i in range(n):
            cell = R.token_row(bt.tolist(), start + i, page, n_pages)
            if cell is not None:
                want[i] = val[cell[0], :, cell[1]]
        assert float(torch.nan_to_num(want.abs(), 0.0).max()) <= 65504
        # exact, NaN codes included, but for codes that no fp16 number has: an e4m3 code has 4 significant bits, so its product
        # is an fp16 number from 2^-14 on, and below that within half a step of the subnormals, 2^-25
        R.within(got[:n], want, torch.where(want.abs() < 2.0 ** -14, 2.0 ** -25 * (dtype != torch.int8), 0.0))
        assert bool((got[n] == 7).all())
    flat = torch.empty(n, n_kv * D, dtype=torch.half, device=DEV)
    K.kv8_read(btd, *c, start, flat, torch.empty_like(flat))
    assert same(flat.view(n, n_kv, D), k[:n])


# ------------------------------------------------------------------------------------------------ attention
def paged_kv(tokens, n_kv, D, page, dtype, g, extra=2, peaky=1.0):
    """A cache that holds `tokens` tokens, arbitrary bytes elsewhere (NaN in an fp16 one): codes, scales (None: fp16), table,
    and the caches' values in fp64."""
    n_pages = -(-tokens // page) + extra
    bt = torch.randperm(n_pages, generator=g).int()
    if dtype == torch.half:
        caches = [torch.full((n_pages, n_kv, page, D), float("nan"), dtype=torch.half) for _ in "kv"]
        scales = [None, None]
    else:
        kc, vc, ks, vs = empty_cache(n_pages, n_kv, page, D, dtype, g)
        caches, scales = [kc, vc], [ks, vs]
    for c, s, size in zip(caches, scales, (peaky, 1.0)):
        rows = (torch.randn(tokens, n_kv, D, generator=g) * size).half()
        for b in range(0, tokens, 16 if page >= 16 else page):
            i, slot = int(bt[b // page]), b % page
            blk = rows[b:b + min(16, page)]
            if s is None:
                c[i, :, slot:slot + blk.size(0)] = blk.transpose(0, 1)
                continue
            for h in range(n_kv):
                sc = R.scale_of(blk[:, h], dtype)
                s[i, h, slot // 16] = sc
                c[i, h, slot:slot + blk.size(0)] = R.to_codes(R.codes_of(blk[:, h], sc, dtype), dtype)
    return caches, scales, bt, [R.values(c, s) for c, s in zip(caches, scales)]


def run(K, q, pos, bt, caches, scales, cap, window=0, sinks=0, ws="full"):
    M, n_kv, D = q.size(0), caches[0].size(1), caches[0].size(3)
    n_q = q.numel() // (M * D)
    dtype = caches[0].dtype
    out = torch.full((M, n_q * D), float("nan"), dtype=torch.half, device=DEV)
    need = K.attention_window_workspace_bytes(M, n_q, n_kv, D, cap, window, sinks, dtype)
    need = {"full": need, "half": need // 2, "none": 0}[ws]
    w = torch.full((need,), 255, dtype=torch.uint8, device=DEV) if need else None
    if dtype == torch.half:
        K.attention_window(q, pos, bt, *caches, cap, out, window, sinks, w)
    else:
        K.attention_kv8(q, pos, bt, *caches, *scales, cap, out, window, sinks, w)
    return out


def check(K, q, pos, bt, caches, scales, vals, cap, window=0, sinks=0, rows=slice(None), ws=("full", "half", "none")):
    want, bound = R.attention(q, pos, bt, *vals, cap, window, sinks)
    a = dev(q, bt, *caches, *scales)
    for w in ws:
        out = run(K, a[0], i32(pos), a[1], a[2:4], a[4:6], cap, window, sinks, w)
        R.within(out[rows], want[rows], bound[rows])
    return out


@pytest.mark.parametrize("dtype", CACHES, ids=name)
@pytest.mark.parametrize("M,n_q,n_kv,D,page,pos,window,sinks", [
    (1, 32, 4, 64, 16, 0, 0, 0), (1, 32, 8, 128, 16, 299, 0, 0), (1, 32, 8, 128, 32, 2047, 0, 0),
    (1, 8, 8, 64, 16, 1000, 100, 4), (1, 8, 1, 128, 16, 777, 200, 70), (1, 4, 2, 128, 64, 1500, 1, 0),
    (2, 16, 2, 128, 16, 500, 64, 3), (4, 8, 2, 64, 32, 333, 0, 0), (5, 32, 4, 64, 16, 295, 37, 5),
    (16, 2, 2, 128, 16, 600, 0, 0), (17, 8, 4, 64, 16, 90, 16, 16), (3, 16, 2, 128, 16, 1800, 512, 1),
    (33, 32, 8, 128, 16, 0, 0, 0), (64, 8, 1, 128, 32, 400, 130, 33), (100, 32, 8, 128, 16, 301, 0, 0),
    (130, 4, 4, 64, 16, 0, 20, 4), (200, 16, 2, 64, 16, 64, 0, 0), (257, 8, 2, 128, 64, 3, 100, 0)])
def test_attention(K, dtype, M, n_q, n_kv, D, page, pos, window, sinks):
    g = gen(M + pos + D + window)
    caches, scales, bt, vals = paged_kv(pos + M, n_kv, D, page, dtype, g)
    q = torch.randn(M, n_q, D, generator=g).half()
    check(K, q, pos, bt, caches, scales, vals, pos + M, window, sinks)


@pytest.mark.parametrize("dtype", CACHES, ids=name)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("M,pos,cap,window", [(1, 900, 900, 0), (1, 900, 5000, 0), (1, 900, 60000, 0), (1, 900, 1 << 22, 0),
                                              (3, 2000, 1 << 22, 700)])
def test_attention_every_plan_of_few_columns(K, dtype, D, M, pos, cap, window):
    """max_ctx and the window choose whether a call of few columns is split, by how many waves, and how K and V are loaded."""
    cap = max(cap, pos + M)
    caches, scales, bt, vals = paged_kv(pos + M, 2, D, 16, dtype, gen(D + M))
    q = torch.randn(M, 8, D, generator=gen(1)).half()
    check(K, q, pos, bt, caches, scales, vals, cap, window, 4 if window else 0)


@pytest.mark.parametrize("dtype", CACHES, ids=name)
@pytest.mark.parametrize("M,pos,window,sinks", [(1, 40, 1 << 30, 0), (3, 40, 43, 0), (3, 40, 5, 1 << 30), (3, 40, 5, 36),
                                                (3, 2, 3, 3), (40, 0, 1, 1), (40, 0, 40, 9), (40, 25, 7, 30)])
def test_attention_windows_that_meet_their_sinks(K, dtype, M, pos, window, sinks):
    caches, scales, bt, vals = paged_kv(pos + M, 2, 64, 16, dtype, gen(M))
    q = torch.randn(M, 8, 64, generator=gen(1)).half()
    check(K, q, pos, bt, caches, scales, vals, pos + M, window, sinks)


@pytest.mark.parametrize("dtype", CACHES, ids=name)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("M,cap", [(1, 5000), (4, 100000), (9, 700), (60, 20000), (150, 5000), (300, 1200)])
def test_attention_caps_and_holes(K, dtype, D, M, cap):
    """max_ctx far above the position (splits without a token), below it, a table that ends early, pages that are not mapped
    (one of them holds the newest token), and *pos < 0."""
    n_q, n_kv, page, pos = 8, 2, 16, 333
    caches, scales, bt, vals = paged_kv(pos + M, n_kv, D, page, dtype, gen(M + D))
    q = torch.randn(M, n_q, D, generator=gen(2)).half()
    bt[3], bt[(pos + M - 1) // page], bt[11] = -1, caches[0].size(0), 1 << 20
    for window, sinks in ((0, 0), (70, 60), (30, 0)):
        check(K, q, pos, bt, caches, scales, vals, cap, window, sinks, ws=("full", "none"))
    check(K, q, pos, bt, caches, scales, vals, 100, 0, 0, ws=("full",))
    check(K, q, pos, bt, caches, scales, vals, 100, 250, 20, ws=("full",))
    check(K, q, pos, bt[:5].contiguous(), caches, scales, vals, cap, 0, 0, ws=("full",))
    check(K, q, pos, torch.full_like(bt, -1), caches, scales, vals, cap, 60, 4, ws=("full",))     # nothing at all: zeros
    check(K, q, -2, bt, caches, scales, vals, cap, 0, 0, ws=("full",))                            # rows 0 and 1 are nowhere
    check(K, q, -(1 << 31), bt, caches, scales, vals, cap, 3, 4, ws=("full",))


@pytest.mark.parametrize("dtype", CACHES, ids=name)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("M,pos,cap,window,sinks,hpg,n_kv", [
    (60, 440, 500, 0, 0, 4, 2), (700, 0, 700, 100, 20, 1, 16), (40, 700, 1 << 20, 0, 0, 4, 2), (800, 0, 800, 0, 0, 8, 8),
    (1500, 0, 1500, 30, 4, 8, 8), (1200, 0, 1200, 200, 70, 1, 32), (130, 900, 60000, 0, 0, 8, 8),
    (300, 500, 20000, 400, 4, 4, 2)])
def test_attention_every_workgroup_shape(K, dtype, D, M, pos, cap, window, sinks, hpg, n_kv):
    """The sizes choose among the shapes of a workgroup, split and not: rows spread over all of them, heads of the first and
    the last kv head, with a page that is not mapped and (fp16, e4m3) a NaN in V of a token that some of the rows attend."""
    page, n_q = 16, hpg * n_kv
    caches, scales, bt, vals = paged_kv(pos + M, n_kv, D, page, dtype, gen(M + D))
    q = torch.randn(M, n_q, D, generator=gen(7)).half()
    bt[(pos + M // 3) // page] = -1
    bad = pos + M // 2 + 30
    if dtype != torch.int8:
        c = R.token_row(bt.tolist(), bad, page, caches[0].size(0))
        for v in (caches, vals):
            v[1][c[0], :, c[1], 9] = float("nan")
    a = dev(q, bt, *caches, *scales)
    half = M // 2
    rows = sorted({0, 1, M // 3 - 1, M // 3, half, half + 29, half + 30, half + 31, M - 1, *range(5, M, max(1, M // 16))})
    for ws in ("full", "none"):
        out = run(K, a[0], i32(pos), a[1], a[2:4], a[4:6], cap, window, sinks, ws).view(M, n_q, D)
        for h in (0, n_kv - 1):
            heads = slice(h * hpg, (h + 1) * hpg)
            for m in (r for r in rows if r < M):
                sees = dtype != torch.int8 and pos + m >= bad and (not window or bad > pos + m - window)
                of = [v[:, h:h + 1] for v in vals]
                want, bound = R.attention(q[m:m + 1, heads], pos + m, bt, *of, cap, window, sinks)
                if sees:
                    assert bool(torch.isnan(out[m, heads, 9]).all()) and bool(torch.isfinite(out[m, heads, :9]).all())
                else:
                    R.within(out[m:m + 1, heads].reshape(1, -1), want, bound)


@pytest.mark.parametrize("dtype", [torch.half, torch.float8_e4m3fn], ids=name)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("M,pos,window,sinks,cap", [
    (6, 90, 0, 0, 96), (12, 400, 0, 0, 5000), (2, 60, 30, 4, 62), (50, 30, 12, 3, 80), (120, 200, 60, 3, 20000),
    (200, 0, 40, 20, 200)])
def test_attention_keeps_unattended_values_out(K, dtype, D, M, pos, window, sinks, cap):
    """NaN in K and V of a token, and NaN (fp16: infinity) in V of two more, among the rows' positions and next to the sinks:
    rows that attend them see them, no other row does."""
    n_q, n_kv, page = 8, 2, 16
    caches, scales, bt, vals = paged_kv(pos + M, n_kv, D, page, dtype, gen(pos + D))
    q = torch.randn(M, n_q, D, generator=gen(4)).half()
    nan, inf = float("nan"), float("inf") if dtype == torch.half else float("nan")
    bad = {pos + M // 2: nan, pos + M // 2 + (M > 4): inf}
    if window:
        bad[sinks + 1] = inf
    for t, b in bad.items():
        c = R.token_row(bt.tolist(), t, page, caches[0].size(0))
        for v in (caches, vals):
            if t == pos + M // 2:
                v[0][c[0], 0, c[1], 3] = b
            v[1][c[0], :, c[1], 9] = b
    see = lambda p, t: t <= p and (not window or t > p - window or t < sinks)
    kept = [m for m in range(M) if not any(see(pos + m, t) for t in bad)]
    hit = [m for m in range(M) if m not in kept]
    assert hit and kept
    clean = [v.clone() for v in vals]
    check(K, q, pos, bt, caches, scales, vals, cap, window, sinks, rows=kept)
    a = dev(q, bt, *caches, *scales)
    out = run(K, a[0], i32(pos), a[1], a[2:4], a[4:6], cap, window, sinks)
    got = out.view(M, n_q, D)[hit][:, n_q // n_kv:]              # the kv head whose K is finite
    assert not bool(torch.isfinite(got[..., 9]).any())
    for t in bad:                                               # the other dims: as if nothing had been there
        c = R.token_row(bt.tolist(), t, page, caches[0].size(0))
        clean[0][c[0], 0, c[1], 3], clean[1][c[0], :, c[1], 9] = 0.0, 0.0
    want, bound = R.attention(q, pos, bt, *clean, cap, window, sinks)
    keep = [d for d in range(D) if d != 9]
    shape = lambda x: x.view(M, n_q, D)[hit][:, n_q // n_kv:][..., keep]
    R.within(shape(out), shape(want), shape(bound))


@pytest.mark.parametrize("dtype", [torch.half, torch.float8_e4m3fn], ids=name)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("M,pos,window,sinks", [(1, 200, 50, 4), (3, 200, 50, 4), (1, 97, 33, 0), (40, 500, 70, 9),
                                                (200, 600, 100, 3)])
def test_attention_nan_outside_every_window(K, dtype, D, M, pos, window, sinks):
    """Tokens that no row attends, next to the windows and the sinks and in the tiles that are read, hold NaN in K and V."""
    n_q, n_kv, page = 8, 2, 16
    caches, scales, bt, vals = paged_kv(pos + M, n_kv, D, page, dtype, gen(pos + D))
    q = torch.randn(M, n_q, D, generator=gen(4)).half()
    lo = pos - window + 1
    for t in {lo - 1, lo - 2, lo - 17, sinks, sinks + 1, sinks + 20}:
        c = R.token_row(bt.tolist(), t, page, caches[0].size(0))
        for x in (*caches, *vals):
            x[c[0], :, c[1]] = float("nan")
    check(K, q, pos, bt, caches, scales, vals, pos + M, window, sinks)


@pytest.mark.parametrize("dtype", CACHES, ids=name)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("M,cap", [(1, 1000), (3, 20000), (70, 1200), (150, 20000)])
@pytest.mark.parametrize("slope", [0.004, 0.05, -0.02])
def test_attention_rising_scores(K, dtype, D, M, cap, slope):
    """Scores that rise or fall steadily with the position: the reference of the weights moves again and again."""
    n_q, n_kv, page, pos = 8, 2, 16, 800
    caches, scales, bt, vals = paged_kv(pos + M, n_kv, D, page, dtype, gen(21))
    q = (torch.randn(M, n_q, D, generator=gen(3)) * 0.1 + 0.5).half()
    kc = torch.zeros_like(vals[0])
    for t in range(pos + M):
        c = R.token_row(bt.tolist(), t, page, caches[0].size(0))
        kc[c[0], :, c[1]] = 0.2 * torch.nan_to_num(vals[0][c[0], :, c[1]]) + slope * t
    if dtype == torch.half:
        caches[0] = kc.half()
    else:
        for b in range(kc.size(0)):
            for h in range(n_kv):
                sc = R.scale_of(kc[b, h].half(), dtype)
                scales[0][b, h, 0] = sc
                caches[0][b, h] = R.to_codes(R.codes_of(kc[b, h].half(), sc, dtype), dtype)
    vals[0] = R.values(caches[0], scales[0])
    check(K, q, pos, bt, caches, scales, vals, cap, 0, 0, ws=("full", "none"))


@pytest.mark.parametrize("dtype", CACHES, ids=name)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("M,pos,cap", [(1, 0, 100), (1, 300, 5000), (4, 300, 384), (20, 700, 1500), (130, 700, 20000)])
@pytest.mark.parametrize("size", [30.0, 1000.0, 16384.0, 57344.0, -2000.0, -57344.0])
def test_attention_far_scores(K, dtype, D, M, pos, cap, size):
    """Scores as large as finite q and K make them. Equal ones weigh alike, whatever their size: the output is the mean of V
    over the tokens that a row sees.

    Tolerance: fp16's half step of the output and of the weight (the same one for every token), and the fp32 sums, a chain of
    at most n + 64 terms of |v| / n. (57344 is a code times a scale in either 8-bit format.)"""
    n_q, n_kv, page = 8, 2, 16
    caches, scales, bt, vals = paged_kv(pos + M, n_kv, D, page, dtype, gen(31))
    g = gen(6)
    q = (abs(size) * (0.5 + 0.5 * torch.rand(M, n_q, D, generator=g))).half()
    row = (size * (0.5 + 0.5 * torch.rand(n_kv, D, generator=g))).half()
    row[:, 0] = size
    if dtype == torch.half:
        caches[0] = row[None, :, None].expand_as(caches[0]).contiguous()
    else:
        for h in range(n_kv):
            sc = R.scale_of(row[h], dtype)
            scales[0][:, h] = sc
            caches[0][:, h] = R.to_codes(R.codes_of(row[h], sc, dtype), dtype)
    cells = [R.token_row(bt.tolist(), t, page, caches[0].size(0)) for t in range(pos + M)]
    v = torch.stack([vals[1][c[0], :, c[1]] for c in cells])                      # [tokens, n_kv, D]
    see = torch.arange(pos + M)[None] <= pos + torch.arange(M)[:, None]
    n = see.sum(1)[:, None, None]
    mean, size_ = ((see.double() @ x.reshape(pos + M, -1)).view(M, n_kv, D) / n for x in (v, v.abs()))
    bound = 2.0 ** -11 * mean.abs() + (2.0 ** -11 + 2.0 ** -24 * (n + 64)) * size_ + 2.0 ** -25
    wide = lambda x: x.repeat_interleave(n_q // n_kv, 1).reshape(M, -1)
    a = dev(q, bt, *caches, *scales)
    for ws in ("full", "none"):
        R.within(run(K, a[0], i32(pos), a[1], a[2:4], a[4:6], cap, ws=ws), wide(mean), wide(bound))


@pytest.mark.parametrize("M,pos,cap", [(1, 300, 2000), (40, 300, 2000)])
def test_attention_infinite_scores(K, M, pos, cap):
    """A score of +infinity, or NaN, leaves no distribution: NaN for the rows that see it, and for no other."""
    n_q, n_kv, D, page = 8, 2, 64, 16
    caches, scales, bt, vals = paged_kv(pos + M, n_kv, D, page, torch.half, gen(5))
    q = (torch.randn(M, n_q, D, generator=gen(5)).abs() + 0.5).half()
    for bad in (float("inf"), float("nan")):
        t = pos + M // 2
        k = caches[0].clone()
        c = R.token_row(bt.tolist(), t, page, k.size(0))
        k[c[0], :, c[1], 1] = bad
        out = run(K, *dev(q), i32(pos), *dev(bt), dev(k, caches[1]), scales, cap)
        assert bool(torch.isnan(out[M // 2:]).all())
        if M > 1:
            check(K, q, pos, bt, [k, caches[1]], scales, vals, cap, rows=slice(0, M // 2), ws=("full",))


@pytest.mark.parametrize("dtype", CACHES, ids=name)
@pytest.mark.parametrize("D,M,window", [(64, 40, 0), (128, 40, 100), (128, 3, 50)])
def test_a_row_does_not_depend_on_later_ones(K, dtype, D, M, window):
    """Not in a bit: the tokens that only later rows attend, and those rows' queries, change."""
    n_q, n_kv, page, pos, m = 8, 2, 16, 500, M // 2
    caches, scales, bt, _ = paged_kv(pos + M, n_kv, D, page, dtype, gen(D))
    q = torch.randn(M, n_q, D, generator=gen(8)).half()
    first = run(K, *dev(q), i32(pos), *dev(bt), dev(*caches), dev(*scales), pos + M, window, 4)
    q[m:] *= 5
    for t in range(pos + m, pos + M):
        c = R.token_row(bt.tolist(), t, page, caches[0].size(0))
        for x in caches:
            y = x[c[0], :, c[1]].view(torch.uint8)
            x[c[0], :, c[1]] = (y ^ 0x80 if x.dtype != torch.half else y).view(x.dtype)
            if x.dtype == torch.half:
                x[c[0], :, c[1]] *= -3
    second = run(K, *dev(q), i32(pos), *dev(bt), dev(*caches), dev(*scales), pos + M, window, 4)
    assert torch.equal(first[:m], second[:m]) and not torch.equal(first[m:], second[m:])


@pytest.mark.parametrize("dtype", CACHES, ids=name)
def test_attention_small_pages_and_strided_q(K, dtype):
    """fp16 pages of one to eight tokens, and q as the first heads of fused rows."""
    M, n_q, n_kv, D, pos = 20, 8, 2, 128, 75
    for page in ((1, 2, 8) if dtype == torch.half else (16, 256)):
        caches, scales, bt, vals = paged_kv(pos + M, n_kv, D, page, dtype, gen(page))
        wide = torch.randn(M, (n_q + 2 * n_kv) * D, generator=gen(1)).half()
        q = wide[:, :n_q * D]
        want, bound = R.attention(q.reshape(M, n_q, D), pos, bt, *vals, pos + M, 40, 4)
        a = dev(wide, bt, *caches, *scales)
        R.within(run(K, a[0][:, :n_q * D], i32(pos), a[1], a[2:4], a[4:6], pos + M, 40, 4), want, bound)
        check(K, q.reshape(M, n_q, D)[:1], pos, bt, caches, scales, vals, pos + M, 40, 4)


@pytest.mark.parametrize("dtype", CACHES, ids=name)
@pytest.mark.parametrize("M,window,sinks", [(1, 0, 0), (1, 300, 4), (24, 0, 0), (24, 64, 4)])
def test_replays_at_other_positions(K, dtype, M, window, sinks):
    """One captured call serves every position up to max_ctx, with eager work between; the eager result is the same."""
    n_q, n_kv, D, cap, page = 32, 8, 128, 3000, 16
    caches, scales, bt, vals = paged_kv(cap, n_kv, D, page, dtype, gen(3))
    q = torch.randn(M, n_q, D, generator=gen(3)).half()
    qd, btd, *c = dev(q, bt, *caches, *scales)
    pos, out = i32(10), torch.empty(M, n_q * D, dtype=torch.half, device=DEV)
    need = K.attention_window_workspace_bytes(M, n_q, n_kv, D, cap, window, sinks, dtype)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)

    def call(o, w):
        if dtype == torch.half:
            K.attention_window(qd, pos, btd, *c[:2], cap, o, window, sinks, w)
        else:
            K.attention_kv8(qd, pos, btd, *c, cap, o, window, sinks, w)

    call(out, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out, ws)
    for p in (0, 10, 64, 999, cap - M, 3):
        pos.fill_(p)
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        eager = torch.empty_like(out)
        call(eager, torch.full_like(ws, 255))
        assert torch.equal(out, eager), p
        want, bound = R.attention(q[:, :4], p, bt, *[v[:, :1] for v in vals], cap, window, sinks)
        R.within(out[:, :4 * D], want, bound)


@pytest.mark.parametrize("dtype", CODES, ids=name)
def test_append_read_and_attend_as_a_sequence(K, dtype):
    """A prompt appended at once and attended, then tokens one by one, each attended, on a side stream; the cache read back.
    The reference holds its own cache from the same rows."""
    n_q, n_kv, D, page, M, n, window, sinks = 8, 2, 64, 16, 37, 30, 25, 3
    g = gen(12)
    kc, vc, ks, vs = empty_cache(6, n_kv, page, D, dtype, g)
    bt = torch.randperm(6, generator=g).int()
    rows = qkv_rows(M + n, n_q, n_kv, D, g, spread=0.5)
    cos, sin = rope_tables(M + n, D)
    ref = [kc, vc, ks, vs]
    cosd, sind, btd, rd, *c = dev(cos, sin, bt, rows, kc, vc, ks, vs)
    pos = i32(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for lo, hi in [(0, M)] + [(t, t + 1) for t in range(M, M + n)]:
        m = hi - lo
        q, ref = R.append(rows[lo:hi], cos, sin, lo, bt, *ref, n_q)
        with torch.cuda.stream(side):
            qd, out = (torch.empty(m, n_q * D, dtype=torch.half, device=DEV) for _ in "qo")
            need = K.attention_window_workspace_bytes(m, n_q, n_kv, D, hi, window, sinks, dtype)
            ws = torch.empty(need, dtype=torch.uint8, device=DEV) if need else None
            pos.fill_(lo)
            K.kv8_append_rows(rd[lo:hi], cosd, sind, pos, btd, *c, n_q, n_kv, qd)
            K.attention_kv8(qd, pos, btd, *c, hi, out, window, sinks, ws)
        side.synchronize()
        assert torch.equal(qd.cpu().view(m, n_q, D), q)
        want, bound = R.attention(q, lo, bt, R.values(ref[0], ref[2]), R.values(ref[1], ref[3]), hi, window, sinks)
        R.within(out, want, bound)
    k, v = (torch.empty(M + n, n_kv, D, dtype=torch.half, device=DEV) for _ in "kv")
    K.kv8_read(btd, *c, 0, k, v)
    for got, code, scale in ((k, ref[0], ref[2]), (v, ref[1], ref[3])):
        val = R.values(code, scale)
        cells = [R.token_row(bt.tolist(), t, page, 6) for t in range(M + n)]
        assert torch.equal(got.cpu().double(), torch.stack([val[a, :, s] for a, s in cells]))


def decode(K, row, cos, sin, pos, bt, c, n_q, n_kv, cap, window=0, sinks=0, ws=True, fill=float("nan")):
    """attention_kv8_decode, in place in the cache c."""
    D = c[0].size(3)
    out = torch.full((n_q * D,), fill, dtype=torch.half, device=DEV)
    need = K.attention_window_workspace_bytes(1, n_q, n_kv, D, cap, window, sinks, c[0].dtype)
    w = torch.full((need,), 255, dtype=torch.uint8, device=DEV) if need and ws else None
    K.attention_kv8_decode(row, cos, sin, i32(pos), bt, *c, n_q, n_kv, cap, out, window, sinks, w)
    return out


@pytest.mark.parametrize("dtype", CODES, ids=name)
@pytest.mark.parametrize("n_q,n_kv,D,page,start,cap,window,sinks", [
    (32, 4, 64, 16, 0, 64, 0, 0), (32, 8, 128, 16, 290, 350, 0, 0), (8, 1, 128, 32, 500, 5000, 0, 0),
    (4, 4, 64, 64, 1000, 1 << 17, 0, 0), (2, 1, 128, 16, 300, 1 << 22, 0, 0), (8, 2, 128, 16, 250, 400, 40, 3),
    (8, 4, 64, 32, 25, 100, 1, 0), (4, 2, 64, 16, 700, 5000, 200, 40), (2, 2, 128, 128, 90, 200, 1000, 4)])
def test_decode_appends_and_attends(K, dtype, n_q, n_kv, D, page, start, cap, window, sinks):
    """Tokens one by one, their sizes going up and down so that blocks grow in the middle: the cache bit for bit the
    reference's, attention within its bound, with and without a workspace, qkv and the pages of others as they were."""
    g, n = gen(start + D + page), 40
    caches, scales, bt, _ = paged_kv(start + n, n_kv, D, page, dtype, g)
    ref = [*caches, *scales]
    size = torch.exp2(torch.randint(-12, 7, (n, 1), generator=g).float())
    size[:3] = 1.0
    rows = (torch.randn(n, (n_q + 2 * n_kv) * D, generator=g) * size).half()
    rows[:, :n_q * D] = torch.randn(n, n_q * D, generator=g).half()
    cos, sin = rope_tables(start + n, D)
    cosd, sind, btd, rd, *c = dev(cos, sin, bt, rows, *ref)
    other = [t.clone() for t in c]
    for i in range(n):
        t = start + i
        q, ref = R.append(rows[i:i + 1], cos, sin, t, bt, *ref, n_q)
        out = decode(K, rd[i], cosd, sind, t, btd, c, n_q, n_kv, cap, window, sinks)
        alone = decode(K, rd[i], cosd, sind, t, btd, other, n_q, n_kv, cap, window, sinks, ws=False)
        if i in (0, 1, 15, 16, 17, 31, 39):
            want, bound = R.attention(q, t, bt, R.values(ref[0], ref[2]), R.values(ref[1], ref[3]), cap, window, sinks)
            R.within(out.view(1, -1), want, bound)
            R.within(alone.view(1, -1), want, bound)
        assert all(same(a, b) for a, b in zip(c, ref)), t
    assert all(same(a, b) for a, b in zip(other, ref)) and same(rd, rows)


@pytest.mark.parametrize("dtype", CODES, ids=name)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("pos,cap,window", [(5, 100, 0), (31, 100, 0), (200, 4000, 0), (200, 4000, 30), (48, 100, 1)])
def test_decode_of_values_that_are_not_finite(K, dtype, D, pos, cap, window):
    """Infinities and NaN in the new K and V, and NaN in codes behind the window: what append and attention give."""
    n_q, n_kv, page = 8, 2, 16
    caches, scales, bt, _ = paged_kv(pos + 1, n_kv, D, page, dtype, gen(pos + D))
    if dtype == torch.float8_e4m3fn and window:
        for t in (0, max(0, pos - 60), max(0, pos - window)):
            i, slot = R.token_row(bt.tolist(), t, page, caches[0].size(0))
            for x in caches:
                x.view(torch.uint8)[i, 0, slot, 3] = 127
    cos, sin = (t.to(DEV) for t in rope_tables(pos + 1, D))
    for edit in range(4):
        row = torch.randn((n_q + 2 * n_kv) * D, generator=gen(edit)).half()
        kv = row[n_q * D:].view(2, n_kv, D)
        if edit == 1:
            kv[1, 0, 5], kv[1, 1, 7] = float("inf"), float("-inf")
        elif edit == 2:
            kv[1, 0, D - 1] = float("nan")
        elif edit == 3:
            kv[0, 1, 2] = float("nan")
        row = row.to(DEV)
        btd, *a = dev(bt, *caches, *scales)
        b = [t.clone() for t in a]
        out = decode(K, row, cos, sin, pos, btd, a, n_q, n_kv, cap, window, 0)
        q = torch.empty(1, n_q * D, dtype=torch.half, device=DEV)
        K.kv8_append_rows(row.view(1, -1), cos, sin, i32(pos), btd, *b, n_q, n_kv, q)
        want = run(K, q, i32(pos), btd, b[:2], b[2:], cap, window, 0)
        assert all(same(x, y) for x, y in zip(a, b))
        torch.testing.assert_close(out, want[0], rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("dtype", CODES, ids=name)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window", [0, 50])
def test_decode_positions_and_pages(K, dtype, D, window):
    """Positions outside the table touch nothing; one past max_ctx, one without a page and one past the block table attend what
    there is."""
    n_q, n_kv, page, tokens = 8, 2, 16, 400
    caches, scales, bt, _ = paged_kv(tokens, n_kv, D, page, dtype, gen(D), extra=0)
    row = torch.randn((n_q + 2 * n_kv) * D, generator=gen(2)).half()
    cos, sin = rope_tables(500, D)
    cosd, sind, rd = dev(cos, sin, row)
    for pos, cap, hole in ((-1, 400, None), (500, 400, None), (1 << 30, 400, None), (399, 100, None), (130, 128, None),
                           (399, 128, None), (399, 5000, 399), (399, 400, 0), (130, 131, 129), (400, 600, None),
                           (499, 600, None), (499, 100, None), (10, 4000, 3)):
        t = bt.clone()
        if hole is not None:
            t[hole // page] = -1 if hole % 2 else caches[0].size(0)
        td, *c = dev(t, *caches, *scales)
        q, ref = R.append(row.view(1, -1), cos, sin, pos, t, *caches, *scales, n_q)
        for ws in (True, False):
            c = dev(*caches, *scales)
            out = decode(K, rd, cosd, sind, pos, td, c, n_q, n_kv, cap, window, 4 if window else 0, ws, fill=7.0)
            assert all(same(a, b) for a, b in zip(c, ref)), pos
            if not 0 <= pos < 500:
                assert bool((out == 7.0).all())
                continue
            want, bound = R.attention(q, pos, t, R.values(ref[0], ref[2]), R.values(ref[1], ref[3]), cap, window,
                                      4 if window else 0)
            R.within(out.view(1, -1), want, bound)


@pytest.mark.parametrize("dtype", CODES, ids=name)
def test_decode_on_two_streams(K, dtype):
    """Two sequences in one cache, each with its block table and workspace, decoded at once: what they give in turn."""
    n_q, n_kv, D, page, cap, n = 32, 8, 128, 16, 2000, 12
    caches, scales, bt, _ = paged_kv(2 * cap, n_kv, D, page, dtype, gen(6))
    tables = [t.contiguous().to(DEV) for t in bt[:2 * (cap // page)].view(2, -1)]
    cos, sin = (t.to(DEV) for t in rope_tables(cap, D))
    rows = (torch.randn(2, n, (n_q + 2 * n_kv) * D, generator=gen(7))
            * torch.exp2(torch.arange(n).float()[:, None] % 5)).half().to(DEV)
    got = []
    for together in (True, False):
        c = dev(*caches, *scales)
        out = torch.empty(2, n, n_q * D, dtype=torch.half, device=DEV)
        pos = torch.arange(1500, 1500 + n, dtype=torch.int32, device=DEV)
        need = K.attention_window_workspace_bytes(1, n_q, n_kv, D, cap, 0, 0, dtype)
        ws = [torch.full((max(need, 16),), 255, dtype=torch.uint8, device=DEV) for _ in range(2)]
        streams = [torch.cuda.Stream() for _ in range(2)] if together else [torch.cuda.current_stream()] * 2
        torch.cuda.synchronize()
        for i in range(n):
            for j, st in enumerate(streams):
                with torch.cuda.stream(st):
                    K.attention_kv8_decode(rows[j, i], cos, sin, pos[i:], tables[j], *c, n_q, n_kv, cap, out[j, i],
                                           workspace=ws[j])
        torch.cuda.synchronize()
        got.append((out, c))
    assert torch.equal(got[0][0], got[1][0]) and all(same(a, b) for a, b in zip(got[0][1], got[1][1]))


@pytest.mark.parametrize("dtype", CODES, ids=name)
def test_decode_replayed(K, dtype):
    """One captured call over a sequence of tokens, with eager work between, beside the append and the attention as two."""
    n_q, n_kv, D, page, cap, start = 32, 8, 128, 16, 1000, 45
    caches, scales, bt, _ = paged_kv(cap, n_kv, D, page, dtype, gen(8))
    cos, sin = (t.to(DEV) for t in rope_tables(cap, D))
    rows = (torch.randn(40, (n_q + 2 * n_kv) * D, generator=gen(9))
            * torch.exp2(torch.arange(40).float()[:, None] % 7)).half().to(DEV)
    btd, *a = dev(bt, *caches, *scales)
    b = [t.clone() for t in a]
    pos, row, out = i32(start), rows[0].clone(), torch.empty(n_q * D, dtype=torch.half, device=DEV)
    ws = torch.empty(K.attention_window_workspace_bytes(1, n_q, n_kv, D, cap, 0, 0, dtype) or 16, dtype=torch.uint8, device=DEV)
    call = lambda: K.attention_kv8_decode(row, cos, sin, pos, btd, *a, n_q, n_kv, cap, out, workspace=ws)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for t, was in zip(a, b):
        t.copy_(was)
    for i in range(40):
        row.copy_(rows[i])
        pos.fill_(start + i)
        graph.replay()
        torch.cuda.synchronize()
        q = torch.empty(1, n_q * D, dtype=torch.half, device=DEV)
        K.kv8_append_rows(rows[i:i + 1], cos, sin, pos, btd, *b, n_q, n_kv, q)
        want = run(K, q, pos, btd, b[:2], b[2:], cap)
        assert all(same(x, y) for x, y in zip(a, b)) and torch.equal(out, want[0]), i


@pytest.mark.parametrize("dtype", CACHES, ids=name)
def test_graphs_share_a_workspace_and_streams(K, dtype):
    """Two captured calls of different sizes with one workspace, replayed in turn, another call on another stream with a
    workspace of its own between; every replay against the eager result."""
    cases = []
    for M, pos, window in ((1, 2500, 0), (30, 900, 200)):
        caches, scales, bt, _ = paged_kv(pos + M, 4, 128, 16, dtype, gen(pos))
        q = torch.randn(M, 16, 128, generator=gen(M)).half()
        qd, btd, *c = dev(q, bt, *caches, *scales)
        out = torch.empty(M, 16 * 128, dtype=torch.half, device=DEV)
        args = (qd, i32(pos), btd, *(c[:2] if dtype == torch.half else c), pos + M, out, window, 4)
        cases.append((args, out, K.attention_window_workspace_bytes(M, 16, 4, 128, pos + M, window, 4, dtype)))
    need = max(c[2] for c in cases)
    ws = [torch.full((max(need, 16),), 255, dtype=torch.uint8, device=DEV) for _ in range(2)]
    op = K.attention_window if dtype == torch.half else K.attention_kv8
    graphs, want = [], []
    for args, out, _ in cases:
        op(*args, ws[0])
        want.append(out.clone())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            op(*args, ws[0])
        graphs.append(g)
    side = torch.cuda.Stream()
    for turn in range(3):
        for i, g in enumerate(graphs):
            cases[i][1].zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(cases[i][1], want[i]), (turn, i)
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                op(*cases[1 - i][0], ws[1])
            torch.cuda.current_stream().wait_stream(side)
            assert torch.equal(cases[1 - i][1], want[1 - i]), (turn, i)


@pytest.mark.parametrize("dtype", CACHES, ids=name)
def test_caches_past_32_bit_offsets(K, dtype):
    """Pages whose bytes lie past 2^32 of the cache (K and V are one cache here): append, read back and attention."""
    n_q, n_kv, D, page, M, pos = 8, 2, 128, 64, 20, 100
    n_pages = (1 << 32) // (n_kv * page * D) + 8
    bt = torch.tensor([n_pages - 1, n_pages - 3], dtype=torch.int32)
    lo = n_pages - 3
    g = gen(5)
    caches, scales, small, vals = paged_kv(pos + M, n_kv, D, page, dtype, g, extra=1)
    small_bt = torch.tensor([2, 0], dtype=torch.int32)
    order = torch.empty(3, dtype=torch.long)
    order[small_bt.long()], order[1] = small[:2].long(), int(small[2])
    big, tiny = [], []
    for c in (*caches, *scales):
        if c is None:
            big.append(None), tiny.append(None)
            continue
        b = torch.empty(n_pages, *c.shape[1:], dtype=c.dtype, device=DEV)
        t = c[order] if c.dtype != torch.float8_e4m3fn else c.view(torch.uint8)[order].view(c.dtype)
        b.view(torch.uint8)[lo:] = t.contiguous().view(torch.uint8).view(b.view(torch.uint8)[lo:].shape).to(DEV)
        big.append(b), tiny.append(t)
    btd = bt.to(DEV)
    q = torch.randn(M, n_q, D, generator=g).half()
    for m in (1, M):
        want, bound = R.attention(q[:m], pos, small_bt, *[R.values(c, s) for c, s in zip(tiny[:2], tiny[2:])], pos + m, 0, 0)
        R.within(run(K, q[:m].to(DEV), i32(pos), btd, big[:2], big[2:], pos + m), want, bound)
    if dtype == torch.half:
        return
    qkv = qkv_rows(M, n_q, n_kv, D, g)
    cos, sin = rope_tables(pos + M, D)
    _, ref = R.append(qkv, cos, sin, pos, small_bt, *tiny, n_q)
    x, cosd, sind = dev(qkv, cos, sin)
    K.kv8_append_rows(x, cosd, sind, i32(pos), btd, *big, n_q, n_kv)
    for a, b in zip(big, ref):
        assert same(a[lo:], b)
    k, v = (torch.empty(pos + M, n_kv, D, dtype=torch.half, device=DEV) for _ in "kv")
    K.kv8_read(btd, *big, 0, k, v)
    val = R.values(ref[0], ref[2])
    assert torch.equal(k.cpu().double(), torch.stack([val[a, :, s] for a, s in
                                                      (R.token_row([2, 0], t, page, 3) for t in range(pos + M))]))
    row, t = qkv_rows(1, n_q, n_kv, D, g), pos + M
    cos, sin = rope_tables(t + 1, D)
    q, ref = R.append(row, cos, sin, t, small_bt, *ref, n_q)
    out = decode(K, row.view(-1).to(DEV), cos.to(DEV), sin.to(DEV), t, btd, big, n_q, n_kv, t + 1)
    for a, b in zip(big, ref):
        assert same(a[lo:], b)
    want, bound = R.attention(q, t, small_bt, R.values(ref[0], ref[2]), R.values(ref[1], ref[3]), t + 1)
    R.within(out.view(1, -1), want, bound)


def test_op_module_refusals(K):
    z = lambda *s, t=torch.half: torch.zeros(*s, dtype=t, device=DEV)
    c8, s8, bt, pos = z(4, 2, 16, 64, t=torch.int8), z(4, 2, 1, t=torch.float32), z(4, t=torch.int32), z(1, t=torch.int32)
    f = z(8, 32, t=torch.float32)
    app = lambda **k: K.kv8_append_rows(**dict(dict(qkv=z(3, 6 * 64), cos_t=f, sin_t=f, pos=pos, bt=bt, kc=c8, vc=c8.clone(),
                                                    ks=s8, vs=s8.clone(), n_q=2, n_kv=2), **k))
    for kw, msg in ((dict(qkv=z(3, 5 * 64)), "qkv must be"), (dict(vc=c8.view(torch.float8_e4m3fn)), "vc must be"),
                    (dict(sin_t=None), "both be"), (dict(cos_t=z(8, 16, t=torch.float32)), "both be"),
                    (dict(pos=z(1, t=torch.int64)), "pos must be"), (dict(ks=z(4, 2, 2, t=torch.float32)), "P / 16"),
                    (dict(q_out=z(3, 64)), "q_out must be"), (dict(q_out=z(3, 256)[:, ::2]), "q_out must be"),
                    (dict(n_kv=1, n_q=4), "qkv must be"), (dict(kc=z(4, 2, 16, 64)), "int8 or float8")):
        with pytest.raises(RuntimeError, match=msg):
            app(**kw)
    with pytest.raises(RuntimeError, match="n >= 1"):
        K.kv8_read(bt, c8, c8, s8, s8, 0, z(0, 2, 64), z(0, 2, 64))
    with pytest.raises(RuntimeError, match="k_out and v_out"):
        K.kv8_read(bt, c8, c8, s8, s8, 0, z(3, 2, 64), z(3, 64))
    with pytest.raises(RuntimeError, match="range"):
        K.kv8_read(bt, c8, c8, s8, s8, -1, z(3, 2, 64), z(3, 2, 64))
    dec = lambda **k: K.attention_kv8_decode(**dict(dict(qkv=z(6 * 64), cos_t=f, sin_t=f, pos=pos, bt=bt, kc=c8, vc=c8.clone(),
                                                         ks=s8, vs=s8.clone(), n_q=2, n_kv=2, max_ctx=10, out=z(128)), **k))
    for kw, msg in ((dict(qkv=z(5 * 64)), "qkv must hold"), (dict(out=z(64)), "qkv must hold"), (dict(cos_t=None), "cos_t and"),
                    (dict(sin_t=z(8, 16, t=torch.float32)), "cos_t and"), (dict(max_ctx=0), "max_ctx"),
                    (dict(max_ctx=1 << 32), "32 bits"), (dict(n_kv=1, n_q=4), "qkv must hold"),
                    (dict(kc=z(4, 2, 16, 64)), "int8 or float8"), (dict(window=-1), "window and sinks|32 bits")):
        with pytest.raises(RuntimeError, match=msg):
            dec(**kw)
    win = lambda **k: K.attention_kv8(**dict(dict(q=z(3, 4, 64), pos=pos, bt=bt, kc=c8, vc=c8, ks=s8, vs=s8, max_ctx=10,
                                                  out=z(3, 256)), **k))
    for kw, msg in ((dict(q=z(3, 6, 64), out=z(3, 384)), "heads-per-group"), (dict(out=z(3, 128)), "out be"),
                    (dict(q=z(3, 4, 32)), "q must be"), (dict(max_ctx=0), "max_ctx"), (dict(window=-1), "window and sinks"),
                    (dict(max_ctx=1 << 32), "32 bits"), (dict(vs=s8.double()), "vs must be"),
                    (dict(workspace=z(64, t=torch.uint8).cpu()), "CUDA tensor")):
        with pytest.raises(RuntimeError, match=msg):
            win(**kw)


@pytest.mark.parametrize("dtype", CACHES, ids=name)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("M,pos,cap,window,sinks,hole", [(40, 100, 140, 75, 4, 0), (20, 51, 71, 1, 82, 2),
                                                         (40, 100, 140, 41, 50, 2), (40, 100, 20000, 41, 50, 3),
                                                         (300, 120, 420, 60, 35, 2), (3, 100, 103, 75, 4, 0)])
def test_attention_holes_among_the_sinks(K, dtype, D, M, pos, cap, window, sinks, hole):
    """A page of the sinks is not mapped, and the window begins in the sinks' last tile or ahead of their end: its tokens are
    attended by no row, whatever the cache's first page holds."""
    caches, scales, bt, vals = paged_kv(pos + M, 2, D, 16, dtype, gen(M + D))
    bt[hole] = -1
    q = torch.randn(M, 8, D, generator=gen(3)).half()
    check(K, q, pos, bt, caches, scales, vals, cap, window, sinks)


@pytest.mark.parametrize("dtype", CODES, ids=name)
@pytest.mark.parametrize("pos,max_pos,M", [(45, 42, 3), (45, 33, 40), (47, 47, 1), (40, 40, 2)])
@pytest.mark.parametrize("scale", [float("nan"), 0.0, 2.0 ** -30])
def test_append_past_the_tables_touches_nothing(K, dtype, pos, max_pos, M, scale):
    """The tables end inside the position's block, whose scale is none that an append leaves: no row is new, and neither the
    scale nor the codes of the rows ahead are taken anew."""
    n_q, n_kv, D, page = 4, 2, 64, 16
    g = gen(pos)
    kc, vc, ks, vs = empty_cache(6, n_kv, page, D, dtype, g, scale)
    bt = torch.tensor([5, 2, 1, 0, 4, 3], dtype=torch.int32)
    qkv = qkv_rows(M, n_q, n_kv, D, g)
    x, cos, sin, btd, *c = dev(qkv, *rope_tables(max_pos, D), bt, kc, vc, ks, vs)
    out = torch.full((M, n_q * D), 7.0, dtype=torch.half, device=DEV)
    K.kv8_append_rows(x, cos, sin, i32(pos), btd, *c, n_q, n_kv, out)
    assert bool((out == 7.0).all()) and all(same(a, b) for a, b in zip(c, (kc, vc, ks, vs)))


@pytest.mark.parametrize("dtype", CODES, ids=name)
@pytest.mark.parametrize("scale", [128.0, 256.0, 512.0, 1024.0])
@pytest.mark.parametrize("D", [64, 128])
def test_append_into_a_block_of_a_large_scale(K, dtype, scale, D):
    """A block of any valid scale takes the largest fp16 values as codes whose values fit fp16, by either way of appending."""
    n_q, n_kv, page, pos = 4, 2, 16, 21
    g = gen(int(scale))
    kc, vc = (R.to_codes(R.codes_of(torch.randn(2, n_kv, page, D, generator=g) * 20000, scale, dtype), dtype) for _ in "kv")
    ks, vs = (torch.full((2, n_kv, 1), scale) for _ in "kv")
    row = torch.randn(1, (n_q + 2 * n_kv) * D, generator=g).half()
    row[0, n_q * D::3], row[0, n_q * D + 1::3], row[0, (n_q + n_kv) * D + 2::9] = 65504.0, -65504.0, float("inf")
    bt, cos, sin = torch.tensor([1, 0], dtype=torch.int32), torch.ones(30, D // 2), torch.zeros(30, D // 2)
    _, want = R.append(row, cos, sin, pos, bt, kc, vc, ks, vs, n_q)
    x, cosd, sind, btd, *a = dev(row, cos, sin, bt, kc, vc, ks, vs)
    b = [t.clone() for t in a]
    decode(K, x[0], cosd, sind, pos, btd, b, n_q, n_kv, pos + 1)
    K.kv8_append_rows(x, cosd, sind, i32(pos), btd, *a, n_q, n_kv)
    for got in (a, b):
        assert all(same(u, v) for u, v in zip(got, want))
    back = [torch.empty(pos + 1, n_kv, D, dtype=torch.half, device=DEV) for _ in "kv"]
    K.kv8_read(btd, *a, 0, *back)
    assert all(bool(torch.isfinite(t).all()) for t in back)


@pytest.mark.parametrize("M,pos,cap", [(1, 300, 301), (1, 300, 5000), (3, 90, 93), (40, 300, 2000)])
def test_attention_of_tokens_without_weight(K, M, pos, cap):
    """A score of -infinity weighs nothing beside others: as if its token were not there. A row that has only such ones gets
    zeros, as one that attends nothing."""
    n_q, n_kv, D, page = 8, 2, 64, 16
    caches, scales, bt, vals = paged_kv(pos + M, n_kv, D, page, torch.half, gen(5))
    q = (torch.randn(M, n_q, D, generator=gen(5)).abs() + 0.5).half()
    a = dev(q, bt, *caches)
    cells = [R.token_row(bt.tolist(), t, page, caches[0].size(0)) for t in range(pos + M)]
    for step in (3, 1):
        k = caches[0].clone()
        for c in cells[::step]:
            k[c[0], :, c[1], 1] = float("-inf")
        for ws in ("full", "none"):
            out = run(K, a[0], i32(pos), a[1], [k.to(DEV), a[3]], scales, cap, ws=ws)
            if step == 1:
                assert bool((out == 0).all())
                continue
            for m in {0, M // 2, M - 1}:
                left = [c for t, c in enumerate(cells[:pos + m + 1]) if t % step]
                kv = [torch.stack([x[c[0], :, c[1]] for c in left], 1)[None] for x in vals]   # one page of the tokens left
                want, bound = R.attention(q[m:m + 1], len(left) - 1, torch.zeros(1, dtype=torch.int32), *kv, len(left))
                R.within(out[m:m + 1], want, bound)


@pytest.mark.parametrize("dtype", CACHES, ids=name)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("M,pos,cap,window,hpg,n_kv", [(1, 17, 18, 0, 8, 2), (1, 40, 5000, 0, 4, 2), (1, 30, 1 << 20, 20, 4, 2),
                                                       (3, 25, 28, 9, 4, 2), (40, 3, 43, 0, 4, 2), (40, 0, 20000, 12, 4, 2),
                                                       (130, 0, 130, 30, 8, 8), (700, 0, 700, 25, 4, 8)])
def test_attention_weights_keep_their_bits(K, dtype, D, M, pos, cap, window, hpg, n_kv):
    """Small scores over few tokens, where a weight's rounding would be the largest error but the output's own. A weight p meets
    V as two fp16 numbers, hi = fp16(p) and fp16(p - hi): |p - hi| <= 2^-11 p, half a step of that is 2^-22 p, or 2^-25 below
    fp16's normal range, which the bound has already. (More than 16 columns over codes: one number, 11 bits.)"""
    bits = 22 if dtype == torch.half or M * hpg <= 16 else 11
    caches, scales, bt, vals = paged_kv(pos + M, n_kv, D, 16, dtype, gen(M + D))
    q = (torch.randn(M, hpg * n_kv, D, generator=gen(5)) * 0.1).half()
    want, bound = R.attention(q, pos, bt, *vals, cap, window, 0)
    size = R.attention(q, pos, bt, vals[0], vals[1].abs(), cap, window, 0)[0]      # sum of w |v|, of which the bound has 2^-11
    bound = bound - (2.0 ** -11 - 2.0 ** -bits) * size
    a = dev(q, bt, *caches, *scales)
    for ws in ("full", "none"):
        R.within(run(K, a[0], i32(pos), a[1], a[2:4], a[4:6], cap, window, 0, ws), want, bound)
