"""64-bit references of the speculative-decoding operators, written from their definitions, and the element-wise error
bounds that the kernels' roundings allow. All on the CPU."""
import math

import torch

NAN = float("nan")


def random_parents(M, branch, g):
    """Parents of a random tree in node order: parents[i] < i, about `branch` children per inner node."""
    p = [-1]
    for i in range(1, M):
        lo = max(0, i - 1 - 3 * branch)
        p.append(i - 1 if branch == 1 else int(torch.randint(lo, i, (1,), generator=g)))
    return p


def token_row(bt, t, page, n_pages, max_ctx=1 << 60):
    """(physical page, slot) of cache token t, None where it has none."""
    if t < 0 or t >= max_ctx or t // page >= len(bt) or not 0 <= bt[t // page] < n_pages:
        return None
    return bt[t // page], t % page


def qk_norm_rope(qkv, q_w, k_w, eps, cos, sin, pos, depth, bt, kc, vc, n_q, n_kv):
    """-> (q, q bound), and fp64 caches with their bounds: rows that are not written keep their value and bound 0."""
    M, D, page = qkv.size(0), kc.size(3), kc.size(2)
    q, kc64, vc64 = torch.full((M, n_q, D), NAN, dtype=torch.float64), kc.double(), vc.double()
    qb, kb = torch.zeros_like(q), torch.zeros_like(kc64)
    bt = bt.tolist()
    touched = []
    for m in range(M):
        t, r = pos + m, pos + (m if depth is None else int(depth[m]))
        touched.append(t >= 0 and 0 <= r < cos.size(0))
        if not touched[-1]:
            continue
        x = qkv[m].double().view(-1, D)

        def turn(y, w):
            if w is not None:
                y = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + eps) * w.double()
            a, b = y[:, :D // 2], y[:, D // 2:]
            c, s = cos[r].double(), sin[r].double()
            z = torch.cat([a * c - b * s, b * c + a * s], -1)
            # fp32 arithmetic on a and b: 2^-18 of their size covers the sum of D squares and a dozen roundings; then
            # one rounding to fp16, half a step of the value or of the smallest subnormal
            size = (a.abs() + b.abs()).repeat(1, 2)
            return z, 2.0 ** -11 * z.abs() + 2.0 ** -18 * size + 2.0 ** -25

        q[m], qb[m] = turn(x[:n_q], q_w)
        row = token_row(bt, t, page, kc.size(0))
        if row is not None:
            kc64[row[0], :, row[1]], kb[row[0], :, row[1]] = turn(x[n_q:n_q + n_kv], k_w)
            vc64[row[0], :, row[1]] = x[n_q + n_kv:]
    return q, qb, kc64, kb, vc64, touched


def mask_rows(parents):
    """bool [M, M]: node j is node i or an ancestor of it."""
    M = len(parents)
    m = torch.zeros(M, M, dtype=torch.bool)
    for i, p in enumerate(parents):
        if p >= 0:
            m[i] = m[p]
        m[i, i] = True
    return m


def mask_words(rows):
    """bool [M, M] -> int64 [M, ceil(M / 64)]."""
    M = rows.size(0)
    W = (M + 63) // 64
    out = torch.zeros(M, W, dtype=torch.int64)
    for i in range(M):
        for j in range(M):
            if rows[i, j]:
                out[i, j // 64] |= (1 << (j % 64)) if j % 64 < 63 else -(1 << 63)
    return out


def attention_tree(q, rows, pos, bt, kc, vc, max_ctx=1 << 60):
    """q [M, n_q, D]; rows bool [M, M] -> (out fp64 [M, n_q * D], bound). A token that a node does not attend is left out
    altogether, whatever its K and V hold."""
    M, n_q, D = q.shape
    n_kv, page, n_pages = kc.size(1), kc.size(2), kc.size(0)
    bt = bt.tolist()
    out, bound = torch.zeros(M, n_q, D, dtype=torch.float64), torch.zeros(M, n_q, D, dtype=torch.float64)
    cells = [token_row(bt, t, page, n_pages, max_ctx) for t in range(max(pos, 0) + M)] if pos >= 0 else []
    for m in range(M):
        toks = [c for t, c in enumerate(cells) if c is not None and (t < pos or rows[m, t - pos])]
        if not toks:
            continue
        pg, sl = torch.tensor([c[0] for c in toks]), torch.tensor([c[1] for c in toks])
        for h in range(n_kv):
            hs = slice(h * (n_q // n_kv), (h + 1) * (n_q // n_kv))
            k, v = kc[pg, h, sl].double(), vc[pg, h, sl].double()
            qh = q[m, hs].double()
            sc = qh @ k.t() / math.sqrt(D)
            p = torch.softmax(sc, -1)
            out[m, hs] = p @ v
            # p is rounded to fp16 (half a step: 2^-11); its score carries D fp32 roundings of |q| . |k| and two of the
            # exponent, in numerator and denominator; the output half a step of its own
            ds = 2.0 ** -24 * ((D + 4) * (qh.abs() @ k.abs().t()) / math.sqrt(D) + 4 * sc.abs()).amax(-1, keepdim=True)
            n = sc.size(1)
            rel = 2.0 ** -11 + 2 * (ds + 2.0 ** -21) + 2.0 ** -24 * (n / 16 + 64)
            bound[m, hs] = 2.0 ** -11 * out[m, hs].abs() + rel * (p @ v.abs()) + 2.0 ** -25
    return out.view(M, -1), bound.view(M, -1)


def token_logprobs(logits, tokens, k):
    """-> logprobs, entropy, top_ids, top_logprobs (fp64), bounds of the fp32 values."""
    x = logits.double()
    M, V = x.shape
    bad = torch.isnan(x).any(1) | (x.amax(1) == math.inf) | (x.amax(1) == -math.inf)
    top = x.amax(1, keepdim=True)
    # about the row's maximum: beside 3e38 even 64 bits have no room for log V
    lp = (x - top) - torch.log(torch.exp(x - top).sum(1, keepdim=True))
    p = lp.exp()
    d = (x - top).clamp(min=-1e30)
    ent = -(torch.where(p > 0, p * lp, torch.zeros_like(p))).sum(1)
    order = torch.sort(torch.nan_to_num(x, nan=math.inf, posinf=1e300, neginf=-math.inf), dim=1, descending=True,
                       stable=True).indices
    nan_first = torch.sort(torch.isnan(x).to(torch.int8).gather(1, order), dim=1, descending=True, stable=True).indices
    order = order.gather(1, nan_first)[:, :k]
    inside = (tokens >= 0) & (tokens < V)
    given = lp.gather(1, tokens.clamp(0, V - 1)[:, None])[:, 0]
    given = torch.where(inside & ~bad, given, torch.full_like(given, NAN))
    ent = torch.where(bad, torch.full_like(ent, NAN), ent)
    tops = torch.where(bad[:, None], torch.full((M, k), NAN, dtype=torch.float64), lp.gather(1, order))
    # sums of V positive fp32 terms in chains of at most V / 64 + 64, each term off by its exponent's two roundings
    rel = 2.0 ** -24 * (V / 64 + 128) + 2.0 ** -22 * (1 + (p * d.abs()).sum(1, keepdim=True))
    size = top.abs().clamp(max=1e30)
    vb = lambda v: rel + 2.0 ** -22 * (v.abs().nan_to_num(0, 0, 0) + 1) + 2.0 ** -23 * size
    eb = rel[:, 0] * (2 + 2 * (p * d.abs()).sum(1)) + 2.0 ** -22 * (1 + ent.abs().nan_to_num(0))
    return given, vb(given[:, None])[:, 0], ent, eb, order, tops, vb(tops)


def tree_accept(tokens, parents, picks, pos, bt, kv):
    """-> path (padded with -1), count, tok, kv after the move (kv [..., pages, n_kv, P, D])."""
    M, path = len(tokens), [0]
    while True:
        nxt = [c for c in range(path[-1] + 1, M) if parents[c] == path[-1] and tokens[c] == picks[path[-1]]]
        if not nxt:
            break
        path.append(nxt[0])
    after = None
    if kv is not None:
        after, bt, page = kv.clone(), bt.tolist(), kv.size(-2)
        for t, p in enumerate(path):
            a, b = (token_row(bt, pos + i, page, kv.size(-4)) for i in (p, t))
            if a is not None and b is not None:
                after[..., b[0], :, b[1], :] = kv[..., a[0], :, a[1], :]
    return path + [-1] * (M - len(path)), len(path), picks[path[-1]], after


def within(out, want, bound):
    """NaN where NaN is wanted, infinities alike, else at most `bound` apart."""
    out, want = out.detach().cpu().double(), want.double()
    assert torch.equal(torch.isnan(out), torch.isnan(want)), "NaN in other places"
    fin = torch.isfinite(want)
    assert torch.equal(out[~fin & ~torch.isnan(want)], want[~fin & ~torch.isnan(want)]), "infinities differ"
    diff = (out - want).abs()[fin] - bound.expand_as(want)[fin]
    assert diff.numel() == 0 or diff.max() <= 0, f"over the bound by {diff.max():.3e}"
