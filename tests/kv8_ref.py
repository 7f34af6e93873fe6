"""References of the 8-bit cache and of attention under a window, in 64 bits and on the CPU, written from their definitions,
with the element-wise error bounds that the kernels' roundings allow."""
import math

import torch

from tree_ref import token_row, within  # noqa: F401  (re-exported)

BLOCK = 16
MOST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
E4M3 = torch.tensor(sorted({f * 2.0 ** -9 if e == 0 else (8 + f) * 2.0 ** (e - 10)
                            for e in range(16) for f in range(8) if (e, f) != (15, 7)}), dtype=torch.float64)


def scale_of(x, dtype):
    """The scale of a block's new values x: 2^k, the smallest k >= -24 with max |x| <= most 2^k (NaN left out, an infinity as
    the largest fp16 value)."""
    top = float(torch.nan_to_num(x.double().abs(), nan=0.0, posinf=65504.0).max())
    k = -24
    while MOST[dtype] * 2.0 ** k < top:
        k += 1
    return 2.0 ** k


def codes_of(x, s, dtype):
    """Values (float64) of the codes of x at scale s: x / s to nearest, ties to even, no further out than 65504 / s."""
    y = torch.nan_to_num(x.double(), nan=float("nan"), posinf=65504.0, neginf=-65504.0) / s
    if dtype == torch.int8:
        most = min(127.0, math.floor(65504.0 / s))
        return torch.nan_to_num(torch.round(y.clamp(-most, most)), nan=0.0)
    grid = E4M3[E4M3 <= 65504.0 / s]
    a = y.abs().clamp(max=float(grid[-1]))
    hi = torch.searchsorted(grid, a.nan_to_num(0.0)).clamp(max=grid.numel() - 1)
    lo = (hi - 1).clamp(min=0)
    # the middle goes to the code of even mantissa: grid entries alternate, the first (0) is even
    up = (grid[hi] - a < a - grid[lo]) | ((grid[hi] - a == a - grid[lo]) & (hi % 2 == 0))
    got = torch.copysign(torch.where(up, grid[hi], grid[lo]), y)
    return torch.where(torch.isnan(y), y, got)


def to_codes(v, dtype):
    """Codes of given code values."""
    return v.to(dtype) if dtype == torch.int8 else v.float().to(dtype)


def values(codes, scales):
    """fp64 values [pages, n_kv, P, D] of a cache; an fp16 one has no scales."""
    x = codes.float().double()
    return x if scales is None else x * scales.double().repeat_interleave(BLOCK, 2)[..., None]


def rope(x, cos, sin):
    """fp16 rotation of x [..., D], products and sums rounded one by one in fp32."""
    a, b = x.float().chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).half()


def append(qkv, cos, sin, pos, bt, kc, vc, ks, vs, n_q):
    """-> (q fp16 [M, n_q, D] with NaN rows where nothing is touched, and copies of the caches and scales)."""
    M, (n_pages, n_kv, P, D) = qkv.size(0), kc.shape
    dtype = kc.dtype
    x = qkv.view(M, -1, D)
    last = cos.size(0) if cos is not None else 1 << 62
    rows = {pos + m: m for m in range(M) if 0 <= pos + m < last}
    q = torch.full((M, n_q, D), float("nan"), dtype=torch.half)
    new = {"k": {}, "v": {}}
    for t, m in rows.items():
        y = x[m, :n_q + n_kv] if cos is None else rope(x[m, :n_q + n_kv], cos[t], sin[t])
        q[m], new["k"][t], new["v"][t] = y[:n_q], y[n_q:], x[m, n_q + n_kv:]
    out = [t.clone() for t in (kc, vc, ks, vs)]
    bt = bt.tolist()
    for code, scale, rows_of in ((out[0], out[2], new["k"]), (out[1], out[3], new["v"])):
        for b in sorted({t // BLOCK for t in rows_of}):
            cell = token_row(bt, b * BLOCK, P, n_pages)
            if cell is None:
                continue
            page, slot = cell
            fresh = [t for t in range(b * BLOCK, (b + 1) * BLOCK) if t in rows_of]
            old = [t for t in range(b * BLOCK, fresh[0]) if t >= 0 and t < pos]
            for h in range(n_kv):
                vals = torch.stack([rows_of[t][h] for t in fresh])
                s = scale_of(vals, dtype)
                had = float(scale[page, h, slot // BLOCK])
                if old and had > s:
                    s = had
                for t, v in zip(fresh, vals):
                    code[page, h, slot + t % BLOCK] = to_codes(codes_of(v, s, dtype), dtype)
                for t in old if s != had else []:
                    at = (page, h, slot + t % BLOCK)
                    code[at] = to_codes(codes_of(code[at].float().double() * had, s, dtype), dtype)
                scale[page, h, slot // BLOCK] = s
    return q, out


def cells_of(pos, M, bt, page, n_pages, max_ctx):
    return [token_row(bt, t, page, n_pages, max_ctx) for t in range(max(pos + M, 0))]


def attention(q, pos, bt, kc, vc, max_ctx, window=0, sinks=0):
    """q [M, n_q, D]; kc, vc values [pages, n_kv, P, D] (fp16 or fp64) -> (out fp64 [M, n_q * D], bound). A token that a row
    does not attend is left out altogether, whatever its K and V hold."""
    M, n_q, D = q.shape
    n_kv, page, n_pages = kc.size(1), kc.size(2), kc.size(0)
    cells = cells_of(pos, M, bt.tolist(), page, n_pages, max_ctx)
    out, bound = (torch.zeros(M, n_q, D, dtype=torch.float64) for _ in range(2))
    hpg = n_q // n_kv
    for m in range(M):
        p = pos + m
        toks = [cells[t] for t in range(min(p + 1, len(cells))) if cells[t] is not None
                and (not window or t > p - window or t < sinks)]
        if not toks:
            continue
        pg, sl = torch.tensor([c[0] for c in toks]), torch.tensor([c[1] for c in toks])
        k, v = kc[pg, :, sl].double().transpose(0, 1), vc[pg, :, sl].double().transpose(0, 1)   # [n_kv, tokens, D]
        qh = q[m].double().view(n_kv, hpg, D)
        sc = qh @ k.transpose(1, 2).contiguous() / math.sqrt(D)
        w = torch.softmax(sc, -1)
        o = w @ v
        # a weight p is rounded to fp16: half a step is 2^-11 of it, or 2^-25 below fp16's smallest normal number. p is 2^7 at
        # the reference, which is the score of a token, so the sum of p is at least 2^7 and the second part at most 2^-32 |v|
        # per token. It counts where V's rows differ widely in size: exact arithmetic with p rounded to fp16 and nothing else is
        # 7.3e-10 past the bound without it for the 18th token of 8 x 4 heads of 64 with V rows of 2^-12 to 2^6. A score
        # carries D fp32 roundings of |q| . |k| and two of the exponent, in numerator and denominator; the sums' chains; the
        # output half a step of its own
        ds = 2.0 ** -24 * ((D + 4) * (qh.abs() @ k.abs().transpose(1, 2).contiguous()) / math.sqrt(D)
                           + 4 * sc.abs()).amax(-1, keepdim=True)
        rel = 2.0 ** -11 + 2 * (ds + 2.0 ** -21) + 2.0 ** -24 * (len(toks) / 16 + 64)
        out[m] = o.view(n_q, D)
        bound[m] = (2.0 ** -11 * o.abs() + rel * (w @ v.abs()) + 2.0 ** -32 * v.abs().sum(1, keepdim=True)
                    + 2.0 ** -25).view(n_q, D)
    return out.view(M, -1), bound.view(M, -1)
