"""Attention over packed sequences and over a paged cache in 64 bits, sequence by
sequence and head by head: what the GPU tests of these operators compare with.

Tolerances.  A value rounded to a type is off by at most u = eps / 2 of it (bf16 2^-8,
fp16 2^-11, fp32 2^-24).  With inputs of unit scale a logit's terms are of unit scale
too, so a rounding of q-hat or k-hat moves P by about u of it, and the 2-norms of a
pass's results are off by at most the roundings on their way:

* O: q-hat, k-hat, P, O: 4 u;   dV: the same with dO for V: 4 u;
* dQ, dK: q-hat, k-hat (P), O (in delta), dS, the other factor, the result: 6 u;
* decode: K is exact, q-hat and P carry a second value (u^2), O: u + 3 u^2 of the
  absolute sum P |V|;
* fp32: no operand is rounded; a logit (log2 units, at most 16 from the row's maximum)
  is off by about 16 + sqrt(D) / 4 units of 2^-24, exp2 by 2, a sum by a few: 32 u,
  and twice that for gradients, which take P and dP.

A single row's norm may be off by twice that, and where terms cancel by the same part
of the tensor's root-mean-square row.  dS = P (dP - delta) can cancel wholly (a row that sees
one key has dS = 0): dP and delta are fp32 sums, off by up to 64 units of 2^-24 of
their terms' absolute sums, and delta is taken from O as stored, off by u |dO| |O|.  So a row
of dQ may also be off by scale * sum_j P_ij (64 * 2^-24 (|dO_i| |V_j| + |dO_i| |O_i|) + u |dO_i|
|O_i|) |k-hat_j| (products of absolute values summed over channels), a row of dK likewise.
"""
from __future__ import annotations

import math

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
ROUNDINGS = {"o": 4, "dv": 4, "dq": 6, "dk": 6}
FP32_UNITS = {"o": 32, "dv": 64, "dq": 64, "dk": 64}


class Table:
    """Any object with tables() serves; ``rows`` positions of one dimension."""

    def __init__(self, rows, D, device="cpu", base=100.0):
        freq = base ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))
        ang = torch.arange(rows, dtype=torch.float64)[:, None] * freq
        self.cos, self.sin = (t.float().to(device).contiguous() for t in (ang.cos(), ang.sin()))

    def tables(self):
        return self.cos, self.sin


def rotate(x, table, index, back=False):
    """x [n, heads, D] in 64 bits, turned by table rows `index` [n]: below 0 not, past the end the last."""
    cos, sin = (t.double().cpu()[index.clamp(0, t.shape[0] - 1)] for t in table.tables())
    cos, sin = torch.where(index[:, None] < 0, 1.0, cos)[:, None], torch.where(index[:, None] < 0, 0.0, sin)[:, None]
    sin = -sin if back else sin
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)


def varlen(q, k, v, do, table, cu, causal, has_cls, positions=None, scale=None):
    """{"o", "dq", "dk", "dv", "lse"} in 64 bits on the CPU; rows of no sequence are zeros.
    "dq+", "dk+": what the rows of dQ and dK may be off by where dS cancels."""
    u = U[q.dtype] if q.dtype in U else 0.0
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    do = None if do is None else do.detach().double().cpu()
    T, H, D = q.shape
    group, c = H // k.shape[1], 1.0 / math.sqrt(D) if scale is None else scale
    out = {"o": torch.zeros_like(q), "dq": torch.zeros_like(q), "dk": torch.zeros_like(k), "dv": torch.zeros_like(v),
           "lse": torch.zeros(H, T, dtype=torch.float64), "dq+": torch.zeros(q.shape[:2], dtype=torch.float64),
           "dk+": torch.zeros(k.shape[:2], dtype=torch.float64)}
    cu = [int(x) for x in cu]
    for a, b in zip(cu[:-1], cu[1:]):
        n = b - a
        if n == 0:
            continue
        index = torch.arange(n) - int(has_cls) if positions is None else positions[a:b].long().cpu()
        qh, kh = rotate(q[a:b], table, index), rotate(k[a:b], table, index)
        gq, gk = torch.zeros_like(qh), torch.zeros_like(kh)
        for h in range(H):
            g = h // group
            s = qh[:, h] @ kh[:, g].t() * c
            if causal:
                s = s.masked_fill(torch.ones(n, n).triu(1).bool(), -math.inf)
            p = torch.softmax(s, dim=1)
            out["lse"][h, a:b] = torch.logsumexp(s, dim=1)
            o = p @ v[a:b, g]
            out["o"][a:b, h] = o
            if do is None:
                continue
            d = do[a:b, h]
            out["dv"][a:b, g] += p.t() @ d
            ds = p * (d @ v[a:b, g].t() - (d * o).sum(1, keepdim=True)) * c
            gq[:, h] = ds @ kh[:, g]
            gk[:, g] += ds.t() @ qh[:, h]
            delta = (d * o).abs().sum(1, keepdim=True)
            off = p * (64 * 2.0 ** -24 * (d.abs() @ v[a:b, g].abs().t() + delta) + u * delta) * abs(c)
            out["dq+"][a:b, h] = (off @ kh[:, g].abs()).norm(dim=1)
            out["dk+"][a:b, g] += (off.t() @ qh[:, h].abs()).norm(dim=1)
        out["dq"][a:b] = rotate(gq, table, index, back=True)
        out["dk"][a:b] = rotate(gk, table, index, back=True)
    return out


def decode(q, k_cache, v_cache, table, pages, lengths, has_cls, positions=None):
    """O and sum P |V| in 64 bits on the CPU, row by row through the page table."""
    q = q.detach().double().cpu()
    kc, vc = k_cache.cpu(), v_cache.cpu()
    B, H, D = q.shape
    Hkv, rows = kc.shape[2], kc.shape[1]
    o, size = torch.zeros_like(q), torch.zeros_like(q)
    for b in range(B):
        n = max(0, min(int(lengths[b]), pages.shape[1] * rows))
        at = [(int(pages[b, i // rows]), i % rows) for i in range(n)]
        at = [(g, r) for g, r in at if 0 <= g < kc.shape[0]]
        if not at:
            continue
        gi, ri = (torch.tensor(x) for x in zip(*at))
        k, v = kc[gi, ri].double(), vc[gi, ri].double()          # [n, Hkv, D]
        index = torch.tensor([n - 1 - int(has_cls)]) if positions is None else positions[b:b + 1].long().cpu()
        qh = rotate(q[b:b + 1], table, index)[0]
        for h in range(H):
            g = h // (H // Hkv)
            p = torch.softmax(k[:, g] @ qh[h] / math.sqrt(D), dim=0)
            o[b, h], size[b, h] = p @ v[:, g], p @ v[:, g].abs()
    return o, size


def rel(x, ref):
    x, ref = x.detach().double().cpu(), ref.double()
    assert torch.isfinite(x).all()
    n = ref.norm()
    return float((x - ref).norm() / n) if n > 0 else float((x - ref).norm())


def check(name, x, refs, dtype):
    """The bounds above for tensor `name` of a pass; returns its relative error."""
    ref = refs[name]
    tol = FP32_UNITS[name] * U[dtype] if dtype == torch.float32 else ROUNDINGS[name] * U[dtype]
    r = rel(x, ref)
    assert r <= tol, f"{name}: 2-norm off by {r:.3e}, {tol:.3e} allowed"
    rows, want = (x.detach().double().cpu() - ref).norm(dim=-1), ref.norm(dim=-1)
    allowed = 2 * tol * (want + want.square().mean().sqrt())
    if name + "+" in refs:
        allowed = allowed + refs[name + "+"]
    assert (rows <= allowed).all(), f"{name}: row off by {float((rows / allowed.clamp(min=1e-300)).max()):.2f} of what is allowed"
    return r
