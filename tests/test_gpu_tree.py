"""GPU: attention of several new tokens per sequence over a paged cache, against 64 bits."""
from __future__ import annotations

import math
import random

import pytest
import torch

from tests import seq_ref
from tests._report import LINES
from triton_fused_rope_flash_attn_amd import (rope_cache_accept, rope_cache_append, rope_cache_fork, sdpa_rope_decode, sdpa_rope_tree,
                                              sdpa_rope_varlen)

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def randn(*shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def page_table(B, per, extra=2, seed=0):
    n = B * per + extra
    order = torch.randperm(n, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    return order[: B * per].reshape(B, per).to(DEV), n


def caches(n, page, Hkv, D, dtype, layout="rows"):
    if layout == "rows":
        return tuple(randn(n, page, Hkv, D, dtype=dtype, seed=s) for s in (1, 2))
    return tuple(randn(n, Hkv, page, D, dtype=dtype, seed=s).transpose(1, 2) for s in (1, 2))


def starts(new):
    return ints([sum(new[:i]) for i in range(len(new) + 1)])


def draft(new, seed, wide=None):
    """A random tree for each sequence as a mask, and the tokens' depths."""
    rng, wide = random.Random(seed), wide or max(new + [1])
    sees, depths = torch.zeros(sum(new), wide, dtype=torch.bool), []
    at = 0
    for m in new:
        d = []
        for i in range(m):
            up = rng.randint(max(-1, i - 5), i - 1) if i else -1
            if up >= 0:
                sees[at + i] = sees[at + up]
            sees[at + i, min(i, wide - 1)] = True
            d.append(0 if up < 0 else d[up] + 1)
        depths.append(d)
        at += m
    return sees.to(DEV), depths


def reference(q, kc, vc, table, pages, lengths, cu, tree=None, has_cls=True, positions=None):
    """O and sum P |V| in 64 bits on the CPU; infinities and NaN of V reach who sees them."""
    q, kc, vc, pages, cu = (x.detach().cpu() for x in (q, kc, vc, pages, cu))
    tree = None if tree is None else tree.cpu()
    H, D = q.shape[1:]
    group, rows = H // kc.shape[2], kc.shape[1]
    o = torch.zeros(q.shape, dtype=torch.float64)
    size = torch.zeros_like(o)
    for b in range(len(cu) - 1):
        n, m = int(lengths[b]), int(cu[b + 1] - cu[b])
        if n < 0 or m <= 0:
            continue
        at = [i for i in range(min(n + m, pages.shape[1] * rows)) if 0 <= int(pages[b, i // rows]) < kc.shape[0]]
        if not at:
            continue
        gi, ri = (torch.tensor(x) for x in zip(*((int(pages[b, i // rows]), i % rows) for i in at)))
        k, v, pos = kc[gi, ri].double(), vc[gi, ri].double(), torch.tensor(at)
        for j in range(m):
            t = int(cu[b]) + j
            if tree is None:
                see = pos <= n + j
            else:
                drafted = torch.cat([tree[t], torch.zeros(max(m, 1), dtype=torch.bool)])
                see = (pos < n) | drafted[(pos - n).clamp(min=0)]
            if not see.any():
                continue
            index = torch.tensor([n + j - int(has_cls)]) if positions is None else positions[t:t + 1].long().cpu()
            qh = seq_ref.rotate(q[t:t + 1].double(), table, index)[0]
            for h in range(H):
                g = h // group
                p = torch.softmax(k[see, g] @ qh[h] / math.sqrt(D), dim=0)
                o[t, h], size[t, h] = p @ v[see, g], p @ v[see, g].abs()
    return o, size


def run(tag, q, kc, vc, table, pages, lengths, cu, **kw):
    """q-hat (with the scale), P and O are rounded to 16 bits, one value each; K and V are exact:
    3 u.  fp32: no operand is rounded: 32 u (seq_ref)."""
    got = sdpa_rope_tree(q, kc, vc, table, pages, lengths, cu, **kw)
    ref, size = reference(q, kc, vc, table, pages, lengths.tolist(), cu, **kw)
    u = seq_ref.U[q.dtype]
    tol = (32 if q.dtype == F32 else 3) * u
    assert torch.isfinite(got).all()
    r = seq_ref.rel(got, ref)
    assert r <= tol, f"2-norm off by {r:.3e}, {tol:.3e} allowed"
    # a row: a rounded q-hat moves a logit by u of its terms (unit scale: sqrt(D) of them of 1 / sqrt(D) each)
    off, allowed = (got.double().cpu() - ref).norm(dim=-1), 2 * tol * size.norm(dim=-1)
    assert (off <= allowed).all(), f"{float((off / allowed.clamp(min=1e-300)).max()):.2f} of what is allowed"
    LINES.append(f"[tree {tag}] rel {r:.2e}")
    return got


@pytest.mark.parametrize("layout", ["rows", "heads"])
@pytest.mark.parametrize("drafted", [False, True])
@pytest.mark.parametrize("dtype,D,H,Hkv,page,lens,new", [
    (BF16, 64, 12, 12, 16, [197], [8]),
    (BF16, 64, 4, 4, 16, [1, 0, 2, 63, 64, 65], [1, 3, 0, 1, 2, 64]),
    (BF16, 128, 16, 4, 64, [500, 1, 0, 2100], [16, 5, 33, 20]),
    (BF16, 128, 24, 1, 7, [129, 300], [17, 4]),
    (BF16, 32, 6, 2, 1, [40, 129], [9, 100]),
    (BF16, 256, 4, 2, 100, [333, 5], [40, 70]),
    (F16, 64, 8, 1, 256, [1000, 255, 256, 257], [1, 1, 1, 1]),
    (F16, 128, 7, 1, 16, [1049], [30]),
    (F16, 256, 2, 2, 16, [17], [1]),
    (F32, 32, 4, 4, 16, [100, 3], [5, 70]),
    (F32, 64, 8, 2, 16, [700, 0, 50], [3, 0, 17]),
    (F32, 128, 3, 3, 5, [258], [66]),
    (F32, 256, 2, 1, 64, [130, 1], [2, 5]),
])
def test_tree(dtype, D, H, Hkv, page, lens, new, drafted, layout):
    B, per = len(lens), -(-max(n + m for n, m in zip(lens, new)) // page) + 1
    for wide in (per, -(-2000 // page)):   # a workgroup a tile, and shares of all tiles
        pages, n = page_table(B, max(per, wide))
        kc, vc = caches(n, page, Hkv, D, dtype, layout)
        q = randn(sum(new), H, D, dtype=dtype, seed=3)
        table = seq_ref.Table(max(lens) + max(new) + 1, D, DEV)
        kw = {}
        if drafted:
            sees, depths = draft(new, 5)
            kw = dict(tree=sees, positions=ints([x + d - 1 for x, row in zip(lens, depths) for d in row]))
        run(f"{dtype} D{D} H{H}/{Hkv} page {page} {lens} {new}", q, kc, vc, table, pages, ints(lens), starts(new), **kw)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_many_sequences(dtype):
    """More sequences than a step of a wave's search covers; many without tokens, some at the end behind all."""
    B, page, D = 150, 16, 32
    rng = random.Random(4)
    lens = [rng.choice([0, 1, 7, 40, 90, 300]) for _ in range(B)]
    new = [rng.choice([0, 0, 1, 2, 9]) for _ in range(B - 3)] + [0] * 3
    for per in (20, 60):
        pages, n = page_table(B, per)
        kc, vc = caches(n, page, 2, D, dtype)
        T = sum(new) + 5
        q = randn(T, 4, D, dtype=dtype, seed=3)
        got = run(f"{B} sequences", q, kc, vc, seq_ref.Table(400, D, DEV), pages, ints(lens), starts(new))
        assert (got[sum(new):] == 0).all()


def test_rows_that_see_nothing():
    """Trees that leave rows empty, narrower and wider than the drafted tokens, without columns; negative lengths."""
    page, D, lens, new = 16, 64, [0, 20, 0, -3, 5], [4, 3, 70, 2, 1]
    for per in (6, 80):
        pages, n = page_table(5, per)
        kc, vc = caches(n, page, 2, D, BF16)
        q = randn(sum(new), 4, D, dtype=BF16, seed=3)
        for wide in (0, 1, 5, 70, 100):
            tree = torch.rand(sum(new), wide, generator=torch.Generator().manual_seed(wide)).to(DEV) < 0.3
            tree[2] = False
            got = run(f"wide {wide}", q, kc, vc, seq_ref.Table(90, D, DEV), pages, ints(lens), starts(new), tree=tree)
            assert (got[2] == 0).all() and (got[77:79] == 0).all()


def test_bad_pages_and_lengths():
    page, D = 16, 64
    for per in (4, 40):
        pages, n = page_table(5, per)
        kc, vc = caches(n, page, 2, D, BF16)
        pages[0, 1], pages[1, 0], pages[2] = -1, n, 1 << 30
        # (the last two run past the table's end: its rows alone are seen)
        lens = [40, 20, 10, per * page - 1, 2 ** 31 - 1]
        new = [3, 9, 2, 4, 2]
        got = sdpa_rope_tree(randn(20, 2, D, dtype=BF16, seed=3), kc, vc, seq_ref.Table(64, D, DEV), pages, ints(lens), starts(new))
        ref, size = reference(randn(20, 2, D, dtype=BF16, seed=3), kc, vc, seq_ref.Table(64, D, DEV), pages, lens, starts(new))
        assert ((got.double().cpu() - ref).norm(dim=-1) <= 6 * 2.0 ** -8 * size.norm(dim=-1)).all()
        assert (got[12:14] == 0).all()


def test_starts_that_do_not_ascend():
    """No values are defined; nothing outside the tensors is touched."""
    page, D = 16, 64
    for per in (4, 40):
        pages, n = page_table(4, per)
        kc, vc = caches(n, page, 1, D, BF16)
        want = kc.clone()
        for cu in ([0, 30, 10, 50, 40], [5, -9, 1 << 30, 7, 60], [40, 30, 20, 10, 0]):
            out = sdpa_rope_tree(randn(60, 2, D, dtype=BF16, seed=3), kc, vc, seq_ref.Table(64, D, DEV), pages, ints([9, 30, 4, 1]), ints(cu))
            assert out.shape == (60, 2, D)
        torch.cuda.synchronize()
        assert torch.equal(kc, want)


@pytest.mark.parametrize("dtype,D", [(BF16, 64), (F16, 128), (F32, 32), (BF16, 256)])
def test_nothing_that_is_not_seen_reaches_a_row(dtype, D):
    """NaN and infinity in rows of no sequence, in other branches of the tree and in later tokens of a chain."""
    page, lens, new = 20, [45, 1, 0, 70], [6, 2, 9, 30]
    table = seq_ref.Table(110, D, DEV)
    sees, depths = draft(new, 7)
    positions = ints([x + d - 1 for x, row in zip(lens, depths) for d in row])
    for per in (6, 60):
        pages, n = page_table(4, per)
        kc, vc = caches(n, page, 2, D, dtype)
        q = randn(sum(new), 4, D, dtype=dtype, seed=3)
        used = torch.zeros(n, page, dtype=torch.bool)
        for b, m in enumerate(lens):
            for i in range(m + new[b]):
                used[pages[b, i // page].item(), i % page] = True
        for kw in (dict(tree=sees, positions=positions), {}):
            clean = run("clean", q, kc, vc, table, pages, ints(lens), starts(new), **kw)
            size = reference(q, kc, vc, table, pages, lens, starts(new), **kw)[1].norm(dim=-1)
            dk, dv = kc.clone(), vc.clone()
            dk[~used.to(DEV)], dv[~used.to(DEV)] = float("nan"), float("inf")
            assert torch.equal(sdpa_rope_tree(q, dk, dv, table, pages, ints(lens), starts(new), **kw), clean)
            # the second new token of each sequence: infinite values, NaN values and keys
            hit = [(pages[b, (lens[b] + 1) // page].item(), (lens[b] + 1) % page) for b in range(4)]
            for value, bad in enumerate([float("inf"), -float("inf"), float("nan")]):
                dk, dv = kc.clone(), vc.clone()
                for g, r in hit:
                    dv[g, r, :, 3] = bad
                    if value == 2:
                        dk[g, r] = bad
                got = sdpa_rope_tree(q, dk, dv, table, pages, ints(lens), starts(new), **kw)
                at = 0
                for b, m in enumerate(new):
                    for j in range(m):
                        sees_it = j >= 1 if not kw else bool(sees[at + j, 1])
                        if not sees_it:
                            assert torch.isfinite(got[at + j]).all(), (b, j)
                            # Another way through the same sums, which may round otherwise: both are within run()'s
                            # 2 tol |sum P |V|| of the formula's values, so within twice that of each other.
                            off = (got[at + j].double() - clean[at + j].double()).cpu().norm(dim=-1)
                            assert (off <= 4 * (32 if dtype == F32 else 3) * seq_ref.U[dtype] * size[at + j]).all()
                        elif value < 2:
                            assert (got[at + j, :, 3] == bad).all() and torch.isfinite(got[at + j, :, 4:]).all()
                        else:
                            assert torch.isnan(got[at + j]).all()
                    at += m


@pytest.mark.parametrize("dtype,D", [(BF16, 64), (F16, 128), (F32, 32), (BF16, 256), (F32, 256)])
def test_nan_queries_give_nan(dtype, D):
    """Of the tokens whose queries they are, and of no others, however many workers share their rows."""
    page, lens, new = 16, [500, 3, 700], [4, 2, 40]
    table = seq_ref.Table(800, D, DEV)
    for per in (48, 20, 120):
        pages, n = page_table(3, per)
        kc, vc = caches(n, page, 2, D, dtype)
        q = randn(sum(new), 4, D, dtype=dtype, seed=3)
        bad = q.clone()
        rows = [1, 5, 9, 44]
        bad[rows] = float("nan")
        sees, _ = draft(new, 7)
        for kw in ({}, dict(tree=sees)):
            want = sdpa_rope_tree(q, kc, vc, table, pages, ints(lens), starts(new), **kw)
            got = sdpa_rope_tree(bad, kc, vc, table, pages, ints(lens), starts(new), **kw)
            rest = [i for i in range(sum(new)) if i not in rows]
            assert torch.equal(got[rest], want[rest])
            assert torch.isnan(got[rows]).all()


@pytest.mark.parametrize("dtype,D", [(BF16, 64), (F16, 128), (F32, 32), (BF16, 256)])
def test_rows_that_see_nothing_feel_nothing(dtype, D):
    """Zeros, whatever the new tokens' rows hold, and on pages that are none."""
    page, lens, new = 16, [0, 0, 30], [6, 70, 4]
    table = seq_ref.Table(120, D, DEV)
    for per in (7, 80):
        pages, n = page_table(3, per)
        kc, vc = (torch.full((n, page, 2, D), x, dtype=dtype, device=DEV) for x in (float("nan"), float("inf")))
        q = randn(sum(new), 4, D, dtype=dtype, seed=3)
        tree = torch.zeros(sum(new), 70, dtype=torch.bool, device=DEV)
        got = sdpa_rope_tree(q, kc, vc, table, pages, ints(lens), starts(new), tree=tree)
        assert (got[:76] == 0).all()
        pages[2] = -1
        got = sdpa_rope_tree(q, kc, vc, table, pages, ints(lens), starts(new), tree=tree)
        assert (got == 0).all()


def test_infinite_values_of_light_rows():
    """An infinite value whose weight is 2^-200 of the largest is infinite in O all the same."""
    page, D = 16, 64
    for per, n in ((8, 100), (200, 3000)):
        pages, pool = page_table(1, per)
        kc, vc = (torch.zeros(pool, page, 1, D, dtype=BF16, device=DEV) for _ in range(2))
        q = torch.zeros(2, 1, D, dtype=BF16, device=DEV)
        q[..., 0] = 16.0
        flat = [(pages[0, i // page].item(), i % page) for i in range(n + 2)]
        for i in (n // 2, n - 1):
            kc[flat[i]][0, 0] = 100.0                    # logits of 200, others 0
        vc[flat[3]][0, 5], vc[flat[9]][0, 6] = float("inf"), float("-inf")
        got = sdpa_rope_tree(q, kc, vc, seq_ref.Table(1, D, DEV), pages, ints([n]), ints([0, 2]), positions=ints([-1, -1]))
        assert (got[..., 5] == float("inf")).all() and (got[..., 6] == float("-inf")).all() and (got[..., :5] == 0).all()


def test_positions_and_strides():
    page, D, lens, new = 16, 64, [50, 9], [3, 4]
    pages, n = page_table(2, 8)
    pages = torch.cat([pages, pages], dim=1)[:, :4]
    kc, vc = caches(n, page, 3, D, F16)
    q = randn(7, D, 6, dtype=F16, seed=3).transpose(1, 2)
    tree = draft(new, 2)[0]
    wide = torch.zeros(7, 9, dtype=torch.bool, device=DEV)
    wide[:, 2:6] = tree
    wide[:, 6:], wide[:, :2] = True, True
    run("positions", q, kc, vc, seq_ref.Table(40, D, DEV), pages, ints(lens), starts(new), positions=ints([12, -1, 0, 5, 70, 3, 39]))
    run("cut table", q, kc, vc, seq_ref.Table(10, D, DEV), pages, ints(lens), starts(new), has_cls=False, tree=wide[:, 2:6])
    every = torch.ones(1, 4, dtype=torch.bool, device=DEV).expand(7, 4)       # one row of the tree for all tokens
    run("one row", q, kc, vc, seq_ref.Table(70, D, DEV), pages, ints(lens), starts(new), tree=every)


def test_large_logits():
    page, D = 16, 64
    for per in (19, 100):
        pages, n = page_table(1, per)
        kc, vc = caches(n, page, 1, D, F32)
        q = randn(2, 2, D, dtype=F32, seed=3)
        q[..., 0] = 100.0
        kc[pages[0, 7].item(), 3, 0, 0] = 3e4
        got = sdpa_rope_tree(q, kc, vc, seq_ref.Table(1, D, DEV), pages, ints([290]), ints([0, 2]), positions=ints([0, 0]))
        for x in got.flatten(0, 1):
            assert torch.allclose(x, vc[pages[0, 7].item(), 3, 0], rtol=1e-5, atol=1e-6)


def test_no_tokens_and_no_sequences():
    kc, vc = caches(3, 16, 1, 64, BF16)
    table, none = seq_ref.Table(4, 64, DEV), randn(0, 2, 64, dtype=BF16, seed=0)
    out = sdpa_rope_tree(none, kc, vc, table, torch.zeros(1, 4, dtype=torch.int32, device=DEV), ints([4]), ints([0, 0]))
    assert out.shape == (0, 2, 64)


def test_one_token_each_is_decode():
    """A chain of one new token is what sdpa_rope_decode computes with the lengths behind it."""
    page, D, lens = 16, 128, [700, 3, 64, 0]
    pages, n = page_table(4, 60)
    kc, vc = caches(n, page, 2, D, BF16)
    q, table = randn(4, 8, D, dtype=BF16, seed=3), seq_ref.Table(800, D, DEV)
    got = run("decode", q, kc, vc, table, pages, ints(lens), starts([1] * 4))
    want = sdpa_rope_decode(q, kc, vc, table, pages, ints(lens) + 1)
    assert seq_ref.rel(got, want.double().cpu()) <= 4 * 2.0 ** -8


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_prompt_in_chunks(dtype):
    """Chunks of prompts, appended and attended to one after the other, give what attention over the whole packs gives."""
    H, Hkv, D, page, lens = 8, 2, 64, 16, [150, 33, 97]
    T = sum(lens)
    q, k, v = (randn(T, h, D, dtype=dtype, seed=s) for h, s in ((H, 7), (Hkv, 8), (Hkv, 9)))
    table = seq_ref.Table(max(lens), D, DEV)
    start = [sum(lens[:i]) for i in range(3)]
    ref = seq_ref.varlen(q, k, v, None, table, [*start, T], True, True)["o"]
    whole = sdpa_rope_varlen(q, k, v, table, ints([*start, T]))
    pages, n = page_table(3, 40)
    kc, vc = (torch.full((n, page, Hkv, D), float("nan"), dtype=dtype, device=DEV) for _ in range(2))
    done, rng = [0] * 3, random.Random(1)
    out = torch.zeros_like(q)
    while done != lens:
        new = [min(rng.randint(0, 60), m - d) for m, d in zip(lens, done)]
        rows = torch.cat([torch.arange(s + d, s + d + c) for s, d, c in zip(start, done, new)])
        if len(rows) == 0:
            continue
        lengths, cu = ints(done), starts(new)
        rope_cache_append(k[rows], v[rows], table, kc, vc, pages, lengths, cu_seqlens=cu)
        out[rows] = sdpa_rope_tree(q[rows], kc, vc, table, pages, lengths, cu)
        done = [d + c for d, c in zip(done, new)]
    tol = 32 * seq_ref.U[F32] if dtype == F32 else 4 * seq_ref.U[dtype]
    assert seq_ref.rel(out, ref) <= tol and seq_ref.rel(whole, ref) <= tol


def test_drafted_and_accepted():
    """Trees are appended, verified and accepted; what is kept gives the outputs of a chain of the kept tokens."""
    H, Hkv, D, page, B = 4, 2, 64, 8, 3
    table, rng = seq_ref.Table(200, D, DEV), random.Random(3)
    pages, n = page_table(B, 20)
    kc, vc = (torch.full((n, page, Hkv, D), float("nan"), dtype=BF16, device=DEV) for _ in range(2))
    lengths, kept = ints([0] * B), [[] for _ in range(B)]
    for step in range(6):
        new = [rng.randint(1, 9) for _ in range(B)]
        sees, depths = draft(new, step)
        cu = starts(new)
        positions = ints([x + d - 1 for x, row in zip(lengths.tolist(), depths) for d in row])
        q, k, v = (randn(sum(new), h, D, dtype=BF16, seed=10 * step + s) for s, h in enumerate((H, Hkv, Hkv)))
        rope_cache_append(k, v, table, kc, vc, pages, lengths, cu_seqlens=cu, positions=positions)
        out = sdpa_rope_tree(q, kc, vc, table, pages, lengths, cu, tree=sees, positions=positions)
        path, at = [], 0
        for b, m in enumerate(new):
            leaf = rng.randrange(m)
            way = [i for i in range(m) if sees[at + leaf, i]]
            path.append(way + [-1] * (9 - len(way)))
            kept[b] += [(q[at + i], k[at + i], v[at + i], out[at + i]) for i in way]
            at += m
        lengths = rope_cache_accept(kc, vc, pages, lengths, ints(path))
        assert lengths.tolist() == [len(x) for x in kept]
    for b in range(B):
        q, k, v, o = (torch.stack(x) for x in zip(*kept[b]))
        ref = seq_ref.varlen(q, k, v, None, table, [0, len(q)], True, True)["o"]
        assert seq_ref.rel(o, ref) <= 4 * 2.0 ** -8


def test_captured_and_replayed():
    H, Hkv, D, page, B = 8, 2, 64, 16, 3
    pages, n = page_table(B, 60)
    table = seq_ref.Table(900, D, DEV)
    kc, vc = caches(n, page, Hkv, D, BF16)
    q, lengths, cu = randn(24, H, D, dtype=BF16, seed=7), ints([0, 10, 400]), starts([8, 8, 8])
    tree = draft([8, 8, 8], 1)[0]

    def step():
        return sdpa_rope_tree(q, kc, vc, table, pages, lengths, cu, tree=tree), sdpa_rope_tree(q, kc, vc, table, pages[:, :9], lengths, cu)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(6):
        q.copy_(randn(24, H, D, dtype=BF16, seed=30 + i))
        lengths.copy_(ints([100 * i, 7 * i, 850 - 90 * i]))
        cu.copy_(starts([[8, 8, 8], [24, 0, 0], [0, 3, 20], [1, 1, 1], [5, 0, 19], [2, 22, 0]][i]))
        tree.copy_(torch.rand(24, 8, generator=torch.Generator().manual_seed(i)) < 0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step())), i


def test_two_graphs_at_once():
    """Each has partial sums of its own: replayed on two streams together they give what each gives alone."""
    page, D = 16, 64
    table = seq_ref.Table(2100, D, DEV)
    sides = []
    for seed in (1, 2):
        pages, n = page_table(2, 130, seed=seed)
        kc, vc = caches(n, page, 2, D, BF16)
        q = randn(40, 8, D, dtype=BF16, seed=seed)
        args = (q, kc, vc, table, pages, ints([2000, 300 * seed]), ints([0, 30, 40]))
        want, stream, graph = sdpa_rope_tree(*args), torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            out = sdpa_rope_tree(*args)
        sides.append((want, stream, graph, out, args))
    for _ in range(5):
        torch.cuda.synchronize()
        for _, stream, graph, out, _ in sides:
            with torch.cuda.stream(stream):
                out.zero_()
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for want, _, _, out, _ in sides)


def test_another_stream():
    page, D = 16, 128
    pages, n = page_table(2, 100)
    kc, vc = caches(n, page, 2, D, F16)
    q, table = randn(40, 4, D, dtype=F16, seed=3), seq_ref.Table(1600, D, DEV)
    args = (q, kc, vc, table, pages, ints([1500, 300]), ints([0, 30, 40]))
    want = sdpa_rope_tree(*args)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = [sdpa_rope_tree(*args) for _ in range(3)]
    s.synchronize()
    assert all(torch.equal(x, want) for x in got)


def test_more_rows_than_a_join_could_take():
    """2^28 query rows and more over short tables, where nothing is joined."""
    B, m, H, page, D = 16384, 257, 64, 64, 32
    kc, vc = caches(8, page, 1, D, BF16)
    table, q = seq_ref.Table(1024, D, DEV), randn(1, H, D, dtype=BF16, seed=3)
    pages, lengths = ints([[3, 1, 4, 0, 5]]).expand(B, 5), ints([40] * B)
    got = sdpa_rope_tree(q.expand(B * m, H, D), kc, vc, table, pages, lengths, torch.arange(B + 1, dtype=torch.int32, device=DEV) * m)
    want = run("one of many", q.expand(m, H, D), kc, vc, table, pages[:1], lengths[:1], ints([0, m]))
    for b in (0, 1, B // 2 + 1, B - 1):
        assert torch.equal(got[b * m:(b + 1) * m], want), b


def test_cache_past_32_bits():
    Hkv, D, page = 8, 128, 64
    n = (1 << 31) // (Hkv * D * page) + 3
    kc, vc = (torch.zeros(n, page, Hkv, D, dtype=BF16, device=DEV) for _ in range(2))
    for g in (n - 1, 0, n - 2):
        kc[g], vc[g] = (randn(page, Hkv, D, dtype=BF16, seed=g % 97 + s) for s in (0, 1000))
    q, table = randn(20, 2 * Hkv, D, dtype=BF16, seed=6), seq_ref.Table(150, D, DEV)
    small_k, small_v = (torch.stack([c[n - 1], c[0], c[n - 2]]) for c in (kc, vc))
    got = sdpa_rope_tree(q, kc, vc, table, ints([[n - 1, 0, n - 2]]), ints([130]), ints([0, 20]))
    want = sdpa_rope_tree(q, small_k, small_v, table, ints([[0, 1, 2]]), ints([130]), ints([0, 20]))
    assert torch.equal(got, want)


def test_op_passes_opcheck():
    kc, vc = caches(10, 16, 2, 64, BF16)
    table = seq_ref.Table(40, 64, DEV)
    q, tree = randn(5, 4, 64, dtype=BF16, seed=3), draft([2, 3], 1)[0]
    args = (q, kc, vc, *table.tables(), ints([[0, 1], [2, 3]]), ints([3, 20]), ints([0, 2, 5]))
    torch.library.opcheck(torch.ops.farope.cache_tree.default, (*args, tree, None, True, 0.125))
    torch.library.opcheck(torch.ops.farope.cache_tree.default, (*args, None, ints([0] * 5), True, 0.125))
    with pytest.raises(RuntimeError, match="no autograd formula"):
        sdpa_rope_tree(q.requires_grad_(), kc, vc, table, *args[5:]).sum().backward()


def test_compiled_steps():
    """Append, tree, accept, fork and windowed decode as one compiled graph, against the same calls."""
    page, D = 16, 64
    table = seq_ref.Table(200, D, DEV)
    new, lens = [4, 6], [30, 3]
    sees, depths = draft(new, 3)
    positions = ints([x + d - 1 for x, row in zip(lens, depths) for d in row])
    q, k, v = (randn(sum(new), h, D, dtype=BF16, seed=s) for s, h in enumerate((4, 2, 2)))
    path, parents, room = ints([[0, 2, -1], [1, 3, 5]]), ints([1, 1]), ints([20, 5])

    def step(kc, vc, pages, lengths, refs, cu):
        rope_cache_append(k, v, table, kc, vc, pages, lengths, cu_seqlens=cu, positions=positions)
        out = sdpa_rope_tree(q, kc, vc, table, pages, lengths, cu, tree=sees, positions=positions)
        chain = sdpa_rope_tree(q, kc, vc, table, pages, lengths, cu)
        lengths.copy_(rope_cache_accept(kc, vc, pages, lengths, path))
        missing = rope_cache_fork(kc, vc, pages, lengths, refs, parents, room=room)
        one = sdpa_rope_decode(q[:2], kc, vc, table, pages, lengths, window=9, sinks=2)
        return out, chain, missing, one

    results = []
    for fn in (step, torch.compile(step, fullgraph=True, backend="aot_eager")):
        kc, vc = caches(20, page, 2, D, BF16)
        state = (kc, vc, ints([[3, 1, 7, -1, -1], [2, 0, -1, -1, -1]]), ints(lens), ints([1, 1, 1, 1, 0, 0, 0, 1] + [0] * 12), starts(new))
        results.append((*fn(*state), *state))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    # (both go on from place 1, 6 rows of one page: the first keeps it and room for 26 rows, the other copies it)
    assert results[0][7].tolist() == [6, 6] and results[0][6].tolist() == [[2, 0, -1, -1, -1], [4, -1, -1, -1, -1]]
