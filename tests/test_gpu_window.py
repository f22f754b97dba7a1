"""GPU: attention over a window and a sequence's first tokens (sinks), packed and over a cache, against 64 bits.
Bounds: those of seq_ref, whose roundings are the same."""
from __future__ import annotations

import math
import random

import pytest
import torch

from tests import seq_ref
from tests._report import LINES
from triton_fused_rope_flash_attn_amd import CosSinTable, rope_cache_append, sdpa_rope_decode, sdpa_rope_varlen

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def starts(lens, device=DEV):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=device)


def randn(*shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def inputs(T, H, Hkv, D, dtype, seed=0, views=False):
    g = torch.Generator().manual_seed(seed)
    if views:   # thirds of one projection's output
        q, k, v = torch.randn(T, H + 2 * Hkv, D, generator=g).to(dtype).to(DEV).split([H, Hkv, Hkv], dim=1)
    else:
        q, k, v = (torch.randn(T, n, D, generator=g).to(dtype).to(DEV) for n in (H, Hkv, Hkv))
    return q, k, v, torch.randn(T, H, D, generator=g).to(dtype).to(DEV)


def visible(n, window, sinks):
    i, j = torch.arange(n)[:, None], torch.arange(n)[None, :]
    return (j <= i) & ((i - j < window) | (j < sinks))


def varlen(q, k, v, do, table, cu, window, sinks, has_cls=True, positions=None, scale=None):
    """As seq_ref.varlen, over what the window leaves."""
    u = seq_ref.U[q.dtype]
    q, k, v, do = (t.detach().double().cpu() for t in (q, k, v, do))
    T, H, D = q.shape
    group, c = H // k.shape[1], 1.0 / math.sqrt(D) if scale is None else scale
    out = {"o": torch.zeros_like(q), "dq": torch.zeros_like(q), "dk": torch.zeros_like(k), "dv": torch.zeros_like(v),
           "dq+": torch.zeros(q.shape[:2], dtype=torch.float64), "dk+": torch.zeros(k.shape[:2], dtype=torch.float64)}
    cu = [int(x) for x in cu]
    for a, b in zip(cu[:-1], cu[1:]):
        n = b - a
        if n == 0:
            continue
        index = torch.arange(n) - int(has_cls) if positions is None else positions[a:b].long().cpu()
        qh, kh = seq_ref.rotate(q[a:b], table, index), seq_ref.rotate(k[a:b], table, index)
        gq, gk = torch.zeros_like(qh), torch.zeros_like(kh)
        hidden = ~visible(n, window, sinks)
        for h in range(H):
            g = h // group
            p = torch.softmax((qh[:, h] @ kh[:, g].t() * c).masked_fill(hidden, -math.inf), dim=1)
            o, d = p @ v[a:b, g], do[a:b, h]
            out["o"][a:b, h] = o
            out["dv"][a:b, g] += p.t() @ d
            ds = p * (d @ v[a:b, g].t() - (d * o).sum(1, keepdim=True)) * c
            gq[:, h] = ds @ kh[:, g]
            gk[:, g] += ds.t() @ qh[:, h]
            delta = (d * o).abs().sum(1, keepdim=True)
            off = p * (64 * 2.0 ** -24 * (d.abs() @ v[a:b, g].abs().t() + delta) + u * delta) * abs(c)
            out["dq+"][a:b, h] = (off @ kh[:, g].abs()).norm(dim=1)
            out["dk+"][a:b, g] += (off.t() @ qh[:, h].abs()).norm(dim=1)
        out["dq"][a:b] = seq_ref.rotate(gq, table, index, back=True)
        out["dk"][a:b] = seq_ref.rotate(gk, table, index, back=True)
    return out


def grads(q, k, v, do, table, cu, **kw):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = sdpa_rope_varlen(*leaves, table, cu, **kw)
    return dict(zip(("o", "dq", "dk", "dv"), (o.detach(), *torch.autograd.grad(o, leaves, do))))


def compare(tag, got, ref, dtype):
    worst = {n: seq_ref.check(n, got[n], ref, dtype) for n in got}
    LINES.append(f"[window {tag}] " + " ".join(f"{n} {e:.2e}" for n, e in worst.items()))


SHORT = [1, 0, 5, 0, 33]
EDGES = [63, 64, 1, 65, 127, 128, 129]
LONG = [197, 3, 577, 300]


@pytest.mark.parametrize("window,sinks", [(1, 1), (2, 0), (16, 4), (64, 0), (65, 1), (100, 70), (130, 4), (576, 0)])
@pytest.mark.parametrize("dtype,D,H,Hkv,lens,views", [
    (BF16, 64, 6, 2, SHORT, True),
    (BF16, 64, 3, 1, EDGES, False),
    (BF16, 128, 4, 2, EDGES, True),
    (BF16, 128, 8, 2, LONG, True),
    (BF16, 32, 4, 1, EDGES, True),
    (BF16, 256, 2, 1, EDGES, False),
    (F16, 64, 12, 12, LONG, True),
    (F16, 128, 7, 1, SHORT, False),
    (F16, 32, 2, 2, LONG, False),
    (F16, 256, 3, 3, LONG, True),
    (F32, 32, 2, 1, EDGES, False),
    (F32, 64, 4, 2, EDGES, True),
    (F32, 128, 2, 2, LONG, False),
    (F32, 256, 2, 1, SHORT, True),
])
def test_window(dtype, D, H, Hkv, lens, views, window, sinks):
    q, k, v, do = inputs(sum(lens), H, Hkv, D, dtype, seed=D + H, views=views)
    table = seq_ref.Table(max(lens), D, DEV)
    ref = varlen(q, k, v, do, table, starts(lens), window, sinks)
    got = grads(q, k, v, do, table, starts(lens), window=window, sinks=sinks)
    compare(f"{dtype} D{D} H{H}/{Hkv} {lens} window {window} sinks {sinks}", got, ref, dtype)


@pytest.mark.parametrize("dtype,D,H,Hkv", [(BF16, 128, 8, 8), (BF16, 64, 16, 16), (F16, 128, 16, 4), (BF16, 256, 8, 8)])
def test_tiles_of_128_rows_and_divided_sinks(dtype, D, H, Hkv):
    """Long sequences beside short ones: tiles of 128 rows, sinks whose queries are divided, more sinks than a tile holds."""
    lens = [3000, 70, 1, 2500]
    q, k, v, do = inputs(sum(lens), H, Hkv, D, dtype, seed=3)
    table = seq_ref.Table(max(lens), D, DEV)
    for window, sinks in ((40, 4), (300, 100), (1500, 1)):
        got = grads(q, k, v, do, table, starts(lens), window=window, sinks=sinks)
        ref = varlen(q, k, v, do, table, starts(lens), window, sinks)
        compare(f"{dtype} D{D} H{H}/{Hkv} long, window {window} sinks {sinks}", got, ref, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_many_sequences(dtype):
    rng = random.Random(3)
    lens = [rng.choice([0, 1, 2, 30, 90]) for _ in range(150)]
    q, k, v, do = inputs(sum(lens) + 9, 2, 1, 32, dtype, seed=3)
    table = seq_ref.Table(90, 32, DEV)
    got = grads(q, k, v, do, table, starts(lens), window=20, sinks=2)
    assert all((t[sum(lens):] == 0).all() for t in got.values())
    compare("many", got, varlen(q, k, v, do, table, starts(lens), 20, 2), dtype)


@pytest.mark.parametrize("dtype,D", [(BF16, 64), (F16, 128), (F32, 32), (BF16, 256)])
def test_a_window_of_one_token(dtype, D):
    """O = V, dQ = dK = 0, dV = dO, summed over the group."""
    lens = [1, 300, 64, 0, 7]
    q, k, v, do = inputs(sum(lens) + 5, 4, 2, D, dtype, seed=2)
    got = grads(q, k, v, do, seq_ref.Table(300, D, DEV), starts(lens), window=1)
    n = sum(lens)
    assert torch.equal(got["o"][:n], v[:n].repeat_interleave(2, dim=1))
    assert (got["dq"] == 0).all() and (got["dk"] == 0).all() and (got["dv"][n:] == 0).all()
    want = do[:n].double().reshape(n, 2, 2, D).sum(2)
    # (a sum of two in fp32, its rounding, and P = exp2 of a difference that is 0 but for the logits' sums: 64 units)
    assert ((got["dv"][:n].double() - want).abs() <= (seq_ref.U[dtype] + 64 * 2.0 ** -24) * do[:n].double().abs().reshape(n, 2, 2, D).sum(2)).all()


def test_windows_that_hold_everything():
    """... are the causal call, bit for bit."""
    lens = [130, 40, 577]
    q, k, v, do = inputs(sum(lens), 4, 2, 64, BF16)
    table = seq_ref.Table(577, 64, DEV)
    want = grads(q, k, v, do, table, starts(lens))
    for window in (sum(lens), 2 ** 31 - 1):
        for sinks in (0, 2 ** 31 - 1):
            got = grads(q, k, v, do, table, starts(lens), window=window, sinks=sinks)
            assert all(torch.equal(got[n], want[n]) for n in want)
    # longer than each sequence, but not than all of them; and sinks that are all tokens
    for window, sinks in ((577, 0), (3, 600)):
        got = grads(q, k, v, do, table, starts(lens), window=window, sinks=sinks)
        compare("everything", got, seq_ref.varlen(q, k, v, do, table, starts(lens), True, True), BF16)


@pytest.mark.parametrize("dtype,D,H,Hkv,lens", [(BF16, 64, 2, 1, [100, 3]), (BF16, 64, 4, 4, [700, 130, 900]), (F16, 128, 4, 2, [90, 20]),
                                                (F16, 128, 16, 4, [4100, 300, 700]), (BF16, 256, 2, 1, [300, 70]), (BF16, 32, 2, 2, [200]),
                                                (F32, 64, 2, 1, [140, 33])])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_rows_do_not_feel_what_they_do_not_see(dtype, D, H, Hkv, lens, value):
    """K and V of a token that is not finite reach the tokens whose windows hold it and no others; a sink reaches all."""
    window, sinks = 50, 2
    q, k, v, _ = inputs(sum(lens), H, Hkv, D, dtype, seed=17)
    table, cu = seq_ref.Table(max(lens), D, DEV), starts(lens)
    kw = dict(window=window, sinks=sinks)
    clean = sdpa_rope_varlen(q, k, v, table, cu, **kw)
    off = (seq_ref.ROUNDINGS["o"] if dtype != F32 else seq_ref.FP32_UNITS["o"]) * seq_ref.U[dtype]
    for where in ("middle", "sink"):
        at = [n * 5 // 8 if where == "middle" else min(1, n - 1) for n in lens]
        bad_k, bad_v, feels = k.clone(), v.clone(), torch.zeros(sum(lens), dtype=torch.bool)
        for a, n, j in zip(cu.tolist(), lens, at):
            bad_v[a + j, :, 3] = value
            bad_k[a + j] = value
            feels[a:a + n] = visible(n, window, sinks)[:, j]
        feels = feels.to(DEV)
        for kk in (k, bad_k):
            got = sdpa_rope_varlen(q, kk, bad_v, table, cu, **kw)
            assert torch.isfinite(got[~feels]).all()
            # (such a row may be computed again in another order: two results, each within the bound)
            err, size = (got[~feels].double() - clean[~feels].double()).norm(dim=-1), clean[~feels].double().norm(dim=-1)
            assert (err <= 4 * off * (size + clean.double().norm(dim=-1).square().mean().sqrt())).all()
            if kk is k:
                assert not torch.isfinite(got[feels][..., 3]).any()
                rest = torch.arange(D, device=DEV) != 3
                assert torch.isfinite(got[..., rest]).all()
            elif value != value:
                assert not torch.isfinite(got[feels]).any()


@pytest.mark.parametrize("dtype,D,window", [(BF16, 64, 5), (F16, 128, 40), (BF16, 256, 12), (F16, 64, 64)])
def test_short_windows_do_not_feel_the_rounding_of_o(dtype, D, window):
    """V with a common offset, as in the test of short rows without a window, everywhere in long sequences."""
    lens = [200, 33]
    q, k, v, do = inputs(sum(lens), 4, 2, D, dtype)
    v = (v.float() + 64.0).to(dtype)
    table = seq_ref.Table(200, D, DEV)
    ref = varlen(q, k, v, do, table, starts(lens), window, 0)
    got = grads(q, k, v, do, table, starts(lens), window=window)
    tol = seq_ref.ROUNDINGS["dq"] * seq_ref.U[dtype] + 64 * 64 * 2.0 ** -24
    for n in ("dq", "dk"):
        assert seq_ref.rel(got[n], ref[n]) <= tol, n


@pytest.mark.parametrize("window,sinks", [(9, 0), (20, 3)])
def test_gradient_against_differences(window, sinks):
    lens, D, eps = [40, 25], 32, 1e-2
    q, k, v, do = inputs(65, 4, 2, D, F32)
    table, kw = seq_ref.Table(40, D, DEV), dict(window=window, sinks=sinks)
    got = grads(q, k, v, do, table, starts(lens), **kw)
    g = torch.Generator().manual_seed(5)
    for i, name in enumerate(("dq", "dk", "dv")):
        x = [q, k, v]
        d = torch.randn(x[i].shape, generator=g).to(DEV)
        up, down = ([t + s * eps * d if j == i else t for j, t in enumerate(x)] for s in (1, -1))
        f = [(sdpa_rope_varlen(*y, table, starts(lens), **kw).double() * do.double()).sum().item() for y in (up, down)]
        slope, want = (f[0] - f[1]) / (2 * eps), (got[name].double() * d.double()).sum().item()
        # third derivatives of order 1 per term: eps^2 of the gradient's norm times the direction's
        scale = got[name].double().norm().item() * d.double().norm().item()
        assert abs(slope - want) <= 4 * eps ** 2 * scale + 1e-5 * scale, (name, slope, want)


def test_strides_positions_and_scales():
    lens, D, T = [150, 20], 64, 170
    table = seq_ref.Table(60, D, DEV)
    q = randn(T, D, 4, dtype=F16, seed=3).transpose(1, 2)                                            # channels apart
    k = randn(2, T, D, dtype=F16, seed=4).transpose(0, 1)
    v = torch.cat([k.new_zeros(1), randn(T, 2, D, dtype=F16, seed=5).reshape(-1)])[1:].view(T, 2, D)   # rows not aligned
    do = randn(1, 4, D, dtype=F16, seed=6).expand(T, 4, D)
    positions = torch.randint(-1, 70, (T,), generator=torch.Generator().manual_seed(1)).to(torch.int32).to(DEV)
    got = grads(q, k, v, do, table, starts(lens), window=30, sinks=3, positions=positions)
    compare("strides", got, varlen(q, k, v, do, table, starts(lens), 30, 3, positions=positions), F16)
    for scale in (0.0, -0.05, 0.25):
        leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
        o, _ = torch.ops.farope.seq_window_fwd(*leaves, *table.tables(), starts(lens), None, True, scale, 30, 3)
        got = dict(zip(("o", "dq", "dk", "dv"), (o.detach(), *torch.autograd.grad(o, leaves, do))))
        if scale == 0:
            assert (got.pop("dq") == 0).all() and (got.pop("dk") == 0).all()
        compare(f"scale {scale}", got, varlen(q, k, v, do, table, starts(lens), 30, 3, scale=scale), F16)


def test_fp16_gradients_of_small_and_large_do():
    lens, D = [300, 90], 128
    q, k, v, do = inputs(390, 8, 2, D, F16, seed=5)
    table = seq_ref.Table(300, D, DEV)
    for size in (1e-4, 1.0, 3e3):
        g = (do.float() * size).to(F16)
        for window, sinks in ((30, 2), (150, 0)):
            ref = varlen(q, k, v, g, table, starts(lens), window, sinks)
            got = grads(q, k, v, g, table, starts(lens), window=window, sinks=sinks)
            for n in ("dq", "dk", "dv"):
                # what fp16 cannot hold is rounded to steps of 2^-24, or not finite
                inside = ref[n].abs() < 65504 * (1 - 6 * 2.0 ** -11)
                off = ((got[n].double().cpu() - ref[n]) * inside).norm() / (ref[n] * inside).norm()
                steps = 2.0 ** -25 * math.sqrt(ref[n].numel()) / float(ref[n].norm())
                assert off <= seq_ref.ROUNDINGS[n] * 2.0 ** -11 + steps, (n, size, window)


def test_starts_out_of_range_stay_inside():
    q, k, v, do = inputs(200, 2, 1, 64, BF16)
    table = seq_ref.Table(200, 64, DEV)
    want = grads(q, k, v, do, table, starts([60, 140]), window=20, sinks=2)
    got = grads(q, k, v, do, table, ints([-5, 60, 1 << 30]), window=20, sinks=2)
    assert all(torch.equal(got[n], want[n]) for n in want)
    for cu in ([0, 150, 20, 180], [190, 100, 90, 0], [3, 3, 300, -1]):   # no values are defined
        grads(q, k, v, do, table, ints(cu), window=20, sinks=70)
    torch.cuda.synchronize()


def test_repeats_are_equal_bit_for_bit():
    q, k, v, do = inputs(1300, 8, 2, 128, BF16, views=True)
    table = seq_ref.Table(1200, 128, DEV)
    first = grads(q, k, v, do, table, starts([1200, 100]), window=100, sinks=4)
    for _ in range(3):
        again = grads(q, k, v, do, table, starts([1200, 100]), window=100, sinks=4)
        assert all(torch.equal(first[n], again[n]) for n in first)


def test_captured_and_replayed_with_other_lengths():
    T, D, kw = 600, 64, dict(window=70, sinks=3)
    q, k, v, do = inputs(T, 4, 2, D, BF16)
    table, cu = seq_ref.Table(T, D, DEV), starts([100, 150, 20])
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    gdo = do.clone()

    def step():
        o = sdpa_rope_varlen(*leaves, table, cu, **kw)
        return (o.detach(), *torch.autograd.grad(o, leaves, gdo))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed, lens in enumerate(([100, 150, 20], [0, 600, 0], [1, 1, 1], [130, 0, 470])):
        x = inputs(T, 4, 2, D, BF16, seed=seed + 20)
        with torch.no_grad():
            for dst, src in zip((*leaves, gdo), x):
                dst.copy_(src)
            cu.copy_(starts(lens))
        graph.replay()
        torch.cuda.synchronize()
        want = grads(*x, table, starts(lens), **kw)
        for g, (n, w) in zip(out, want.items()):
            assert torch.equal(g, w), (n, lens)


def test_two_streams_at_once():
    q, k, v, do = inputs(500, 4, 2, 64, BF16)
    table, cu = seq_ref.Table(300, 64, DEV), starts([300, 200])
    want = grads(q, k, v, do, table, cu, window=40, sinks=4)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(grads(q, k, v, do, table, cu, window=40, sinks=4))
    torch.cuda.synchronize()
    assert all(torch.equal(g[n], want[n]) for g in got for n in want)


def test_autocast_compile_and_opcheck():
    lens, D, kw = [90, 40], 64, dict(window=33, sinks=1)
    q, k, v, do = inputs(130, 2, 1, D, F32)
    table = CosSinTable(100.0, 10, D, device=DEV)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    with torch.autocast("cuda", torch.bfloat16):
        o = sdpa_rope_varlen(*leaves, table, starts(lens), **kw)
    assert o.dtype == F32
    fn = torch.compile(lambda a, b, c, cu: sdpa_rope_varlen(a, b, c, table, cu, **kw) * 2, fullgraph=True, backend="aot_eager")
    o = fn(*leaves, starts(lens))
    g = torch.autograd.grad(o, leaves, do)
    want = grads(q, k, v, do * 2, table, starts(lens), **kw)
    assert torch.equal(o, want["o"] * 2) and all(torch.equal(a, want[n]) for a, n in zip(g, ("dq", "dk", "dv")))
    args = (*leaves, *seq_ref.Table(40, 64, DEV).tables(), starts([13, 20]), None, True, 0.125, 7, 2)
    torch.library.opcheck(torch.ops.farope.seq_window_fwd.default, args)


def test_second_derivative_refused():
    q, k, v, do = inputs(20, 1, 1, 64, F32)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = sdpa_rope_varlen(*leaves, seq_ref.Table(20, 64, DEV), starts([20]), window=5)
    g = torch.autograd.grad(o, leaves, do, create_graph=True)
    with pytest.raises(RuntimeError, match="no autograd formula"):
        g[0].sum().backward()


# ---------------------------------------------------------------------------
# over a cache
# ---------------------------------------------------------------------------
def page_table(B, per, extra=2, seed=0):
    n = B * per + extra
    order = torch.randperm(n, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    return order[: B * per].reshape(B, per).to(DEV), n


def decode_ref(q, kc, vc, table, pages, lengths, window, sinks, positions=None):
    q, kc, vc, pages = (x.detach().cpu() for x in (q, kc, vc, pages))
    B, H, D = q.shape
    group, rows = H // kc.shape[2], kc.shape[1]
    o, size = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for b in range(B):
        n = max(0, min(int(lengths[b]), pages.shape[1] * rows))
        at = [i for i in range(n) if (i >= n - window or i < sinks) and 0 <= int(pages[b, i // rows]) < kc.shape[0]]
        if not at:
            continue
        gi, ri = (torch.tensor(x) for x in zip(*((int(pages[b, i // rows]), i % rows) for i in at)))
        k, v = kc[gi, ri].double(), vc[gi, ri].double()
        index = torch.tensor([n - 2]) if positions is None else positions[b:b + 1].long().cpu()
        qh = seq_ref.rotate(q[b:b + 1].double(), table, index)[0]
        for h in range(H):
            p = torch.softmax(k[:, h // group] @ qh[h] / math.sqrt(D), dim=0)
            o[b, h], size[b, h] = p @ v[:, h // group], p @ v[:, h // group].abs()
    return o, size


def run_decode(tag, q, kc, vc, table, pages, lengths, window, sinks, **kw):
    got = sdpa_rope_decode(q, kc, vc, table, pages, ints(lengths), window=window, sinks=sinks, **kw)
    ref, size = decode_ref(q, kc, vc, table, pages, lengths, window, sinks, **kw)
    u = seq_ref.U[q.dtype]
    allowed = u * ref.norm(dim=-1) + (32 * u if q.dtype == F32 else 3 * u * u + 32 * 2.0 ** -24) * size.norm(dim=-1)
    assert torch.isfinite(got).all()
    off = (got.double().cpu() - ref).norm(dim=-1)
    assert (off <= allowed).all(), f"{float((off / allowed.clamp(min=1e-300)).max()):.2f} of what is allowed"
    LINES.append(f"[window decode {tag}] rel {seq_ref.rel(got, ref):.2e}")
    return got


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (31, 4), (32, 0), (64, 33), (100, 4), (700, 70)])
@pytest.mark.parametrize("dtype,D,H,Hkv,page,lens", [
    (BF16, 64, 4, 4, 16, [1, 0, 2, 31, 32, 33, 900]),
    (BF16, 128, 16, 4, 64, [500, 1, 0, 2097]),
    (BF16, 128, 24, 1, 7, [129, 300]),
    (BF16, 32, 6, 2, 1, [40, 129]),
    (F16, 64, 8, 1, 256, [1000, 255, 256, 257]),
    (F16, 256, 2, 2, 16, [417]),
    (F32, 64, 8, 2, 16, [700, 0, 50]),
    (F32, 256, 2, 1, 64, [130, 1]),
])
def test_decode(dtype, D, H, Hkv, page, lens, window, sinks):
    B = len(lens)
    for per in (-(-max(lens) // page) + 1, -(-3000 // page)):   # a worker a sequence, and shares of all of them
        pages, n = page_table(B, per)
        kc, vc = (randn(n, page, Hkv, D, dtype=dtype, seed=s) for s in (1, 2))
        q = randn(B, H, D, dtype=dtype, seed=3)
        run_decode(f"{dtype} D{D} {lens} {window} {sinks}", q, kc, vc, seq_ref.Table(max(lens) + 1, D, DEV), pages, lens, window, sinks)


def test_decode_of_a_long_window():
    """Windows that several workers share, sinks far before them, most sequences short."""
    page, D = 16, 64
    lens = [9000, 0, 5, 4100, 100, 4097]
    pages, n = page_table(6, 600)
    kc, vc = (randn(n, page, 2, D, dtype=BF16, seed=s) for s in (1, 2))
    q, table = randn(6, 4, D, dtype=BF16, seed=3), seq_ref.Table(9000, D, DEV)
    for window, sinks in ((4096, 4), (4096, 0), (2500, 200), (8990, 5)):
        run_decode(f"long {window} {sinks}", q, kc, vc, table, pages, lens, window, sinks)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_decode_reads_nothing_between_sinks_and_window(dtype):
    """NaN and infinity in every row that does not count, pages there given back: the same values."""
    lens, page, D, window, sinks = [345, 1, 0, 700], 20, 64, 50, 7
    pages, n = page_table(4, 40)
    kc, vc = (randn(n, page, 2, D, dtype=dtype, seed=s) for s in (1, 2))
    q, table = randn(4, 4, D, dtype=dtype, seed=3), seq_ref.Table(700, D, DEV)
    want = run_decode("clean", q, kc, vc, table, pages, lens, window, sinks)
    used = torch.zeros(n, page, dtype=torch.bool)
    for b, m in enumerate(lens):
        for i in range(m):
            if i >= m - window or i < sinks:
                used[pages[b, i // page].item(), i % page] = True
    kc[~used.to(DEV)], vc[~used.to(DEV)] = float("nan"), float("inf")
    assert torch.equal(sdpa_rope_decode(q, kc, vc, table, pages, ints(lens), window=window, sinks=sinks), want)
    gone = ~used.any(1)
    pages = torch.where(gone.to(DEV)[pages.long()], -1, pages)
    assert torch.equal(sdpa_rope_decode(q, kc, vc, table, pages, ints(lens), window=window, sinks=sinks), want)


def test_decode_windows_that_hold_everything():
    pages, n = page_table(3, 40)
    kc, vc = (randn(n, 16, 2, 64, dtype=BF16, seed=s) for s in (1, 2))
    q, table, lens = randn(3, 4, 64, dtype=BF16, seed=3), seq_ref.Table(640, 64, DEV), ints([640, 3, 100])
    want = sdpa_rope_decode(q, kc, vc, table, pages, lens)
    for window in (640, 2 ** 31 - 1):
        assert torch.equal(sdpa_rope_decode(q, kc, vc, table, pages, lens, window=window, sinks=2 ** 31 - 1), want)
    got = sdpa_rope_decode(q, kc, vc, table, pages, lens, window=639, sinks=2 ** 31 - 1)
    assert seq_ref.rel(got, want.double().cpu()) <= 2 * 2.0 ** -8


def test_decode_bad_lengths_and_positions():
    pages, n = page_table(4, 40)
    kc, vc = (randn(n, 16, 2, 64, dtype=F16, seed=s) for s in (1, 2))
    q, table = randn(4, 4, 64, dtype=F16, seed=3), seq_ref.Table(300, 64, DEV)
    pages[0, 30:] = -1
    run_decode("positions", q, kc, vc, table, pages, [500, -7, 2 ** 31 - 1, 30], 40, 3, positions=ints([3, 4, -1, 999]))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_prompt_then_tokens(dtype):
    """Every step's output is the row that windowed attention over the whole sequences gives."""
    H, Hkv, D, page, window, sinks = 8, 2, 64, 16, 24, 3
    prompt, steps = [20, 1, 33], 12
    lens = [n + steps for n in prompt]
    T = sum(lens)
    q, k, v = (randn(T, h, D, dtype=dtype, seed=s) for h, s in ((H, 7), (Hkv, 8), (Hkv, 9)))
    table, start = seq_ref.Table(max(lens), D, DEV), [sum(lens[:i]) for i in range(3)]
    ref = varlen(q, k, v, q, table, [*start, T], window, sinks)["o"]
    whole = sdpa_rope_varlen(q, k, v, table, ints([*start, T]), window=window, sinks=sinks)
    pages, n = page_table(3, 40)
    kc, vc = (torch.full((n, page, Hkv, D), float("nan"), dtype=dtype, device=DEV) for _ in range(2))
    rows = torch.cat([torch.arange(s, s + m) for s, m in zip(start, prompt)])
    lengths = ints([0, 0, 0])
    rope_cache_append(k[rows], v[rows], table, kc, vc, pages, lengths, cu_seqlens=starts(prompt))
    lengths += ints(prompt)
    tol = 32 * seq_ref.U[F32] if dtype == F32 else 4 * seq_ref.U[dtype]
    for i in range(steps):
        at = torch.tensor([s + m + i for s, m in zip(start, prompt)])
        rope_cache_append(k[at], v[at], table, kc, vc, pages, lengths)
        lengths += 1
        got = sdpa_rope_decode(q[at], kc, vc, table, pages, lengths, window=window, sinks=sinks)
        assert seq_ref.rel(got, ref[at]) <= tol and seq_ref.rel(whole[at], ref[at]) <= tol


def test_decode_captured_and_replayed():
    page, D, B = 16, 64, 3
    pages, n = page_table(B, 60)
    table = seq_ref.Table(960, D, DEV)
    kc, vc = (randn(n, page, 2, D, dtype=BF16, seed=s) for s in (1, 2))
    q, lengths = randn(B, 8, D, dtype=BF16, seed=7), ints([0, 10, 900])

    def step():
        return sdpa_rope_decode(q, kc, vc, table, pages, lengths, window=300, sinks=5)

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
        q.copy_(randn(B, 8, D, dtype=BF16, seed=30 + i))
        lengths.copy_(ints([190 * i, 7 * i, 900 - 90 * i]))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step()), i


def test_decode_opcheck_and_gradients_refused():
    pages, n = page_table(2, 3)
    kc, vc = (randn(n, 16, 2, 64, dtype=BF16, seed=s) for s in (1, 2))
    q, table = randn(2, 4, 64, dtype=BF16, seed=3), seq_ref.Table(40, 64, DEV)
    torch.library.opcheck(torch.ops.farope.cache_attn_window.default, (q, kc, vc, *table.tables(), pages, ints([40, 3]), None, True, 0.125, 9, 2))
    with pytest.raises(RuntimeError, match="no autograd formula"):
        sdpa_rope_decode(q.requires_grad_(), kc, vc, table, pages, ints([40, 3]), window=9).sum().backward()


# ---------------------------------------------------------------------------
# sinks as many as tokens, ragged packs
# ---------------------------------------------------------------------------
def test_many_short_sequences_with_more_sinks_than_tokens():
    """Their key tiles all hold sinks; the backward takes what the forward does."""
    rng = random.Random(6)
    lens = [rng.choice([1, 20, 30, 40, 65]) for _ in range(300)]
    q, k, v, do = inputs(sum(lens), 8, 8, 32, BF16, seed=4)
    table = seq_ref.Table(65, 32, DEV)
    for window, sinks in ((8, 2 ** 31 - 1), (8, 20)):
        got = grads(q, k, v, do, table, starts(lens), window=window, sinks=sinks)
        compare(f"300 sequences, {sinks} sinks", got, varlen(q, k, v, do, table, starts(lens), window, sinks), BF16)


@pytest.mark.parametrize("lens,H,Hkv,window,sinks", [([3000, 2800], 2, 2, 100, 600), ([4000], 4, 1, 70, 3000), ([2500] + [50] * 40, 4, 2, 90, 3),
                                                     ([900] * 6, 16, 16, 64, 70)])
def test_many_sinks_and_ragged_packs(lens, H, Hkv, window, sinks):
    """Sinks over many key tiles, in few parts or undivided, and of one long sequence beside many short ones."""
    q, k, v, do = inputs(sum(lens), H, Hkv, 64, BF16, seed=9)
    table = seq_ref.Table(max(lens), 64, DEV)
    got = grads(q, k, v, do, table, starts(lens), window=window, sinks=sinks)
    compare(f"{len(lens)} up to {max(lens)}, {sinks} sinks", got, varlen(q, k, v, do, table, starts(lens), window, sinks), BF16)


@pytest.mark.parametrize("dtype,D,H,Hkv,lens", [(BF16, 64, 2, 1, [300, 200]), (BF16, 128, 4, 2, [700, 130]), (F16, 128, 4, 4, [700, 130]),
                                                (F16, 64, 4, 2, [1700, 30]), (BF16, 256, 2, 1, [500]), (F32, 64, 2, 1, [400, 33]),
                                                (BF16, 32, 16, 16, [1300, 600]), (F32, 128, 2, 2, [400]),
                                                # (key tiles with sinks that are not divided)
                                                (BF16, 128, 16, 16, [330] * 33), (F16, 64, 32, 32, [330] * 33)])
@pytest.mark.parametrize("what", ["dO", "Q"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_gradients_do_not_feel_rows_far_from_theirs(dtype, D, H, Hkv, lens, what, value):
    """dO or Q of a token that is not finite reach dK and dV of the keys that it sees, and none whose own queries all are more than
    126 tokens from it: not those in a tile with the sinks either."""
    window, sinks = 50, 2
    q, k, v, do = inputs(sum(lens), H, Hkv, D, dtype, seed=17)
    table, cu = seq_ref.Table(max(lens), D, DEV), starts(lens)
    clean = grads(q, k, v, do, table, cu, window=window, sinks=sinks)
    bad_q, bad_do = q.clone(), do.clone()
    sees, near = (torch.zeros(sum(lens), dtype=torch.bool) for _ in range(2))
    for a, n in zip(cu.tolist(), lens):
        i = n - 20
        (bad_q if what == "Q" else bad_do)[a + i] = value
        seen = visible(n, window, sinks)
        sees[a:a + n] = seen[i]
        near[a:a + n] = seen[max(0, i - 126):i + 127].any(0)
    got = grads(bad_q, k, v, bad_do, table, cu, window=window, sinks=sinks)
    sees, far = sees.to(DEV), ~near.to(DEV)
    assert far.sum() > 60
    for name in ("dk", "dv"):
        assert torch.isfinite(got[name][far]).all(), name
        units = seq_ref.FP32_UNITS if dtype == F32 else seq_ref.ROUNDINGS
        tol = 4 * units[name] * seq_ref.U[dtype]
        off = (got[name][far].double() - clean[name][far].double()).norm(dim=-1)
        size = clean[name][far].double().norm(dim=-1)
        assert (off <= tol * (size + clean[name].double().norm(dim=-1).square().mean().sqrt())).all(), name
        if value != value:
            assert not torch.isfinite(got[name][sees]).any(), name
    rest = torch.ones(sum(lens), dtype=torch.bool, device=DEV)
    for a, n in zip(cu.tolist(), lens):
        rest[a + n - 20] = False
    assert torch.isfinite(got["dq"][rest]).all()
