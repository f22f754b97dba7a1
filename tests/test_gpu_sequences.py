"""GPU: attention over packed sequences (sdpa_rope_varlen) against 64 bits."""
from __future__ import annotations

import pytest
import torch

from tests import seq_ref
from tests._report import LINES
from triton_fused_rope_flash_attn_amd import CosSinTable, sdpa_rope_varlen, sdpa_triton_fa_rope

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def starts(lens, device=DEV):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=device)


def inputs(T, H, Hkv, D, dtype, seed=0, views=False):
    g = torch.Generator().manual_seed(seed)
    if views:   # thirds of one projection's output
        q, k, v = torch.randn(T, H + 2 * Hkv, D, generator=g).to(dtype).to(DEV).split([H, Hkv, Hkv], dim=1)
    else:
        q, k, v = (torch.randn(T, n, D, generator=g).to(dtype).to(DEV) for n in (H, Hkv, Hkv))
    return q, k, v, torch.randn(T, H, D, generator=g).to(dtype).to(DEV)


def grads(q, k, v, do, table, cu, **kw):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = sdpa_rope_varlen(*leaves, table, cu, **kw)
    return dict(zip(("o", "dq", "dk", "dv"), (o.detach(), *torch.autograd.grad(o, leaves, do))))


def compare(tag, got, ref, dtype):
    worst = {n: seq_ref.check(n, got[n], ref, dtype) for n in got}
    LINES.append(f"[varlen {tag}] " + " ".join(f"{n} {e:.2e}" for n, e in worst.items()))


SHORT = [1, 0, 5, 0, 33]
EDGES = [63, 64, 1, 65, 127, 128, 129]
LONG = [197, 3, 577, 300]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,D,H,Hkv,lens,views", [
    (BF16, 64, 4, 4, [1], False),
    (BF16, 64, 6, 2, SHORT, True),
    (BF16, 64, 3, 1, EDGES, False),
    (BF16, 128, 4, 2, EDGES, True),
    (BF16, 128, 8, 2, LONG, True),
    (BF16, 32, 4, 1, EDGES, True),
    (BF16, 256, 2, 1, EDGES, False),
    (F16, 64, 12, 12, LONG, True),
    (F16, 128, 7, 1, SHORT, False),
    (F16, 32, 2, 2, LONG, False),
    (F16, 256, 3, 3, SHORT, True),
    (F32, 32, 2, 1, EDGES, False),
    (F32, 64, 4, 2, EDGES, True),
    (F32, 128, 2, 2, LONG, False),
    (F32, 256, 2, 1, SHORT, True),
])
def test_varlen(dtype, D, H, Hkv, lens, views, causal):
    T = sum(lens)
    q, k, v, do = inputs(T, H, Hkv, D, dtype, seed=D + H, views=views)
    table = seq_ref.Table(max(lens), D, DEV)
    ref = seq_ref.varlen(q, k, v, do, table, starts(lens), causal, True)
    got = grads(q, k, v, do, table, starts(lens), causal=causal)
    compare(f"{dtype} D{D} H{H}/{Hkv} {lens} causal={causal}", got, ref, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_tokens_behind_the_last_sequence_are_zeros(dtype):
    """... and what they hold, and what other sequences hold, reaches nothing."""
    lens, T, D = [70, 0, 130], 333, 64
    q, k, v, do = inputs(T, 4, 2, D, dtype)
    table = seq_ref.Table(130, D, DEV)
    ref = seq_ref.varlen(q[:200], k[:200], v[:200], do[:200], table, starts(lens), True, False)
    for t in (q, k, v, do):
        t[200:] = float("nan")
    got = grads(q, k, v, do, table, starts(lens), has_cls=False)
    for t in got.values():
        assert (t[200:] == 0).all()
    compare(f"behind the last {dtype}", {n: t[:200] for n, t in got.items()}, ref, dtype)
    for t in (q, k, v, do):
        t[:70] = float("inf")
    again = grads(q, k, v, do, table, starts(lens), has_cls=False)
    for n in got:
        assert torch.equal(got[n][70:], again[n][70:]), n


@pytest.mark.parametrize("dtype,D,H,Hkv,lens", [(BF16, 64, 2, 1, [100, 3]), (BF16, 64, 4, 4, [700, 130, 900]), (F16, 128, 4, 2, [90, 20]),
                                                (F16, 128, 16, 4, [4100, 300, 700, 64, 2000, 1500]), (BF16, 256, 2, 1, [300, 70]),
                                                (BF16, 32, 2, 2, [200]), (F32, 64, 2, 1, [140, 33]), (F32, 256, 1, 1, [70])])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_rows_do_not_feel_the_tokens_behind_them(dtype, D, H, Hkv, lens, value):
    """Causal: K and V of some tokens not finite; the rows before them have the values that they have
    without, the rows behind see them.  (V alone: channels that it does not touch stay as they are.)"""
    T = sum(lens)
    q, k, v, _ = inputs(T, H, Hkv, D, dtype, seed=17)
    table, cu = seq_ref.Table(max(lens), D, DEV), starts(lens)
    clean = sdpa_rope_varlen(q, k, v, table, cu)
    at = [(a, i) for a, n in zip(cu.tolist(), lens) for i in (n * 5 // 8,)]
    bad_v, bad_k = v.clone(), k.clone()
    for a, i in at:
        bad_v[a + i, :, 3] = value
        bad_k[a + i] = value
    behind = torch.zeros(T, dtype=torch.bool)
    for (a, i), n in zip(at, lens):
        behind[a + i:a + n] = True
    behind = behind.to(DEV)
    off = seq_ref.ROUNDINGS["o"] * seq_ref.U[dtype] if dtype != F32 else seq_ref.FP32_UNITS["o"] * seq_ref.U[dtype]
    for kk in (k, bad_k):
        got = sdpa_rope_varlen(q, kk, bad_v, table, cu)
        assert torch.isfinite(got[~behind]).all()
        # (such a row may be computed again in another order: two results, each within the bound)
        err, size = (got[~behind].double() - clean[~behind].double()).norm(dim=-1), clean[~behind].double().norm(dim=-1)
        assert (err <= 4 * off * (size + size.square().mean().sqrt())).all()
        if kk is k:
            assert not torch.isfinite(got[behind][..., 3]).any()
            rest = torch.arange(D, device=DEV) != 3
            assert torch.isfinite(got[..., rest]).all()
            assert (got[behind][..., 3].isnan() | (got[behind][..., 3] == value)).all()
        elif value != value:
            assert not torch.isfinite(got[behind]).any()


def test_a_tensor_of_nan():
    """V not a number from a token on: every row from it on, no row before it; nothing is searched for long."""
    T, D = 20000, 64
    q, k, v, _ = inputs(T, 2, 1, D, BF16, seed=23)
    v[5001:] = float("nan")
    o = sdpa_rope_varlen(q, k, v, seq_ref.Table(T, D, DEV), starts([T]))
    assert o[5001:].isnan().all() and torch.isfinite(o[:5001]).all()


def test_all_sequences_empty():
    q, k, v, do = inputs(9, 2, 2, 64, BF16)
    got = grads(q, k, v, do, seq_ref.Table(4, 64, DEV), starts([0, 0]))
    assert all((t == 0).all() for t in got.values())


@pytest.mark.parametrize("dtype,D,B,low,high", [(BF16, 32, 4300, 0, 3), (F32, 64, 70, 0, 20), (F16, 128, 256, 120, 150), (BF16, 128, 257, 120, 150)])
def test_many_sequences(dtype, D, B, low, high):
    """More sequences than a step of a wave's search covers, and more than the order by work takes."""
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(low, high + 1, (B,), generator=g).tolist()
    T = sum(lens) + 5
    q, k, v, do = inputs(T, 2, 1, D, dtype, seed=13)
    table = seq_ref.Table(200, D, DEV)
    cu = starts(lens)
    compare(f"{B} sequences {dtype} D{D}", grads(q, k, v, do, table, cu), seq_ref.varlen(q, k, v, do, table, cu, True, True), dtype)


@pytest.mark.parametrize("dtype,D,H,lens", [(F16, 32, 36, [4105]), (BF16, 64, 34, [4200]), (F16, 128, 64, [1500, 650]), (BF16, 256, 64, [700, 400])])
def test_tiles_of_128_rows(dtype, D, H, lens):
    """Calls large enough for the wider tiles; two of the heads against 64 bits."""
    q, k, v, do = inputs(sum(lens), H, H, D, dtype, seed=19)
    table, cu = seq_ref.Table(max(lens), D, DEV), starts(lens)
    got = grads(q, k, v, do, table, cu)
    heads = [1, H - 1]
    ref = seq_ref.varlen(*(t[:, heads] for t in (q, k, v, do)), table, cu, True, True)
    compare(f"128 rows {dtype} D{D}", {n: x[:, heads] for n, x in got.items()}, ref, dtype)


def test_rows_past_32_bits():
    """Q, O, dO and dQ of more than 2^31 elements: the last sequences against 64 bits."""
    H, Hkv, D, n = 256, 2, 128, 32
    T = (1 << 31) // (H * D) // n * n + 2 * n
    lens = [n] * (T // n - 1) + [n - 5]
    g = torch.Generator(device=DEV).manual_seed(1)
    q, k, v, do = (torch.randn(T, h, D, generator=g, device=DEV, dtype=BF16) for h in (H, Hkv, Hkv, H))
    table = seq_ref.Table(n, D, DEV)
    got = grads(q, k, v, do, table, starts(lens))
    a = T - 2 * n
    ref = seq_ref.varlen(*(t[a:] for t in (q, k, v, do)), table, starts(lens[-2:]), True, True)
    compare("past 32 bits", {m: got[m][a:] for m in got}, ref, BF16)
    assert (got["o"][T - 5:] == 0).all() and (got["dq"][T - 5:] == 0).all()


def test_no_tokens():
    q, k, v, do = inputs(0, 2, 2, 64, BF16)
    got = grads(q, k, v, do, seq_ref.Table(4, 64, DEV), starts([0]))
    assert all(t.numel() == 0 for t in got.values())


def _strided(kind, T, H, Hkv, D, dtype):
    q, k, v, do = inputs(T, H, Hkv, D, dtype, seed=3)
    if kind == "heads first":
        return [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v, do)]
    if kind == "channels apart":
        return [torch.stack([t, t], dim=-1)[..., 1] for t in (q, k, v, do)]
    if kind == "odd offset":   # rows not 16-byte aligned
        flat = [torch.cat([t.new_zeros(1), t.reshape(-1)]) for t in (q, k, v, do)]
        return [f[1:].view(t.shape) for f, t in zip(flat, (q, k, v, do))]
    if kind == "one row":   # every token has the same k, v and dO row
        return [q, *(t[:1].expand(T, -1, -1) for t in (k, v, do))]
    if kind == "one head":
        return [q[:, :1].expand(-1, H, -1), k[:, :1].expand(-1, Hkv, -1), v[:, :1].expand(-1, Hkv, -1), do[:, :1].expand(-1, H, -1)]
    raise AssertionError(kind)


@pytest.mark.parametrize("dtype,D", [(BF16, 64), (F16, 128), (F32, 64)])
@pytest.mark.parametrize("kind", ["heads first", "channels apart", "odd offset", "one row", "one head"])
def test_strides(kind, dtype, D):
    lens = [130, 1, 77]
    q, k, v, do = _strided(kind, sum(lens), 4, 2, D, dtype)
    table = seq_ref.Table(130, D, DEV)
    ref = seq_ref.varlen(q, k, v, do, table, starts(lens), True, True)
    got = grads(q, k, v, do, table, starts(lens))
    names = got if kind != "one row" else ("o", "dv")   # (equal keys: P's rows are exact, dQ and dK cancel to rounding)
    compare(f"{kind} {dtype}", {n: got[n] for n in names}, ref, dtype)


def test_gradient_of_a_sum():
    """dO of o.sum(): one value expanded over the tensor."""
    lens, D = [100, 61], 64
    q, k, v, _ = inputs(161, 4, 2, D, BF16)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    table = seq_ref.Table(100, D, DEV)
    sdpa_rope_varlen(*leaves, table, starts(lens)).sum().backward()
    ref = seq_ref.varlen(q, k, v, torch.ones_like(q), table, starts(lens), True, True)
    compare("sum", dict(dq=leaves[0].grad, dk=leaves[1].grad, dv=leaves[2].grad), ref, BF16)


def test_positions_and_a_short_table():
    lens, D = [50, 20], 64
    q, k, v, do = inputs(70, 2, 1, D, F16)
    table = seq_ref.Table(31, D, DEV)
    pos = torch.randint(-2, 40, (70,), generator=torch.Generator().manual_seed(1), dtype=torch.int32).to(DEV)
    ref = seq_ref.varlen(q, k, v, do, table, starts(lens), True, True, positions=pos)
    compare("positions", grads(q, k, v, do, table, starts(lens), positions=pos), ref, F16)
    ref = seq_ref.varlen(q, k, v, do, table, starts(lens), True, False)   # (rows 31 .. 49 take row 30)
    compare("short table", grads(q, k, v, do, table, starts(lens), has_cls=False), ref, F16)


@pytest.mark.parametrize("value", [3e4, -3e4])
def test_large_logits(value):
    """One key that takes every later row's whole softmax, and one that none looks at."""
    lens, D = [140], 64
    q, k, v, do = inputs(140, 2, 2, D, F32)
    q[:, :, 0] = 8.0
    k[3, :, 0] = value
    table = seq_ref.Table(1, D, DEV)   # (row 0 turns by nothing)
    ref = seq_ref.varlen(q, k, v, do, table, starts(lens), True, True)
    got = grads(q, k, v, do, table, starts(lens))
    # The backward takes P = exp2(s - LSE) with both at 4.3e4 (log2 units), where half a step of fp32
    # is 2^-9: K's scaling, the product, its sum, LSE's two terms, its two conversions and the
    # difference are 8 roundings, of 2^-9 ln 2 of P each.
    assert seq_ref.rel(got["o"], ref["o"]) <= 32 * 2.0 ** -24
    assert seq_ref.rel(got["dv"], ref["dv"]) <= 8 * 2.0 ** -9 * 0.6932
    assert all(torch.isfinite(t).all() for t in got.values())


def test_equals_the_dense_op():
    """Not causal, equal lengths, one key head per query head: the dense op's values."""
    B, H, side, D = 3, 4, 9, 64
    N = side * side + 1
    table = CosSinTable(100.0, side, D, device=DEV)
    q, k, v, do = inputs(B * N, H, H, D, BF16)
    dense = [t.view(B, N, H, D).transpose(1, 2).detach().requires_grad_() for t in (q, k, v)]
    o = sdpa_triton_fa_rope(*dense, table)
    want = [o.detach(), *torch.autograd.grad(o, dense, do.view(B, N, H, D).transpose(1, 2))]
    got = grads(q, k, v, do, table, starts([N] * B), causal=False)
    for (n, t), w in zip(got.items(), want):   # (each within its bound of the exact value)
        w = w.transpose(1, 2).reshape(t.shape)
        assert seq_ref.rel(t, w.double().cpu()) <= 2 * seq_ref.ROUNDINGS[n] * seq_ref.U[BF16], n


def test_autocast():
    lens, D = [90, 40], 64
    q, k, v, do = inputs(130, 2, 1, D, F32)
    table = seq_ref.Table(90, D, DEV)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    with torch.autocast("cuda", torch.bfloat16):
        o = sdpa_rope_varlen(*leaves, table, starts(lens))
    assert o.dtype == F32
    g = torch.autograd.grad(o, leaves, do)
    assert all(x.dtype == F32 for x in g)
    # (the casts of q, k, v and dO are roundings too)
    ref = seq_ref.varlen(*(t.detach().bfloat16() for t in (q, k, v)), do.bfloat16(), table, starts(lens), True, True)
    compare("autocast", dict(zip(("o", "dq", "dk", "dv"), (o, *g))), ref, BF16)


@pytest.mark.parametrize("dtype,D,causal", [(BF16, 64, True), (F16, 128, False), (BF16, 256, True)])
def test_short_rows_do_not_feel_the_rounding_of_o(dtype, D, causal):
    """V with a common offset: dP - delta cancels it, where delta does not come from O as stored
    (u |dO| |O| = 64 u sqrt(D) here, dS of unit scale: several times dQ itself)."""
    lens = [2, 17, 32, 1]
    q, k, v, do = inputs(sum(lens), 4, 2, D, dtype)
    v = (v.float() + 64.0).to(dtype)
    table = seq_ref.Table(64, D, DEV)
    ref = seq_ref.varlen(q, k, v, do, table, starts(lens), causal, True)
    got = grads(q, k, v, do, table, starts(lens), causal=causal)
    # dP's terms are 64 times dS's scale: sqrt(D) 64 units of 2^-24 of it
    tol = seq_ref.ROUNDINGS["dq"] * seq_ref.U[dtype] + 64 * 64 * 2.0 ** -24
    for n in ("dq", "dk"):
        assert seq_ref.rel(got[n], ref[n]) <= tol, n


@pytest.mark.parametrize("scale", [0.0, -0.05, 0.25])
@pytest.mark.parametrize("dtype,lens", [(F16, [40, 9]), (BF16, [300, 70]), (F32, [100, 3])])
def test_softmax_scale_of_the_op(dtype, lens, scale):
    """The op takes any scale; at 0 every key weighs the same and dQ and dK are zeros."""
    T, D = sum(lens), 64
    q, k, v, do = inputs(T, 4, 2, D, dtype, seed=9)
    table = seq_ref.Table(300, D, DEV)
    ref = seq_ref.varlen(q, k, v, do, table, starts(lens), True, True, scale=scale)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o, _ = torch.ops.farope.seq_fwd(*leaves, *table.tables(), starts(lens), None, True, True, scale)
    got = dict(zip(("o", "dq", "dk", "dv"), (o.detach(), *torch.autograd.grad(o, leaves, do))))
    if scale == 0:
        assert (got.pop("dq") == 0).all() and (got.pop("dk") == 0).all()
    compare(f"scale {scale} {dtype}", got, ref, dtype)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,D,lens", [(BF16, 64, [1, 40, 1]), (F16, 128, [1, 1, 3]), (F16, 128, [300, 1, 700]), (BF16, 256, [1, 65]),
                                          (F32, 32, [1, 1]), (F32, 64, [200, 1]), (BF16, 32, [1000, 1, 500])])
def test_rows_that_see_one_key(dtype, D, lens, causal):
    """P = 1 whatever the logit: dQ of the row is zero, and dK of a key that no other row sees."""
    T = sum(lens)
    q, k, v, do = inputs(T, 4, 2, D, dtype, seed=11)
    table = seq_ref.Table(1000, D, DEV)
    got = grads(q, k, v, do, table, starts(lens), causal=causal)
    names = ("o", "dv") if max(lens) == 1 else tuple(got)   # (dQ and dK are zeros then)
    ref = seq_ref.varlen(q, k, v, do, table, starts(lens), causal, True)
    compare(f"one key {dtype} D{D} {lens}", {n: got[n] for n in names}, ref, dtype)
    for a, n in zip(starts(lens, "cpu").tolist(), lens):
        if causal or n == 1:
            assert (got["dq"][a] == 0).all()
        if n == 1:
            assert (got["dk"][a] == 0).all()
            assert torch.equal(got["o"][a], v[a].repeat_interleave(2, dim=0))


def test_gradient_against_differences():
    """Central differences of the fp32 forward along random directions."""
    lens, D, eps = [40, 25], 32, 1e-2
    q, k, v, do = inputs(65, 4, 2, D, F32)
    table = seq_ref.Table(40, D, DEV)
    got = grads(q, k, v, do, table, starts(lens))
    g = torch.Generator().manual_seed(5)
    for i, name in enumerate(("dq", "dk", "dv")):
        x = [q, k, v]
        d = torch.randn(x[i].shape, generator=g).to(DEV)
        up, down = ([t + s * eps * d if j == i else t for j, t in enumerate(x)] for s in (1, -1))
        f = [(sdpa_rope_varlen(*y, table, starts(lens)).double() * do.double()).sum().item() for y in (up, down)]
        slope, want = (f[0] - f[1]) / (2 * eps), (got[name].double() * d.double()).sum().item()
        # third derivatives of order 1 per term: eps^2 of the gradient's norm times the direction's
        scale = got[name].double().norm().item() * d.double().norm().item()
        assert abs(slope - want) <= 4 * eps ** 2 * scale + 1e-5 * scale, (name, slope, want)


def test_repeats_are_equal_bit_for_bit():
    lens, D = [257, 64, 100], 128
    q, k, v, do = inputs(421, 8, 2, D, BF16, views=True)
    table = seq_ref.Table(257, D, DEV)
    first = grads(q, k, v, do, table, starts(lens))
    for _ in range(3):
        again = grads(q, k, v, do, table, starts(lens))
        assert all(torch.equal(first[n], again[n]) for n in first)


def test_captured_and_replayed_with_other_lengths():
    """One graph of forward and gradients; inputs and sequence starts change between replays."""
    T, D = 300, 64
    q, k, v, do = inputs(T, 4, 2, D, BF16)
    table = seq_ref.Table(T, D, DEV)
    cu = starts([100, 150, 20])
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    gdo = do.clone()

    def step():
        o = sdpa_rope_varlen(*leaves, table, cu)
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
    for seed, lens in enumerate(([100, 150, 20], [0, 300, 0], [1, 1, 1], [130, 0, 170])):
        x = inputs(T, 4, 2, D, BF16, seed=seed + 20)
        with torch.no_grad():
            for dst, src in zip((*leaves, gdo), x):
                dst.copy_(src)
            cu.copy_(starts(lens))
        graph.replay()
        torch.cuda.synchronize()
        want = grads(*x, table, starts(lens))
        for g, (n, w) in zip(out, want.items()):
            assert torch.equal(g, w), (n, lens)


def test_two_streams_at_once():
    q, k, v, do = inputs(500, 4, 2, 64, BF16)
    table = seq_ref.Table(300, 64, DEV)
    cu = starts([300, 200])
    want = grads(q, k, v, do, table, cu)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(grads(q, k, v, do, table, cu))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(g[n], want[n]) for n in want)


def test_starts_out_of_range_stay_inside():
    """Values of cu_seqlens are clamped to the tensors: no error, nothing outside is touched."""
    q, k, v, do = inputs(100, 2, 1, 64, BF16)
    table = seq_ref.Table(100, 64, DEV)
    want = grads(q, k, v, do, table, starts([60, 40]))
    cu = torch.tensor([-5, 60, 1 << 30], dtype=torch.int32, device=DEV)
    got = grads(q, k, v, do, table, cu)
    assert all(torch.equal(got[n], want[n]) for n in want)


def test_compiles_fullgraph():
    lens, D = [90, 40], 64
    q, k, v, do = inputs(130, 2, 1, D, BF16)
    table = CosSinTable(100.0, 10, D, device=DEV)
    fn = torch.compile(lambda a, b, c, cu: sdpa_rope_varlen(a, b, c, table, cu) * 2, fullgraph=True, backend="aot_eager")
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = fn(*leaves, starts(lens))
    g = torch.autograd.grad(o, leaves, do)
    want = grads(q, k, v, do * 2, table, starts(lens))
    assert torch.equal(o, want["o"] * 2)
    assert all(torch.equal(a, want[n]) for a, n in zip(g, ("dq", "dk", "dv")))


def test_op_passes_opcheck():
    q, k, v, _ = inputs(40, 2, 1, 64, F16)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    torch.library.opcheck(torch.ops.farope.seq_fwd.default,
                          (*leaves, *seq_ref.Table(40, 64, DEV).tables(), starts([13, 20]), None, True, True, 0.125))


def test_second_derivative_refused():
    q, k, v, do = inputs(20, 1, 1, 64, F32)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = sdpa_rope_varlen(*leaves, seq_ref.Table(20, 64, DEV), starts([20]))
    (dq,) = torch.autograd.grad(o, leaves[:1], do, create_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable again"):
        dq.sum().backward()


@pytest.mark.parametrize("D,H,Hkv,lens", [
    (128, 2, 1, [4096]), (128, 64, 64, [1500, 650]), (64, 2, 1, [2048, 1000]), (64, 34, 34, [4200]), (32, 36, 36, [4105]),
    (256, 2, 1, [1500]), (256, 64, 64, [700, 400]), (64, 4, 4, [100, 60, 1, 30]), (32, 4, 2, [30, 2, 17]), (128, 2, 2, [90, 20]),
])
@pytest.mark.parametrize("sizes", ["dO of 1e-4", "dO of 2e-5", "rows of dO apart", "large dO and V"])
def test_fp16_gradients_over_its_range(D, H, Hkv, lens, sizes):
    """dS = P (dP - delta) reaches the products with its eleven bits where P or dO is small, and does not
    overflow where dO V is large.  The results as stored: half a step, 2^-25, of fp16's subnormals each."""
    T, g = sum(lens), torch.Generator().manual_seed(27)
    q, k, v, do = (t.float() for t in inputs(T, H, Hkv, D, F32, seed=29))
    if sizes == "large dO and V":
        q, k, v, do = 0.05 * q, 0.05 * k, 32 * v, 500 * do
    elif sizes == "rows of dO apart":
        do = do * (10.0 ** (6 * torch.rand(T, 1, 1, generator=g) - 4)).to(DEV)
    else:
        do = do * float(sizes[6:])
    q, k, v, do = (t.to(F16) for t in (q, k, v, do))
    table, cu = seq_ref.Table(max(lens), D, DEV), starts(lens)
    got = grads(q, k, v, do, table, cu)
    if H > 4:
        heads = [H - 1]
        got, (q, k, v, do) = {n: x[:, heads] for n, x in got.items()}, (t[:, heads] for t in (q, k, v, do))
    ref = seq_ref.varlen(q, k, v, do, table, cu, True, True)
    for n in ("dq", "dk", "dv"):
        off = (got[n].double().cpu() - ref[n]).norm(dim=-1)
        tol = seq_ref.ROUNDINGS[n] * seq_ref.U[F16]
        stored = 2.0 ** -25 * D ** 0.5   # of a row
        total = tol * ref[n].norm() + stored * off.numel() ** 0.5
        assert off.norm() <= total, (n, float(off.norm() / total))
        if n == "dq":   # each row by its own size
            allowed = 2 * tol * ref[n].norm(dim=-1) + stored + ref["dq+"]
            assert (off <= allowed).all(), (n, float((off / allowed).max()))


@pytest.mark.parametrize("dtype,D,H,short,long,causal", [
    (BF16, 128, 4, [40, 50, 64, 33], [], True), (BF16, 128, 4, [40, 50, 64, 33], [], False), (BF16, 256, 2, [40, 64], [], True),
    (BF16, 64, 4, [40, 50, 64, 33], [], True), (F32, 128, 2, [40, 64], [], True), (F32, 128, 2, [40, 60, 64, 1], [], False),
    (BF16, 128, 32, [2, 17, 32, 1, 33, 64], [1100] * 6, True), (F16, 128, 32, [2, 17, 32, 1, 33, 64], [1100] * 6, False),
    (BF16, 256, 32, [2, 17, 64], [900] * 3, True), (F16, 256, 32, [2, 17, 64], [900] * 3, False),
    (F16, 64, 16, [2, 64], [13000], True), (F32, 256, 1, [3, 40, 64], [400], True), (BF16, 32, 16, [2, 64], [13000], True),
])
def test_short_rows_whatever_their_neighbours(dtype, D, H, short, long, causal):
    """V with a common offset: the gradients of rows that see 64 keys at most do not feel the rounding of O, in
    packs of every tile size (as in the test of short rows above; causal: a long sequence's first rows too)."""
    lens = short + long
    q, k, v, do = inputs(sum(lens), H, 2 if H > 2 else 1, D, dtype, seed=31)
    v = (v.float() + 64.0).to(dtype)
    table, cu = seq_ref.Table(max(lens), D, DEV), starts(lens)
    got = grads(q, k, v, do, table, cu, causal=causal)
    n = sum(short)
    ref = seq_ref.varlen(*(t[:n] for t in (q, k, v, do)), table, starts(short), causal, True)
    tol = seq_ref.ROUNDINGS["dq"] * seq_ref.U[dtype] + 64 * 64 * 2.0 ** -24 if dtype != F32 else 64 * 64 * 2.0 ** -24
    for m in ("dq", "dk"):
        assert seq_ref.rel(got[m][:n], ref[m]) <= tol, m
    if long and causal:   # a first row of a long sequence depends on the rows before it alone
        a = n + 64
        ref = seq_ref.varlen(*(t[n:a] for t in (q, k, v, do)), table, starts([64]), True, True)
        assert seq_ref.rel(got["dq"][n:a], ref["dq"]) <= tol


@pytest.mark.parametrize("grad", [False, True], ids=["no_grad", "grad"])
@pytest.mark.parametrize("which", ["Q", "K", "V", "table"])
def test_tangents_are_refused(which, grad):
    """Forward mode: no derivative is implemented, and none is dropped."""
    from torch.autograd import forward_ad

    q, k, v, _ = inputs(20, 2, 1, 64, BF16)
    table = seq_ref.Table(20, 64, DEV)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        if which == "table":
            table.cos = dual(table.cos)
        x = [dual(t) if n == which else t for n, t in zip("QKV", (q, k, v))]
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            sdpa_rope_varlen(*x, table, starts([20]))
    sdpa_rope_varlen(q, k, v, seq_ref.Table(20, 64, DEV), starts([20]))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_many_small_weights(dtype):
    """One key that weighs 2^25 times each of the others, 2^17 - 1 of them: together they are 0.4% of the row.
    (Their weights are below the half of fp16's least value.)"""
    T, D = 1 << 17, 32
    q, k, v, do = (torch.zeros(T, 1, D, dtype=dtype, device=DEV) for _ in range(4))
    logit = 25.03125 * 0.693147   # log2 units; q k / sqrt(D), in values that both types hold
    q[..., 0] = 8.0
    k[0, 0, 0] = logit * D ** 0.5 / 8
    w = (T - 1) * torch.exp(-8.0 * k[0, 0, 0].double() / D ** 0.5).item()
    assert dtype == BF16 or w / (T - 1) < 2.0 ** -25
    v[:] = 1.0
    v[0] = -1.0
    do[:] = 0.25
    got = grads(q, k, v, do, seq_ref.Table(1, D, DEV), starts([T]), causal=False)
    u = seq_ref.U[dtype]
    off = (got["o"].double() - (w - 1) / (1 + w)).abs().max().item()
    # q-hat k-hat rounds as 25 * 2^-24 would (k-hat carries the scale: one rounding, u of the logit)
    assert off <= 4 * u + 2 * w * (25 * 0.7 * u), off
    each = 0.25 * T * (w / (T - 1)) / (1 + w)
    off = (got["dv"][1:].double() - each).abs().max().item()
    assert off <= (4 * u + 25 * 0.7 * u) * each + 2.0 ** -25, (off, each)
    assert all(torch.isfinite(x).all() for x in got.values())


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("dtype,D,H,Hkv", [(F16, 64, 2, 1), (F16, 128, 2, 1), (F16, 128, 48, 48), (F16, 256, 2, 2), (BF16, 128, 2, 1)])
def test_one_row_of_do_that_is_not_finite(dtype, D, H, Hkv, value):
    """Its own dQ row and the keys that it sees are not finite; the scale of the others' dS does not follow it."""
    T, i = 700, 300
    q, k, v, do = inputs(T, H, Hkv, D, dtype, seed=37)
    do[i] = 0.0
    table = seq_ref.Table(T, D, DEV)
    heads = [0, H - 1] if H == Hkv else list(range(H))
    keys = heads if H == Hkv else [0]
    ref = seq_ref.varlen(q[:, heads], k[:, keys], v[:, keys], do[:, heads], table, starts([T]), True, True)
    do[i] = value
    got = grads(q, k, v, do, table, starts([T]))
    assert not torch.isfinite(got["dq"][i]).any()
    assert not torch.isfinite(got["dk"][:i + 1]).any() and not torch.isfinite(got["dv"][:i + 1]).any()
    tol = {n: seq_ref.ROUNDINGS[n] * seq_ref.U[dtype] for n in ("dq", "dk", "dv")}
    rows = torch.arange(T) != i
    assert seq_ref.rel(got["dq"][:, heads][rows.to(DEV)], ref["dq"][rows]) <= tol["dq"]
    assert seq_ref.rel(got["dk"][i + 1:][:, keys], ref["dk"][i + 1:]) <= tol["dk"]
    assert seq_ref.rel(got["dv"][i + 64:][:, keys], ref["dv"][i + 64:]) <= tol["dv"]   # (0 times it, up to 63 tokens away)
