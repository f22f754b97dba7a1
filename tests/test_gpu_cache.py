"""GPU: appends to a paged cache and attention over it, against 64 bits."""
from __future__ import annotations

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


def randn(*shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def page_table(B, per, extra=2, seed=0):
    n = B * per + extra
    order = torch.randperm(n, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    return order[: B * per].reshape(B, per).to(DEV), n


def caches(n, page, Hkv, D, dtype, layout="rows"):
    if layout == "rows":
        return tuple(randn(n, page, Hkv, D, dtype=dtype, seed=s) for s in (1, 2))
    return tuple(randn(n, Hkv, page, D, dtype=dtype, seed=s).transpose(1, 2) for s in (1, 2))   # "heads"


def run_decode(tag, q, kc, vc, table, pages, lengths, has_cls=True, positions=None):
    got = sdpa_rope_decode(q, kc, vc, table, pages, lengths, has_cls=has_cls, positions=positions)
    ref, size = seq_ref.decode(q, kc, vc, table, pages, lengths, has_cls, positions)
    u = seq_ref.U[q.dtype]
    allowed = u * ref.norm(dim=-1) + (32 * u if q.dtype == F32 else 3 * u * u + 32 * 2.0 ** -24) * size.norm(dim=-1)
    assert torch.isfinite(got).all()
    off = (got.double().cpu() - ref).norm(dim=-1)
    assert (off <= allowed).all(), f"{float((off / allowed.clamp(min=1e-300)).max()):.2f} of what is allowed"
    LINES.append(f"[decode {tag}] rel {seq_ref.rel(got, ref):.2e}")
    return got


@pytest.mark.parametrize("layout", ["rows", "heads"])
@pytest.mark.parametrize("dtype,D,H,Hkv,page,lens", [
    (BF16, 64, 12, 12, 16, [197]),
    (BF16, 64, 4, 4, 16, [1, 0, 2, 31, 32, 33]),
    (BF16, 128, 16, 4, 64, [500, 1, 0, 4097]),
    (BF16, 128, 24, 1, 7, [129, 300]),            # more query heads per key head than one tile
    (BF16, 128, 34, 2, 32, [64, 65]),
    (BF16, 32, 6, 2, 1, [40, 129]),
    (BF16, 256, 4, 2, 100, [333, 5]),
    (F16, 64, 8, 1, 256, [1000, 255, 256, 257]),
    (F16, 128, 7, 1, 16, [2049]),
    (F16, 256, 2, 2, 16, [17]),
    (F32, 32, 4, 4, 16, [100, 3]),
    (F32, 64, 8, 2, 16, [700, 0, 50]),
    (F32, 128, 3, 3, 5, [258]),
    (F32, 256, 2, 1, 64, [130, 1]),
])
def test_decode(dtype, D, H, Hkv, page, lens, layout):
    B, per = len(lens), -(-max(lens) // page) + 1
    pages, n = page_table(B, per)
    kc, vc = caches(n, page, Hkv, D, dtype, layout)
    q = randn(B, H, D, dtype=dtype, seed=3)
    run_decode(f"{dtype} D{D} H{H}/{Hkv} page {page} {lens}", q, kc, vc, seq_ref.Table(max(lens) + 1, D, DEV), pages, ints(lens))


@pytest.mark.parametrize("B,Hkv", [(1, 1), (300, 4)])
def test_decode_in_many_parts_and_in_one(B, Hkv):
    lens = [(37 * i) % 700 for i in range(B)] if B > 1 else [20000]
    page, D = 32, 64
    pages, n = page_table(B, -(-max(lens) // page))
    kc, vc = caches(n, page, Hkv, D, BF16)
    run_decode(f"B{B}", randn(B, 2 * Hkv, D, dtype=BF16, seed=3), kc, vc, seq_ref.Table(30, D, DEV), pages, ints(lens), has_cls=False)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_decode_reads_nothing_but_the_sequence(dtype):
    """NaN and infinity in every cache row of no sequence; pages that end inside a block."""
    lens, page, D = [45, 1, 0, 70], 20, 64
    pages, n = page_table(4, 5)
    kc, vc = caches(n, page, 2, D, dtype)
    q = randn(4, 4, D, dtype=dtype, seed=3)
    table = seq_ref.Table(80, D, DEV)
    want = run_decode("clean", q, kc, vc, table, pages, ints(lens))
    used = torch.zeros(n, page, dtype=torch.bool)
    for b, m in enumerate(lens):
        for i in range(m):
            used[pages[b, i // page].item(), i % page] = True
    kc[~used.to(DEV)] = float("nan")
    vc[~used.to(DEV)] = float("inf")
    got = sdpa_rope_decode(q, kc, vc, table, pages, ints(lens))
    assert torch.equal(got, want)


def test_decode_bad_pages_and_lengths():
    """Rows on no page of the cache are left out; a length past the table's end, or below 0, is cut."""
    page, D = 16, 64
    pages, n = page_table(5, 4)
    kc, vc = caches(n, page, 2, D, BF16)
    pages[0, 1], pages[1, 0], pages[2] = -1, n, 1 << 30
    lens = [60, 40, 64, 1000, -7]
    got = run_decode("bad pages", randn(5, 2, D, dtype=BF16, seed=3), kc, vc, seq_ref.Table(64, D, DEV), pages, ints(lens))
    assert (got[2] == 0).all() and (got[4] == 0).all()


def test_decode_positions_and_strides():
    lens, page, D = [50, 9], 16, 64
    pages, n = page_table(2, 8)
    wide = pages.clone()
    pages = torch.cat([wide, wide], dim=1)[:, :4]            # rows of the page table apart
    kc, vc = caches(n, page, 3, D, F16)
    q = randn(2, D, 6, dtype=F16, seed=3).transpose(1, 2)    # channels apart
    run_decode("positions", q, kc, vc, seq_ref.Table(40, D, DEV), pages, ints(lens), positions=ints([12, -1]))
    run_decode("cut table", q, kc, vc, seq_ref.Table(10, D, DEV), pages, ints(lens), has_cls=False)


def test_decode_large_logits():
    lens, page, D = [300], 16, 64
    pages, n = page_table(1, 19)
    kc, vc = caches(n, page, 1, D, F32)
    q = randn(1, 2, D, dtype=F32, seed=3)
    q[..., 0] = 100.0
    kc[pages[0, 7].item(), 3, 0, 0] = 3e4
    got = sdpa_rope_decode(q, kc, vc, seq_ref.Table(1, D, DEV), pages, ints(lens))
    assert torch.allclose(got[0, 0], vc[pages[0, 7].item(), 3, 0], rtol=1e-5, atol=1e-6)


def test_decode_no_sequences():
    kc, vc = caches(3, 16, 1, 64, BF16)
    out = sdpa_rope_decode(randn(0, 2, 64, dtype=BF16, seed=0), kc, vc, seq_ref.Table(4, 64, DEV),
                           torch.zeros(0, 4, dtype=torch.int32, device=DEV), ints([]))
    assert out.shape == (0, 2, 64)


def _append_ref(k, v, table, kc, vc, pages, lengths, lens, has_cls, positions=None):
    """The caches after the append (64 bits) and how far each value may be off."""
    kc, vc, off = kc.double().cpu(), vc.double().cpu(), torch.zeros(kc.shape, dtype=torch.float64)
    page, at = kc.shape[1], 0
    for b, n in enumerate(lens):
        for j in range(n):
            t, pos = at + j, int(lengths[b]) + j
            if int(lengths[b]) < 0 or pos // page >= pages.shape[1]:
                continue
            g = int(pages[b, pos // page])
            if not 0 <= g < kc.shape[0]:
                continue
            index = torch.tensor([pos - int(has_cls)]) if positions is None else positions[t:t + 1].long().cpu()
            x = k[t:t + 1].double().cpu()
            kc[g, pos % page] = seq_ref.rotate(x, table, index)[0]
            vc[g, pos % page] = v[t].double().cpu()
            size = x[0, :, 0::2].abs() + x[0, :, 1::2].abs()
            # two products and a sum in fp32, then the rounding to the cache's type
            off[g, pos % page] = seq_ref.U[k.dtype] * kc[g, pos % page].abs() + 2.0 ** -22 * size.repeat_interleave(2, dim=-1)
        at += n
    return kc, vc, off


def run_append(k, v, table, kc, vc, pages, lengths, lens=None, **kw):
    want_k, want_v, off = _append_ref(k, v, table, kc, vc, pages, lengths, lens or [1] * len(lengths), kw.get("has_cls", True),
                                      kw.get("positions"))
    version = kc._version
    rope_cache_append(k, v, table, kc, vc, pages, lengths, **kw)
    assert kc._version > version
    assert ((kc.double().cpu() - want_k).abs() <= off).all()   # (rows that are not written: off = 0)
    assert torch.equal(vc.double().cpu(), want_v)


@pytest.mark.parametrize("layout", ["rows", "heads"])
@pytest.mark.parametrize("dtype,D,Hkv,page", [(BF16, 64, 12, 16), (BF16, 128, 1, 7), (F16, 32, 5, 1), (F16, 256, 2, 64),
                                              (F32, 64, 4, 16), (F32, 128, 9, 100)])
def test_append_one_token_each(dtype, D, Hkv, page, layout):
    lengths = [0, 5, 196, page, page - 1]
    pages, n = page_table(5, 197 // page + 1)
    kc, vc = caches(n, page, Hkv, D, dtype, layout)
    k, v = randn(5, 2, Hkv, D, dtype=dtype, seed=4).unbind(1)
    run_append(k, v, seq_ref.Table(200, D, DEV), kc, vc, pages, ints(lengths))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_append_prompts(dtype):
    """Prompts of different lengths behind what is there, empty ones, and tokens of no sequence."""
    lens, before, page, D = [33, 0, 1, 100], [0, 7, 50, 3], 16, 64
    pages, n = page_table(4, 8)
    kc, vc = caches(n, page, 3, D, dtype)
    k, v = (randn(140, 3, D, dtype=dtype, seed=s) for s in (4, 5))
    cu = ints([0, 33, 33, 34, 134])
    run_append(k, v, seq_ref.Table(60, D, DEV), kc, vc, pages, ints(before), lens, cu_seqlens=cu, has_cls=False)


def test_append_to_many_sequences():
    """More sequences than a step of a wave's search covers, many of them without a token."""
    page, D, B = 4, 32, 4300
    g = torch.Generator().manual_seed(2)
    lens, before = (torch.randint(0, 3, (B,), generator=g).tolist() for _ in range(2))
    pages, n = page_table(B, 1)
    kc, vc = caches(n, page, 1, D, BF16)
    k, v = (randn(sum(lens), 1, D, dtype=BF16, seed=s) for s in (4, 5))
    cu = ints([0, *torch.tensor(lens).cumsum(0).tolist()])
    run_append(k, v, seq_ref.Table(8, D, DEV), kc, vc, pages, ints(before), lens, cu_seqlens=cu)


@pytest.mark.parametrize("per", [4, 40])
def test_decode_of_many_sequences(per):
    """A thousand sequences, most of them short or empty: one worker each, and shares over all of them."""
    page, D, B = 16, 32, 1100
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 12, (B,), generator=g)
    lens[::97] = torch.randint(0, per * page + 1, (len(lens[::97]),), generator=g)
    pages, n = page_table(B, per)
    kc, vc = caches(n, page, 1, D, BF16)
    run_decode(f"{B} sequences", randn(B, 2, D, dtype=BF16, seed=3), kc, vc, seq_ref.Table(700, D, DEV), pages, ints(lens.tolist()))


def test_append_left_out():
    """Tokens past the page table, on no page of the cache, or of a negative length are not stored."""
    page, D = 16, 64
    pages, n = page_table(6, 2)
    pages[1, 0], pages[2, 1] = -1, n
    kc, vc = caches(n, page, 2, D, BF16)
    k, v = (randn(6, 2, D, dtype=BF16, seed=s) for s in (4, 5))
    run_append(k, v, seq_ref.Table(60, D, DEV), kc, vc, pages, ints([31, 3, 20, 32, -1, 2 ** 31 - 1]))


def test_append_positions_and_strides():
    page, D = 16, 64
    pages, n = page_table(3, 2)
    kc, vc = caches(n, page, 2, D, F16)
    k = randn(3, D, 2, dtype=F16, seed=4).transpose(1, 2)
    v = torch.cat([k.new_zeros(1), randn(3, 2, D, dtype=F16, seed=5).reshape(-1)])[1:].view(3, 2, D)   # rows not aligned
    run_append(k, v, seq_ref.Table(9, D, DEV), kc, vc, pages, ints([1, 2, 3]), positions=ints([-1, 4, 30]))


def test_append_no_tokens():
    kc, vc = caches(3, 16, 2, 64, BF16)
    want = kc.clone()
    none = randn(0, 2, 64, dtype=BF16, seed=0)
    rope_cache_append(none, none, seq_ref.Table(9, 64, DEV), kc, vc, torch.zeros(1, 2, dtype=torch.int32, device=DEV), ints([0]),
                      cu_seqlens=ints([0, 0]))
    assert torch.equal(kc, want)


def test_cache_past_32_bits():
    """A cache of more than 2^31 elements: its last page is written and read."""
    Hkv, D, page = 8, 128, 64
    n = (1 << 31) // (Hkv * D * page) + 3
    kc, vc = (torch.zeros(n, page, Hkv, D, dtype=BF16, device=DEV) for _ in range(2))
    pages = ints([[n - 1, 0, n - 2]])
    k, v = (randn(150, Hkv, D, dtype=BF16, seed=s) for s in (4, 5))
    table = seq_ref.Table(150, D, DEV)
    rope_cache_append(k, v, table, kc, vc, pages, ints([0]), cu_seqlens=ints([0, 150]))
    assert torch.equal(vc[n - 1], v[:64]) and torch.equal(vc[0], v[64:128]) and torch.equal(vc[n - 2, :22], v[128:])
    q = randn(1, Hkv, D, dtype=BF16, seed=6)
    small_k, small_v = (torch.stack([c[n - 1], c[0], c[n - 2]]) for c in (kc, vc))
    got = sdpa_rope_decode(q, kc, vc, table, pages, ints([150]))
    want = sdpa_rope_decode(q, small_k, small_v, table, ints([[0, 1, 2]]), ints([150]))
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_prompt_then_tokens(dtype):
    """Prompts enter the cache, then tokens one by one: every step's output is the row that
    attention over the whole sequences gives."""
    H, Hkv, D, page = 8, 2, 64, 16
    prompt, steps = [20, 1, 33], 5
    lens = [n + steps for n in prompt]
    T = sum(lens)
    q, k, v = (randn(T, h, D, dtype=dtype, seed=s) for h, s in ((H, 7), (Hkv, 8), (Hkv, 9)))
    table = seq_ref.Table(max(lens), D, DEV)
    start = [sum(lens[:i]) for i in range(len(lens))]
    ref = seq_ref.varlen(q, k, v, None, table, [*start, T], True, True)["o"]
    whole = sdpa_rope_varlen(q, k, v, table, ints([*start, T]))

    pages, n = page_table(3, -(-max(lens) // page))
    kc, vc = (torch.full((n, page, Hkv, D), float("nan"), dtype=dtype, device=DEV) for _ in range(2))
    rows = torch.cat([torch.arange(s, s + m) for s, m in zip(start, prompt)])
    cu = ints([0, *(sum(prompt[: i + 1]) for i in range(3))])
    lengths = ints([0, 0, 0])
    rope_cache_append(k[rows], v[rows], table, kc, vc, pages, lengths, cu_seqlens=cu)
    lengths += ints(prompt)
    tol = 32 * seq_ref.U[F32] if dtype == F32 else 4 * seq_ref.U[dtype]
    for i in range(steps):
        at = torch.tensor([s + m + i for s, m in zip(start, prompt)])
        rope_cache_append(k[at], v[at], table, kc, vc, pages, lengths)
        lengths += 1
        got = sdpa_rope_decode(q[at], kc, vc, table, pages, lengths)
        assert seq_ref.rel(got, ref[at]) <= tol and seq_ref.rel(whole[at], ref[at]) <= tol


def test_step_captured_and_replayed():
    """One graph of append and attention serves every later step: lengths grow on the device."""
    H, Hkv, D, page, B = 8, 2, 64, 16, 3
    pages, n = page_table(B, 4)
    table = seq_ref.Table(64, D, DEV)
    kc, vc = caches(n, page, Hkv, D, BF16)
    q, k, v = (randn(B, h, D, dtype=BF16, seed=s) for h, s in ((H, 7), (Hkv, 8), (Hkv, 9)))
    lengths = ints([0, 10, 40])

    def step():
        rope_cache_append(k, v, table, kc, vc, pages, lengths)
        lengths.add_(1)
        return sdpa_rope_decode(q, kc, vc, table, pages, lengths)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    lengths.copy_(ints([0, 10, 40]))
    ek, ev, el = kc.clone(), vc.clone(), lengths.clone()
    for i in range(12):
        q.copy_(randn(B, H, D, dtype=BF16, seed=30 + i))
        k.copy_(randn(B, Hkv, D, dtype=BF16, seed=60 + i))
        v.copy_(randn(B, Hkv, D, dtype=BF16, seed=90 + i))
        graph.replay()
        torch.cuda.synchronize()
        rope_cache_append(k, v, table, ek, ev, pages, el)
        el += 1
        assert torch.equal(out, sdpa_rope_decode(q, ek, ev, table, pages, el)), i
    assert torch.equal(kc, ek) and torch.equal(vc, ev)


@pytest.mark.parametrize("one", [False, True], ids=["two caches", "halves of one tensor"])
def test_step_compiles_fullgraph(one):
    H, Hkv, D, page, B = 4, 2, 64, 16, 3
    pages, n = page_table(B, 4)
    table = CosSinTable(100.0, 8, D, device=DEV)
    both = torch.stack(caches(n, page, Hkv, D, BF16))
    q, k, v = (randn(B, h, D, dtype=BF16, seed=s) for h, s in ((H, 7), (Hkv, 8), (Hkv, 9)))
    lengths = ints([0, 10, 40])

    def step(q, k, v, kc, vc, lengths):
        rope_cache_append(k, v, table, kc, vc, pages, lengths)
        return sdpa_rope_decode(q, kc, vc, table, pages, lengths + 1) * 2

    ek, ev = both[0].clone(), both[1].clone()
    want = step(q, k, v, ek, ev, lengths)
    kc, vc = (both[0], both[1]) if one else (both[0].clone(), both[1].clone())
    got = torch.compile(step, fullgraph=True, backend="aot_eager")(q, k, v, kc, vc, lengths)
    assert torch.equal(got, want) and torch.equal(kc, ek) and torch.equal(vc, ev)


def test_ops_pass_opcheck():
    page, D = 16, 64
    pages, n = page_table(2, 3)
    kc, vc = caches(n, page, 2, D, BF16)
    q, k, v = (randn(2, h, D, dtype=BF16, seed=s) for h, s in ((4, 7), (2, 8), (2, 9)))
    tables = seq_ref.Table(40, D, DEV).tables()
    torch.library.opcheck(torch.ops.farope.cache_append.default, (k, v, *tables, kc, vc, pages, ints([0, 20]), None, None, True))
    torch.library.opcheck(torch.ops.farope.cache_attn.default, (q, kc, vc, *tables, pages, ints([1, 21]), None, True, 0.125))


def test_pages_shared_by_sequences():
    """Sequences that share the pages of a common beginning, and one read twice."""
    page, D = 16, 64
    pages, n = page_table(4, 40)
    pages[1, :30] = pages[0, :30]
    pages[2] = pages[0]
    kc, vc = caches(n, page, 2, D, BF16)
    q = randn(4, 8, D, dtype=BF16, seed=3)
    run_decode("shared pages", q, kc, vc, seq_ref.Table(640, D, DEV), pages, ints([600, 500, 600, 640]))


def test_two_streams_at_once():
    lens, page, D = [500, 40, 700], 16, 128
    pages, n = page_table(3, 44)
    kc, vc = caches(n, page, 2, D, BF16)
    q = randn(3, 8, D, dtype=BF16, seed=3)
    table = seq_ref.Table(700, D, DEV)
    lengths = ints(lens)
    want = sdpa_rope_decode(q, kc, vc, table, pages, lengths)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(sdpa_rope_decode(q, kc, vc, table, pages, lengths))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_gradients_are_refused():
    kc, vc = caches(3, 16, 2, 64, BF16)
    pages, table = ints([[0, 1]]), seq_ref.Table(9, 64, DEV)
    k = randn(1, 2, 64, dtype=BF16, seed=1).requires_grad_()
    with pytest.raises(RuntimeError, match="not differentiable"):
        rope_cache_append(k, k, table, kc, vc, pages, ints([0]))
    with torch.no_grad():
        rope_cache_append(k, k, table, kc, vc, pages, ints([0]))
    o = sdpa_rope_decode(k, kc, vc, table, pages, ints([1]))
    with pytest.raises(RuntimeError, match="no gradients"):
        o.sum().backward()


@pytest.mark.parametrize("which", ["k", "v", "kc", "vc", "q"])
def test_tangents_are_refused(which):
    from torch.autograd import forward_ad

    kc, vc = caches(3, 16, 2, 64, BF16)
    pages, table = ints([[0, 1]]), seq_ref.Table(9, 64, DEV)
    q, k, v = (randn(1, h, 64, dtype=BF16, seed=h) for h in (4, 2, 2))
    with forward_ad.dual_level():
        a = dict(q=q, k=k, v=v, kc=kc, vc=vc)
        a[which] = forward_ad.make_dual(a[which], torch.ones_like(a[which]))
        calls = [lambda: rope_cache_append(a["k"], a["v"], table, a["kc"], a["vc"], pages, ints([0]))] if which != "q" else []
        calls += [lambda: sdpa_rope_decode(a["q"], a["kc"], a["vc"], table, pages, ints([1]))] if which in ("q", "kc", "vc") else []
        for call in calls:
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                call()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_decode_many_small_weights(dtype):
    """As in the packed call's test: one key, and 2^17 - 1 that weigh 2^-25 of it each; so many key heads (one,
    expanded) that one worker takes a head's rows."""
    N, D, H, page = 1 << 17, 32, 1024, 64
    kc, vc = (torch.zeros(N // page, page, 1, D, dtype=dtype, device=DEV) for _ in range(2))
    kc[0, 0, 0, 0] = 25.03125 * 0.693147 * D ** 0.5 / 8
    vc[:] = 1.0
    vc[0, 0] = -1.0
    q = torch.zeros(1, H, D, dtype=dtype, device=DEV)
    q[..., 0] = 8.0
    w = (N - 1) * torch.exp(-8.0 * kc[0, 0, 0, 0].double() / D ** 0.5).item()
    assert dtype == BF16 or w / (N - 1) < 2.0 ** -25
    kc, vc = (t.expand(-1, -1, H, -1) for t in (kc, vc))
    pages = torch.arange(N // page, dtype=torch.int32, device=DEV).view(1, -1)
    got = sdpa_rope_decode(q, kc, vc, seq_ref.Table(1, D, DEV), pages, ints([N]))
    u = seq_ref.U[dtype]
    # the bound of run_decode; the logit in fp32 (log2 units, 25) and exp2: 32 units of 2^-24 of the weights
    off = (got.double() - (w - 1) / (1 + w)).abs().max().item()
    assert off <= u + 3 * u * u + 32 * 2.0 ** -24, off


@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("dtype,D,H,Hkv,lens", [(BF16, 64, 16, 4, [300, 40]), (F16, 128, 32, 2, [130, 2]), (BF16, 128, 8, 8, [3000, 900]),
                                                (F16, 64, 8, 2, [5000]), (BF16, 256, 4, 1, [600]), (F16, 32, 40, 2, [1500]), (F32, 64, 8, 2, [700, 90])])
def test_decode_of_rows_that_are_not_finite(dtype, D, H, Hkv, lens, value):
    """One channel of a K row (a logit of an infinity: a weight of 0, or of no value), then of a V row: the formula's
    values, finite or not, in every head and channel."""
    page = 16
    pages, n = page_table(len(lens), -(-max(lens) // page))
    kc, vc = caches(n, page, Hkv, D, dtype)
    q = randn(len(lens), H, D, dtype=dtype, seed=3)
    table = seq_ref.Table(max(lens), D, DEV)
    for which in "KV":
        bad = {"K": kc.clone(), "V": vc.clone()}
        for b, m in enumerate(lens):
            i = m * 5 // 8
            bad[which][pages[b, i // page].item(), i % page, :, 5] = value
        got = sdpa_rope_decode(q, bad["K"], bad["V"], table, pages, ints(lens)).double().cpu()
        ref, _ = seq_ref.decode(q, bad["K"], bad["V"], table, pages, lens, True)
        assert torch.equal(torch.isnan(got), torch.isnan(ref)), which
        assert torch.equal(got[torch.isinf(ref)], ref[torch.isinf(ref)]) and torch.equal(torch.isinf(got), torch.isinf(ref))
        if which == "K" and value == value:
            assert torch.isfinite(ref).any()
        ok = torch.isfinite(ref)
        # run_decode's bound, for the rows' finite channels (|V| up to 5: sum P |V| no larger)
        u = seq_ref.U[dtype]
        off = torch.where(ok, got - ref, 0.0).norm(dim=-1)
        allowed = u * torch.where(ok, ref, 0.0).norm(dim=-1) + (32 * u if dtype == F32 else 3 * u * u + 32 * 2.0 ** -24) * 5 * D ** 0.5
        assert (off <= allowed).all()
