"""GPU: accepted rows and forked pages of a cache, against the same done row by row on the CPU."""
from __future__ import annotations

import random

import pytest
import torch

from tests import seq_ref
from triton_fused_rope_flash_attn_amd import rope_cache_accept, rope_cache_append, rope_cache_fork, sdpa_rope_decode

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def ints(x, shape=None):
    t = torch.tensor(x, dtype=torch.int32, device=DEV)
    return t if shape is None else t.reshape(shape)


def caches(n, page, Hkv, D, dtype, layout="rows"):
    def one(seed):
        g = torch.Generator().manual_seed(seed)
        shape = (n, page, Hkv, D) if layout == "rows" else (n, Hkv, page, D)
        x = torch.randn(shape, generator=g).to(dtype).to(DEV)
        return x if layout == "rows" else x.transpose(1, 2)
    return one(1), one(2)


def accept_ref(cache, pages, lengths, path):
    out, page = cache.clone(), cache.shape[1]

    def place(b, pos):
        if pos // page >= len(pages[b]):
            return None
        g = pages[b][pos // page]
        return (g, pos % page) if 0 <= g < cache.shape[0] else None

    for b, row in enumerate(path):
        row = row[: next((i for i, x in enumerate(row) if x < 0), len(row))]
        if lengths[b] < 0:
            continue
        for i, j in enumerate(row):
            s, t = place(b, lengths[b] + j), place(b, lengths[b] + i)
            if s and t:
                out[t] = cache[s]
    return out


def run_accept(kc, vc, pages, lengths, path):
    want = [accept_ref(x.cpu(), pages.tolist(), lengths.tolist(), path.tolist()) for x in (kc, vc)]
    count = [next((i for i, x in enumerate(r) if x < 0), len(r)) for r in path.tolist()]
    after = [n if n < 0 else min(n + c, 2 ** 31 - 1) for n, c in zip(lengths.tolist(), count)]
    versions = kc._version, vc._version, lengths._version
    got = rope_cache_accept(kc, vc, pages, lengths, path)
    assert got.dtype == torch.int32 and got.tolist() == after
    assert torch.equal(kc.cpu(), want[0]) and torch.equal(vc.cpu(), want[1])
    assert kc._version > versions[0] and vc._version > versions[1] and lengths._version == versions[2]


@pytest.mark.parametrize("layout", ["rows", "heads"])
@pytest.mark.parametrize("dtype,D,Hkv,page,cols", [(BF16, 64, 12, 16, 8), (F16, 128, 8, 32, 5), (F32, 256, 2, 7, 16),
                                                    (BF16, 32, 1, 1, 64), (F32, 32, 5, 100, 1), (BF16, 128, 3, 16, 65)])
def test_accept(dtype, D, Hkv, page, cols, layout):
    B, rng = 5, random.Random(cols)
    lengths = [0, 17, 3, page - 1, 40]
    per = -(-(40 + 2 * cols) // page)
    order = torch.randperm(B * per + 2, generator=torch.Generator().manual_seed(3)).to(torch.int32)
    pages = order[: B * per].reshape(B, per).to(DEV)
    path = []
    for b in range(B):   # rows in order, then any order, then none and all of them
        n = [cols, cols // 2, 0, cols, 1][b]
        row = sorted(rng.sample(range(2 * cols), n)) if b < 3 else [rng.randrange(2 * cols) for _ in range(n)]
        path.append(row + [-1] * (cols - n))
    kc, vc = caches(B * per + 2, page, Hkv, D, dtype, layout)
    run_accept(kc, vc, pages, ints(lengths), ints(path))


def test_accept_of_what_is_not_in_the_cache():
    """Sources and rows past the table, on no page, negative lengths, entries behind the first -1."""
    kc, vc = caches(9, 4, 2, 64, BF16)
    pages = ints([[0, 1], [2, -1], [9, 3], [4, 5], [6, 7]])
    path = ints([[1, 9, 3, 2 ** 31 - 1], [0, 3, 1, -1], [0, 4, 5, -1], [3, 2, 1, 0], [2, -1, 5, 6]])
    run_accept(kc, vc, pages, ints([5, 2, 0, -3, 1]), path)
    run_accept(kc, vc, pages, ints([2 ** 31 - 1, 2 ** 31 - 3, 8, 7, 6]), path)


def test_accept_strides_and_empty_calls():
    kc, vc = caches(8, 16, 2, 64, F16)
    wide = ints([[0, 1, 2, 3], [4, 5, 6, 7]])
    path = ints([[3, 1, 9, 9], [2, 5, 9, 9]])[:, :2]     # rows of the path apart, and of the table
    run_accept(kc, vc, wide[:, :3], ints([10, 30]), path)
    run_accept(kc, vc, wide, ints([10, 30]), path[:, :0])
    none = rope_cache_accept(kc, vc, wide[:0], ints([]), path[:0])
    assert none.shape == (0,)


def test_accept_many_columns():
    """As many columns as there may be, turned round: every row is read before one is written."""
    for cols in (1000, 2048):
        kc, vc = caches(2, cols, 1, 64, BF16)
        run_accept(kc, vc, ints([[1], [0]]), ints([0, 0]), ints([list(range(cols))[::-1]] * 2))


def fork_ref(caches_, pages, lengths, refs, parents, room):
    """The documented rules, place by place."""
    n_pages, page = caches_[0].shape[:2]
    old, out = [x.clone() for x in caches_], [x.clone() for x in caches_]
    B, M = len(pages), len(pages[0])
    free = [g for g in range(n_pages) if refs[g] == 0]
    table, after, seen, missing, delta = [], [], set(), 0, [0] * n_pages
    for b, p in enumerate(parents):
        row = [-1] * M
        table.append(row)
        if not 0 <= p < B:
            after.append(0)
            continue
        n = max(0, min(lengths[p], M * page))
        after.append(n)
        full, need = n // page, min(M, -(-(n + max(0, room[b] if room else 0)) // page))
        for i, g in enumerate(pages[p]):
            g = g if 0 <= g < n_pages else -1
            if i < full:
                row[i] = g
            elif g >= 0 and p not in seen and refs[g] == 1:
                row[i] = g
            elif i < need:
                if free:
                    row[i] = free.pop(0)
                    if i == full and g >= 0:
                        for a, c in zip(old, out):
                            c[row[i], : n % page] = a[g, : n % page]
                else:
                    missing += 1
        seen.add(p)
    for rows, sign in ((pages, -1), (table, 1)):
        for row in rows:
            for g in row:
                if 0 <= g < n_pages:
                    delta[g] += sign
    return table, after, [r + d for r, d in zip(refs, delta)], out, missing


def run_fork(kc, vc, pages, lengths, refs, parents, room=None):
    want = fork_ref([kc.cpu(), vc.cpu()], pages.tolist(), lengths.tolist(), refs.tolist(), parents.tolist(),
                    None if room is None else room.tolist())
    tensors = (kc, vc, pages, lengths, refs)
    versions = [t._version for t in tensors]
    missing = rope_cache_fork(kc, vc, pages, lengths, refs, parents, room=room)
    assert pages.tolist() == want[0]
    assert lengths.tolist() == want[1] and refs.tolist() == want[2]
    assert torch.equal(kc.cpu(), want[3][0]) and torch.equal(vc.cpu(), want[3][1])
    assert missing.tolist() == [want[4]]
    assert all(t._version > v for t, v in zip(tensors, versions))
    return want


def counts(pages, n):
    g = torch.tensor([x for row in pages.tolist() for x in row if 0 <= x < n], dtype=torch.long)
    return torch.bincount(g, minlength=n).to(torch.int32).to(DEV)


@pytest.mark.parametrize("layout", ["rows", "heads"])
@pytest.mark.parametrize("dtype,D,Hkv,page", [(BF16, 64, 12, 16), (F16, 128, 8, 64), (F32, 256, 1, 5), (BF16, 32, 3, 1),
                                              (F32, 64, 2, 300)])
def test_fork_in_steps(dtype, D, Hkv, page, layout):
    """A batch that grows, forks, shrinks and grows again, from an empty cache."""
    B, M, rng = 6, 9, random.Random(page)
    kc, vc = caches(40, page, Hkv, D, dtype, layout)
    pages, lengths, refs = torch.full((B, M), -1, dtype=torch.int32, device=DEV), ints([0] * B), ints([0] * 40)
    own = list(range(B))
    plans = [(own, [2 * page + 3, 0, 1, page, page - 1, 4 * page]), ([0, 0, 2, 0, 4, 5], [1] * B), ([0, 1, 1, 3, 3, -1], [1, 0, 2, 1, 1, 9]),
             (own, [page + 1] * B), ([5, 4, 3, 2, 1, 0], None), (own, [1] * B), ([-1, B, 2, 2, 2, 2], [-5] * B), ([2, 2, 2, 2, 2, 2], [3 * page] * B)]
    for parents, room in plans:
        run_fork(kc, vc, pages, lengths, refs, ints(parents), None if room is None else ints(room))
        assert refs.tolist() == counts(pages, 40).tolist()
        # some of the reserved rows are filled
        lengths += ints([rng.randint(0, 1 + (r if r and r > 0 else 0)) for r in (room or [0] * B)])


def test_fork_frees_and_gives_out_again():
    kc, vc = caches(6, 8, 1, 32, BF16)
    pages, lengths, refs = torch.full((2, 4), -1, dtype=torch.int32, device=DEV), ints([0, 0]), ints([0] * 6)
    run_fork(kc, vc, pages, lengths, refs, ints([0, 1]), ints([24, 24]))
    assert pages.tolist() == [[0, 1, 2, -1], [3, 4, 5, -1]]
    lengths += ints([20, 24])
    run_fork(kc, vc, pages, lengths, refs, ints([0, -1]), ints([9, 0]))      # what this call gives back is not there yet
    assert pages.tolist() == [[0, 1, 2, -1], [-1] * 4] and refs.tolist() == [1, 1, 1, 0, 0, 0]
    want = run_fork(kc, vc, pages, lengths, refs, ints([0, 0]), ints([12, 12]))
    assert want[4] == 0 and pages.tolist() == [[0, 1, 2, 3], [0, 1, 4, 5]]


def test_fork_without_enough_pages():
    kc, vc = caches(4, 8, 2, 64, F16)
    pages, lengths, refs = ints([[0, 1, -1], [2, -1, -1], [-1] * 3]), ints([12, 3, 0]), ints([1, 1, 1, 0])
    want = run_fork(kc, vc, pages, lengths, refs, ints([0, 0, 0]), ints([1, 1, 8]))
    assert want[4] == 2


def test_fork_of_shared_and_odd_pages():
    """Lengths cut back onto shared pages, counts of other holders, numbers that are no page, lengths out of range."""
    kc, vc = caches(30, 4, 2, 64, BF16)
    pages = ints([[0, 1, 2, 3], [0, 1, 4, -1], [-1, 30, 5, 1 << 30], [6, 7, 8, 9], [10, -7, 11, -1]])
    refs = counts(pages, 30)
    refs[6:9] += 1                                           # something else holds them
    lengths = ints([6, 5, 9, 1000, -4])
    run_fork(kc, vc, pages, lengths, refs, ints([0, 1, 2, 3, 4]), ints([4, 4, 4, 4, 4]))
    lengths.copy_(ints([15, 9, 9, 9, 2]))
    run_fork(kc, vc, pages, lengths, refs, ints([3, 3, 0, 0, 4]), ints([0, 2 ** 31 - 1, 1, 1, 1]))


def test_fork_of_wide_tables_and_many_places():
    """More pages, places and entries than a step of a search covers; rows of the table apart."""
    B, M, page, n = 300, 700, 2, 70000
    kc, vc = caches(n, page, 1, 32, BF16)
    wide = torch.full((B, M + 1), -1, dtype=torch.int32, device=DEV)
    pages, lengths, refs = wide[:, :M], ints([0] * B), ints([0] * n)
    refs[torch.randperm(n, generator=torch.Generator().manual_seed(1))[: n // 2].to(DEV)] = 3
    g = torch.Generator().manual_seed(2)
    room = torch.randint(0, 250, (B,), generator=g).to(torch.int32)
    room[::50] = 2 * M
    room = room.to(DEV)
    run_fork(kc, vc, pages, lengths, refs, ints(list(range(B))), room)
    lengths += room
    parents = torch.randint(-20, B + 20, (B,), generator=g).to(torch.int32).to(DEV)
    run_fork(kc, vc, pages, lengths, refs, parents, ints([1] * B))
    run_fork(kc, vc, pages, lengths, refs, ints([0] * B), ints([1000] * B))
    assert (wide[:, M] == -1).all()


def test_cache_past_32_bits():
    """Rows past 2^31 elements move and are copied."""
    Hkv, D, page = 8, 128, 64
    n = (1 << 31) // (Hkv * D * page) + 4
    kc, vc = (torch.zeros(n, page, Hkv, D, dtype=BF16, device=DEV) for _ in range(2))
    kc[n - 1], vc[n - 1] = torch.randn(page, Hkv, D, device=DEV), torch.randn(page, Hkv, D, device=DEV)
    before = kc[n - 1].clone(), vc[n - 1].clone()
    after = rope_cache_accept(kc, vc, ints([[n - 1]]), ints([10]), ints([[40, 20]]))
    assert after.tolist() == [12]
    assert torch.equal(kc[n - 1, 10], before[0][50]) and torch.equal(vc[n - 1, 11], before[1][30])
    refs = torch.ones(n, dtype=torch.int32, device=DEV)
    refs[n - 2] = 0
    pages, lengths = ints([[n - 1], [-1]]), ints([12, 0])
    assert rope_cache_fork(kc, vc, pages, lengths, refs, ints([0, 0])).tolist() == [0]
    assert pages.tolist() == [[n - 1], [n - 2]]
    assert torch.equal(kc[n - 2, :12], kc[n - 1, :12]) and torch.equal(vc[n - 2, :12], vc[n - 1, :12])
    assert (kc[n - 2, 12:] == 0).all()


def test_forked_sequences_go_on_apart():
    """A beam: tokens appended after a fork do not reach the other places' sequences."""
    H, Hkv, D, page, B = 4, 2, 64, 16, 4
    table = seq_ref.Table(80, D, DEV)
    kc, vc = caches(40, page, Hkv, D, BF16)
    pages, lengths, refs = torch.full((B, 5), -1, dtype=torch.int32, device=DEV), ints([0] * B), ints([0] * 40)
    rng, history = torch.Generator().manual_seed(5), [[] for _ in range(B)]

    def randn(*shape):
        return torch.randn(shape, generator=rng).to(BF16).to(DEV)

    for step in range(40):
        parents = [0] * B if step == 20 else torch.randint(0, B, (B,), generator=rng).tolist() if step % 7 == 3 else list(range(B))
        assert rope_cache_fork(kc, vc, pages, lengths, refs, ints(parents), room=ints([1] * B)).tolist() == [0]
        history = [list(history[p]) for p in parents]
        k, v, q = randn(B, Hkv, D), randn(B, Hkv, D), randn(B, H, D)
        rope_cache_append(k, v, table, kc, vc, pages, lengths)
        lengths += 1
        for b in range(B):
            history[b].append((k[b], v[b]))
        if step % 9 == 8 or step == 21:
            n = len(history[0])
            fresh = [torch.zeros(B, n, Hkv, D, dtype=BF16, device=DEV) for _ in range(2)]
            own = ints([[b] for b in range(B)])
            starts = ints([n * b for b in range(B + 1)])
            ks, vs = (torch.stack([x[i] for row in history for x in row]) for i in (0, 1))
            rope_cache_append(ks, vs, table, *fresh, own, ints([0] * B), cu_seqlens=starts)
            got = sdpa_rope_decode(q, kc, vc, table, pages, lengths)
            want = sdpa_rope_decode(q, *fresh, table, own, lengths)
            # (the same rows in other blocks of the pool: only the workers' shares may differ)
            assert (got.float() - want.float()).abs().max() <= 2 * 2.0 ** -8 * want.float().abs().max()
    assert refs.tolist() == counts(pages, 40).tolist()


def test_captured_and_replayed():
    """One graph of fork, append and accept serves every later step."""
    Hkv, D, page, B = 2, 64, 8, 4
    table = seq_ref.Table(80, D, DEV)

    def fresh():
        kc, vc = caches(60, page, Hkv, D, BF16)
        return [kc, vc, torch.full((B, 9), -1, dtype=torch.int32, device=DEV), ints([0] * B), ints([0] * 60)]

    k, v = (torch.zeros(B * 3, Hkv, D, dtype=BF16, device=DEV) for _ in range(2))
    parents, path, room, starts = ints([0] * B), ints([[0, -1]] * B), ints([3] * B), ints([0, 3, 6, 9, 12])

    def step(kc, vc, pages, lengths, refs):
        missing = rope_cache_fork(kc, vc, pages, lengths, refs, parents, room=room)
        rope_cache_append(k, v, table, kc, vc, pages, lengths, cu_seqlens=starts)
        lengths.copy_(rope_cache_accept(kc, vc, pages, lengths, path))
        return missing

    state, other = fresh(), fresh()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(*fresh())
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*state)
    for i in range(14):
        g = torch.Generator().manual_seed(i)
        k.copy_(torch.randn(k.shape, generator=g))
        v.copy_(torch.randn(v.shape, generator=g))
        parents.copy_(torch.randint(-1 if i == 9 else 0, B, (B,), generator=g))
        path.copy_(torch.randint(-1, 3, (B, 2), generator=g))
        graph.replay()
        torch.cuda.synchronize()
        want = step(*other)
        assert torch.equal(out, want), i
        assert all(torch.equal(a, b) for a, b in zip(state, other)), i


def test_ops_pass_opcheck_and_compile():
    kc, vc = caches(10, 16, 2, 64, BF16)
    pages, lengths = ints([[0, 1], [2, 3]]), ints([10, 20])
    refs = counts(pages, 10)
    torch.library.opcheck(torch.ops.farope.cache_accept.default, (kc, vc, pages, lengths, ints([[1, 2], [3, -1]])))
    torch.library.opcheck(torch.ops.farope.cache_fork.default, (kc, vc, pages, lengths, refs, ints([0, 0]), ints([1, 1])))


def test_gradients_are_refused():
    kc, vc = caches(10, 16, 2, 64, BF16)
    pages, lengths, refs = ints([[0, 1], [2, 3]]), ints([10, 20]), ints([0] * 10)
    with pytest.raises(RuntimeError, match="not differentiable"):
        rope_cache_accept(kc.clone().requires_grad_(), vc, pages, lengths, ints([[1], [2]]))
    with pytest.raises(RuntimeError, match="not differentiable"):
        rope_cache_fork(kc, vc.clone().requires_grad_(), pages, lengths, refs, ints([0, 1]))
    assert (refs == 0).all() and pages.tolist() == [[0, 1], [2, 3]]
