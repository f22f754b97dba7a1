"""The calls that the speed of windowed attention, of drafted tokens and of a cache's pages is judged by.

A case is one pass through one of the operators of sequence models with rotary positions:

* ``prompt``: windowed attention within packed sequences, the first tokens (sinks) staying visible;
* ``train``: the same with its gradients;
* ``decode``: one new token per sequence over the window and the sinks of its cached keys;
* ``tree``: several new tokens per sequence over the cache: a drafted tree, or a chunk of a prompt;
* ``accept``: the cached rows of the drafted tokens that were accepted move up behind the sequence;
* ``fork``: places of a batch continue others' sequences: pages shared, copied, reserved and freed.

``listed`` names twelve of them; ``draw`` gives further ones of the same ranges:

* head_dim 32, 64, 128 and 256; bf16, fp16 and fp32; 1 to 16 query heads per key head; pages of 1 to 256 rows;
* packs of 1 to 128 sequences of 1 to 16 K tokens, windows of 1 to 4 K tokens, 0 to 70 sinks;
* caches of up to 128 K rows a sequence, 1 to 256 sequences of different lengths;
* trees of 1 to 64 drafted tokens, chunks of 1 to 2 K tokens;
* 1 to 256 places, up to 16 of them continuing the same prompt.

Tables are those of a square token grid (the class token in front of it is not
rotated).  Queries, keys and values of a prompt are views of one projection's output.
"""
import math
import random

import torch

own = False

ROPE_BASE = 100.0
DEVICE = "cuda"

# seqs, longest: the sequences and the longest one's length (decode: after the new token; tree, accept: before
# the drafted ones); ragged: the others are shorter; window, sinks: of prompt, train and decode; new: drafted
# tokens of a sequence at most (chunk: they are a chain, no tree); width: places that continue one prompt;
# page: rows a page holds; pad: the last sequence (fork: the last prompt's places) is an empty place of the batch
_DEFAULT = dict(kind="train", seqs=1, longest=197, ragged=False, H=12, Hkv=12, D=64, dtype="bf16", cls=True, page=16,
                window=64, sinks=0, new=0, chunk=False, width=1, pad=False)


def _case(name, **kw):
    return dict(_DEFAULT, name=name, **kw)


def listed():
    return [
        # Prompts of a served batch, shared key heads, fp16.
        _case("window_prompt_fp16", kind="prompt", seqs=16, longest=4096, ragged=True, H=16, Hkv=4, D=128, dtype="fp16",
              window=512, sinks=4),
        # Training on one long sequence, four query heads per key head.
        _case("window_train_long", longest=16384, H=8, Hkv=2, D=128, cls=False, window=1024, sinks=4),
        # A small training step in plain fp32; the class token is the sink.
        _case("window_train_fp32", seqs=3, longest=513, ragged=True, H=8, Hkv=4, dtype="fp32", window=100, sinks=1),
        # One token of one long sequence: the latency of a step.
        _case("window_decode_one", kind="decode", longest=9000, window=1024, sinks=1),
        # A served batch at different stages, one of its places empty.
        _case("window_decode_batch", kind="decode", seqs=64, longest=16384, ragged=True, H=32, Hkv=8, D=128, page=32,
              window=2048, sinks=4, pad=True),
        # A few drafted tokens of one sequence are verified.
        _case("tree_one", kind="tree", longest=1024, new=8),
        # A served batch verifies a tree of drafted tokens for each of its sequences.
        _case("tree_batch", kind="tree", seqs=32, longest=8192, ragged=True, H=32, Hkv=8, D=128, page=32, new=32),
        # Long prompts arrive in chunks, behind what of them is cached.
        _case("tree_chunk_fp16", kind="tree", seqs=4, longest=8192, ragged=True, H=32, Hkv=8, D=128, dtype="fp16", page=64,
              new=1024, chunk=True),
        # The accepted tokens of one small tree.
        _case("accept_one", kind="accept", longest=1024, new=8),
        # The accepted tokens of a served batch's trees.
        _case("accept_batch", kind="accept", seqs=128, longest=512, ragged=True, Hkv=8, D=128, new=64),
        # A beam of four continuations of one prompt.
        _case("fork_beam", kind="fork", seqs=4, width=4, longest=200, page=16),
        # Many prompts with eight continuations each, in large pages; one prompt is finished.
        _case("fork_batch_fp16", kind="fork", seqs=256, width=8, longest=1024, ragged=True, Hkv=8, D=128, dtype="fp16",
              page=128, pad=True),
    ]


# What no drawn case may exceed: about the listed cases' largest operation count, traffic and
# score matrix of the plain form.
_MOST_FLOPS = 6.0e11
_MOST_BYTES = 6.0e8
_MOST_SCORES = 2.1e9


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    while True:
        c = dict(_DEFAULT)
        c["kind"] = rng.choice(["prompt", "train", "train", "decode", "tree", "tree", "accept", "fork"])
        c["D"] = rng.choice([32, 64, 64, 128, 128, 128, 256])
        c["dtype"] = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp16", "fp32"])
        c["Hkv"] = rng.choice([1, 2, 3, 4, 6, 8, 8, 12])
        c["H"] = c["Hkv"] * rng.choice([1, 1, 2, 3, 4, 4, 7, 8, 16])
        c["cls"] = rng.random() < 0.6
        c["ragged"] = rng.random() < 0.8
        c["page"] = rng.choice([1, 7, 16, 16, 32, 64, 100, 128, 256])
        if c["kind"] in ("prompt", "train", "decode"):
            c["window"] = _log_int(rng, 1, 4096)
            c["sinks"] = rng.choice([0, 1, 4, 4, 7, 70])
        if c["kind"] in ("prompt", "train"):
            c["seqs"], c["longest"] = _log_int(rng, 1, 128), _log_int(rng, 1, 16384)
        elif c["kind"] == "decode":
            c["seqs"], c["longest"] = _log_int(rng, 1, 256), _log_int(rng, 1, 131072)
            c["pad"] = c["seqs"] > 2 and rng.random() < 0.3
        elif c["kind"] == "tree":
            c["chunk"] = rng.random() < 0.4
            c["seqs"], c["longest"] = _log_int(rng, 1, 32 if c["chunk"] else 128), _log_int(rng, 1, 32768)
            c["new"] = _log_int(rng, 1, 2048 if c["chunk"] else 64)
            c["pad"] = c["seqs"] > 2 and rng.random() < 0.3
        elif c["kind"] == "accept":
            c["H"] = c["Hkv"]
            c["seqs"], c["longest"], c["new"] = _log_int(rng, 1, 256), _log_int(rng, 1, 1024), _log_int(rng, 1, 64)
        else:
            c["H"] = c["Hkv"]
            c["width"] = rng.choice([1, 2, 4, 8, 16])
            c["seqs"], c["longest"] = c["width"] * _log_int(rng, 1, 256 // c["width"]), _log_int(rng, 1, 2048)
            c["pad"] = c["seqs"] > 2 * c["width"] and rng.random() < 0.3
        w = work(c)
        slow = 12 if c["dtype"] == "fp32" else 1
        wide = {"prompt": c["longest"], "train": c["longest"], "tree": c["new"]}.get(c["kind"], 1)
        scores = c["seqs"] * c["H"] * wide * (c["longest"] + c["new"])
        cache = c["seqs"] * (c["longest"] + c["new"] + c["page"]) * c["Hkv"] * c["D"] * 4
        most = 4e8 if c["kind"] in ("accept", "fork") else 4e9
        if w["flops"] * slow <= _MOST_FLOPS and w["bytes"] <= _MOST_BYTES and scores <= _MOST_SCORES and cache <= most:
            return c


# ---------------------------------------------------------------------------
# what a case's shape is, the same for every seed
# ---------------------------------------------------------------------------
def _rng(case):
    return random.Random("%s %d %d %d" % (case["kind"], case["seqs"], case["longest"], case["new"]))


def _lengths(case):
    """The sequences' lengths; of a fork the places', those of a prompt alike."""
    rng, most, width = _rng(case), case["longest"], case["width"]
    n = case["seqs"] // width
    if not case["ragged"]:
        lens = [most] * n
    else:
        lens = [max(min(1, most), int(most * 16.0 ** -rng.random())) for _ in range(n)]
        lens[rng.randrange(n)] = most
    if case["pad"] and case["kind"] == "decode":
        lens[-1] = 0
    return [x for x in lens for _ in range(width)]


def _drafted(case):
    """New tokens of each sequence."""
    rng, n = _rng(case), case["seqs"]
    new = [case["new"] - rng.randint(0, case["new"] // 2) if case["ragged"] else case["new"] for _ in range(n)]
    if case["pad"]:
        new[-1] = 0
    return new


def _trees(case):
    """Each sequence's tree: a token's parent among the tokens before it (-1: the cached sequence's end)."""
    rng = _rng(case)
    return [[-1 if i == 0 else rng.randint(max(-1, i - 9), i - 1) for i in range(m)] for m in _drafted(case)]


def _depths(tree):
    depth = []
    for up in tree:
        depth.append(0 if up < 0 else depth[up] + 1)
    return depth


def _paths(case):
    """Each sequence's accepted tokens: the front part of the way to its deepest token."""
    rng, out = _rng(case), []
    for tree in _trees(case):
        depth, way = _depths(tree), []
        at = depth.index(max(depth)) if tree else -1
        while at >= 0:
            way.append(at)
            at = tree[at]
        way.reverse()
        out.append(way[: rng.randint(len(way) // 2, len(way))])
    return out


def _dtype(case):
    return {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[case["dtype"]]


class _Table:
    """Cosines and sines [side * side, D/2] of a square grid: row angles first, then the column's."""

    def __init__(self, rows, D):
        side, pairs = max(1, math.isqrt(max(0, rows - 1)) + 1), D // 4
        freq = ROPE_BASE ** (-torch.arange(pairs, dtype=torch.float64, device=DEVICE) / pairs)
        at = torch.arange(side * side, device=DEVICE)
        ang = torch.cat([(at // side).double()[:, None] * freq, (at % side).double()[:, None] * freq], dim=1)
        self.cos, self.sin = ang.cos().float(), ang.sin().float()

    def tables(self):
        return self.cos, self.sin


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _starts(values):
    return _ints([sum(values[:i]) for i in range(len(values) + 1)])


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    kind, H, Hkv, D, dt = case["kind"], case["H"], case["Hkv"], case["D"], _dtype(case)
    lens, page = _lengths(case), case["page"]

    def randn(*shape):
        return torch.randn(shape, generator=gen, device=DEVICE).to(dt)

    state = {"case": dict(case), "most": max(lens)}
    if kind in ("prompt", "train"):
        T = sum(lens)
        qkv = randn(T, H + 2 * Hkv, D)
        state["q"], state["k"], state["v"] = (
            t.detach().requires_grad_(kind == "train") for t in qkv.split([H, Hkv, Hkv], dim=1))
        if kind == "train":
            state["do"] = randn(T, H, D)
        state["starts"], state["table"] = _starts(lens), _Table(state["most"], D)
        return state
    if kind == "fork":
        return _prepare_fork(case, state, lens, gen, randn)
    capacity = max(lens) + (1 if kind == "decode" else case["new"])
    per = max(1, -(-capacity // page))
    total = len(lens) * per + 3
    order = torch.randperm(total, generator=gen, device=DEVICE).to(torch.int32)
    state["pages"] = order[: len(lens) * per].reshape(len(lens), per).contiguous()
    state["k_cache"], state["v_cache"] = randn(total, page, Hkv, D), randn(total, page, Hkv, D)
    state["lengths"], state["table"] = _ints(lens), _Table(capacity, D)
    if kind == "decode":
        state["q"] = randn(len(lens), H, D)
    elif kind == "tree":
        new = _drafted(case)
        state["q"], state["starts"], state["most_new"] = randn(sum(new), H, D), _starts(new), max(new)
        if case["chunk"]:
            state["tree"] = state["positions"] = None
        else:   # ancestors of every drafted token, itself among them; its table row goes by its depth
            sees = torch.zeros(sum(new), max(new), dtype=torch.bool)
            rows, at = [], 0
            for n, tree in zip(lens, _trees(case)):
                for i, up in enumerate(tree):
                    if up >= 0:
                        sees[at + i] = sees[at + up]
                    sees[at + i, i] = True
                rows += [n + d - int(case["cls"]) for d in _depths(tree)]
                at += len(tree)
            state["tree"], state["positions"] = sees.to(DEVICE), _ints(rows)
    else:
        paths = _paths(case)
        wide = max(len(x) for x in paths)
        state["path"] = _ints([x + [-1] * (wide - len(x)) for x in paths])
    return state


def _prepare_fork(case, state, lens, gen, randn):
    """Places that continued one prompt before share its whole pages; each has its own last one."""
    width, page, B = case["width"], case["page"], len(lens)
    per = max(lens) // page + 2
    owned, table, refs = 0, [], []
    for first in range(0, B, width):
        full = lens[first] // page
        shared = list(range(owned, owned + full))
        refs += [width] * full
        owned += full
        for _ in range(width):
            table.append(shared + [owned] + [-1] * (per - full - 1))
            refs.append(1)
            owned += 1
    total = owned + 3 * B + 5   # (the last page belongs to none of the places: nobody's rows, and never handed out)
    order = torch.randperm(total, generator=gen, device=DEVICE).to(torch.int32)
    table, refs = _ints(table), _ints(refs + [0] * (total - owned - 1) + [1])
    state["pages"] = torch.where(table >= 0, order[table.clamp(min=0).long()], -1).to(torch.int32)
    state["refs"] = torch.zeros_like(refs)
    state["refs"][order.long()] = refs
    state["spare"] = int(order[-1])
    state["lengths"], state["room"] = _ints(lens), _ints([1] * B)
    group = torch.arange(B, device=DEVICE) // width * width
    parents = group + torch.randint(0, width, (B,), generator=gen, device=DEVICE)
    if case["pad"]:
        parents[-width:] = -1
    state["parents"] = parents.to(torch.int32)
    state["k_cache"], state["v_cache"] = (randn(total, page, case["Hkv"], case["D"]) for _ in range(2))
    return state


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _cos_sin(state, row):
    """Rows of the table, [..., 1, D/2]: below 0 is not rotated."""
    cos, sin = state["table"].tables()
    at = row.long()
    none = (at < 0)[..., None]
    at = at.clamp(0, cos.shape[0] - 1)
    return torch.where(none, 1.0, cos[at])[..., None, :], torch.where(none, 0.0, sin[at])[..., None, :]


def _rotate(x, cos, sin):
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)


def _token_places(starts, n):
    """Sequence and index within it of each of the n packed tokens."""
    at = torch.arange(n, device=DEVICE)
    seq = torch.searchsorted(starts[1:].long(), at, right=True)
    return seq, at - starts.long()[seq]


def _softmax(s, keep):
    s = torch.where(keep, s, -torch.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isfinite(top), top, 0.0))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total > 0, total, 1.0)


def _cached(state, name, keep):
    """The sequences' rows [B, Hkv, rows, D] of a cache in 32 bits, zeros where they are not in use."""
    c = state[name]
    x = c[state["pages"].long()].float().reshape(state["pages"].shape[0], -1, *c.shape[2:])
    return torch.where(keep[..., None, None], x, 0.0).transpose(1, 2)


def _decode(state):
    case, q, lengths = state["case"], state["q"], state["lengths"].long()
    B, H, D = q.shape
    Hkv = case["Hkv"]
    at = torch.arange(state["pages"].shape[1] * case["page"], device=DEVICE)
    keep = (at < lengths[:, None]) & ((at >= lengths[:, None] - case["window"]) | (at < case["sinks"]))
    keys, values = (_cached(state, n, keep) for n in ("k_cache", "v_cache"))
    qh = _rotate(q.float(), *_cos_sin(state, lengths.clamp(min=1) - 1 - int(case["cls"]))).reshape(B, Hkv, H // Hkv, D)
    s = torch.matmul(qh, keys.transpose(2, 3).contiguous()) * D ** -0.5
    p = _softmax(s, keep[:, None, None, :])
    return torch.matmul(p, values).reshape(B, H, D).to(q.dtype)


def _tree(state):
    case, q, lengths, starts = state["case"], state["q"], state["lengths"].long(), state["starts"].long()
    (T, H, D), most, Hkv, B = q.shape, state["most_new"], case["Hkv"], case["seqs"]
    new = starts[1:] - starts[:-1]
    at = torch.arange(state["pages"].shape[1] * case["page"], device=DEVICE)
    keys, values = (_cached(state, n, at < (lengths + new)[:, None]) for n in ("k_cache", "v_cache"))
    j = torch.arange(most, device=DEVICE)
    place = (starts[:-1, None] + j).clamp(max=T - 1)                        # [B, M]
    row = lengths[:, None] + j - int(case["cls"]) if state["positions"] is None else state["positions"].long()[place]
    qh = _rotate(q[place].float(), *_cos_sin(state, row))                   # [B, M, H, D]
    qh = qh.reshape(B, most, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    i = at[None, :] - lengths[:, None]                                      # a position's drafted token
    if state["tree"] is None:
        keep = i[:, None, :] <= j[:, None]
    else:
        keep = (i < 0)[:, None, :] | torch.gather(state["tree"][place], 2, i.clamp(0, most - 1)[:, None, :].expand(-1, most, -1))
    keep = keep & (i < new[:, None])[:, None, :]                            # [B, M, rows]
    s = torch.matmul(qh, keys.transpose(2, 3).contiguous()).mul_(D ** -0.5).reshape(B, H, most, -1)
    p = _softmax(s, keep[:, None]).reshape(B, Hkv, -1, at.numel())
    o = torch.matmul(p, values).reshape(B, H, most, D).transpose(1, 2)
    seq, i = _token_places(state["starts"], T)
    return o[seq, i].to(q.dtype)


def _accept(state):
    page, pages, path = state["case"]["page"], state["pages"], state["path"]
    lengths = state["lengths"]
    take = (path >= 0).long().cumprod(1).bool()
    pos = torch.where(take, lengths[:, None] + path, 0)                     # (rows not taken: row 0 onto itself)
    to = torch.where(take, lengths[:, None] + torch.arange(path.shape[1], device=DEVICE), 0)
    seq = torch.arange(path.shape[0], device=DEVICE)[:, None]
    pos, to = (pages[seq, x // page].long() * page + x % page for x in (pos, to))
    for n in ("k_cache", "v_cache"):
        flat = state[n].view(-1, *state[n].shape[2:])
        flat[to] = flat[pos]
    return state["k_cache"], state["v_cache"], (lengths + take.sum(1)).to(torch.int32)


def _fork(state):
    page, table, refs = state["case"]["page"], state["pages"], state["refs"]
    B, M = table.shape
    parents, n = state["parents"].long(), state["lengths"].long()
    alive = parents >= 0
    p = parents.clamp(min=0)
    n = torch.where(alive, n[p], 0)
    twin = (parents[:, None] == parents[None, :]).tril(-1).any(1)           # an earlier place has the same parent
    full, part = n // page, n % page
    need = torch.where(alive, (n + state["room"] + page - 1) // page, 0)
    at = torch.arange(M, device=DEVICE)
    held = table[p].long()
    there = alive[:, None] & (held >= 0)
    shared = there & (at < full[:, None])
    kept = there & (at >= full[:, None]) & ~twin[:, None] & (refs[held.clamp(min=0)] == 1)
    want = (at >= full[:, None]) & (at < need[:, None]) & ~kept
    free = torch.sort((refs != 0).to(torch.int32), stable=True).indices
    number = torch.cumsum(want.flatten().long(), 0).reshape(B, M) - 1
    got = want & (number < (refs == 0).sum())
    fresh = free[number.clamp(0, free.numel() - 1)]
    new = torch.where(shared | kept, held, torch.where(got, fresh, -1))
    # the rows in use of a page that is not kept; the others copy a row of the spare page onto itself
    row = torch.arange(page, device=DEVICE)
    last = full.clamp(max=M - 1)[:, None]
    copy = torch.gather(got & there, 1, last) & (row < part[:, None])
    source = torch.where(copy, torch.gather(held, 1, last), state["spare"]) * page + row
    target = torch.where(copy, torch.gather(new, 1, last), state["spare"]) * page + row
    for name in ("k_cache", "v_cache"):
        flat = state[name].view(-1, *state[name].shape[2:])
        flat[target] = flat[source]
    one = torch.ones(B * M, dtype=torch.int32, device=DEVICE)
    for t, sign in ((table.long(), -1), (new, 1)):
        refs.index_add_(0, t.clamp(min=0).flatten(), torch.where(t.flatten() >= 0, sign * one, 0))
    table.copy_(new)
    state["lengths"].copy_(n)
    missing = (want.sum() - got.sum()).to(torch.int32).reshape(1)
    return table, state["lengths"], refs, state["k_cache"], state["v_cache"], missing


def _attention(state):
    case, q, starts, most = state["case"], state["q"], state["starts"].long(), state["most"]
    T, H, D = q.shape
    Hkv, group = state["k"].shape[1], H // state["k"].shape[1]
    at = torch.arange(most, device=DEVICE)
    place = (starts[:-1, None] + at).clamp(max=T - 1)                     # [B, L]
    inside = at < (starts[1:] - starts[:-1])[:, None]
    cos, sin = _cos_sin(state, at - int(case["cls"]))

    def padded(x, rotated):
        x = x.detach()[place].float()
        x = _rotate(x, cos, sin) if rotated else x
        x = x.transpose(1, 2).repeat_interleave(H // x.shape[2], dim=1)
        return torch.where(inside[:, None, :, None], x, 0.0)              # [B, H, L, D]

    def packed(x, rotated):
        x = x.transpose(1, 2)
        x = _rotate(x, cos, -sin) if rotated else x
        seq, i = _token_places(state["starts"], T)
        return x[seq, i].to(q.dtype)

    qh, kh, vh = padded(state["q"], True), padded(state["k"], True), padded(state["v"], False)
    back = at[:, None] - at[None, :]
    keep = inside[:, None, None, :] & (back >= 0) & ((back < case["window"]) | (at[None, :] < case["sinks"]))
    p = _softmax(torch.matmul(qh, kh.transpose(2, 3).contiguous()) * D ** -0.5, keep)
    o = torch.matmul(p, vh)
    if case["kind"] == "prompt":
        return (packed(o, False),)
    g = padded(state["do"], False)
    dv = torch.matmul(p.transpose(2, 3), g)
    ds = torch.matmul(g, vh.transpose(2, 3).contiguous()) - (g * o).sum(-1, keepdim=True)
    ds = ds.mul_(p).mul_(D ** -0.5)
    del p
    dq, dk = torch.matmul(ds, kh), torch.matmul(ds.transpose(2, 3), qh)
    dk, dv = (x.reshape(-1, Hkv, group, most, D).sum(2) for x in (dk, dv))
    return packed(o, False), packed(dq, True), packed(dk, True), packed(dv, False)


def _own(state):
    import triton_fused_rope_flash_attn_amd as farope

    case, kind = state["case"], state["case"]["kind"]
    if kind in ("prompt", "train"):
        args = (state["q"], state["k"], state["v"], state["table"], state["starts"])
        out = farope.sdpa_rope_varlen(*args, has_cls=case["cls"], window=case["window"], sinks=case["sinks"])
        if kind == "prompt":
            return (out,)
        return (out.detach(), *torch.autograd.grad(out, args[:3], state["do"]))
    caches = (state["k_cache"], state["v_cache"])
    if kind == "decode":
        return (farope.sdpa_rope_decode(state["q"], *caches, state["table"], state["pages"], state["lengths"],
                                        has_cls=case["cls"], window=case["window"], sinks=case["sinks"]),)
    if kind == "tree":
        return (farope.sdpa_rope_tree(state["q"], *caches, state["table"], state["pages"], state["lengths"], state["starts"],
                                      tree=state["tree"], has_cls=case["cls"], positions=state["positions"]),)
    if kind == "accept":
        return (*caches, farope.rope_cache_accept(*caches, state["pages"], state["lengths"], state["path"]))
    missing = farope.rope_cache_fork(*caches, state["pages"], state["lengths"], state["refs"], state["parents"],
                                     room=state["room"])
    return state["pages"], state["lengths"], state["refs"], *caches, missing


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    if kind in ("prompt", "train"):
        return _attention(state)
    if kind == "decode":
        return (_decode(state),)
    if kind == "tree":
        return (_tree(state),)
    return _accept(state) if kind == "accept" else _fork(state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def _seen(n, window, sinks):
    """Keys that the tokens 0 .. n - 1 of a sequence see, added up."""
    w = min(n, window)
    near = w * (w + 1) // 2 + (n - w) * w
    m = min(sinks, max(0, n - window))
    return near + m * (m + 1) // 2 + max(0, n - window - sinks) * m


def work(case):
    H, Hkv, D, e = case["H"], case["Hkv"], case["D"], 4 if case["dtype"] == "fp32" else 2
    lens, kind, row = _lengths(case), case["kind"], 2 * case["Hkv"] * case["D"] * (4 if case["dtype"] == "fp32" else 2)
    if kind in ("prompt", "train"):
        train = kind == "train"
        pairs = sum(_seen(n, case["window"], case["sinks"]) for n in lens)
        return {"bytes": (2 if train else 1) * 2 * sum(lens) * (H + Hkv) * D * e + 4 * case["longest"] * D,
                "flops": (14 if train else 4) * pairs * H * D}
    if kind == "decode":
        rows = sum(min(n, case["window"]) + min(case["sinks"], max(0, n - case["window"])) for n in lens)
        return {"bytes": rows * row + case["seqs"] * (2 * H * D * e + 4 * D) + 4 * rows // case["page"], "flops": 4 * rows * H * D}
    if kind == "tree":
        new = _drafted(case)
        rows = sum(n + m for n, m in zip(lens, new) if m)
        if case["chunk"]:
            among, mask = sum(m * (m + 1) // 2 for m in new), 0
        else:
            among, mask = sum(d + 1 for t in _trees(case) for d in _depths(t)), sum(new) * max(new)
        pairs = sum(n * m for n, m in zip(lens, new)) + among
        return {"bytes": rows * row + sum(new) * (2 * H * D * e + 4 * D) + mask + 4 * rows // case["page"], "flops": 4 * pairs * H * D}
    if kind == "accept":
        paths = _paths(case)
        moved = sum(i != x for way in paths for i, x in enumerate(way))
        return {"bytes": 2 * moved * row + 4 * sum(len(x) for x in paths) + 8 * len(paths), "flops": sum(len(x) for x in paths) + 1}
    # about one place in each width keeps its last page
    page, width = case["page"], case["width"]
    copied = sum((width - 1) * (n % page) for n in lens[::width])
    table = len(lens) * (max(lens) // page + 2)
    return {"bytes": 2 * copied * row + 8 * table + 24 * len(lens), "flops": table}


# ---------------------------------------------------------------------------
# the same passes in 64 bits (attention) or token by token (pages)
# ---------------------------------------------------------------------------
def _turn(x, table, index, back=False):
    """Pairs (2p, 2p+1) of x [n, heads, D] as complex numbers times e^(i angle); index < 0: as they are."""
    cos, sin = (t.double()[index.clamp(0, t.shape[0] - 1)] for t in table.tables())
    turn = torch.complex(cos, -sin if back else sin)
    turn[index < 0] = 1.0
    z = torch.view_as_complex(x.double().reshape(*x.shape[:-1], x.shape[-1] // 2, 2).contiguous()) * turn[:, None, :]
    return torch.view_as_real(z).reshape(x.shape)


def _exact_windows(case, state):
    """Sequence by sequence, head by head, 1024 queries at a time over the keys that one of them sees."""
    table, D, cls, W, S = state["table"], case["D"], int(case["cls"]), case["window"], case["sinks"]
    train, group, step = case["kind"] == "train", case["H"] // case["Hkv"], 1024
    outs = [torch.zeros_like(state["q"], dtype=torch.float64).detach()]
    if train:
        outs += [torch.zeros_like(state[n], dtype=torch.float64).detach() for n in ("q", "k", "v")]
    at = 0
    for n in _lengths(case):
        index = torch.arange(n, device=DEVICE) - cls
        q, k = (_turn(state[x].detach()[at:at + n], table, index) for x in ("q", "k"))
        v = state["v"].detach()[at:at + n].double()
        grads = [torch.zeros_like(x) for x in (q, k, v)]
        for i0 in range(0, n, step):
            i = torch.arange(i0, min(n, i0 + step), device=DEVICE)
            low = max(0, i0 - W + 1)
            j = torch.cat([torch.arange(min(S, low), device=DEVICE), torch.arange(low, int(i[-1]) + 1, device=DEVICE)])
            hidden = (j > i[:, None]) | ((i[:, None] - j >= W) & (j >= S))
            for h in range(case["H"]):
                qh, kh, vh = q[i, h], k[j, h // group], v[j, h // group]
                p = torch.softmax((qh @ kh.t() / math.sqrt(D)).masked_fill_(hidden, -math.inf), dim=-1)
                o = p @ vh
                outs[0][at + i, h] = o
                if not train:
                    continue
                g = state["do"][at + i, h].double()
                ds = p * (g @ vh.t() - (g * o).sum(1, keepdim=True)) / math.sqrt(D)
                grads[0][i, h] = ds @ kh
                grads[1][:, h // group].index_add_(0, j, ds.t() @ qh)
                grads[2][:, h // group].index_add_(0, j, p.t() @ g)
        if train:
            outs[1][at:at + n] = _turn(grads[0], table, index, back=True)
            outs[2][at:at + n] = _turn(grads[1], table, index, back=True)
            outs[3][at:at + n] = grads[2]
        at += n
    return tuple(outs)


def _exact_cached(case, state):
    """Sequence by sequence, key head by key head: decode's one token and the tokens of a tree or chunk."""
    lens, page, D, cls = _lengths(case), case["page"], case["D"], int(case["cls"])
    group, tree = case["H"] // case["Hkv"], case["kind"] == "tree"
    new = _drafted(case) if tree else [1] * len(lens)
    out, at = torch.zeros_like(state["q"], dtype=torch.float64), 0
    for b, (n, m) in enumerate(zip(lens, new)):
        total = n + m if tree else n
        if m == 0 or total == 0:
            at += m
            continue
        row = torch.arange(total, device=DEVICE)
        k, v = (state[c][state["pages"][b].long()].flatten(0, 1)[:total].double() for c in ("k_cache", "v_cache"))
        if not tree:
            index = torch.tensor([n - 1 - cls], device=DEVICE)
            hidden = ((row < n - case["window"]) & (row >= case["sinks"]))[None]
        elif case["chunk"]:
            index = torch.arange(n, total, device=DEVICE) - cls
            hidden = row[None] > torch.arange(n, total, device=DEVICE)[:, None]
        else:
            parents = _trees(case)[b]
            sees = []
            for i in range(m):
                way = {i}
                while parents[i] >= 0:
                    i = parents[i]
                    way.add(i)
                sees.append([x not in way for x in range(m)])
            index = torch.tensor([n + d - cls for d in _depths(parents)], device=DEVICE)
            hidden = torch.cat([torch.zeros(m, n, dtype=torch.bool), torch.tensor(sees)], dim=1).to(DEVICE)
        q = _turn(state["q"][at:at + m], state["table"], index)
        for h in range(case["H"]):
            s = (q[:, h] @ k[:, h // group].t() / math.sqrt(D)).masked_fill_(hidden, -math.inf)
            out[at:at + m, h] = torch.softmax(s, dim=-1) @ v[:, h // group]
        at += m
    return (out,)


def _exact_pages(case, state):
    page, pages = case["page"], state["pages"].tolist()
    lengths = state["lengths"].tolist()
    old = [state[n].clone() for n in ("k_cache", "v_cache")]
    out = [x.clone() for x in old]

    def copy(pairs):
        if pairs:
            (sg, sr), (tg, tr) = (torch.tensor(x, device=DEVICE).t() for x in zip(*pairs))
            for a, b in zip(old, out):
                b[tg, tr] = a[sg, sr]

    if case["kind"] == "accept":
        pairs, after = [], []
        for b, way in enumerate(state["path"].tolist()):
            way = way[: way.index(-1)] if -1 in way else way
            places = [[(pages[b][x // page], x % page) for x in (lengths[b] + j, lengths[b] + i)] for i, j in enumerate(way)]
            pairs += [(s, t) for s, t in places]
            after.append(lengths[b] + len(way))
        copy(pairs)
        return out[0], out[1], _ints(after)
    refs, room = state["refs"].tolist(), state["room"].tolist()
    free = [g for g, r in enumerate(refs) if r == 0]
    table, after, pairs, seen, missing = [], [], [], set(), 0
    for b, p in enumerate(state["parents"].tolist()):
        row = [-1] * len(pages[b])
        table.append(row)
        after.append(0 if p < 0 else lengths[p])
        if p < 0:
            continue
        full, used = divmod(lengths[p], page)
        for i, g in enumerate(pages[p]):
            if i < full or (g >= 0 and p not in seen and refs[g] == 1):
                row[i] = g
            elif i * page < lengths[p] + room[b]:
                if not free:
                    missing += 1
                    continue
                row[i] = free.pop(0)
                if i == full and g >= 0:
                    pairs += [((g, r), (row[i], r)) for r in range(used)]
        seen.add(p)
    copy(pairs)
    for rows, sign in ((pages, -1), (table, 1)):
        for row in rows:
            for g in row:
                if g >= 0:
                    refs[g] += sign
    return _ints(table), _ints(after), _ints(refs), out[0], out[1], _ints([missing])


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] in ("prompt", "train"):
        return _exact_windows(case, state)
    return _exact_cached(case, state) if case["kind"] in ("decode", "tree") else _exact_pages(case, state)
