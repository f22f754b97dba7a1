"""The calls that the speed of the packed and cached attention is judged by.

A case is one pass through one of the operators of autoregressive models with
rotary positions (an image generator over its token grid, a text decoder):

* ``append``: new keys and values go to a paged cache, the keys rotated on the way;
* ``decode``: one new token per sequence attends to its cached keys;
* ``prompt``: attention over whole packed sequences, the forward alone;
* ``train``: the same with its gradients.

``listed`` names twelve of them; ``draw`` gives further ones of the same ranges:

* head_dim 32, 64, 128 and 256; bf16, fp16 and fp32; 1 to 16 query heads per key head;
* appends of one token per sequence, or of whole prompts, up to 16 K tokens; pages of 1 to 256 rows;
* caches from one row to 128 K rows a sequence, 1 to 256 sequences of different lengths;
* packs of 1 to 128 sequences of 1 to 16 K tokens, causal or not.

Tables are those of a square token grid (the class token in front of it is not
rotated).  Queries, keys and values of a prompt are views of one projection's output.
"""
import math
import random

import torch

own = False

ROPE_BASE = 100.0
DEVICE = "cuda"

# seqs, longest: the sequences and the longest one's length (append: the cached tokens before
# the call; decode: after it); ragged: the others are shorter; new: appended tokens (0: one per
# sequence); page: rows a page holds; pad: the last sequence is an empty place of the batch
_DEFAULT = dict(kind="train", seqs=1, longest=197, ragged=False, H=12, Hkv=12, D=64, dtype="bf16",
                causal=True, cls=True, page=16, new=0, pad=False)


def _case(name, **kw):
    return dict(_DEFAULT, name=name, **kw)


def listed():
    return [
        # The next token of one sequence: the latency of an append.
        _case("append_one", kind="append", longest=196),
        # One step of a served batch.
        _case("append_step_fp16", kind="append", seqs=64, longest=2048, ragged=True, Hkv=8, D=128, dtype="fp16", page=32),
        # The keys of a batch of prompts enter an empty cache.
        _case("append_prompt", kind="append", seqs=9, longest=0, new=8200, Hkv=8, D=128, page=64),
        # One token of one short sequence (a 14x14 token grid behind a class token).
        _case("decode_one", kind="decode", longest=197),
        # A served batch at different stages, one of its places empty, shared key heads.
        _case("decode_batch", kind="decode", seqs=48, longest=4097, ragged=True, H=16, Hkv=4, D=128, pad=True),
        # Two long documents: few sequences, so the cache's length is what there is to divide.
        _case("decode_long", kind="decode", seqs=2, longest=100000, ragged=True, H=32, Hkv=8, D=128, page=64),
        # A reference run in plain fp32.
        _case("decode_fp32", kind="decode", seqs=5, longest=1025, ragged=True, H=8, Hkv=8, dtype="fp32"),
        # One short prompt served alone.
        _case("prompt_one", kind="prompt"),
        # Prompts of a served batch, shared key heads, fp16.
        _case("prompt_packed_fp16", kind="prompt", seqs=24, longest=2048, ragged=True, H=16, Hkv=4, D=128, dtype="fp16"),
        # A training batch of token grids up to 24x24 + class token.
        _case("train_packed", seqs=64, longest=577, ragged=True),
        # Training on one long sequence, four query heads per key head.
        _case("train_long", longest=16384, H=8, Hkv=2, D=128, cls=False),
        # A small training step in plain fp32 (a debugging or reference run).
        _case("train_fp32", seqs=3, longest=257, ragged=True, H=8, Hkv=4, dtype="fp32"),
    ]


# What no drawn case may exceed: the listed cases' largest operation count and traffic, and the
# score matrix that the plain form holds.
_MOST_FLOPS = 1.9e12
_MOST_BYTES = 8.0e8
_MOST_SCORES = 2.1e9


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    while True:
        c = dict(_DEFAULT)
        c["kind"] = rng.choice(["append", "decode", "decode", "prompt", "train", "train"])
        c["D"] = rng.choice([32, 64, 64, 128, 128, 128, 256])
        c["dtype"] = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp16", "fp32"])
        c["Hkv"] = rng.choice([1, 2, 3, 4, 6, 8, 8, 12])
        c["H"] = c["Hkv"] * rng.choice([1, 1, 2, 3, 4, 4, 7, 8, 16])
        c["cls"] = rng.random() < 0.6
        c["ragged"] = rng.random() < 0.8
        c["page"] = rng.choice([1, 7, 16, 16, 32, 64, 100, 128, 256])
        if c["kind"] == "append":
            c["H"] = c["Hkv"]
            if rng.random() < 0.5:
                c["seqs"], c["longest"] = _log_int(rng, 1, 256), _log_int(rng, 1, 8192)
            else:
                c["seqs"], c["longest"], c["new"] = _log_int(rng, 1, 32), rng.choice([0, 0, 333]), _log_int(rng, 1, 16384)
                c["seqs"] = min(c["seqs"], c["new"])
        elif c["kind"] == "decode":
            c["seqs"], c["longest"] = _log_int(rng, 1, 256), _log_int(rng, 1, 131072)
            c["pad"] = c["seqs"] > 2 and rng.random() < 0.3
        else:
            c["seqs"], c["longest"] = _log_int(rng, 1, 128), _log_int(rng, 1, 16384)
            c["causal"] = rng.random() < 0.8
        w = work(c)
        slow = 12 if c["dtype"] == "fp32" else 1
        scores = c["seqs"] * c["H"] * max(1, c["longest"]) ** (2 if c["kind"] in ("prompt", "train") else 1)
        cache = c["seqs"] * (max(_lengths(c)) + c["page"]) * c["Hkv"] * c["D"] * (4 if c["kind"] == "decode" else 16)
        if w["flops"] * slow <= _MOST_FLOPS and w["bytes"] <= _MOST_BYTES and scores <= _MOST_SCORES and cache <= 4e9:
            return c


def _lengths(case):
    """The sequences' lengths (append of prompts: the new tokens), the same for every seed."""
    n, most = case["seqs"], case["longest"]
    rng = random.Random("%d %d %d" % (n, most, case["new"]))
    if case["kind"] == "append" and case["new"]:
        cuts = sorted(rng.randint(0, case["new"]) for _ in range(n - 1))
        return [b - a for a, b in zip([0] + cuts, cuts + [case["new"]])]
    if not case["ragged"]:
        lens = [most] * n
    else:
        lens = [max(min(1, most), int(most * 16.0 ** -rng.random())) for _ in range(n)]
        lens[rng.randrange(n)] = most
    if case["pad"]:
        lens[-1] = 0
    return lens


def _pairs(case):
    return sum(n * (n + 1) // 2 if case["causal"] else n * n for n in _lengths(case))


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


def _pages(case, capacity, gen):
    """A page table [seqs, pages] over a shuffled pool, and the pool's size."""
    per = max(1, -(-capacity // case["page"]))
    total = case["seqs"] * per + 3
    order = torch.randperm(total, generator=gen, device=DEVICE).to(torch.int32)
    return order[: case["seqs"] * per].reshape(case["seqs"], per).contiguous(), total


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    kind, H, Hkv, D, dt = case["kind"], case["H"], case["Hkv"], case["D"], _dtype(case)
    lens = _lengths(case)

    def randn(*shape):
        return torch.randn(shape, generator=gen, device=DEVICE).to(dt)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=DEVICE)

    def starts(values):
        return ints([sum(values[:i]) for i in range(len(values) + 1)])

    state = {"case": dict(case), "most": max(lens)}
    if kind in ("append", "decode"):
        prompt = kind == "append" and case["new"] > 0
        before = [case["longest"]] * len(lens) if prompt else lens
        capacity = max(a + b for a, b in zip(before, lens if prompt else [1] * len(lens)))
        table, total = _pages(case, capacity, gen)
        state["k_cache"], state["v_cache"] = randn(total, case["page"], Hkv, D), randn(total, case["page"], Hkv, D)
        state["pages"], state["lengths"] = table, ints(before)
        state["table"] = _Table(capacity, D)
        if kind == "decode":
            state["q"] = randn(len(lens), H, D)
        else:
            state["starts"] = starts(lens) if prompt else None
            new = sum(lens) if prompt else len(lens)
            state["k"], state["v"] = randn(new, 2, Hkv, D).unbind(1)
        return state
    T = sum(lens)
    qkv = randn(T, H + 2 * Hkv, D)
    state["q"], state["k"], state["v"] = (
        t.detach().requires_grad_(kind == "train") for t in qkv.split([H, Hkv, Hkv], dim=1))
    if kind == "train":
        state["do"] = randn(T, H, D)
    state["starts"], state["table"] = starts(lens), _Table(state["most"], D)
    return state


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _cos_sin(state, pos):
    """Rows of the table for token indexes `pos`, [..., 1, D/2]: the class token is not rotated."""
    cos, sin = state["table"].tables()
    at = pos.long() - int(state["case"]["cls"])
    row = at.clamp(0, cos.shape[0] - 1)
    none = (at < 0)[..., None]
    return torch.where(none, 1.0, cos[row])[..., None, :], torch.where(none, 0.0, sin[row])[..., None, :]


def _rotate(x, cos, sin):
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)


def _token_places(starts, n):
    """Sequence and index within it of each of the n packed tokens."""
    at = torch.arange(n, device=DEVICE)
    seq = torch.searchsorted(starts[1:].long(), at, right=True)
    return seq, at - starts.long()[seq]


def _append(state):
    k, v, page, pages = state["k"], state["v"], state["case"]["page"], state["pages"]
    if state["starts"] is None:
        seq = torch.arange(k.shape[0], device=DEVICE)
        pos = state["lengths"].long()
    else:
        seq, at = _token_places(state["starts"], k.shape[0])
        pos = state["lengths"].long()[seq] + at
    slot = pages[seq, pos // page].long() * page + pos % page
    rotated = _rotate(k.float(), *_cos_sin(state, pos)).to(k.dtype)
    state["k_cache"].view(-1, *k.shape[1:])[slot] = rotated
    state["v_cache"].view(-1, *v.shape[1:])[slot] = v
    return state["k_cache"], state["v_cache"]


def _softmax(s, keep):
    s = torch.where(keep, s, -torch.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isfinite(top), top, 0.0))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total > 0, total, 1.0)


def _decode(state):
    q, lengths = state["q"], state["lengths"]
    B, H, D = q.shape
    Hkv = state["k_cache"].shape[2]
    keys, values = (state[n][state["pages"].long()].float().reshape(B, -1, Hkv, D) for n in ("k_cache", "v_cache"))
    qh = _rotate(q.float(), *_cos_sin(state, lengths.clamp(min=1) - 1)).reshape(B, Hkv, H // Hkv, D)
    keep = torch.arange(keys.shape[1], device=DEVICE) < lengths[:, None]
    keys = torch.where(keep[..., None, None], keys, 0.0)
    values = torch.where(keep[..., None, None], values, 0.0)
    s = torch.matmul(qh, keys.permute(0, 2, 3, 1)) * D ** -0.5
    p = _softmax(s, keep[:, None, None, :])
    return torch.matmul(p, values.permute(0, 2, 1, 3)).reshape(B, H, D).to(q.dtype)


def _attention(state):
    case, q, starts, most = state["case"], state["q"], state["starts"].long(), state["most"]
    T, H, D = q.shape
    Hkv, group = state["k"].shape[1], H // state["k"].shape[1]
    at = torch.arange(most, device=DEVICE)
    place = (starts[:-1, None] + at).clamp(max=T - 1)                     # [B, L]
    inside = at < (starts[1:] - starts[:-1])[:, None]
    cos, sin = _cos_sin(state, at)

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
    keep = inside[:, None, None, :]
    keep = keep & (at[None, :] <= at[:, None]) if case["causal"] else keep
    p = _softmax(torch.matmul(qh, kh.transpose(2, 3)) * D ** -0.5, keep)
    o = torch.matmul(p, vh)
    if case["kind"] == "prompt":
        return (packed(o, False),)
    g = padded(state["do"], False)
    dv = torch.matmul(p.transpose(2, 3), g)
    ds = torch.matmul(g, vh.transpose(2, 3)) - (g * o).sum(-1, keepdim=True)
    ds = ds.mul_(p).mul_(D ** -0.5)
    del p
    dq, dk = torch.matmul(ds, kh), torch.matmul(ds.transpose(2, 3), qh)
    dk, dv = (x.reshape(-1, Hkv, group, most, D).sum(2) for x in (dk, dv))
    return packed(o, False), packed(dq, True), packed(dk, True), packed(dv, False)


def _own(state):
    from triton_fused_rope_flash_attn_amd import rope_cache_append, sdpa_rope_decode, sdpa_rope_varlen

    case = state["case"]
    if case["kind"] == "append":
        rope_cache_append(state["k"], state["v"], state["table"], state["k_cache"], state["v_cache"], state["pages"],
                          state["lengths"], cu_seqlens=state["starts"], has_cls=case["cls"])
        return state["k_cache"], state["v_cache"]
    if case["kind"] == "decode":
        return (sdpa_rope_decode(state["q"], state["k_cache"], state["v_cache"], state["table"], state["pages"],
                                 state["lengths"], has_cls=case["cls"]),)
    args = (state["q"], state["k"], state["v"], state["table"], state["starts"])
    out = sdpa_rope_varlen(*args, causal=case["causal"], has_cls=case["cls"])
    if case["kind"] == "prompt":
        return (out,)
    return (out.detach(), *torch.autograd.grad(out, args[:3], state["do"]))


def run(state):
    if own:
        return _own(state)
    if state["case"]["kind"] == "append":
        return _append(state)
    if state["case"]["kind"] == "decode":
        return (_decode(state),)
    return _attention(state)


def work(case):
    H, Hkv, D, e = case["H"], case["Hkv"], case["D"], 4 if case["dtype"] == "fp32" else 2
    n = sum(_lengths(case))
    if case["kind"] == "append":
        n = case["new"] or case["seqs"]
        return {"bytes": n * (4 * Hkv * D * e + 4 * D + 4), "flops": 3 * n * Hkv * D}
    if case["kind"] == "decode":
        return {"bytes": 2 * n * Hkv * D * e + case["seqs"] * (2 * H * D * e + 4 * D) + 4 * n // case["page"],
                "flops": 4 * n * H * D}
    train = case["kind"] == "train"
    return {"bytes": (2 if train else 1) * 2 * n * (H + Hkv) * D * e + 4 * case["longest"] * D,
            "flops": (14 if train else 4) * _pairs(case) * H * D}


# ---------------------------------------------------------------------------
# the same passes in 64 bits, sequence by sequence
# ---------------------------------------------------------------------------
def _turn(x, table, index, back=False):
    """Pairs (2p, 2p+1) of x [n, heads, D] as complex numbers times e^(i angle); index < 0: as they are."""
    cos, sin = (t.double()[index.clamp(min=0)] for t in table.tables())
    turn = torch.complex(cos, -sin if back else sin)
    turn[index < 0] = 1.0
    z = torch.view_as_complex(x.double().reshape(*x.shape[:-1], x.shape[-1] // 2, 2).contiguous()) * turn[:, None, :]
    return torch.view_as_real(z).reshape(x.shape)


def exact(case, seed):
    state = prepare(case, seed)
    table, lens, D, cls = state["table"], _lengths(case), case["D"], int(case["cls"])
    group = case["H"] // case["Hkv"]
    if case["kind"] == "append":
        out = [state[n].double().clone() for n in ("k_cache", "v_cache")]
        at, pages, page = 0, state["pages"].tolist(), case["page"]
        for b, before in enumerate(state["lengths"].tolist()):
            n = lens[b] if case["new"] else 1
            pos = range(before, before + n)
            kh = _turn(state["k"][at:at + n], table, torch.arange(before, before + n, device=DEVICE) - cls)
            where = torch.tensor([pages[b][p // page] * page + p % page for p in pos], dtype=torch.long, device=DEVICE)
            out[0].view(-1, case["Hkv"], D)[where] = kh
            out[1].view(-1, case["Hkv"], D)[where] = state["v"][at:at + n].double()
            at += n
        return tuple(out)
    if case["kind"] == "decode":
        rows = []
        for b, n in enumerate(lens):
            if n == 0:
                rows.append(torch.zeros(case["H"], D, dtype=torch.float64, device=DEVICE))
                continue
            k, v = (state[c][state["pages"][b].long()].reshape(-1, case["Hkv"], D)[:n].double().transpose(0, 1)
                    for c in ("k_cache", "v_cache"))
            q = _turn(state["q"][b:b + 1], table, torch.tensor([n - 1 - cls], device=DEVICE))
            q = q.reshape(case["Hkv"], group, D)
            p = torch.softmax(torch.bmm(q, k.transpose(1, 2).contiguous()) / math.sqrt(D), dim=-1)
            rows.append(torch.bmm(p, v.contiguous()).reshape(case["H"], D))
        return (torch.stack(rows),)
    if case["kind"] == "train" and work(case)["flops"] > 2.0e12:
        return None
    train = case["kind"] == "train"
    outs = [torch.zeros_like(state["q"], dtype=torch.float64).detach()]
    if train:
        outs += [torch.zeros_like(state[n], dtype=torch.float64).detach() for n in ("q", "k", "v")]
    at = 0
    for n in lens:
        index = torch.arange(n, device=DEVICE) - cls
        q, k = (_turn(state[x].detach()[at:at + n], table, index) for x in ("q", "k"))
        v = state["v"].detach()[at:at + n].double()
        later = torch.arange(n, device=DEVICE)[None, :] > torch.arange(n, device=DEVICE)[:, None]
        grads = [torch.zeros_like(x) for x in (q, k, v)]
        for h in range(case["H"]):
            qh, kh, vh = q[:, h].contiguous(), k[:, h // group].contiguous(), v[:, h // group].contiguous()
            s = qh @ kh.t() / math.sqrt(D)
            if case["causal"]:
                s.masked_fill_(later, -math.inf)
            p = torch.softmax(s, dim=-1)
            del s
            o = p @ vh
            outs[0][at:at + n, h] = o
            if not train:
                continue
            g = state["do"][at:at + n, h].double()
            grads[2][:, h // group] += p.t() @ g
            ds = p * (g @ vh.t() - (g * o).sum(1, keepdim=True)) / math.sqrt(D)
            grads[0][:, h] = ds @ kh
            grads[1][:, h // group] += ds.t() @ qh
        if train:
            outs[1][at:at + n] = _turn(grads[0], table, index, back=True)
            outs[2][at:at + n] = _turn(grads[1], table, index, back=True)
            outs[3][at:at + n] = grads[2]
        at += n
    return tuple(outs)
