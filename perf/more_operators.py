"""Performance cases of the stretch between the packed q, k, v projection and the output projection when a model answers token by
token: heads normed and rotated, keys and values kept in a paged cache, drafted tokens attending over it.

  heads   root-mean-square norm of every query and key head and the rotation by its token's position, in one pass;
  append  the same on the way into a paged cache: keys (normed, rotated) and values of new tokens, the queries beside them;
  attend  a tree of drafted tokens of each sequence over its cache; one token per sequence is its smallest form.

Formulas (all in 32 bits or more, rounded once where they are stored):
  n = x * (mean(x^2) + eps)^-1/2 * weight
  pairs (a, b) = (i, i + R/2), or interleaved (2i, 2i + 1):  n_a cos_i - n_b sin_i,  n_b cos_i + n_a sin_i;  i < R/2
  token t of a sequence is entry length + t of its cache: page table[entry div P], row entry mod P
  out = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - max), over the cached entries and those drafted tokens whose bit is
  set in the token's mask; zeros where there is none

``listed()`` are fixed cases, ``draw(rng)`` gives further ones of the same ranges, ``prepare`` makes what a program holds
before the call, ``run`` is one pass: through elementary torch operations, or with ``own`` through the package.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _heads(name, batch, tokens, hq, hk, d, rotary, dtype="bf16", norm=True, interleaved=False, packed=True):
    c = dict(kind="heads", batch=batch, tokens=tokens, hq=hq, hk=hk, d=d, rotary=rotary, dtype=dtype, norm=norm,
             interleaved=interleaved, packed=packed)
    return dict(c, name=name) if name else c


def _append(name, batch, tokens, hq, hk, d, rotary, length, page, dtype="bf16", norm=True, interleaved=False, ragged=False):
    c = dict(kind="append", batch=batch, tokens=tokens, hq=hq, hk=hk, d=d, rotary=rotary, length=length, page=page, dtype=dtype,
             norm=norm, interleaved=interleaved, ragged=ragged)
    return dict(c, name=name) if name else c


def _attend(name, batch, tokens, hq, hk, d, length, page, dtype="bf16", tree=False, ragged=False):
    c = dict(kind="attend", batch=batch, tokens=tokens, hq=hq, hk=hk, d=d, length=length, page=page, dtype=dtype, tree=tree,
             ragged=ragged)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token of a generating model of 768 channels, nothing cached: latency alone
        _heads("heads_1x12x64", 1, 1, 12, 12, 64, 64),
        # 256 images of 197 tokens, ViT-Tiny's heads as a slice of the packed projection
        _heads("heads_50432x3x64", 256, 197, 3, 3, 64, 64),
        # eight sequences of 16384 tokens, 768 channels: the longest of the layer benchmark
        _heads("heads_131072x12x64", 8, 16384, 12, 12, 64, 64),
        # float32, an odd number of tokens, one shared key head, half of the channels rotated, neighbours as pairs, no norm
        _heads("heads_fp32_4099x5x80", 1, 4099, 5, 1, 80, 40, dtype="fp32", norm=False, interleaved=True),
        # the next token of one sequence: latency alone
        _append("append_1x1", 1, 1, 32, 8, 128, 128, 5000, 64),
        # eight prompts of 4096 tokens behind what is cached
        _append("append_8x4096", 8, 4096, 32, 8, 128, 128, 1000, 64),
        # float32 trees of up to 37 tokens, some shorter, in odd pages, neighbours as pairs, half rotated
        _append("append_fp32_5x37", 5, 37, 6, 2, 80, 40, 3000, 20, dtype="fp32", interleaved=True, ragged=True),
        # the next token of one short sequence, as many key as query heads: latency alone
        _attend("attend_1x1x1000", 1, 1, 12, 12, 64, 1000, 64),
        # a few dozen sequences of different lengths in decoding
        _attend("attend_48x1x16384", 48, 1, 32, 8, 128, 16384, 64, ragged=True),
        # one very long sequence
        _attend("attend_1x1x131072", 1, 1, 32, 8, 128, 131072, 64),
        # trees of 64 drafted tokens
        _attend("attend_tree_16x64x16384", 16, 64, 32, 8, 128, 16384, 64, tree=True, ragged=True),
        # float32, small, odd in every direction
        _attend("attend_fp32_tree_3x13x1777", 3, 13, 6, 2, 80, 1777, 20, dtype="fp32", tree=True, ragged=True),
    ]


MOST_HEADS = 8 * 4096 * 48 * 128                    # values that pass through heads or append
MOST_CACHED = 48 * 16384 * 8 * 128                  # keys of a cache
MOST_SCORES = 16 * 64 * 32 * 16384 * 128            # products of queries and keys


def _between(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["heads", "append", "attend", "attend"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    hk = rng.choice([1, 2, 3, 4, 8, 12])
    hq = hk * rng.choice([1, 1, 2, 3, 4, 7, 8])
    d = rng.choice([64, 64, 80, 96, 128, 128, 192, 256])
    rotary = rng.choice([d, d, d // 2])
    page = rng.choice([16, 32, 64, 128, 20, 48])
    norm, interleaved, ragged = rng.random() < 0.7, rng.random() < 0.3, rng.random() < 0.6
    half = 2 if dtype == "fp32" else 1
    if kind == "heads":
        rows = _between(rng, 1, MOST_HEADS // (half * (hq + hk) * d))
        batch = min(rows, _between(rng, 1, 256))
        return _heads(None, batch, rows // batch, hq, hk, d, rotary, dtype, norm, interleaved, rng.random() < 0.7)
    if kind == "append":
        rows = _between(rng, 1, MOST_HEADS // (half * (hq + 2 * hk) * d))
        batch = min(rows, _between(rng, 1, 64))
        room = MOST_CACHED // (half * batch * hk * d) - rows // batch
        length = _between(rng, 1, max(1, min(8192, room)))
        return _append(None, batch, rows // batch, hq, hk, d, rotary, length, page, dtype, norm, interleaved, ragged)
    batch, tokens = _between(rng, 1, 64), rng.choice([1, 1, _between(rng, 2, 64)])
    # (float32 products run off the tensor cores: a sixteenth of the work)
    most = min(131072, MOST_CACHED // (half * batch * hk * d), MOST_SCORES // (batch * tokens * hq * d) // (16 if dtype == "fp32" else 1))
    length = _between(rng, 16, max(16, most))
    return _attend(None, batch, tokens, hq, hk, d, length, page, dtype, tokens > 1 and rng.random() < 0.7, ragged)


# ---- what a program holds -------------------------------------------------------------------------------------------

def _table(rows, rotary):
    """cos | sin of the positions' angles, computed in 64 bits."""
    at = torch.arange(rows, device="cuda", dtype=torch.float64)
    freq = 10000.0 ** (-torch.arange(rotary // 2, device="cuda", dtype=torch.float64) / (rotary // 2))
    angle = at[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def _lengths(case, rng):
    b, top = case["batch"], case["length"]
    return rng.randint(top // 4, top + 1, b) if case["ragged"] else np.full(b, top)


def _drafted(case, lengths, rng):
    """Positions, masks and counts of trees of drafted tokens: each token's parent is one of the last few before it."""
    b, t = case["batch"], case["tokens"]
    depth, mask = np.zeros((b, t), np.int64), np.zeros((b, t), np.uint64)
    mask[:, 0] = 1
    every = np.arange(b)
    for i in range(1, min(t, 64)):
        parent = np.maximum(0, i - 1 - rng.geometric(0.4, b) + 1)
        depth[:, i] = depth[every, parent] + 1
        mask[:, i] = mask[every, parent] | np.uint64(1 << i)
    counts = rng.randint((t + 1) // 2, t + 1, b) if case["ragged"] else np.full(b, t)
    cuda = lambda a, dtype: torch.from_numpy(np.ascontiguousarray(a)).to(dtype).cuda()  # noqa: E731
    return cuda(lengths[:, None] + depth, torch.int32), cuda(mask.view(np.int64), torch.int64), cuda(counts, torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.RandomState(seed % (1 << 32))
    dtype, b, t, hq, hk, d = TYPES[case["dtype"]], case["batch"], case["tokens"], case["hq"], case["hk"], case["d"]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    s = dict(case, dtype=dtype, positions=None)
    if case["kind"] == "heads":
        # (`packed`: slices of the projection's rows, values behind them)
        rows = (randn(b, t, hq + (2 if case["packed"] else 1) * hk, d) * 1.5).to(dtype)
        s.update(q=rows[:, :, :hq], k=rows[:, :, hq:hq + hk])
        if not case["packed"]:
            s.update(q=s["q"].contiguous(), k=s["k"].contiguous())
        s["rope"] = _table(t, case["rotary"])
    else:
        lengths = _lengths(case, rng)
        s["lengths"] = torch.from_numpy(lengths).to(torch.int32).cuda()
        pages = -(-(case["length"] + t) // case["page"])
        order = rng.permutation(b * pages).reshape(b, pages)
        s["table"] = torch.from_numpy(order).to(torch.int32).cuda()
        s["cache_k"], s["cache_v"] = (randn(b * pages, hk, case["page"], d).to(dtype) for _ in range(2))
        s["tree"] = s["counts"] = None
        if case["kind"] == "append":
            rows = (randn(b, t, hq + 2 * hk, d) * 1.5).to(dtype)
            s.update(q=rows[:, :, :hq], k=rows[:, :, hq:hq + hk], v=rows[:, :, hq + hk:])
            s["rope"] = _table(case["length"] + t, case["rotary"])
            if case["ragged"]:
                positions, _, s["counts"] = _drafted(case, lengths, rng)
                s["positions"] = positions if t <= 64 else None
        else:
            s["q"] = randn(b, t, hq, d).to(dtype)
            if case["tree"]:
                _, s["tree"], s["counts"] = _drafted(case, lengths, rng)
    if case["kind"] != "attend":
        s["q_weight"], s["k_weight"] = ((1.0 + 0.2 * randn(d)).to(dtype) if case["norm"] else None for _ in range(2))
    return s


def run(state):
    s = state
    if own:
        from convnn_b200 import ops
        if s["kind"] == "heads":
            return ops.qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["rope"], eps=EPS, interleaved=s["interleaved"])
        cache = ops.PagedCache(s["cache_k"], s["cache_v"], s["table"])
        if s["kind"] == "append":
            q = ops.append_kv(cache, s["k"], s["v"], s["lengths"], q=s["q"], q_weight=s["q_weight"], k_weight=s["k_weight"],
                              rope=s["rope"], positions=s["positions"], counts=s["counts"], eps=EPS, interleaved=s["interleaved"])
            return q, s["cache_k"], s["cache_v"]
        return ops.tree_attention(s["q"], cache, s["lengths"], tree=s["tree"], counts=s["counts"])
    if s["kind"] == "heads":
        at = torch.arange(s["q"].shape[1], device="cuda")
        return tuple(_plain_heads(s[x], s[x + "_weight"], s["rope"][at], s["interleaved"]) for x in "qk")
    return _plain_append(s) if s["kind"] == "append" else _plain_attend(s)


# ---- the plain form -------------------------------------------------------------------------------------------------

def _plain_heads(x, weight, rope, interleaved):
    """x (..., tokens, heads, d), rope (..., tokens, rotary)."""
    n, half = x.float(), rope.shape[-1] // 2
    if weight is not None:
        n = n * torch.rsqrt((n * n).mean(dim=-1, keepdim=True) + EPS) * weight.float()
    cos, sin = rope[..., None, :half], rope[..., None, half:]
    y = n.clone()
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    y[..., a] = n[..., a] * cos - n[..., b] * sin
    y[..., b] = n[..., b] * cos + n[..., a] * sin
    return y.to(x.dtype)


def _plain_append(s):
    b, t, page = s["batch"], s["tokens"], s["page"]
    new = torch.arange(t, device="cuda")
    entry = s["lengths"].long()[:, None] + new
    rope = s["rope"][entry if s["positions"] is None else s["positions"].long()]
    live = torch.ones(b, t, dtype=torch.bool, device="cuda") if s["counts"] is None else new < s["counts"][:, None]
    seq = torch.arange(b, device="cuda")[:, None].expand(b, t)[live]
    entry = entry[live]
    at, row = s["table"][seq, entry // page].long(), entry % page
    s["cache_k"][at, :, row] = _plain_heads(s["k"], s["k_weight"], rope, s["interleaved"])[live]
    s["cache_v"][at, :, row] = s["v"][live]
    q = _plain_heads(s["q"], s["q_weight"], rope, s["interleaved"])
    return q.masked_fill_(~live[..., None, None], 0), s["cache_k"], s["cache_v"]


def _visible(s, entries):
    """(batch, tokens, entries): what each drafted token sees."""
    t = s["tokens"]
    counts = torch.full_like(s["lengths"], t) if s["counts"] is None else s["counts"]
    drafted = torch.arange(entries, device="cuda") - s["lengths"][:, None]                   # (batch, entries)
    bits = s["tree"]
    if bits is None:                                       # a chain: what came before, and itself
        bits = (torch.bitwise_left_shift(torch.full((t,), 2, device="cuda"), torch.arange(t, device="cuda")) - 1).expand(s["batch"], t)
    seen = torch.bitwise_right_shift(bits[:, :, None], drafted.clamp(0, 63)[:, None]) & 1
    new = (drafted >= 0) & (drafted < counts[:, None])
    live = torch.arange(t, device="cuda") < counts[:, None]
    return ((drafted < 0)[:, None] | (new[:, None] & (seen == 1))) & live[..., None]


def _plain_attend(s):
    b, t, hq, hk, d = s["batch"], s["tokens"], s["hq"], s["hk"], s["d"]
    table = s["table"].long()
    k, v = (s[c][table].float().transpose(1, 2).reshape(b, hk, -1, d) for c in ("cache_k", "cache_v"))
    q = s["q"].float().view(b, t, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)
    scores = (q @ k.transpose(2, 3)).view(b, hk, hq // hk, t, -1) * d ** -0.5
    seen = _visible(s, k.shape[2])[:, None, None]
    scores = scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(dim=-1, keepdim=True).clamp(min=-1e30)
    p = scores.sub_(top).exp_()
    total = p.sum(dim=-1, keepdim=True)
    out = (p.view(b, hk, -1, k.shape[2]) @ v).view(b, hk, hq // hk, t, d) / total.clamp(min=1e-30)
    return out.permute(0, 3, 1, 2, 4).reshape(b, t, hq, d).to(s["dtype"])


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

def work(case):
    elt = 4 if case["dtype"] == "fp32" else 2
    b, t, hq, hk, d = case["batch"], case["tokens"], case["hq"], case["hk"], case["d"]
    if case["kind"] == "attend":
        entries = b * ((0.625 if case["ragged"] else 1.0) * case["length"] + t)
        return {"bytes": elt * (2 * entries * hk * d + 2 * b * t * hq * d), "flops": 4 * entries * t * hq * d}
    values = b * t * (hq + hk) * d
    moved = 2 * elt * values
    if case["kind"] == "append":
        moved += 2 * elt * b * t * hk * d
        table = b * t
    else:
        table = t
    return {"bytes": moved + 4 * table * case["rotary"], "flops": (4 * case["norm"] + 3) * values}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------

def _exact_heads(x, weight, cos, sin, interleaved):
    """Pairs as complex numbers, turned by (cos + i sin)."""
    x = x.double()
    if weight is not None:
        square = torch.einsum("...d,...d->...", x, x) / x.shape[-1]
        x = torch.einsum("...d,d,...->...d", x, weight.double(), 1.0 / torch.sqrt(square + EPS))
    turn, half = torch.complex(cos.double(), sin.double()).unsqueeze(-2), cos.shape[-1]
    if interleaved:
        pair = torch.view_as_complex(x[..., :2 * half].reshape(*x.shape[:-1], half, 2).contiguous()) * turn
        first = torch.view_as_real(pair).flatten(-2)
    else:
        pair = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * turn
        first = torch.cat([pair.real, pair.imag], -1)
    return torch.cat([first, x[..., 2 * half:]], -1)


def exact(case, seed):
    s = prepare(case, seed)
    b, t, hq, hk, d, page = s["batch"], s["tokens"], s["hq"], s["hk"], s["d"], case.get("page")
    half = case.get("rotary", 0) // 2
    if case["kind"] == "heads":
        out = []
        for x in "qk":
            rows = [_exact_heads(s[x][i], s[x + "_weight"], s["rope"][:, :half], s["rope"][:, half:], s["interleaved"]) for i in range(b)]
            out.append(torch.stack(rows))
        return out
    lengths = s["lengths"].tolist()
    counts = [t] * b if s["counts"] is None else s["counts"].tolist()
    if case["kind"] == "append":
        q_out = torch.zeros(b, t, hq, d, dtype=torch.float64, device="cuda")
        keys, values = s["cache_k"].double(), s["cache_v"].double()
        for i in range(b):
            n, first = counts[i], lengths[i]
            at = torch.arange(first, first + n, device="cuda")
            rope = s["rope"][at if s["positions"] is None else s["positions"][i, :n].long()]
            turned = [_exact_heads(s[x][i, :n], s[x + "_weight"], rope[:, :half], rope[:, half:], s["interleaved"]) for x in "qk"]
            q_out[i, :n] = turned[0]
            where = s["table"][i].long()[torch.div(at, page, rounding_mode="floor")]
            keys.index_put_((where[:, None], torch.arange(hk, device="cuda")[None], (at % page)[:, None]), turned[1])
            values.index_put_((where[:, None], torch.arange(hk, device="cuda")[None], (at % page)[:, None]), s["v"][i, :n].double())
        return [q_out, keys, values]
    out = torch.zeros(b, t, hq, d, dtype=torch.float64, device="cuda")
    for i in range(b):
        n, first = counts[i], lengths[i]
        pages = s["table"][i].long()[:-(-(first + n) // page)]
        k, v = (s[c][pages].double().transpose(0, 1).flatten(1, 2)[:, :first + n] for c in ("cache_k", "cache_v"))
        masks = s["tree"][i].tolist() if s["tree"] is not None else [(2 << j) - 1 for j in range(n)]
        seen = torch.ones(n, first + n, dtype=torch.bool)
        for j in range(n):
            seen[j, first:] = torch.tensor([masks[j] >> e & 1 == 1 for e in range(n)])
        hidden = ~seen.cuda()
        for h in range(hk):
            group = slice(h * (hq // hk), (h + 1) * (hq // hk))
            logits = torch.einsum("tgd,ed->gte", s["q"][i, :n, group].double(), k[h]) / math.sqrt(d)
            share = torch.softmax(logits.masked_fill(hidden, -math.inf), -1)
            out[i, :n, group] = torch.einsum("gte,ed->tgd", share, v[h])
    return out
