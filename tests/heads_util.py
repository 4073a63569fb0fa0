"""The formulas of the heads' norm and rotation, of the paged cache and of attention over it, in 64 bits, and how far a kernel may be
off them.

Tolerances.  A rounding is off by half a step at most, relative to the value: ``HALF`` (bfloat16 2^-8, float32 2^-24).  Float32 sums of n
terms are off by n * 2^-24 of the sum of magnitudes (2^-23, truncated, on the tensor cores)."""
import torch

U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: U}


def randn(*shape, seed=0, dtype=torch.float32, scale=1.0, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    return (torch.randn(*shape, device=device, generator=g) * scale).to(dtype)


def rope_table(rows, rotary, device="cuda"):
    at = torch.arange(rows, device=device, dtype=torch.float64)
    angle = at[:, None] * 10000.0 ** (-torch.arange(rotary // 2, device=device, dtype=torch.float64) / max(1, rotary // 2))
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def turned(x, weight, rows, eps, interleaved):
    """x (..., tokens, heads, D), rows (..., tokens, R) of the table or None -> (exact, off): off bounds the error before rounding."""
    n = x.double()
    D = n.shape[-1]
    if weight is not None:
        n = n / torch.sqrt((n * n).mean(-1, keepdim=True) + eps) * weight.double()
    y, size = n.clone(), n.abs()
    if rows is not None:
        half = rows.shape[-1] // 2
        cos, sin = rows[..., None, :half].double(), rows[..., None, half:].double()
        a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
        y[..., a], y[..., b] = n[..., a] * cos - n[..., b] * sin, n[..., b] * cos + n[..., a] * sin
        size = size.clone()
        size[..., a], size[..., b] = (n[..., a] * cos).abs() + (n[..., b] * sin).abs(), (n[..., b] * cos).abs() + (n[..., a] * sin).abs()
    # the sum of D squares, the mean and eps; rsqrt (2 ulp), two products; a product and a fused one
    return y, ((D + 12) * U if weight is not None else 4 * U) * size


def check_heads(got, x, weight, rows, eps, interleaved):
    want, off = turned(x, weight, rows, eps, interleaved)
    assert got.dtype == x.dtype and got.shape == x.shape
    if weight is None and rows is None:
        assert torch.equal(got, x)
        return
    assert torch.all((got.double() - want).abs() <= HALF[x.dtype] * want.abs() + 1.01 * off + 1e-38)


def entries(pages, table_row, total):
    """(pages, H, P, D), the pages of a sequence -> (total, H, D) in 64 bits; a page that is not there: zeros."""
    P = pages.shape[2]
    at = table_row.long()[:-(-total // P)] if total else table_row.long()[:0]
    there = (at >= 0) & (at < pages.shape[0])
    picked = pages[at.clamp(0, pages.shape[0] - 1)].double() * 1.0
    picked = torch.where(there[:, None, None, None], picked, torch.zeros((), dtype=torch.float64, device=pages.device))
    return picked.transpose(1, 2).reshape(-1, pages.shape[1], pages.shape[3])[:total]


def attention(q, cache_k, cache_v, table, lengths, tree, counts, scale):
    """-> (exact, off) of tree_attention."""
    B, T, Hq, D = q.shape
    Hk = cache_k.shape[1]
    G = Hq // Hk
    out, off = torch.zeros(B, T, Hq, D, dtype=torch.float64, device=q.device), torch.zeros(B, T, Hq, D, dtype=torch.float64, device=q.device)
    room = table.shape[1] * cache_k.shape[2]
    for b in range(B):
        length = min(max(int(lengths[b]), 0), room)
        n = min(max(T if counts is None else int(counts[b]), 0), T)
        total = min(length + n, room)
        k, v = entries(cache_k, table[b], total), entries(cache_v, table[b], total)
        for t in range(n):
            bits = (2 << t) - 1 if tree is None else int(tree[b, t]) & (2 ** 64 - 1)
            seen = torch.tensor([True] * length + [bool(bits >> j & 1) for j in range(total - length)], dtype=torch.bool, device=q.device)
            if not seen.any():
                continue
            ks, vs = k[seen], v[seen]                                             # (entries, Hk, D)
            qq = q[b, t].double().view(Hk, G, D)
            logits = torch.einsum("hgd,ehd->hge", qq, ks) * scale
            p = torch.softmax(logits, -1)
            out[b, t] = torch.einsum("hge,ehd->hgd", p, vs).reshape(Hq, D)
            # (a value that is not finite makes its own channel so, and a key its head's scores: nothing is bounded there)
            ks, vs = (torch.where(torch.isfinite(x), x, torch.zeros_like(x)) for x in (ks, vs))
            size = torch.einsum("hge,ehd->hgd", p, vs.abs()).reshape(Hq, D)
            # a score: D truncated products and the scale's; its exponential: that, its argument's roundings, 2^-22 of ex2
            s_off = (abs(scale) * torch.einsum("hgd,ehd->hge", qq.abs(), ks.abs()).amax(-1) * (D + 4) * 2 * U
                     + logits.abs().amax(-1) * 4 * U).reshape(Hq, 1) + 2.0 ** -22
            # a weight: in bfloat16 the sum of two (a step below it, 2^-7 at most, and the rest to half a step of its own, 2^-8), or where
            # more than 16 rows share the keys one; sums over all entries
            weight = 0.0 if q.dtype == torch.float32 else 2.0 ** -15 if T * G <= 16 else 2.0 ** -8
            off[b, t] = size * (2 * s_off + weight + (total + 96) * 2 * U)
    return out, off


def check_attention(got, q, cache, lengths, tree=None, counts=None, scale=None):
    want, off = attention(q, *cache, lengths, tree, counts, q.shape[-1] ** -0.5 if scale is None else scale)
    assert got.dtype == q.dtype and got.shape == q.shape
    finite = torch.isfinite(want)
    assert torch.equal(finite, torch.isfinite(got)), "finite where it should not be, or the other way round"
    far = (torch.where(finite, got.double() - want, 0)).abs() - (HALF[q.dtype] * want.abs() + 1.01 * off + 1e-38)
    assert torch.all(far[finite] <= 0), f"{float(far[finite].max())} beyond the bound"
    if not finite.all():
        a, b = got[~finite].double(), want[~finite]
        assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a[~torch.isnan(a)], b[~torch.isnan(b)])
