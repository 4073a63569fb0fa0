"""Attention of drafted tokens over a paged cache against its formula in 64 bits, and as part of a decoding step."""
import threading

import pytest
import torch

from convnn_b200 import _capi, ops
from heads_util import check_attention, check_heads, randn, rope_table

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _no_grad():
    with torch.no_grad():
        yield
    assert _capi.device_status() == 0


def ints(*values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def cache_of(B, H, P, D, entries, dtype=BF16, seed=0, rows_first=False):
    width = -(-entries // P)
    g = torch.Generator().manual_seed(seed)
    pages = B * width + 2
    table = torch.randperm(pages, generator=g)[:B * width].view(B, width).to(torch.int32).cuda()
    shape = (pages, P, H, D) if rows_first else (pages, H, P, D)
    k, v = (randn(*shape, seed=seed + i + 1, dtype=dtype) for i in range(2))
    return ops.PagedCache(*(t.transpose(1, 2) if rows_first else t for t in (k, v)), table)


def trees(B, T, seed=0):
    g = torch.Generator().manual_seed(seed)
    masks = torch.zeros(B, T, dtype=torch.int64)
    for b in range(B):
        for i in range(T):
            bit = 1 << i if i < 63 else -2 ** 63
            parent = int(torch.randint(-1, i, (1,), generator=g)) if i else -1
            masks[b, i] = (int(masks[b, parent]) if parent >= 0 else 0) | bit
    return masks.cuda()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [8, 16, 40, 64, 72, 80, 96, 128, 136, 192, 256])
@pytest.mark.parametrize("T,G", [(1, 1), (1, 4), (3, 2), (5, 7)])
def test_widths(dtype, D, T, G):
    B, H, P = 2, 2, 16
    cache = cache_of(B, H, P, D, 300 + T, dtype)
    q = randn(B, T, H * G, D, seed=9, dtype=dtype)
    lengths = ints(300, 61)
    check_attention(ops.tree_attention(q, cache, lengths), q, cache, lengths)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("P", [1, 3, 16, 20, 48, 64, 128])
@pytest.mark.parametrize("rows_first", [False, True])
def test_pages(dtype, P, rows_first):
    B, H, D, T = 4, 2, 64, 2
    cache = cache_of(B, H, P, D, 260, dtype, rows_first=rows_first)
    q = randn(B, T, 6, D, seed=9, dtype=dtype)
    lengths = ints(0, 63, 129, 250)
    check_attention(ops.tree_attention(q, cache, lengths), q, cache, lengths)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,G", [(2, 1), (16, 1), (17, 1), (13, 3), (64, 1), (64, 4), (33, 8)])
@pytest.mark.parametrize("chain", [False, True])
def test_trees(dtype, T, G, chain):
    B, H, D = 3, 2, 64
    cache = cache_of(B, H, 16, D, 200 + T, dtype)
    q = randn(B, T, H * G, D, seed=9, dtype=dtype)
    lengths, counts = ints(200, 0, 77), ints(T, T - 1, (T + 1) // 2)
    tree = None if chain else trees(B, T)
    check_attention(ops.tree_attention(q, cache, lengths, tree, counts), q, cache, lengths, tree, counts)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_lengths(dtype):
    """One more and one fewer than the tiles' sizes, all in one batch."""
    lengths = [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 513, 1023, 1025]
    B, H, D = len(lengths), 1, 64
    cache = cache_of(B, H, 16, D, 1040, dtype)
    q = randn(B, 1, 4, D, seed=9, dtype=dtype)
    at = ints(*lengths)
    check_attention(ops.tree_attention(q, cache, at), q, cache, at)
    # and the same without the token itself
    alone = torch.zeros(B, 1, dtype=torch.int64, device="cuda")
    got = ops.tree_attention(q, cache, at, alone)
    check_attention(got, q, cache, at, alone)
    assert not got[0].any()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,T,H,G,D,length", [(1, 1, 8, 4, 128, 20000), (1, 1, 1, 1, 64, 9999), (2, 9, 2, 3, 128, 5001), (40, 1, 2, 4, 64, 700),
                                              (1, 40, 1, 8, 128, 6000)])
def test_units_of_several_ctas(dtype, B, T, H, G, D, length):
    cache = cache_of(B, H, 64, D, length + T, dtype)
    q = randn(B, T, H * G, D, seed=9, dtype=dtype)
    lengths = ints(*[length - (b * 37) % length for b in range(B)])
    got = ops.tree_attention(q, cache, lengths)
    check_attention(got, q, cache, lengths)
    assert torch.equal(got, ops.tree_attention(q, cache, lengths))      # (the order of its sums does not change)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [4, 20])
def test_nothing_to_attend_to(dtype, T):
    B, H, D = 5, 2, 64
    cache = cache_of(B, H, 16, D, 100, dtype)
    q = randn(B, T, 4, D, seed=9, dtype=dtype)
    lengths, counts = ints(0, 40, -5, 0, 80), ints(T, 0, T, -3, T + 70)
    tree = trees(B, T)
    tree[0, 1] = 0
    tree[2] = 0
    got = ops.tree_attention(q, cache, lengths, tree, counts)
    check_attention(got, q, cache, lengths, tree, counts)
    assert not got[0, 1].any() and not got[1].any() and not got[2].any() and not got[3].any() and got[4].any()
    nothing = cache._replace(table=cache.table[:, :0])
    assert not ops.tree_attention(q, nothing, lengths, tree, counts).any()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [4, 20])
def test_tables_that_end_and_pages_that_are_not_there(dtype, T):
    B, H, D, P = 4, 2, 64, 16
    cache = cache_of(B, H, P, D, 96, dtype)
    cache.table[1, 2], cache.table[2, 0], cache.table[2, 5] = -1, cache.k.shape[0], 2 ** 31 - 1
    q = randn(B, T, 4, D, seed=9, dtype=dtype)
    lengths = ints(96 - T // 2, 60, 90 - T, 2 ** 31 - 1)
    check_attention(ops.tree_attention(q, cache, lengths), q, cache, lengths)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,length", [(6, 30), (20, 30), (6, 4000)])
@pytest.mark.parametrize("value", [float("inf"), float("nan"), -float("inf")])
def test_what_is_not_seen_may_hold_anything(dtype, T, length, value):
    """Drafted tokens of other branches, and whatever is behind the last entry."""
    B, H, D, P = 1, 2, 64, 16
    cache = cache_of(B, H, P, D, length + T + 40, dtype)
    q = randn(B, T, 4, D, seed=9, dtype=dtype)
    lengths, tree = ints(length), trees(B, T, seed=3)
    tree &= ~2                                               # nobody sees token 1
    tree[0, 2] |= 2                                          # but token 2
    at = torch.arange(length + T, length + T + 40)
    for c, every in ((cache.k, value), (cache.v, value)):
        for e in at.tolist():
            c[int(cache.table[0, e // P]), :, e % P] = every
    e = length + 1
    page = int(cache.table[0, e // P])
    cache.k[page, 0, e % P, 3] = value
    cache.v[page, 1, e % P, 5] = value
    cache.v[page, 1, e % P, 9] = -value
    got = ops.tree_attention(q, cache, lengths, tree)
    others = [t for t in range(T) if t != 2]
    assert torch.isfinite(got[:, others]).all()
    whole = got
    # key head 1: the value itself arrives where its row sees it
    assert not torch.isfinite(whole[0, 2, 2:, 5]).any() and not torch.isfinite(whole[0, 2, 2:, 9]).any()
    keep = [c for c in range(D) if c not in (5, 9)]
    assert torch.isfinite(whole[0, 2, 2:][:, keep]).all()
    # the rest is what it is without them
    clean = [t.clone() for t in (cache.k, cache.v)]
    clean[0][page, 0, e % P, 3] = clean[1][page, 1, e % P, 5] = clean[1][page, 1, e % P, 9] = 0
    again = ops.tree_attention(q, ops.PagedCache(*clean, cache.table), lengths, tree)
    assert torch.equal(again[:, others], got[:, others])
    assert torch.equal(again[0, 2, 2:][:, keep], got[0, 2, 2:][:, keep])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_not_finite_where_it_is_seen(dtype):
    cache = cache_of(2, 1, 16, 64, 400, dtype)
    q = randn(2, 3, 2, 64, seed=9, dtype=dtype)
    cache.v[int(cache.table[0, 3]), 0, 5, 7] = float("inf")
    lengths = ints(300, 200)
    got = ops.tree_attention(q, cache, lengths)
    check_attention(got, q, cache, lengths)
    assert torch.isinf(got[0, :, :, 7]).all() and torch.isfinite(got[1]).all()
    cache.k[int(cache.table[1, 2]), 0, 1, 1] = float("nan")
    assert torch.isnan(ops.tree_attention(q, cache, lengths)[1]).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_scales(dtype):
    cache = cache_of(1, 2, 16, 64, 300, dtype)
    q = randn(1, 2, 4, 64, seed=9, dtype=dtype)
    for scale in (1.0, 0.0, -0.2, 1e-3):
        got = ops.tree_attention(q, cache, ints(290), scale=scale)
        check_attention(got, q, cache, ints(290), scale=scale)
    # far apart scores: one entry takes all
    q, cache = q * 30, cache._replace(k=cache.k * 30)
    check_attention(ops.tree_attention(q, cache, ints(290)), q, cache, ints(290))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strides(dtype):
    cache = cache_of(2, 2, 16, 64, 100, dtype)
    rows = randn(2, 3, 10, 64, seed=9, dtype=dtype)
    lengths = ints(90, 33)
    q = rows[:, :, 2:8]
    want = ops.tree_attention(q.contiguous(), cache, lengths)
    assert torch.equal(ops.tree_attention(q, cache, lengths), want)
    apart = q.transpose(2, 3).contiguous().transpose(2, 3)
    assert torch.equal(ops.tree_attention(apart, cache, lengths), want)
    odd = torch.empty(2 * 3 * 6 * 64 + 1, dtype=dtype, device="cuda")[1:].view(2, 3, 6, 64)
    odd.copy_(q)
    assert torch.equal(ops.tree_attention(odd, cache, lengths), want)
    room = torch.full((2, 3, 10, 64), 7.0, dtype=dtype, device="cuda")
    got = ops.tree_attention(q, cache, lengths, out=room[:, :, 1:7])
    assert got.data_ptr() == room[:, :, 1:7].data_ptr() and torch.equal(got, want)
    assert (room[:, :, 0] == 7).all() and (room[:, :, 7:] == 7).all()
    unaligned = torch.full((2 * 3 * 6 * 64 + 2,), 7.0, dtype=dtype, device="cuda")
    got = ops.tree_attention(q, cache, lengths, out=unaligned[1:-1].view(2, 3, 6, 64))
    assert torch.equal(got, want) and unaligned[0] == 7 and unaligned[-1] == 7
    tree, counts = trees(2, 3), ints(3, 2)
    want = ops.tree_attention(q, cache, lengths, tree, counts)
    wide = torch.stack([tree, tree + 1], -1)[..., 0]
    assert torch.equal(ops.tree_attention(q, cache, torch.stack([lengths, lengths], 1)[:, 0], wide, counts), want)
    assert torch.equal(ops.tree_attention(q, cache, lengths, tree[:1].expand(2, 3)), ops.tree_attention(q, cache, lengths, tree[0]))


def test_shared_pages():
    """Two sequences with one beginning."""
    cache = cache_of(2, 2, 16, 64, 200)
    cache.table[1, :5] = cache.table[0, :5]
    q = randn(2, 1, 4, 64, seed=9, dtype=BF16)
    check_attention(ops.tree_attention(q, cache, ints(180, 83)), q, cache, ints(180, 83))


def test_far_into_a_large_cache():
    """Offsets beyond 2^32 bytes and 2^31 values."""
    P, H, D = 64, 4, 128
    pages = (1 << 31) // (P * H * D) + 40
    k, v = (torch.zeros(pages, H, P, D, dtype=BF16, device="cuda") for _ in range(2))
    k[-40:], v[-40:] = randn(40, H, P, D, seed=1, dtype=BF16), randn(40, H, P, D, seed=2, dtype=BF16)
    table = torch.arange(pages - 40, pages, dtype=torch.int32, device="cuda")[None]
    small = ops.PagedCache(k[-40:].clone(), v[-40:].clone(), torch.arange(40, dtype=torch.int32, device="cuda")[None])
    for T, G in ((1, 4), (30, 2)):
        q = randn(1, T, H * G, D, seed=3, dtype=BF16)
        want = ops.tree_attention(q, small, ints(2500))
        check_attention(want, q, small, ints(2500))
        assert torch.equal(ops.tree_attention(q, ops.PagedCache(k, v, table), ints(2500)), want)


@pytest.mark.parametrize("T", [1, 20])
def test_streams_and_threads(T):
    cache = cache_of(3, 2, 16, 64, 3000)
    q, lengths = randn(3, T, 8, 64, seed=9, dtype=BF16), ints(2900, 100, 1700)
    want = ops.tree_attention(q, cache, lengths)
    torch.cuda.synchronize()
    failed = []

    def several():
        try:
            with torch.no_grad(), torch.cuda.stream(torch.cuda.Stream()):
                got = [ops.tree_attention(q, cache, lengths) for _ in range(30)]
                torch.cuda.current_stream().synchronize()
                assert all(torch.equal(g, want) for g in got)
        except BaseException as e:
            failed.append(e)

    threads = [threading.Thread(target=several) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


@pytest.mark.parametrize("T", [1, 20])
def test_two_graphs_with_new_lengths(T):
    """A captured call reads lengths, counts and table when it is replayed; two graphs side by side do not share what they write."""
    cache = cache_of(2, 2, 16, 64, 3000)
    lengths, counts = ints(5, 7), ints(1, 1)
    qs = [randn(2, T, 8, 64, seed=9 + i, dtype=BF16) for i in range(2)]
    for q in qs:
        ops.tree_attention(q, cache, lengths, counts=counts)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.tree_attention(q, cache, lengths, counts=counts))
        graphs.append(g)
    lengths.copy_(ints(2950, 1234))
    counts.copy_(ints(T, max(1, T - 3)))
    want = [ops.tree_attention(q, cache, lengths, counts=counts) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for q, o, w in zip(qs, outs, want):
        assert torch.equal(o, w)
        check_attention(o, q, cache, lengths, None, counts)


# ---- a decoding step --------------------------------------------------------------------------------------------------

def test_a_step_of_decoding():
    """Norm, 8-bit projection, heads into the cache, attention, 8-bit projection: token by token, and as one tree whose accepted path is
    the same tokens."""
    B, H, Hk, D, width = 2, 8, 2, 64, 512
    g = randn(width, seed=1, dtype=BF16, scale=0.1) + 1
    w_qkv = ops.quantize_fp8(randn((H + 2 * Hk) * D, width, seed=2, dtype=BF16, scale=width ** -0.5), 128)
    w_o = ops.quantize_fp8(randn(width, H * D, seed=3, dtype=BF16, scale=width ** -0.5), 128)
    wq, wk = randn(D, seed=4, dtype=BF16, scale=0.1) + 1, randn(D, seed=5, dtype=BF16, scale=0.1) + 1
    rope = rope_table(256, D)
    cache = cache_of(B, Hk, 16, D, 256)
    tree_cache = ops.PagedCache(cache.k.clone(), cache.v.clone(), cache.table)
    lengths = ints(100, 37)

    def block(x, cache, lengths, positions=None, tree=None):
        T = x.shape[1]
        rows = ops.linear_fp8(ops.rms_norm(x, g, quantize=True), w_qkv).view(B, T, -1, D)
        q, k, v = rows.split((H, Hk, Hk), 2)
        q = ops.append_kv(cache, k, v, lengths, q=q, q_weight=wq, k_weight=wk, rope=rope, positions=positions)
        o = ops.tree_attention(q, cache, lengths, tree)
        check_attention(o, q, cache, lengths, tree)
        return ops.linear_fp8(ops.quantize_fp8(o.flatten(2)), w_o, residual=x), rows

    path, x = [0, 2, 3], randn(B, 5, width, seed=6, dtype=BF16)
    single = []
    for i, t in enumerate(path):
        y, rows = block(x[:, t:t + 1].contiguous(), cache, lengths + i)
        single.append(y[:, 0])
    depth, parent = [0, 1, 1, 2, 2], [-1, 0, 0, 2, 1]
    masks = []
    for t in range(5):
        masks.append((masks[parent[t]] if parent[t] >= 0 else 0) | 1 << t)
    y, rows = block(x, tree_cache, lengths, lengths[:, None] + ints(*depth), ints(*masks, dtype=torch.int64).expand(B, 5))
    # the heads are the same bits, entry by entry; the sums over them run in another order
    P = 16
    for i, t in enumerate(path):
        for b in range(B):
            a, c = int(lengths[b]) + i, int(lengths[b]) + t
            for one, other in ((cache.k, tree_cache.k), (cache.v, tree_cache.v)):
                assert torch.equal(one[int(cache.table[b, a // P]), :, a % P], other[int(cache.table[b, c // P]), :, c % P])
        # attention rounded to bfloat16 and then 8 bits: a step of either in few values
        off = (y[:, t].double() - single[i].double()).norm() / single[i].double().norm()
        assert off < 2.0 ** -4
    check_heads(tree_cache.k[int(cache.table[0, 100 // P]), :, 100 % P][None, None], rows[:1, :1, H:H + Hk], wk, rope[None, 100:101], 1e-6, False)


# ---- many rows --------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("T,G", [(17, 1), (32, 4), (43, 3), (64, 4), (33, 8), (64, 8)])
@pytest.mark.parametrize("D", [8, 40, 64, 72, 80, 104, 128])
def test_tiles_of_rows(T, G, D):
    B, H, P = 3, 2, 16
    cache = cache_of(B, H, P, D, 400 + T)
    q = randn(B, T, H * G, D, seed=9, dtype=BF16)
    lengths, counts, tree = ints(400, 129, 0), ints(T, (T + 1) // 2, 1), trees(B, T)
    check_attention(ops.tree_attention(q, cache, lengths, tree, counts), q, cache, lengths, tree, counts)


@pytest.mark.parametrize("P", [1, 8, 16, 20, 48, 64, 96, 128, 256, 512])
@pytest.mark.parametrize("T,G", [(20, 1), (50, 4)])
@pytest.mark.parametrize("rows_first", [False, True])
def test_tiles_of_rows_and_pages(P, T, G, rows_first):
    B, H, D = 3, 2, 64
    cache = cache_of(B, H, P, D, 700 + T, rows_first=rows_first)
    q = randn(B, T, H * G, D, seed=9, dtype=BF16)
    lengths = ints(700, 127, 128)
    check_attention(ops.tree_attention(q, cache, lengths), q, cache, lengths)


@pytest.mark.parametrize("G", [2, 8])
def test_tiles_of_rows_at_every_length(G):
    lengths = [0, 1, 63, 64, 65, 107, 108, 109, 127, 128, 129, 235, 236, 237, 255, 256, 257, 383, 384, 511, 512, 513]
    B, H, D, T = len(lengths), 1, 64, 20
    cache = cache_of(B, H, 32, D, 540)
    q = randn(B, T, H * G, D, seed=9, dtype=BF16)
    at, tree = ints(*lengths), trees(B, T)
    check_attention(ops.tree_attention(q, cache, at, tree), q, cache, at, tree)


@pytest.mark.parametrize("G", [2, 8])
@pytest.mark.parametrize("growth", [0.02, 1.0])
def test_maxima_that_grow(G, growth):
    """Scores that rise along the keys, a little or by far more than 2^8 a tile; and fall."""
    B, H, D, T, n = 2, 1, 64, 20, 1500
    cache = cache_of(B, H, 16, D, n + T)
    q = randn(B, T, H * G, D, seed=9, dtype=BF16).abs()
    for b, order in ((0, 1), (1, -1)):
        for j in range(n):
            e = j if order == 1 else n - 1 - j
            cache.k[int(cache.table[b, e // 16]), 0, e % 16] = growth * j / 10
    lengths = ints(n, n)
    check_attention(ops.tree_attention(q, cache, lengths, scale=1 / 64), q, cache, lengths, scale=1 / 64)


@pytest.mark.parametrize("T,G", [(30, 2), (40, 4), (64, 8)])
def test_tiles_of_rows_of_several_ctas(T, G):
    B, H, D = 3, 2, 128
    cache = cache_of(B, H, 64, D, 5000 + T)
    q = randn(B, T, H * G, D, seed=9, dtype=BF16)
    lengths, counts, tree = ints(5000, 0, 3333), ints(T - 1, T, T // 2), trees(B, T)
    got = ops.tree_attention(q, cache, lengths, tree, counts)
    check_attention(got, q, cache, lengths, tree, counts)
    assert torch.equal(got, ops.tree_attention(q, cache, lengths, tree, counts))


@pytest.mark.parametrize("T,G", [(20, 2), (40, 4)])
@pytest.mark.parametrize("length", [40, 3000])
def test_tiles_of_rows_and_what_is_not_seen(T, G, length):
    """Nothing in the pages behind the last entry, and values of other branches that are not finite."""
    B, H, D, P = 1, 2, 128, 64
    cache = cache_of(B, H, P, D, length + T + 200)
    q = randn(B, T, H * G, D, seed=9, dtype=BF16)
    lengths, tree = ints(length), trees(B, T, seed=3)
    tree[0] &= ~2
    tree[0, 2] |= 2
    want = ops.tree_attention(q, cache, lengths, tree)
    check_attention(want, q, cache, lengths, tree)
    for e in range(length + T, length + T + 200):
        for c in (cache.k, cache.v):
            c[int(cache.table[0, e // P]), :, e % P] = float("nan")
    e = length + 1
    cache.v[int(cache.table[0, e // P]), 1, e % P, 70] = float("inf")
    got = ops.tree_attention(q, cache, lengths, tree)
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[0, 2, G:, 70] = True
    assert torch.equal(got[~hit], want[~hit]) and torch.isinf(got[hit]).all()


@pytest.mark.parametrize("T,G", [(20, 2), (40, 4)])
@pytest.mark.parametrize("scale", [1.0, 0.0, -0.2])
def test_tiles_of_rows_and_scales(T, G, scale):
    cache = cache_of(1, 2, 16, 64, 400)
    q = randn(1, T, 2 * G, 64, seed=9, dtype=BF16)
    check_attention(ops.tree_attention(q, cache, ints(300), scale=scale), q, cache, ints(300), scale=scale)


# ---- the even division ------------------------------------------------------------------------------------------------

def widened(cache, entries=1 << 20):
    """The same cache with room in its tables for far more entries than there are: the work is divided over all CTAs, and joined by a second
    kernel, by what the tables could hold."""
    more = entries // cache.k.shape[2]
    return cache._replace(table=torch.cat([cache.table, torch.full((cache.table.shape[0], more), -1, dtype=torch.int32, device="cuda")], 1))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [8, 40, 64, 80, 96, 128, 136, 256])
@pytest.mark.parametrize("T,G", [(1, 1), (1, 8), (3, 3)])
def test_division_widths(dtype, D, T, G):
    cache = widened(cache_of(2, 3, 16, D, 900 + T, dtype))
    q = randn(2, T, 3 * G, D, seed=9, dtype=dtype)
    lengths = ints(900, 444)
    got = ops.tree_attention(q, cache, lengths)
    check_attention(got, q, cache, lengths)
    assert torch.equal(got, ops.tree_attention(q, cache, lengths))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,G", [(1, 4), (6, 3)])
def test_division_lengths(dtype, T, G):
    lengths = [0, 1, 31, 32, 33, 63, 64, 65, 0, 127, 128, 129, 1000, 257, 2, 511, 513, 0, 0, 1023, 1025, 7, 64, 64, 64, 64, 1, 1, 1, 1, 1, 1, 1, 3000, 0, 1]
    B, H, D = len(lengths), 2, 64
    cache = widened(cache_of(B, H, 16, D, 3010, dtype))
    q = randn(B, T, H * G, D, seed=9, dtype=dtype)
    at, counts, tree = ints(*lengths), ints(*[(b * 5) % (T + 1) for b in range(B)]), trees(B, T)
    check_attention(ops.tree_attention(q, cache, at), q, cache, at)
    check_attention(ops.tree_attention(q, cache, at, tree, counts), q, cache, at, tree, counts)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [4, 20])
def test_division_of_nothing(dtype, T):
    cache = widened(cache_of(3, 2, 16, 64, 60, dtype))
    q = randn(3, T, 4, 64, seed=9, dtype=dtype)
    nobody = torch.zeros(3, T, dtype=torch.int64, device="cuda")
    for lengths, counts in ((ints(0, 0, 0), ints(0, 0, 0)), (ints(9, 9, 9), ints(0, -1, 0)), (ints(0, 0, 0), ints(T, T, T))):
        got = ops.tree_attention(q, cache, lengths, nobody, counts, out=torch.full_like(q, 7.0))
        assert not got.any()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("length", [5, 3000])
def test_division_and_what_is_not_seen(dtype, wide, length):
    B, H, D, P, T = 1, 2, 64, 16, 6
    cache = cache_of(B, H, P, D, length + T, dtype)
    cache = widened(cache) if wide else cache
    q = randn(B, T, 4, D, seed=9, dtype=dtype)
    lengths, tree = ints(length), trees(B, T, seed=3)
    tree[0] &= ~2
    tree[0, 2] |= 2
    want = ops.tree_attention(q, cache, lengths, tree)
    check_attention(want, q, cache, lengths, tree)
    e = length + 1
    cache.v[int(cache.table[0, e // P]), 1, e % P, 7] = -float("inf")
    got = ops.tree_attention(q, cache, lengths, tree)
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[0, 2, 2:, 7] = True
    assert torch.equal(got[~hit], want[~hit]) and (got[hit] == -float("inf")).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,T,H,G,D,length", [(1, 1, 8, 4, 128, 20000), (3, 1, 40, 1, 64, 900), (100, 1, 3, 2, 64, 300), (2, 5, 2, 3, 192, 3001)])
def test_division_and_clusters_agree(dtype, B, T, H, G, D, length):
    cache = cache_of(B, H, 64, D, length + T, dtype)
    q = randn(B, T, H * G, D, seed=9, dtype=dtype)
    lengths = ints(*[length - (b * 37) % length for b in range(B)])
    for c in (cache, widened(cache)):
        check_attention(ops.tree_attention(q, c, lengths), q, c, lengths)


# ---- ways to call -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("D", [4, 12, 20, 36, 60, 68, 100, 132, 160, 188, 252])
@pytest.mark.parametrize("T,G", [(1, 2), (7, 2)])
def test_float32_widths(D, T, G):
    cache = cache_of(2, 2, 16, D, 150 + T, F32)
    q = randn(2, T, 2 * G, D, seed=9)
    for c in (cache, widened(cache)):
        check_attention(ops.tree_attention(q, c, ints(150, 61)), q, c, ints(150, 61))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_calls_through_python_are_the_same(dtype, monkeypatch):
    """What the host module does, the Python form does, to the bit."""
    H, Hk, D, T = 6, 2, 64, 3
    rows = randn(2, T, H + 2 * Hk, D, seed=4, dtype=dtype)
    q, k, v = rows.split((H, Hk, Hk), 2)
    w, rope = randn(D, seed=5, dtype=dtype) + 1, rope_table(200, D)
    lengths, counts, tree = ints(100, 7), ints(T, T - 1), trees(2, T)

    def all_of_them():
        cache = cache_of(2, Hk, 16, D, 120, dtype)
        a = ops.qk_norm_rope(q, k, w, None, rope)
        b = ops.append_kv(cache, k, v, lengths, q=q, q_weight=w, k_weight=w, rope=rope, positions=lengths[:, None] + ints(0, 1, 1), counts=counts)
        nothing = ops.append_kv(cache, k, v, lengths)
        c = ops.tree_attention(b, cache, lengths, tree, counts)
        d = ops.tree_attention(b, cache, lengths, scale=0.3)
        assert nothing is None
        return [*a, b, cache.k, cache.v, c, d]

    fast = all_of_them()
    monkeypatch.setattr(ops, "_calls", ops._GeneralCalls)
    for x, y in zip(fast, all_of_them()):
        assert x.dtype == y.dtype and x.stride() == y.stride() and torch.equal(x, y)


def test_modes_and_flags():
    q, cache = randn(1, 1, 4, 64, seed=9, dtype=BF16), cache_of(1, 2, 16, 64, 50)
    with torch.inference_mode():
        y = ops.tree_attention(q, cache, ints(30))
        assert y.is_inference()
    with torch.enable_grad():
        z = ops.tree_attention(q, cache, ints(30))
        assert not z.requires_grad and not z.is_inference() and torch.equal(z, y)
        with pytest.raises(RuntimeError, match="forward-only"):
            ops.tree_attention(q.clone().requires_grad_(), cache, ints(30))
        with pytest.raises(RuntimeError, match="forward-only"):
            ops.qk_norm_rope(q.clone().requires_grad_(), None)
    assert z.is_contiguous() and z.add_(1).shape == q.shape


def test_no_tokens():
    cache = cache_of(2, 2, 16, 64, 50)
    assert ops.tree_attention(torch.empty(2, 0, 4, 64, dtype=BF16, device="cuda"), cache, ints(3, 4)).shape == (2, 0, 4, 64)
    none = cache._replace(table=cache.table[:0])
    assert ops.tree_attention(torch.empty(0, 3, 4, 64, dtype=BF16, device="cuda"), none, ints()).shape == (0, 3, 4, 64)


@pytest.mark.parametrize("T", [1, 20, 64])
def test_first_call_under_capture(T):
    """A width that no other test has: the kernels' limits are set while a graph is captured."""
    D = {1: 112, 20: 88, 64: 120}[T]
    cache, q, lengths = cache_of(1, 1, 16, D, 500), randn(1, T, 4, D, seed=9, dtype=BF16), ints(400)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.tree_attention(q, cache, lengths)
    graph.replay()
    torch.cuda.synchronize()
    check_attention(out, q, cache, lengths)


def test_many_sequences():
    B, H, D = 700, 1, 64
    cache = cache_of(B, H, 16, D, 40)
    q = randn(B, 2, 2, D, seed=9, dtype=BF16)
    lengths = torch.arange(B, dtype=torch.int32, device="cuda") % 38
    for c in (cache, widened(cache)):
        check_attention(ops.tree_attention(q, c, lengths), q, c, lengths)
    q = randn(B, 17, 2, D, seed=9, dtype=BF16)
    lengths = lengths % 20
    check_attention(ops.tree_attention(q, cache, lengths), q, cache, lengths)
