"""Norm and rotation of heads, and their way into a paged cache, against the formulas in 64 bits."""
import pytest
import torch

from convnn_b200 import _capi, ops
from heads_util import check_heads, randn, rope_table

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _no_grad():
    with torch.no_grad():
        yield
    assert _capi.device_status() == 0


def weights(D, dtype, seed=5):
    return tuple((1.0 + 0.3 * randn(D, seed=seed + i)).to(dtype) for i in range(2))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D,R", [(1, 0), (2, 2), (7, 4), (16, 16), (33, 32), (40, 24), (64, 64), (64, 32), (72, 72), (80, 40), (96, 96),
                                 (128, 128), (128, 16), (192, 192), (250, 100), (256, 256)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_widths(dtype, D, R, interleaved, norm):
    tokens, Hq, Hk = 37, 5, 2
    q, k = randn(tokens, Hq, D, seed=1, dtype=dtype, scale=3.0), randn(tokens, Hk, D, seed=2, dtype=dtype)
    wq, wk = weights(D, dtype) if norm else (None, None)
    rope = rope_table(tokens, R) if R else None
    yq, yk = ops.qk_norm_rope(q, k, wq, wk, rope, interleaved=interleaved)
    check_heads(yq, q, wq, rope, 1e-6, interleaved)
    check_heads(yk, k, wk, rope, 1e-6, interleaved)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape", [(1, 1), (1, 3), (3, 1), (5, 197), (2, 5000), (600, 3)])
@pytest.mark.parametrize("Hq,Hk,D", [(1, 1, 64), (12, 12, 64), (32, 8, 128), (7, 1, 80)])
def test_packed_projections(dtype, shape, Hq, Hk, D):
    """Slices of the projection's rows; every token of a batch at its own index."""
    rows = randn(*shape, (Hq + 2 * Hk) * D, seed=3, dtype=dtype).unflatten(-1, (-1, D))
    q, k = rows[:, :, :Hq], rows[:, :, Hq:Hq + Hk]
    before = rows.clone()
    wq, wk = weights(D, dtype)
    rope = rope_table(shape[1], D)
    yq, yk = ops.qk_norm_rope(q, k, wq, wk, rope)
    check_heads(yq, q, wq, rope, 1e-6, False)
    check_heads(yk, k, wk, rope, 1e-6, False)
    assert torch.equal(rows, before)
    # over themselves; the values behind them stay
    again = ops.qk_norm_rope(q, k, wq, wk, rope, out=(q, k))
    assert again[0] is q and torch.equal(q, yq) and torch.equal(k, yk)
    assert torch.equal(rows[:, :, Hq + Hk:], before[:, :, Hq + Hk:])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rows_that_start_anywhere(dtype, interleaved):
    D, R, tokens = 64, 48, 19
    wq, wk = weights(D, dtype)
    table = rope_table(64, R)
    base_q, base_k = randn(tokens * 3 * D + 8, seed=8, dtype=dtype), randn(tokens * 5 * (D + 2) + 8, seed=9, dtype=dtype)
    wide = torch.zeros(64, R + 7, device="cuda")
    wide[:, 3:3 + R] = table
    want = None
    for off in (0, 1, 2, 4):
        q = base_q[off:off + tokens * 3 * D].view(tokens, 3, D)
        k = base_k.as_strided((tokens, 2, D), (5 * (D + 2), D + 2, 1), off)
        for rope in (table, wide[:, 3:3 + R]):
            yq, yk = ops.qk_norm_rope(q, k, wq, wk, rope, interleaved=interleaved)
            check_heads(yq, q, wq, table[:tokens], 1e-6, interleaved)
            check_heads(yk, k, wk, table[:tokens], 1e-6, interleaved)
        if off == 0:
            want = yq
    # channels that do not lie side by side
    q = base_q[:tokens * 3 * D].view(tokens, 3, D)
    apart = q.transpose(1, 2).contiguous().transpose(1, 2)
    got = ops.qk_norm_rope(apart, None, wq, None, table, interleaved=interleaved)
    assert got[1] is None
    check_heads(got[0], q, wq, table[:tokens], 1e-6, interleaved)
    assert want is not None


def test_positions():
    D, rows = 64, 70000
    table = rope_table(rows, D)
    q, k = randn(2, 5, 3, D, seed=1, dtype=BF16), randn(2, 5, 1, D, seed=2, dtype=BF16)
    at = torch.tensor([[0, 69999, 5, 5, 40000], [1, 2, 3, 65536, 0]], dtype=torch.int32, device="cuda")
    for positions in (at, at[0], at.t().contiguous().t(), torch.stack([at, at], -1)[..., 0]):
        yq, yk = ops.qk_norm_rope(q, k, rope=table, positions=positions)
        rows_of = table[positions.expand(2, 5).long()]
        check_heads(yq, q, None, rows_of, 1e-6, False)
        check_heads(yk, k, None, rows_of, 1e-6, False)
    # outside the table: NaN in the turned channels of those tokens, and there alone
    at[0, 1], at[1, 3], at[1, 4] = rows, -1, -2 ** 31
    bad = torch.zeros(2, 5, dtype=torch.bool, device="cuda")
    bad[0, 1] = bad[1, 3] = bad[1, 4] = True
    half = rope_table(rows, D // 2)
    yq, _ = ops.qk_norm_rope(q, k, rope=half, positions=at)
    assert torch.isnan(yq[bad][..., :D // 2]).all() and torch.equal(yq[bad][..., D // 2:], q[bad][..., D // 2:])
    check_heads(yq[~bad][:, None], q[~bad][:, None], None, half[at[~bad].long()][:, None], 1e-6, False)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_values_out_of_the_ordinary(dtype):
    D = 64
    q = randn(8, 2, D, seed=1, dtype=dtype)
    q[0] = 0
    q[1, 0, 3] = float("inf")
    q[2, 0, 5] = float("nan")
    q[3] = 1e-30
    q[4] = 1e15
    w = weights(D, dtype)[0]
    y, _ = ops.qk_norm_rope(q, None, w, eps=0.0)
    assert torch.isnan(y[0]).all()                           # 0 / 0, as the formula has it
    y, _ = ops.qk_norm_rope(q, None, w)
    assert torch.equal(y[0], torch.zeros_like(y[0]))
    assert torch.isnan(y[1, 0, 3]) and torch.isnan(y[2, 0]).all()
    for i in (1, 2):                                         # other heads do not notice
        check_heads(y[i:i + 1, 1:], q[i:i + 1, 1:], w, None, 1e-6, False)
    for i in (0, 3, 4, 5):
        check_heads(y[i:i + 1], q[i:i + 1], w, None, 1e-6, False)


def test_no_tokens():
    q, k = (torch.empty(0, 5, h, 64, dtype=BF16, device="cuda") for h in (3, 1))
    yq, yk = ops.qk_norm_rope(q, k)
    assert yq.shape == q.shape and yk.shape == k.shape


# ---- into a cache ---------------------------------------------------------------------------------------------------

def cache_of(pages, H, P, D, dtype, table, seed=20, rows_first=False):
    shape = (pages, P, H, D) if rows_first else (pages, H, P, D)
    k, v = (randn(*shape, seed=seed + i, dtype=dtype) for i in range(2))
    return ops.PagedCache(*(t.transpose(1, 2) if rows_first else t for t in (k, v)), table)


def spread(B, width, extra=3, seed=0):
    """Pages of B sequences, in no order, some of them nobody's."""
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(B * width + extra, generator=g)[:B * width].view(B, width).to(torch.int32).cuda(), B * width + extra


def check_append(cache, before, q, k, v, lengths, counts, wq, wk, rope, positions, interleaved, got):
    B, T = k.shape[:2]
    P, want_k, want_v = cache.k.shape[2], before[0].clone(), before[1].clone()
    for b in range(B):
        for t in range(T):
            entry = max(int(lengths[b]), 0) + t
            live = counts is None or t < int(counts[b])
            position = entry if positions is None else int(positions[b, t])
            row = None if rope is None else rope[None, position:position + 1]
            if q is not None and not live:
                assert not got[b, t].any()
            elif q is not None:
                check_heads(got[b:b + 1, t:t + 1], q[b:b + 1, t:t + 1], wq, row, 1e-6, interleaved)
            slot = entry // P
            page = int(cache.table[b, slot]) if slot < cache.table.shape[1] else -1
            if not live or not 0 <= page < cache.k.shape[0]:
                continue
            check_heads(cache.k[page, :, entry % P][None, None], k[b:b + 1, t:t + 1], wk, row, 1e-6, interleaved)
            want_k[page, :, entry % P] = cache.k[page, :, entry % P]
            want_v[page, :, entry % P] = v[b, t]
    assert torch.equal(cache.k, want_k) and torch.equal(cache.v, want_v)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,T,Hq,Hk,D,R,P,width", [
    (1, 1, 1, 1, 64, 64, 1, 9), (1, 1, 32, 8, 128, 128, 64, 2), (3, 5, 6, 2, 80, 40, 20, 3), (5, 7, 4, 4, 64, 64, 3, 9),
    (2, 70, 3, 1, 72, 72, 16, 6), (4, 1, 8, 1, 256, 128, 32, 1), (2, 3, 2, 2, 33, 32, 5, 4)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append(dtype, B, T, Hq, Hk, D, R, P, width, interleaved):
    table, pages = spread(B, width)
    cache = cache_of(pages, Hk, P, D, dtype, table)
    before = cache.k.clone(), cache.v.clone()
    rows = randn(B, T, Hq + 2 * Hk, D, seed=4, dtype=dtype)
    q, k, v = rows[:, :, :Hq], rows[:, :, Hq:Hq + Hk], rows[:, :, Hq + Hk:]
    wq, wk = weights(D, dtype)
    rope = rope_table(width * P + T, R)
    lengths = torch.tensor([(5 * b) % max(1, width * P - T) for b in range(B)], dtype=torch.int32, device="cuda")
    got = ops.append_kv(cache, k, v, lengths, q=q, q_weight=wq, k_weight=wk, rope=rope, interleaved=interleaved)
    check_append(cache, before, q, k, v, lengths, None, wq, wk, rope, None, interleaved, got)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows_first", [False, True])
def test_append_what_is_not_there(dtype, rows_first):
    """Counts, a table that ends, pages that do not exist, lengths out of range, positions of a tree; no queries."""
    B, T, H, D, P, width = 6, 5, 2, 64, 4, 3
    table, pages = spread(B, width)
    table[2, 1], table[3, 0], table[3, 1] = -1, pages, 2 ** 31 - 1
    cache = cache_of(pages, H, P, D, dtype, table, rows_first=rows_first)
    before = cache.k.clone(), cache.v.clone()
    k, v = randn(B, T, H, D, seed=4, dtype=dtype), randn(B, T, H, D, seed=5, dtype=dtype)
    lengths = torch.tensor([0, 9, 3, 2, 2 ** 31 - 1, -7], dtype=torch.int32, device="cuda")
    counts = torch.tensor([0, 5, 4, 99, 5, 2], dtype=torch.int32, device="cuda")
    positions = torch.arange(B * T, dtype=torch.int32, device="cuda").view(B, T) % 7
    rope = rope_table(7, D)
    assert ops.append_kv(cache, k, v, lengths, rope=rope, positions=positions, counts=counts) is None
    check_append(cache, before, None, k, v, lengths, counts, None, None, rope, positions, False, None)


def test_append_nothing():
    table, pages = spread(2, 2)
    cache = cache_of(pages, 1, 4, 64, BF16, table)
    before = cache.k.clone()
    none = torch.empty(2, 0, 1, 64, dtype=BF16, device="cuda")
    q = ops.append_kv(cache, none, none, torch.zeros(2, dtype=torch.int32, device="cuda"), q=torch.empty(2, 0, 3, 64, dtype=BF16, device="cuda"))
    assert q.shape == (2, 0, 3, 64) and torch.equal(cache.k, before)


def test_append_far_into_a_large_cache():
    """Offsets beyond 2^32 bytes and 2^31 values."""
    P, H, D = 64, 4, 128
    pages = (1 << 31) // (P * H * D) + 40                    # of 64 KiB: 4.3 GB each
    k = torch.zeros(pages, H, P, D, dtype=BF16, device="cuda")
    cache = ops.PagedCache(k, torch.zeros_like(k), torch.tensor([[pages - 1, 1, pages - 3]], dtype=torch.int32, device="cuda"))
    new = randn(1, 3, H, D, seed=1, dtype=BF16), randn(1, 3, H, D, seed=2, dtype=BF16)
    ops.append_kv(cache, *new, torch.tensor([62], dtype=torch.int32, device="cuda"))
    ops.append_kv(cache, *new, torch.tensor([128], dtype=torch.int32, device="cuda"))
    for at, x in ((cache.k, new[0]), (cache.v, new[1])):
        assert torch.equal(at[pages - 1, :, 62], x[0, 0]) and torch.equal(at[pages - 1, :, 63], x[0, 1])
        assert torch.equal(at[1, :, 0], x[0, 2])
        assert torch.equal(at[pages - 3, :, :3], x[0].transpose(0, 1))
        assert int(torch.count_nonzero(at[pages - 1, :, 63])) == H * D and int(torch.count_nonzero(at[:pages - 40])) == H * D


def test_streams_threads_and_graphs():
    import threading
    D, table = 64, rope_table(40, 64)
    q, k = randn(3, 33, 4, D, seed=1, dtype=BF16), randn(3, 33, 2, D, seed=2, dtype=BF16)
    w = weights(D, BF16)
    want = ops.qk_norm_rope(q, k, *w, table)
    torch.cuda.synchronize()
    failed = []

    def several():
        try:
            with torch.no_grad(), torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(50):
                    got = ops.qk_norm_rope(q, k, *w, table)
                torch.cuda.current_stream().synchronize()
                assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        except BaseException as e:
            failed.append(e)

    threads = [threading.Thread(target=several) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.qk_norm_rope(q, k, *w, table)
    q.copy_(randn(3, 33, 4, D, seed=7, dtype=BF16))
    graph.replay()
    check_heads(got[0], q, w[0], table[:33], 1e-6, False)
    assert torch.equal(got[1], want[1])
