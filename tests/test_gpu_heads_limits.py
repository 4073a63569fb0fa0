"""Calls of the heads' norm and rotation, the paged cache and the attention over it that their documentation allows and that lie at an edge:
tables without rows, values that are not finite under weights that vanish, tensors that autograd watches."""
import os
import subprocess
import sys

import pytest
import torch
from torch.autograd import forward_ad

from convnn_b200 import _capi, ops
from heads_util import HALF, check_attention, randn, rope_table, turned
from test_gpu_tree_attention import cache_of, ints

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _no_grad():
    with torch.no_grad():
        yield
    assert _capi.device_status() == 0


@pytest.fixture(params=["host module", "Python"])
def both_ways(request, monkeypatch):
    """Every call by the host module, and through Python."""
    if request.param == "Python":
        monkeypatch.setattr(ops, "_calls", ops._GeneralCalls)


def check_turned_by_no_row(got, x, weight, R):
    """NaN in the channels that are turned; the others normed."""
    want, off = turned(x, weight, None, 1e-6, False)
    near = (got.double() - want).abs() <= HALF[x.dtype] * want.abs() + 1.01 * off
    assert torch.isnan(got[..., :R]).all() and near[..., R:].all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("R", [64, 24, 2])
def test_a_rotation_table_without_rows(both_ways, dtype, R):
    """Every position is outside of it."""
    q, k = randn(2, 3, 4, 64, seed=1, dtype=dtype), randn(2, 3, 2, 64, seed=2, dtype=dtype)
    w, rope = randn(64, seed=3, dtype=dtype) + 1, torch.empty(0, R, device="cuda")
    for got, x in zip(ops.qk_norm_rope(q, k, w, w, rope), (q, k)):
        check_turned_by_no_row(got, x, w, R)
    cache = cache_of(2, 2, 16, 64, 60, dtype)
    got = ops.append_kv(cache, k, k, ints(5, 30), q=q, k_weight=w, q_weight=w, rope=rope)
    check_turned_by_no_row(got, q, w, R)
    for b, length in enumerate((5, 30)):
        for i in range(3):
            page, row = int(cache.table[b, (length + i) // 16]), (length + i) % 16
            check_turned_by_no_row(cache.k[page, :, row], k[b, i], w, R)
            assert torch.equal(cache.v[page, :, row], k[b, i])


# ---- values that are not finite -----------------------------------------------------------------------------------------

def place(cache, entry):
    return int(cache.table[0, entry // cache.k.shape[2]]), entry % cache.k.shape[2]


def far_below(dtype, length, T, G, D=64, wide=False):
    """Queries and a cache in which an entry with the key -40 has a weight that float32 does not hold."""
    cache = cache_of(1, 2, 16, D, length + T, dtype)
    if wide:
        cache = cache._replace(table=torch.cat([cache.table, torch.full((1, 1 << 16), -1, dtype=torch.int32, device="cuda")], 1))
    return randn(1, T, 2 * G, D, seed=9, dtype=dtype).abs() + 0.5, cache


@pytest.mark.parametrize("dtype,T,G", [(F32, 1, 1), (F32, 3, 2), (F32, 7, 4), (BF16, 1, 1), (BF16, 3, 2), (BF16, 20, 2), (BF16, 40, 4)])
@pytest.mark.parametrize("length", [31, 32, 33, 60, 64, 65, 127, 130, 400])
@pytest.mark.parametrize("wide", [False, True])
def test_a_cached_value_that_is_not_finite_shows(dtype, T, G, length, wide):
    """An entry that all rows see leaves its trace in its channel wherever it lies, however small its weight."""
    q, cache = far_below(dtype, length, T, G, wide=wide)
    lengths, D = ints(length), 64
    for entry in {0, 5, max(0, length // 32 * 32 - 1), length - 1}:
        page, row = place(cache, entry)
        key, value = cache.k[page, 1, row].clone(), cache.v[page, 1, row].clone()
        cache.k[page, 1, row] = -40
        cache.v[page, 1, row] = 0
        want = ops.tree_attention(q, cache, lengths)
        for bad in (float("inf"), float("nan")):
            cache.v[page, 1, row, 7] = bad
            got = ops.tree_attention(q, cache, lengths)
            hit = torch.zeros_like(got, dtype=torch.bool)
            hit[:, :, G:, 7] = True
            assert torch.isfinite(want).all() and not torch.isfinite(got[hit]).any(), (entry, bad)
            assert torch.equal(got[~hit], want[~hit]), (entry, bad)
        cache.k[page, 1, row], cache.v[page, 1, row] = key, value


@pytest.mark.parametrize("dtype,T,G", [(F32, 3, 2), (F32, 7, 4), (F32, 33, 1), (BF16, 3, 2), (BF16, 20, 2), (BF16, 40, 4)])
@pytest.mark.parametrize("length", [0, 29, 31, 62, 126, 400, 3000])
@pytest.mark.parametrize("wide", [False, True])
def test_a_drafted_value_that_is_not_finite_shows_where_it_is_seen(dtype, T, G, length, wide):
    """The value itself, however small its weight, and nothing of it anywhere else."""
    q, cache = far_below(dtype, length, T, G, wide=wide)
    lengths = ints(length)
    tree = torch.tensor([[1 | 1 << t | (2 if t == 2 else 0) for t in range(T)]], dtype=torch.int64, device="cuda")
    tree[0, 1] = 1                                           # token 1 is seen by token 2 alone
    page, row = place(cache, length + 1)
    cache.k[page, 1, row] = -40
    cache.v[page, 1, row] = 0
    want = ops.tree_attention(q, cache, lengths, tree)
    for bad in (float("inf"), -float("inf"), float("nan")):
        cache.v[page, 1, row, 7] = bad
        got = ops.tree_attention(q, cache, lengths, tree)
        hit = torch.zeros_like(got, dtype=torch.bool)
        hit[0, 2, G:, 7] = True
        assert torch.equal(got[~hit], want[~hit]) and torch.isfinite(want).all()
        assert torch.isnan(got[hit]).all() if bad != bad else (got[hit] == bad).all()


@pytest.mark.parametrize("dtype,T,G", [(F32, 3, 2), (F32, 7, 4), (BF16, 3, 2), (BF16, 20, 2), (BF16, 40, 4)])
@pytest.mark.parametrize("wide", [False, True])
def test_scores_of_minus_infinity(dtype, T, G, wide):
    """Among others they are weights of zero; where a token sees nothing else there is no softmax, and the result says so."""
    B, D = 5, 64
    cache = cache_of(B, 2, 16, D, 200 + T, dtype)
    if wide:
        cache = cache._replace(table=torch.cat([cache.table, torch.full((B, 1 << 16), -1, dtype=torch.int32, device="cuda")], 1))
    q = randn(B, T, 2 * G, D, seed=9, dtype=dtype).abs() + 0.5
    lengths, counts = ints(1, 1, 0, 200, 0), ints(T, T - 1, T, T, T)
    tree = torch.zeros(B, T, dtype=torch.int64, device="cuda")
    tree[0] = torch.arange(T, device="cuda") % 2            # one or two entries
    tree[2, 1] = 4                                          # a token that sees the third alone
    for b, entry in ((0, 0), (1, 0), (2, 2), (3, 7)):
        cache.k[int(cache.table[b, entry // 16]), 1, entry % 16, 3] = -float("inf")
    got = ops.tree_attention(q, cache, lengths, tree, counts)
    check_attention(got, q, cache, lengths, tree, counts)
    assert torch.isnan(got[0, ::2, G:]).all() and torch.isfinite(got[0, 1::2]).all() and torch.isnan(got[1, :T - 1, G:]).all()
    assert not got[1, T - 1:].any() and torch.isnan(got[2, 1, G:]).all() and torch.isfinite(got[3]).all()
    assert not got[2, [t for t in range(T) if t != 1]].any() and not got[4].any()


# ---- long sums ----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("G,T", [(1, 1), (4, 1), (8, 1), (3, 5)])
def test_long_sums_in_float32(G, T):
    """Equal weights and values that a sum of thousands of them rounds the same way each time.  Tiles of 32 keys are summed before they are
    added to what came before: 32 roundings of a tile's sum, one for each of 512 tiles, and at most 40 of pieces and of what follows, half a
    step of 2^-24 each; 16384 of them one after the other are off by more than three times that."""
    n, D, B, v = 16384, 256, 160, 1 + 2.0 ** -12
    k = randn(n // 64, 1, 64, D, seed=1)
    cache = ops.PagedCache(k, torch.full_like(k, v), torch.arange(n // 64, dtype=torch.int32, device="cuda").repeat(B, 1))
    got = ops.tree_attention(torch.zeros(B, T, G, D, device="cuda"), cache, torch.full((B,), n - T, dtype=torch.int32, device="cuda"))
    assert float((got.double() / v - 1).abs().max()) <= (32 + n // 32 + 40) * 2.0 ** -24


# ---- tensors that autograd watches --------------------------------------------------------------------------------------

def appended(cache, n=2):
    new = randn(2, n, 2, 64, seed=3, dtype=cache.k.dtype)
    ops.append_kv(cache, new, new, ints(5, 30))


@pytest.mark.parametrize("which", ["k", "v"])
def test_a_cache_that_autograd_has_kept(both_ways, which):
    cache = cache_of(2, 2, 16, 64, 60)
    w = torch.ones(64, dtype=BF16, device="cuda", requires_grad=True)
    with torch.enable_grad():
        y = (getattr(cache, which) * w).sum()
    appended(cache)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    # slices of one buffer: its own version
    both = randn(2, 9, 2, 16, 64, seed=1, dtype=BF16)
    before = both._version
    appended(cache._replace(k=both[0], v=both[1]))
    assert both._version > before
    # no version to move
    with torch.inference_mode():
        cache = cache_of(2, 2, 16, 64, 60)
    appended(cache)
    with torch.inference_mode():
        appended(cache)
        appended(cache_of(2, 2, 16, 64, 60))


def test_results_that_autograd_has_kept(both_ways):
    cache, q = cache_of(2, 2, 16, 64, 60), randn(2, 1, 4, 64, seed=9, dtype=BF16)
    w = torch.ones(64, dtype=BF16, device="cuda", requires_grad=True)
    odd = torch.empty(q.numel() + 1, dtype=BF16, device="cuda")[1:].view(q.shape)
    for out in (torch.ones_like(q), odd.fill_(1)):
        for write in (lambda: ops.tree_attention(q, cache, ints(5, 30), out=out), lambda: ops.qk_norm_rope(q, None, out=(out, None))):
            with torch.enable_grad():
                y = (out * w).sum()
            write()
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                y.backward()
    with torch.enable_grad():
        for write in (lambda o: ops.tree_attention(q, cache, ints(5, 30), out=o), lambda o: ops.qk_norm_rope(q, None, out=(o, None))):
            with pytest.raises(RuntimeError, match="forward-only"):
                write(torch.ones_like(q).requires_grad_())


def test_a_layers_result_that_autograd_has_kept():
    x, w = randn(2, 40, 64, seed=1, dtype=BF16), torch.ones(64, dtype=BF16, device="cuda", requires_grad=True)
    w_qkv, w_o = randn(3, 64, 64, seed=2, dtype=BF16, scale=0.1), randn(64, 64, seed=3, dtype=BF16, scale=0.1)
    out = torch.ones_like(x)
    with torch.enable_grad():
        y = (out * w).sum()
    ops.softmax_attention(x, w_qkv, w_o, 2, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(both_ways, grad):
    cache, q, k, w = cache_of(2, 2, 16, 64, 60), randn(2, 1, 4, 64, seed=9, dtype=BF16), randn(2, 1, 2, 64, seed=8, dtype=BF16), randn(64, dtype=BF16)
    lengths = ints(5, 30)
    want = ops.tree_attention(q, cache, lengths)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        def dual(x):
            return forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: ops.qk_norm_rope(dual(q), k, w, w), lambda: ops.qk_norm_rope(q, dual(k)[:, :, :1]),
                     lambda: ops.append_kv(cache, k, k, lengths, q=dual(q)), lambda: ops.append_kv(cache, k, dual(k), lengths),
                     lambda: ops.tree_attention(dual(q), cache, lengths), lambda: ops.rms_norm(dual(q), w), lambda: ops.rms_norm(q, w, residual=dual(q)),
                     lambda: ops.quantize_fp8(dual(q)),
                     lambda: ops.linear_fp8(ops.quantize_fp8(q[:, 0, 0]), ops.quantize_fp8(q[:, 0, 0], 128), bias=dual(w[:2]))):
            with pytest.raises(RuntimeError, match="no tangents"):
                call()
        assert torch.equal(ops.tree_attention(q, cache, lengths), want)
        # without forward mode a dual tensor is what it holds
        with forward_ad._set_fwd_grad_enabled(False):
            assert torch.equal(ops.tree_attention(dual(q), cache, lengths), want)


def test_layers_refuse_tangents():
    import convnn_b200
    layer = convnn_b200.MultiHeadAttention(64, 2, 0.0).cuda().to(BF16).eval()
    x = randn(2, 40, 64, seed=1, dtype=BF16)
    want = layer(x)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="no tangents"):
            layer(forward_ad.make_dual(x, torch.ones_like(x)))
        assert torch.equal(layer(x), want)


# ---- what a call asks and launches --------------------------------------------------------------------------------------

def recorded(*calls):
    """Names of what the calls launch and of what they ask of the driver."""
    torch.cuda.synchronize()
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU, torch.profiler.ProfilerActivity.CUDA]) as seen:
        for call in calls:
            call()
        torch.cuda.synchronize()
    return [e.name for e in seen.events()]


@pytest.mark.parametrize("dtype,widths", [(F32, range(68, 257, 12)), (BF16, range(136, 257, 8))])
def test_the_driver_is_asked_once_for_every_width(dtype, widths):
    """How many clusters run at once goes by the heads' width; a size that does not fit is remembered too."""
    calls = []
    for D in widths:
        cache, q, lengths = cache_of(1, 12, 16, D, 1000, dtype), randn(1, 1, 12, D, dtype=dtype), ints(900)
        calls.append(lambda q=q, cache=cache, lengths=lengths: ops.tree_attention(q, cache, lengths))
        calls[-1]()
    names = recorded(*calls)
    assert sum("rows_kernel" in n or "scalar_kernel" in n for n in names) == len(calls), set(names)
    assert not [n for n in names if "Occupancy" in n or "FuncSetAttribute" in n]


def kernels(call):
    return [n for n in recorded(call) if "_kernel" in n]


@pytest.mark.parametrize("dtype,tiles,worth", [(BF16, 64, 6), (F32, 32, 2)])
def test_clusters_on_one_side_of_the_line_and_the_even_division_on_the_other(dtype, tiles, worth):
    """Two units: sixteen CTAs each, while those have no more than `worth` tiles of what the table could hold."""
    q, lengths = randn(1, 2, 2, 64, seed=9, dtype=dtype), ints(500)
    for room, clusters in ((16 * worth * tiles, True), (16 * worth * tiles + 16, False)):
        cache = cache_of(1, 2, 16, 64, room, dtype)
        call = lambda: ops.tree_attention(q, cache, lengths)         # noqa: E731
        check_attention(call(), q, cache, lengths)
        names = kernels(call)
        assert len(names) == (1 if clusters else 2), names
        assert ("true>" if clusters else "false>") in names[0] and ("rows_kernel" if dtype == BF16 else "scalar_kernel") in names[0]
        assert clusters or "join_kernel" in names[1]


@pytest.mark.parametrize("T,G,D,P,kernel", [(16, 1, 128, 16, "rows_kernel"), (17, 1, 128, 16, "tiles_kernel<2, 3, 3, false>"),
                                            (32, 4, 64, 16, "tiles_kernel<1, 6, 6, false>"), (43, 3, 64, 48, "tiles_kernel<1, 6, 5, true>"),
                                            (43, 3, 72, 128, "tiles_kernel<2, 3, 2, true>"), (17, 1, 136, 16, "rows_kernel"),
                                            (17, 1, 128, 20, "rows_kernel"), (17, 1, 128, 8, "rows_kernel")])
def test_rows_channels_and_pages_decide_which_kernel(T, G, D, P, kernel):
    cache, q, lengths = cache_of(2, 2, P, D, 300 + T), randn(2, T, 2 * G, D, seed=9, dtype=BF16), ints(300, 41)
    call = lambda: ops.tree_attention(q, cache, lengths)             # noqa: E731
    check_attention(call(), q, cache, lengths)
    names = kernels(call)
    assert kernel in names[0] and ("join_tiles_kernel" in names[1] if "tiles" in kernel else True), names


# ---- ways to call -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF16, F32])
def test_the_host_module_answers(dtype):
    """Ordinary calls are its, and its results those of the Python form."""
    calls = ops._bind_calls()
    assert calls is not ops._GeneralCalls
    rows = randn(2, 3, 10, 64, seed=4, dtype=dtype)
    q, k, v = rows.split((6, 2, 2), 2)
    w, rope, lengths, counts = randn(64, seed=5, dtype=dtype) + 1, rope_table(200, 64), ints(100, 7), ints(3, 2)
    tree, positions = torch.ones(2, 3, dtype=torch.int64, device="cuda"), lengths[:, None] + ints(0, 1, 1)

    def answers(by):
        cache = cache_of(2, 2, 16, 64, 120, dtype)
        a = by.qk_norm_rope(q, k, w, None, rope, None, 1e-6, False, None)
        b = by.append_kv(cache, k, v, lengths, q, w, w, rope, positions, counts, 1e-6, True)
        nothing = by.append_kv(cache, k, v, lengths, None, None, None, None, None, None, 1e-6, False)
        c = by.tree_attention(q, cache, lengths, tree, counts, None, None)
        d = by.tree_attention(q, cache, lengths, None, None, 0.3, None)
        assert a is not None and b is not None and c is not None and d is not None and not nothing
        return [*a, b, *cache[:2], c, d], nothing

    (host, done), (python, none) = answers(calls), answers(ops)
    assert done is False and none is None
    for x, y in zip(host, python):
        assert x.dtype == y.dtype and x.stride() == y.stride() and torch.equal(x, y)


@pytest.mark.parametrize("dtype,T,G", [(BF16, 1, 4), (BF16, 3, 3), (BF16, 20, 2), (BF16, 64, 4), (F32, 1, 4), (F32, 9, 3)])
@pytest.mark.parametrize("wide", [False, True])
def test_results_over_the_queries(dtype, T, G, wide):
    cache = cache_of(3, 2, 16, 64, 3000, dtype)
    if wide:
        cache = cache._replace(table=torch.cat([cache.table, torch.full((3, 1 << 16), -1, dtype=torch.int32, device="cuda")], 1))
    rows, lengths, counts = randn(3, T, 2 * G + 1, 64, seed=9, dtype=dtype), ints(2900, 0, 40), ints(T, T, max(0, T - 1))
    q, last = rows[:, :, :-1], rows[:, :, -1].clone()
    want = ops.tree_attention(q, cache, lengths, counts=counts)
    got = ops.tree_attention(q, cache, lengths, counts=counts, out=q)
    assert got is q and torch.equal(q, want) and torch.equal(rows[:, :, -1], last)


CAPTURE = """
import sys
sys.path[:0] = {path!r}
import torch
from convnn_b200 import _capi, ops
from heads_util import check_attention, randn, rope_table
torch.set_grad_enabled(False)
def ints(*x): return torch.tensor(x, dtype=torch.int32, device="cuda")
made = []
# one call of each kernel; the width of the table decides between clusters and the even division
for name, dtype, T, G, D, width in (("rows", torch.bfloat16, 1, 2, 256, 32), ("rows, divided", torch.bfloat16, 1, 2, 64, 4096),
                                    ("float32", torch.float32, 2, 2, 256, 32), ("float32, divided", torch.float32, 2, 2, 64, 4096),
                                    ("tiles", torch.bfloat16, 20, 2, 128, 32), ("two tiles", torch.bfloat16, 64, 4, 64, 32)):
    k = randn(64, 2, 16, D, seed=1, dtype=dtype)
    table = torch.full((1, width), -1, dtype=torch.int32, device="cuda")
    table[0, :32] = torch.arange(32, 64)
    made.append((name, randn(1, T, 2 * G, D, seed=3, dtype=dtype), ops.PagedCache(k, k.flip(0).contiguous(), table), ints(400)))
rope, new = rope_table(512, 64), randn(1, 3, 2, 64, seed=4, dtype=torch.bfloat16)
cache = ops.PagedCache(*(torch.zeros(64, 2, 16, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2)), made[0][2].table)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    outs = [ops.tree_attention(q, c, lengths) for _, q, c, lengths in made]
    turned = ops.append_kv(cache, new, new, made[0][3], q=new, rope=rope)
graph.replay()
torch.cuda.synchronize()
for (name, q, c, lengths), out in zip(made, outs):
    check_attention(out, q, c, lengths)
assert torch.equal(turned[:, 0].transpose(0, 1), cache.k[32 + 25, :, :1]) and torch.equal(cache.v[32 + 25, :, :3], new[0].transpose(0, 1))
assert _capi.device_status() == 0
print("captured", len(outs))
"""


def test_first_calls_of_a_process_under_capture():
    """Kernels are loaded, their limits raised and the driver asked while a graph is captured."""
    here = os.path.dirname(os.path.abspath(__file__))
    done = subprocess.run([sys.executable, "-c", CAPTURE.format(path=[os.path.dirname(here), here])], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "captured 6" in done.stdout, done.stdout + done.stderr
