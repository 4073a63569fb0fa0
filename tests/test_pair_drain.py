"""The way out of the 8-bit product's CTA pairs after a wait that gave up: whatever the two producers have asked for has landed before
either CTA leaves.  No wait is made to give up here: the self-test stops the producers of a ring at chosen places."""
import pytest
import torch

from convnn_b200 import _capi

STAGES, PIECE = 4, 2048


def drain(even, odd, src, dst, status, stream=None):
    return _capi.lib().convnn_b200_selftest_pair_drain(even, odd, src, dst, status, stream)


@pytest.mark.parametrize("even,odd", [(9, 8), (8, 9), (-1, 0), (0, -1), (5, 0), (8, 3), (3, 8), (0, 5)])
def test_counts_that_no_ring_reaches_are_refused(even, odd):
    assert drain(even, odd, 1 << 20, 1 << 20, 1 << 20) == _capi.E_INVALID


def test_pointers_are_checked():
    p = 1 << 20
    for args, status in (((None, p, p), _capi.E_NULL), ((p, None, p), _capi.E_NULL), ((p, p, None), _capi.E_NULL),
                         ((p + 8, p, p), _capi.E_ALIGN), ((p, p + 8, p), _capi.E_ALIGN), ((p, p, p + 2), _capi.E_ALIGN)):
        assert drain(1, 1, *args) == status


def ring_model(even, odd):
    """The same arithmetic on the host: barriers as (phase, pending arrivals, bytes), copies that land after the drain has begun.
    -> whether each wait of the drain ends, and only once both CTAs' last copies of its stage have landed."""
    phase, pending, tx = [0] * STAGES, [1] * STAGES, [0] * STAGES
    flying = []

    def settle(s):
        if pending[s] == 0 and tx[s] == 0:
            phase[s] += 1
            pending[s] = 1

    def arm(s, n):
        tx[s] += n
        pending[s] -= 1
        settle(s)

    def land(f):
        tx[f % STAGES] -= 1
        settle(f % STAGES)

    for first, last in ((0, STAGES), (STAGES, 2 * STAGES)):
        for f in range(first, last):
            if f < even:
                arm(f % STAGES, 2)
            for cta, fills in enumerate((even, odd)):
                if f < fills:
                    flying.append((f, cta))
        if first == 0:                                       # (what both did the first time round has landed before the second)
            for f, cta in [x for x in flying if x[0] < min(even, odd)]:
                flying.remove((f, cta))
                land(f)
    fills = max(even, odd)
    for f in range(max(0, fills - STAGES), fills):
        s = f % STAGES
        if f >= odd:
            tx[s] -= 1
            settle(s)
        elif f >= even:
            arm(s, 1)
        mine = [x for x in flying if x[0] == f]
        if mine and phase[s] != f // STAGES:
            return False                                     # the wait would have ended too early
        for x in mine:
            flying.remove(x)
            land(f)
        if phase[s] != f // STAGES + 1:
            return False                                     # the wait would not end
    return not flying


FILLS = [(e, o) for e in range(9) for o in range(9) if abs(e - o) <= STAGES]


@pytest.mark.parametrize("even,odd", FILLS)
def test_the_counts_add_up(even, odd):
    assert ring_model(even, odd)


@pytest.mark.gpu
@pytest.mark.parametrize("even,odd", FILLS)
def test_everything_has_landed(even, odd):
    src = torch.randint(1, 256, (16, PIECE), dtype=torch.uint8, device="cuda", generator=torch.Generator("cuda").manual_seed(even * 9 + odd))
    dst = torch.full((2, STAGES, PIECE), 7, dtype=torch.uint8, device="cuda")
    status = torch.full((1,), -1, dtype=torch.int32, device="cuda")
    _capi.check(drain(even, odd, src.data_ptr(), dst.data_ptr(), status.data_ptr(), torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert status.item() == 0
    want = torch.zeros_like(dst)
    for cta, fills in enumerate((even, odd)):
        for f in range(fills):
            want[cta, f % STAGES] = src[2 * f + cta]
    assert torch.equal(dst, want)
    assert _capi.device_status() == 0
