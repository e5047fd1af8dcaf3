"""GPU tests of waits that run out: the kernels report it, return with nothing in flight, and leave the context usable.  The
limit is the host's; nothing faults, nothing hangs."""
import contextlib

import pytest
import torch

from tests.test_gpu_serving import F16, Step, _int, _normal, _packed

pytestmark = pytest.mark.gpu


@contextlib.contextmanager
def _limit(pk, nanoseconds):
    pk.lib.lib.pk100_set_wait_limit(nanoseconds)
    try:
        yield
    finally:
        pk.lib.lib.pk100_set_wait_limit(-1)


def _gives_up_and_recovers(pk, call):
    """call(status) -> output.  With a limit of 0 some wait for a copy or a product runs out; before and behind it all is well."""
    status = _int([0])
    want = call(status).clone()
    assert int(status) == 0
    with _limit(pk, 0):
        for _ in range(3):
            status.zero_()
            call(status)
            torch.cuda.synchronize()
            assert int(status) == 1
    status.zero_()
    assert torch.equal(call(status), want) and int(status) == 0
    with _limit(pk, 10 ** 9):                            # a second: a limit that no wait reaches
        assert torch.equal(call(status), want) and int(status) == 0


@pytest.mark.parametrize("dim", [64, 128])
def test_single_tokens_whose_copies_are_not_there(pk, cuda, dim):
    """One block of 64 keys each: the warp that loads never waits, those that compute do, and say so."""
    s = Step([1] * 20, [40] * 20, 8, 4, dim, 64, F16)
    _gives_up_and_recovers(pk, lambda status: s.run(pk, max_new=1, status=status))


@pytest.mark.parametrize("dim", [64, 128])
def test_single_tokens_over_long_contexts(pk, cuda, dim):
    s = Step([1] * 9, [4000] * 9, 8, 4, dim, 32, F16)
    _gives_up_and_recovers(pk, lambda status: s.run(pk, max_new=1, status=status))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,cached", [([300], [0]), ([130, 1, 700], [2000, 900, 0]), ([40] * 40, [300] * 40)])
def test_chunks(pk, cuda, dim, new, cached):
    s = Step(new, cached, 8, 4, dim, 32, F16)
    _gives_up_and_recovers(pk, lambda status: s.run(pk, status=status))


@pytest.mark.parametrize("k", [128, 1152, 4096])
def test_wide_product(pk, cuda, k):
    codes, scales = _packed(20000, k, 1, cuda)
    x = _normal(2, 5, k)
    _gives_up_and_recovers(pk, lambda status: pk.ops.gemv_w4g128(x, codes, scales, status=status))
