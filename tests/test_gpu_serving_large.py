"""GPU tests of the serving operators at sizes whose kernels and loops the smaller tests do not reach, and of requests alone against
requests together."""
import numpy as np
import pytest
import torch

from tests import serving_reference as R
from tests.test_gpu_serving import BF16, F16, Step, _check_norm, _int, _normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,width", [(16384, 4096), (16383, 2568), (40000, 1024), (9000, 512), (50001, 264), (20000, 8), (9001, 1023), (5000, 12000)])
def test_norm_of_many_rows(pk, cuda, dtype, rows, width):
    """Four chunks a thread, a row a warp or a block; two in between; odd widths and last blocks that are not full."""
    L = pk.lib
    x, r = _normal(rows + width, rows, width, dtype=dtype), _normal(7, rows, width, dtype=dtype, scale=4.0)
    gamma = _normal(8, width, dtype=dtype, scale=0.2) + 1.0
    for mode in (L.LN_F16, L.LN_E4M3_FIXED, L.LN_E4M3_ROW, L.LN_S8_ROW):
        _check_norm(pk, x, gamma, r, mode, inv_scale=56.0)
        _check_norm(pk, x, gamma, None, mode, inv_scale=56.0)


@pytest.mark.parametrize("page", [16, 24, 128])
def test_plan_of_more_tokens_than_a_pass(pk, cuda, page):
    """A warp's run of tokens takes several passes from 303 000 tokens on: requests that are empty, that end on either side of a pass, and
    long ones; padding behind them."""
    rng = np.random.default_rng(page)
    new = [int(n) for n in rng.choice([0, 1, 2, 31, 32, 33, 127, 128, 129, 255, 257, 1000, 3999], 1300)]
    new[5] = 40000
    cached = [int(c) for c in rng.choice([0, 1, 15, 16, 17, 300, 4001], 1300)]
    tokens, padding = sum(new), 12345
    assert tokens > 320000
    most = max(-(-(c + n) // page) for c, n in zip(cached, new))
    ids = rng.permutation(sum(-(-(c + n) // page) for c, n in zip(cached, new)) + 3).tolist()
    table = [[-1] * most for _ in cached]
    for r, c in enumerate(cached):
        for i in range(-(-c // page)):
            table[r][i] = ids.pop()
    want = R.plan(cached, new, table, ids, page)
    t, status = _int(table), _int([0])
    p = pk.ops.paged_plan(_int(cached), _int(new), t, _int(ids), _int([len(ids)]), tokens=tokens + padding, page_size=page, status=status)
    same = lambda got, values: np.array_equal(got.cpu().numpy(), np.array(values))
    assert int(status) == 0 and same(t, want[0]) and same(p.starts, want[1]) and same(p.lengths, want[2]) and int(p.used) == want[5]
    assert same(p.positions[:tokens], want[3]) and same(p.slots[:tokens], want[4])
    assert bool((p.positions[tokens:] == -1).all()) and bool((p.slots[tokens:] == -1).all())


@pytest.mark.parametrize("dim,kv", [(128, 2), (64, 4)])
def test_attention_of_requests_together_and_alone(pk, cuda, dim, kv):
    """Single tokens and chunks in one step: each request's rows are those of a step of its own, but for the roundings that sharing
    the work out differently moves (each side is within the tolerance of the 64-bit rows)."""
    new = [1] * 12 + [300, 3, 90] + [1] * 4
    cached = [100 * i for i in range(12)] + [1300, 50, 0] + [37 * i for i in range(4)]
    s = Step(new, cached, 8, kv, dim, 32, BF16, seed=3)
    together = s.run(pk).clone()
    s.check(together)
    at = 0
    for r, n in enumerate(new):
        alone = pk.ops.paged_attention(s.q[at:at + n], s.k_cache, s.v_cache, s.table[r:r + 1], _int([0, n]), s.lengths[r:r + 1])
        k, v = (R.paged(cache, s.table[r], cached[r] + n) for cache in (s.k_cache, s.v_cache))
        want, _, spread, off = R.attention(s.q[at:at + n], k, v, torch.arange(cached[r], cached[r] + n, device="cuda"), True, 0, dim ** -0.5)
        tolerance = R.attention_tolerance(want, spread, off, v, cached[r] + n, BF16)
        assert bool(((alone.double() - together[at:at + n].double()).abs() <= 2 * tolerance).all()), r
        at += n
