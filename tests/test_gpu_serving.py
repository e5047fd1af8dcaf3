"""GPU parity of the serving operators: RMS norm with 8-bit outputs, few-row INT4 products, the paged plan, attention
over a paged cache, and a decoder layer made of them.  Against plain 64-bit statements (tests/serving_reference.py)."""
import math

import numpy as np
import pytest
import torch

from tests import serving_reference as R

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _normal(seed, *shape, dtype=F16, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _within(got, want, tolerance, what=""):
    off = (got.double() - want).abs()
    worst = float((off / tolerance).max()) if off.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.2f} times the tolerance"
    assert torch.isfinite(got.float()).all()


# ------------------------------------------------------------- norm
def _check_norm(pk, x, gamma, residual, mode, eps=1e-5, inv_scale=0.0, **kw):
    L, dtype = pk.lib, x.dtype
    s, y = R.rms_norm(x, gamma, residual, eps)
    out, scales, total = pk.ops.add_rms_norm(x, gamma, residual=residual, mode=mode, eps=eps, inv_scale=inv_scale, **kw)
    torch.cuda.synchronize()
    assert torch.equal(total.double(), s)
    if mode == L.LN_F16:
        _within(out, y, (R.HALF[dtype] + R.NORM_REL) * y.abs() + R.TINY[dtype] + 1e-30)
        return
    if mode == L.LN_E4M3_FIXED:
        q, code = y * inv_scale, out.view(torch.float8_e4m3fn).double()
        q = q.clamp(-448, 448)
    else:
        peak = y.abs().amax(1)
        want = torch.where(peak > 0, peak / (448.0 if mode == L.LN_E4M3_ROW else 127.0), torch.ones_like(peak))
        _within(scales, want, R.NORM_REL * want)
        q = y / want[:, None]
        code = out.view(torch.float8_e4m3fn).double() if mode == L.LN_E4M3_ROW else out.double()
    half = 0.5 if mode == L.LN_S8_ROW else (2.0 ** -4 * q.abs()).clamp(min=2.0 ** -10)
    _within(code, q, half + 4 * R.NORM_REL * q.abs() + 1e-12)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,width", [(1, 8), (3, 1), (5, 13), (2, 255), (7, 256), (9, 264), (33, 1024), (700, 2560), (601, 4096),
                                        (3, 8192), (2, 16384), (2, 20000), (1, 32768), (5, 32767)])
def test_norm_modes_and_widths(pk, cuda, dtype, rows, width):
    L = pk.lib
    x, r = _normal(rows + width, rows, width, dtype=dtype), _normal(7, rows, width, dtype=dtype, scale=4.0)
    gamma = _normal(8, width, dtype=dtype, scale=0.2) + 1.0
    for mode in (L.LN_F16, L.LN_E4M3_FIXED, L.LN_E4M3_ROW, L.LN_S8_ROW):
        _check_norm(pk, x, gamma, r, mode, inv_scale=56.0)
    _check_norm(pk, x, gamma, None, L.LN_S8_ROW)


@pytest.mark.parametrize("offset,stride", [(0, 300), (1, 300), (8, 304), (3, 257)])
def test_norm_strides_and_alignment(pk, cuda, offset, stride):
    L, rows, width = pk.lib, 11, 256
    base, other = _normal(1, rows * stride + 8), _normal(2, rows * stride + 8)
    x = base[offset:offset + rows * stride].view(rows, stride)[:, :width]
    r = other[offset:offset + rows * stride].view(rows, stride)[:, :width]
    gamma = _normal(3, width + 1)[1:]
    kept = base.clone()
    for mode in (L.LN_F16, L.LN_E4M3_ROW, L.LN_S8_ROW):
        dtype = {L.LN_F16: F16, L.LN_E4M3_ROW: torch.uint8, L.LN_S8_ROW: torch.int8}[mode]
        big = torch.full((rows, stride + 5), 77, device=cuda).to(dtype)
        _check_norm(pk, x, gamma, r, mode, out=big[:, 5:5 + width])
        assert (big[:, :5].float() == 77).all() and (big[:, 5 + width:].float() == 77).all()
    assert torch.equal(base, kept)


def test_norm_in_place(pk, cuda):
    L = pk.lib
    for alias in ("x", "residual"):
        x, r, gamma = _normal(1, 6, 512), _normal(2, 6, 512), _normal(3, 512)
        s, y = R.rms_norm(x, gamma, r, 1e-5)
        target = x if alias == "x" else r
        out, _, total = pk.ops.add_rms_norm(x, gamma, residual=r, residual_out=target)
        assert total is target and torch.equal(target.double(), s)
        _within(out, y, (R.HALF[F16] + R.NORM_REL) * y.abs() + R.TINY[F16])


def test_norm_rows_of_zeros_and_of_what_is_no_number(pk, cuda):
    L = pk.lib
    x, gamma = _normal(1, 6, 320), _normal(2, 320, scale=0.1) + 1.0
    x[1] = 0
    x[2, 5] = math.nan
    x[3, 7] = math.inf
    x[4] = 60000.0
    r = torch.zeros_like(x)
    r[4] = 60000.0                                  # the sum overflows fp16
    for mode in (L.LN_E4M3_ROW, L.LN_S8_ROW):
        out, scales, _ = pk.ops.add_rms_norm(x, gamma, residual=r, mode=mode)
        assert float(scales[1]) == 1.0 and int(out[1].to(torch.int32).abs().sum()) == 0
        assert torch.isfinite(scales).all() and (scales > 0).all()
        values = out.view(torch.float8_e4m3fn).float() if mode == L.LN_E4M3_ROW else out.float()
        if mode == L.LN_S8_ROW:
            assert (values[2:5] == 0).all()
        else:
            assert torch.isnan(values[2]).all() and torch.isnan(values[3, 7]) and torch.isnan(values[4]).all()
            assert (values[3, :7] == 0).all() and (values[3, 8:] == 0).all()
        clean, clean_scales, _ = pk.ops.add_rms_norm(x[:1], gamma, residual=r[:1], mode=mode)
        assert torch.equal(out[:1], clean) and torch.equal(scales[:1], clean_scales)
    assert pk.ops.add_rms_norm(x[:0], gamma)[0].shape == (0, 320)


def test_norm_feeds_the_8_bit_products(pk, cuda):
    L, m, k, n = pk.lib, 130, 1024, 256
    x, r, gamma, w = _normal(1, m, k), _normal(2, m, k), _normal(3, k, scale=0.1) + 1.0, _normal(4, n, k, scale=0.02)
    for mode, kind, fmt in ((L.LN_S8_ROW, L.KIND_S8, L.PACK_S8), (L.LN_E4M3_ROW, L.KIND_E4M3, L.PACK_E4M3)):
        q, s, _ = pk.ops.add_rms_norm(x, gamma, residual=r, mode=mode)
        wq, ws = pk.ops.pack_weight_rows(w, fmt)
        out = torch.empty(m, n, device=cuda, dtype=F16)
        pk.ops.gemm(q, wq, kind=kind, row_scales=s, col_scales=ws, out=out)
        value = (lambda t: t.view(torch.float8_e4m3fn).double()) if mode == L.LN_E4M3_ROW else (lambda t: t.double())
        a, b = value(q) * s.double()[:, None], value(wq) * ws.double()[:, None]
        want = a @ b.t()
        _within(out, want, (R.HALF[F16] + 1e-6) * want.abs() + k / 16 * 2.0 ** -22 * (a.abs() @ b.abs().t()) + R.TINY[F16])


# ------------------------------------------------------------- few-row INT4 products
def _w4(pk, n, k, seed=0):
    return pk.ops.pack_weight_rows(_normal(seed, n, k, scale=0.02), pk.lib.PACK_S4_G128)


def _packed(n, k, seed, cuda):
    """Codes of the whole range, -8 among them, and scales of mixed size."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 256, (n, k // 2), generator=gen, device=cuda, dtype=torch.int32).to(torch.uint8)
    return codes, (torch.rand(k // 128, n, generator=gen, device=cuda) * 0.02 + 1e-4).half()


@pytest.mark.parametrize("m,n,k", [(1, 1, 128), (1, 16, 256), (2, 17, 128), (3, 100, 1024), (8, 64, 2048), (9, 63, 1152), (16, 257, 4096),
                                   (1, 1024, 4096), (7, 9473, 384), (16, 9500, 1280), (13, 4096, 16384), (1, 70001, 1024),
                                   (16, 16390, 9088), (5, 33000, 2176), (2, 20000, 128),
                                   (3, 16400, 16384), (9, 16400, 16512)])
def test_gemv_sizes(pk, cuda, m, n, k):
    codes, scales = _packed(n, k, m + n + k, cuda)
    w, x = R.w4_weights(codes, scales), _normal(5, m, k)
    for out_type, dtype in ((pk.lib.OUT_F16, F16), (pk.lib.OUT_F32, torch.float32)):
        got = pk.ops.gemv_w4g128(x, codes, scales, out_type=out_type)
        want = x.double() @ w.t()
        _within(got, want, R.gemv_tolerance(x, w, want, dtype))
        assert torch.equal(got, pk.ops.gemv_w4g128(x, codes, scales, out_type=out_type))          # the same bits again


def test_gemv_epilogue_and_strides(pk, cuda):
    L, m, n, k = pk.lib, 5, 150, 512
    codes, scales = _packed(n, k, 1, cuda)
    w = R.w4_weights(codes, scales)
    x = _normal(2, m, k + 40)[:, 8:8 + k]
    rs, cs, bias = (torch.rand(s, device=cuda) + 0.5 for s in (m, n, n))
    v = (x.double() @ w.t()) * rs.double()[:, None] * cs.double() + bias.double()
    for act, f in ((L.ACT_NONE, lambda t: t), (L.ACT_SILU, lambda t: t * torch.sigmoid(t)), (L.ACT_RELU, lambda t: t.clamp(min=0))):
        stream = _normal(3, m, n + 7)
        residual = stream[:, 3:3 + n]
        want = residual.double() + 0.5 * f(v)
        want[4] = 0
        near = R.gemv_tolerance(x, w, want, F16) * 4 + 1e-5 * v.abs()      # scales below 1.5 each, SiLU's slope below 1.1
        guard = stream.clone()
        got = pk.ops.gemv_w4g128(x, codes, scales, row_scales=rs, col_scales=cs, bias=bias, act=act, residual=residual, alpha=0.5,
                                 valid_rows=4, out=residual)                    # in place
        _within(got, want, near)
        assert torch.equal(stream[:, :3], guard[:, :3]) and torch.equal(stream[:, 3 + n:], guard[:, 3 + n:])


def test_gemv_is_the_product_of_the_gemm(pk, cuda):
    L, n, k = pk.lib, 1024, 1024
    codes, scales = _w4(pk, n, k)
    x = _normal(2, 16, k)
    out = torch.empty(16, n, device=cuda, dtype=F16)
    pk.ops.gemm(x, codes, kind=L.KIND_F16_W4G128, out=out, b_group_scales=scales)
    got = pk.ops.gemv_w4g128(x, codes, scales)
    w = R.w4_weights(codes, scales)
    _within(got, out.double(), 2 * R.gemv_tolerance(x, w, out.double(), F16))
    assert torch.equal(pk.ops.gemv_w4g128(x[3:4], codes, scales), got[3:4])      # a row's bits do not depend on its neighbours


def test_gemv_rows_that_are_no_numbers_stay_alone(pk, cuda):
    codes, scales = _w4(pk, 128, 512)
    x = _normal(2, 3, 512)
    clean = pk.ops.gemv_w4g128(x, codes, scales)
    x[1, 100] = math.nan
    got = pk.ops.gemv_w4g128(x, codes, scales)
    assert torch.isnan(got[1]).all() and torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2])


def test_gemv_refuses_what_it_does_not_hold(pk, cuda):
    codes, scales = _w4(pk, 128, 512)
    with pytest.raises(pk.lib.Pk100Error):
        pk.ops.gemv_w4g128(_normal(1, 17, 512), codes, scales)
    with pytest.raises(ValueError):
        pk.ops.gemv_w4g128(_normal(1, 2, 256), codes, scales)
    with pytest.raises(TypeError):
        pk.ops.gemv_w4g128(_normal(1, 2, 512, dtype=BF16), codes, scales)
    assert pk.ops.gemv_w4g128(_normal(1, 0, 512), codes, scales).shape == (0, 128)


# ------------------------------------------------------------- plan
def _int(values, cuda="cuda"):
    return torch.tensor(values, dtype=torch.int32, device=cuda)


def _check_plan(pk, cached, new, page, max_pages, spare=3, padding=0):
    rng = np.random.default_rng(len(cached))
    need = sum(-(-(c + n) // page) for c, n in zip(cached, new))
    ids = rng.permutation(need + spare).tolist()
    table = [[-1] * max_pages for _ in cached]
    for r, c in enumerate(cached):
        for i in range(-(-c // page)):
            table[r][i] = ids.pop()
    want = R.plan(cached, new, table, ids, page)
    t, status, tokens = _int(table).reshape(len(cached), max_pages), torch.zeros(1, dtype=torch.int32, device="cuda"), sum(new) + padding
    p = pk.ops.paged_plan(_int(cached), _int(new), t, _int(ids), _int([len(ids)]), tokens=tokens, page_size=page, status=status)
    assert int(status) == 0 and t.tolist() == want[0]
    assert p.starts.tolist() == want[1] and p.lengths.tolist() == want[2] and p.used.tolist() == [want[5]]
    assert p.positions.tolist() == want[3] + [-1] * padding and p.slots.tolist() == want[4] + [-1] * padding


@pytest.mark.parametrize("cached,new,page", [
    ([0], [1], 16), ([15], [1], 16), ([16], [1], 16), ([0], [0], 16), ([5, 0, 31], [0, 0, 0], 16), ([0, 40, 7], [33, 1, 0], 8),
    ([100, 0, 3, 64], [1, 700, 61, 128], 64), ([9, 2], [3, 5], 1), ([1] * 513, [1] * 513, 3), ([0] * 1030, [2] * 1030, 16)])
def test_plan(pk, cuda, cached, new, page):
    most = max(-(-(c + n) // page) for c, n in zip(cached, new))
    _check_plan(pk, cached, new, page, max(most, 1))
    _check_plan(pk, cached, new, page, most + 5, spare=0, padding=37)


def test_plan_of_the_largest_batch(pk, cuda):
    rng = np.random.default_rng(3)
    _check_plan(pk, rng.integers(0, 100, 4096).tolist(), rng.integers(0, 9, 4096).tolist(), 16, 8, padding=5)


@pytest.mark.parametrize("cached,new,max_pages,free,tokens", [
    ([10, 16], [1, 1], 4, 0, 2), ([0, 0], [40, 8], 2, 9, 48), ([0, 0], [9, 8], 4, 9, 16), ([-1, 0], [1, 1], 4, 9, 2),
    ([0, 5], [3, -1], 4, 9, 8), ([2147483647, 0], [1, 1], 4, 9, 2)])
def test_plan_refuses_a_step_that_does_not_fit(pk, cuda, cached, new, max_pages, free, tokens):
    table = _int([[50 + 10 * r + i for i in range(max_pages)] for r in range(2)])
    before, status = table.clone(), _int([0])
    p = pk.ops.paged_plan(_int(cached), _int(new), table, _int(list(range(9))), _int([free]), tokens=tokens, page_size=16, status=status)
    assert int(status) == pk.lib.STATUS_PLAN and torch.equal(table, before)
    assert p.starts.tolist() == [0, 0, 0] and p.lengths.tolist() == cached and p.used.tolist() == [0]
    assert (p.positions == -1).all() and (p.slots == -1).all()


def test_plan_reads_no_further_than_the_free_list(pk, cuda):
    """A count that is larger than the list: what the list does not hold is not there."""
    table, status = _int([[-1] * 4]), _int([0])
    p = pk.ops.paged_plan(_int([0]), _int([40]), table, _int([5, 6]), _int([1000]), tokens=40, page_size=16, status=status)
    assert int(status) == pk.lib.STATUS_PLAN and p.used.tolist() == [0] and (table == -1).all()


def test_plan_captured_and_replayed(pk, cuda):
    cached, new, table, free, count = _int([0, 20]), _int([1, 1]), _int([[-1] * 4, [7, 3, -1, -1]]), _int(list(range(10, 20))), _int([10])
    before = table.clone()
    pk.ops.paged_plan(cached, new, table, free, count, tokens=8, page_size=16)
    table.copy_(before)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p = pk.ops.paged_plan(cached, new, table, free, count, tokens=8, page_size=16)
    for c, n in (([0, 20], [1, 1]), ([0, 20], [5, 3]), ([0, 31], [0, 2])):
        cached.copy_(_int(c))
        new.copy_(_int(n))
        table.copy_(before)
        graph.replay()
        want = R.plan(c, n, before.tolist(), free.tolist(), 16)
        pad = 8 - sum(n)
        assert table.tolist() == want[0] and p.starts.tolist() == want[1] and p.slots.tolist() == want[4] + [-1] * pad and p.used.tolist() == [want[5]]


def test_plan_without_requests_or_tokens(pk, cuda):
    none = torch.empty(0, dtype=torch.int32, device=cuda)
    p = pk.ops.paged_plan(none, none, none.reshape(0, 4), none, _int([0]), tokens=3, page_size=16)
    assert p.starts.tolist() == [0] and p.slots.tolist() == [-1] * 3
    p = pk.ops.paged_plan(_int([5]), _int([0]), _int([[2]]), none, _int([0]), tokens=0, page_size=16)
    assert p.starts.tolist() == [0, 0] and p.lengths.tolist() == [5]


# ------------------------------------------------------------- attention
class Step:
    """A cache in use and one step on it; what nobody owns holds NaN and infinities."""

    def __init__(self, new, cached, heads, kv_heads, dim, page, dtype, seed=0, spare=3, by_head=False, extra_pages=0):
        rng = np.random.default_rng(seed)
        self.new, self.cached, self.page, self.dtype = new, cached, page, dtype
        self.heads, self.kv, self.dim = heads, kv_heads, dim
        counts = [-(-(c + n) // page) for c, n in zip(cached, new)]
        pages = sum(counts) + spare
        ids = rng.permutation(pages)
        self.table = torch.full((len(new), max(counts + [1]) + extra_pages), -1, dtype=torch.int32)
        at = 0
        for r, n in enumerate(counts):
            self.table[r, :n] = torch.from_numpy(ids[at:at + n].astype(np.int32))
            at += n
        self.table = self.table.cuda()
        self.tokens = sum(new)
        self.starts = _int([0] + np.cumsum(new).tolist())
        self.lengths = _int([c + n for c, n in zip(cached, new)])
        shape = (pages, kv_heads, page, dim) if by_head else (pages, page, kv_heads, dim)
        caches = [_normal(seed + 1 + i, *shape, dtype=dtype) for i in range(2)]
        if by_head:
            caches = [c.transpose(1, 2) for c in caches]
        self.k_cache, self.v_cache = caches
        qkv = _normal(seed + 3, self.tokens, (heads + 2 * kv_heads) * dim, dtype=dtype)
        q, k, v = qkv.split([heads * dim, kv_heads * dim, kv_heads * dim], 1)
        self.q, self.k, self.v = (t.unflatten(1, (-1, dim)) for t in (q, k, v))
        slots = []
        for r, (n, c) in enumerate(zip(new, cached)):
            row = self.table[r].tolist()
            slots += [row[p // page] * page + p % page for p in range(c, c + n)]
        self.slots = torch.tensor(slots, dtype=torch.int64, device="cuda")
        # places that hold no position of a request
        owned = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
        for r, (n, c) in enumerate(zip(new, cached)):
            place = torch.arange(c, device="cuda")
            owned[self.table[r, place // page].long(), place % page] = True
        junk = torch.tensor([math.nan, math.inf, -math.inf], device="cuda").to(dtype)
        for cache in caches:
            cache[~owned] = junk[torch.randint(0, 3, cache[~owned].shape, device="cuda")]

    def run(self, pk, **kw):
        kw = dict(dict(key=self.k, value=self.v, slots=self.slots), **kw)
        return pk.ops.paged_attention(self.q, self.k_cache, self.v_cache, self.table, self.starts, self.lengths, **kw)

    def check(self, out, lse=None, causal=True, window=0, scale=None, lengths=None):
        scale, at = 1 / math.sqrt(self.dim) if scale is None else scale, 0
        for r, (n, c) in enumerate(zip(self.new, self.cached)):
            length = c + n if lengths is None else lengths[r]
            k, v = (R.paged(cache, self.table[r], length) for cache in (self.k_cache, self.v_cache))
            positions = torch.arange(length - n, length, device="cuda")
            want, want_lse, spread, off = R.attention(self.q[at:at + n], k, v, positions, causal, window, scale)
            _within(out[at:at + n], want, R.attention_tolerance(want, spread, off, v, length, self.dtype), f"request {r}")
            if lse is not None and n:
                got, inf = lse[at:at + n].double(), torch.isinf(want_lse)
                assert torch.equal(got[inf], want_lse[inf])
                assert float((got - want_lse)[~inf].abs().max() if (~inf).any() else 0.0) <= 24 * 2.0 ** -22 * off + 1e-5 * (1 + off)
            at += n


LAYOUTS = [(8, 8, 128), (8, 1, 64), (6, 2, 128), (20, 4, 64), (16, 2, 128), (34, 2, 64)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,kv,dim", LAYOUTS)
def test_attention_single_tokens(pk, cuda, heads, kv, dim, dtype):
    s = Step([1] * 9, [0, 1, 15, 16, 63, 64, 65, 700, 2049], heads, kv, dim, 16, dtype)
    out, lse = torch.empty_like(s.q), torch.empty(9, heads, device=cuda)
    s.run(pk, lse=lse, max_new=1, out=out)
    s.check(out, lse)
    assert torch.equal(s.run(pk, max_new=1), out)                     # the same bits again


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (4, 4, 64), (5, 1, 128)])
def test_attention_chunks(pk, cuda, heads, kv, dim, page):
    s = Step([3, 0, 130, 1, 17, 300, 0, 64], [0, 40, 5, 333, 127, 260, 0, 64], heads, kv, dim, page, BF16, seed=page)
    lse = torch.empty(s.tokens, heads, device=cuda)
    s.check(s.run(pk, lse=lse), lse)


@pytest.mark.parametrize("causal,window", [(True, 1), (True, 7), (True, 64), (True, 200), (False, 0), (False, 100)])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_masks(pk, cuda, causal, window, dim):
    s = Step([1, 50, 300, 2], [400, 300, 100, 0], 8, 2, dim, 32, F16, seed=window)
    lse = torch.empty(s.tokens, 8, device=cuda)
    s.check(s.run(pk, lse=lse, causal=causal, window=window, scale=0.2), lse, causal, window, 0.2)


def test_attention_long_prompt(pk, cuda):
    s = Step([1500, 777], [0, 2100], 8, 2, 128, 64, F16, seed=4)
    s.check(s.run(pk))


def test_attention_writes_the_cache_and_nothing_else(pk, cuda):
    s = Step([3, 1, 40], [30, 16, 9], 8, 2, 64, 16, F16, by_head=True)
    want_k, want_v = s.k_cache.contiguous().clone(), s.v_cache.contiguous().clone()
    want_k.view(-1, 2, 64)[s.slots] = s.k
    want_v.view(-1, 2, 64)[s.slots] = s.v
    s.check(s.run(pk))
    for got, want in ((s.k_cache, want_k), (s.v_cache, want_v)):
        assert torch.equal(got.contiguous().view(torch.int16), want.view(torch.int16))
    # a call that brings no keys reads the cache alone, and answers the same
    a, b = s.run(pk), s.run(pk, key=None, value=None, slots=None)
    assert torch.equal(a, b)


def test_attention_without_requests_writes_the_new_keys(pk, cuda):
    key, value = _normal(90, 4, 2, 64), _normal(91, 4, 2, 64)
    cache_k, cache_v = _normal(92, 3, 16, 2, 64), _normal(93, 3, 16, 2, 64)
    want_k, want_v = cache_k.clone(), cache_v.clone()
    want_k[1, 5], want_k[2, 15], want_v[1, 5], want_v[2, 15] = key[0], key[3], value[0], value[3]
    empty = torch.zeros(0, dtype=torch.int32, device="cuda")
    out = torch.full((4, 8, 64), 7.0, dtype=F16, device="cuda")
    pk.ops.paged_attention(_normal(95, 4, 8, 64), cache_k, cache_v, empty.view(0, 5), torch.zeros(1, dtype=torch.int32, device="cuda"), empty, key=key,
                           value=value, slots=torch.tensor([21, -1, -1, 47], device="cuda"), out=out)
    torch.cuda.synchronize()
    assert torch.equal(cache_k, want_k) and torch.equal(cache_v, want_v) and bool((out == 7.0).all())


def test_attention_rows_that_see_nothing(pk, cuda):
    """Lengths below the number of new tokens: the first rows stand before the first key.  No length at all."""
    s = Step([5, 200, 3], [20, 100, 0], 8, 2, 128, 16, F16)
    s.run(pk)
    lengths = [2, 150, 0]
    s.lengths = _int(lengths)
    lse = torch.empty(s.tokens, 8, device=cuda)
    out = s.run(pk, key=None, value=None, slots=None, lse=lse)
    assert (out[:3] == 0).all() and (lse[:3] == -math.inf).all() and (out[205:] == 0).all()
    s.check(out, lse, lengths=lengths)


def test_attention_leaves_the_rows_behind_the_last_request(pk, cuda):
    for new, cached in (([1, 1, 1], [70, 3, 500]), ([40, 1, 200], [70, 3, 500])):
        s = Step(new, cached, 8, 2, 128, 16, F16)
        pad = 9
        q = torch.cat([s.q, torch.full((pad, 8, 128), math.nan, device=cuda, dtype=F16)])
        k, v = (torch.cat([t, t[:1].expand(pad, -1, -1)]) for t in (s.k, s.v))
        slots = torch.cat([s.slots, torch.full((pad,), -1, dtype=torch.int64, device=cuda)])
        out, lse = torch.full((s.tokens + pad, 8, 128), 7.0, device=cuda, dtype=F16), torch.full((s.tokens + pad, 8), 7.0, device=cuda)
        kept = s.k_cache.clone()
        kept.view(-1, 2, 128)[s.slots] = s.k
        pk.ops.paged_attention(q, s.k_cache, s.v_cache, s.table, s.starts, s.lengths, key=k, value=v, slots=slots, out=out, lse=lse)
        s.check(out[:s.tokens], lse[:s.tokens])
        assert (out[s.tokens:] == 7).all() and (lse[s.tokens:] == 7).all()
        assert torch.equal(s.k_cache.view(torch.int16), kept.view(torch.int16))


def test_attention_reports_what_lies_outside_the_cache(pk, cuda):
    def fresh():
        s = Step([1, 30], [100, 90], 8, 2, 128, 16, F16, extra_pages=1)
        return s, _int([0])
    s, status = fresh()
    want = s.run(pk, status=status).clone()
    assert int(status) == 0
    for bad in (-1, s.k_cache.shape[0], 1 << 30, -(1 << 31)):
        s, status = fresh()
        s.table[0, 2] = bad
        out = s.run(pk, status=status)
        assert int(status) == pk.lib.STATUS_PAGE and torch.equal(out[1:], want[1:]) and torch.isfinite(out).all()
    s, status = fresh()
    s.lengths[0] = 1 << 30
    out = s.run(pk, status=status)
    # (other lengths share the work out differently: two roundings of P and of the output, |out| and the mean |v| below 2)
    assert int(status) == pk.lib.STATUS_PAGE and float((out[1:].float() - want[1:].float()).abs().max()) <= 4 * 2 * R.HALF[F16]
    s, status = fresh()
    s.slots[0] = s.k_cache.shape[0] * 16
    kept = s.v_cache.clone()
    kept.view(-1, 2, 128)[s.slots[1:]] = s.v[1:]
    s.run(pk, status=status)
    assert int(status) == pk.lib.STATUS_PAGE and torch.equal(s.v_cache.view(torch.int16), kept.view(torch.int16))


def test_attention_scores_of_any_size(pk, cuda):
    """Large scores, one dominant key, rows whose maximum grows block by block."""
    s = Step([1, 70], [500, 600], 4, 2, 128, 32, BF16, seed=2)
    s.run(pk)
    for r in range(2):
        length = int(s.lengths[r])
        for j in range(length):
            s.k_cache[s.table[r, j // 32].long(), j % 32] *= 0.02 * j
    s.k = s.k * 4
    s.check(s.run(pk))
    s.check(s.run(pk, scale=-0.3), scale=-0.3)
    s.check(s.run(pk, scale=0.0), scale=0.0)


def test_attention_cache_beyond_32_bit_offsets(pk, cuda):
    """Elements behind 2^32 of a cache: (page * page_size + token) * heads * dim does not fit 32 bits."""
    pages, page, kv, dim = 70000, 64, 8, 128                      # 4.6 G elements each
    k_cache, v_cache = (torch.empty(pages, page, kv, dim, device=cuda, dtype=BF16) for _ in range(2))
    ids = [pages - 1, 3, pages - 2, 66000, 40000]
    for i, p in enumerate(ids):
        k_cache[p], v_cache[p] = _normal(i, page, kv, dim, dtype=BF16), _normal(50 + i, page, kv, dim, dtype=BF16)
    s = Step([1, 130], [99, 29], 16, kv, dim, page, BF16)
    s.k_cache, s.v_cache, s.table = k_cache, v_cache, _int([[ids[0], ids[1], -1], [ids[2], ids[3], ids[4]]])
    s.slots = torch.tensor([s.table[r, p // page] * page + p % page for r, c, n in ((0, 99, 1), (1, 29, 130)) for p in range(c, c + n)],
                           dtype=torch.int64, device=cuda)
    s.check(s.run(pk))


def test_attention_does_not_depend_on_the_hint(pk, cuda):
    s = Step([1, 2, 1, 1], [300, 10, 0, 2000], 8, 2, 128, 16, F16)
    for hint in (0, 1, 2, 8, 1000):
        s.check(s.run(pk, max_new=hint))


def test_attention_captured_and_replayed_on_other_lengths(pk, cuda):
    s = Step([1] * 4, [900, 20, 333, 64], 8, 2, 128, 16, BF16, extra_pages=1)
    out = torch.empty_like(s.q)
    s.run(pk, out=out, max_new=1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.run(pk, out=out, max_new=1)
    for cached in ([900, 20, 333, 64], [10, 21, 300, 0]):
        s.cached = cached
        s.lengths.copy_(_int([c + 1 for c in cached]))
        s.slots.copy_(torch.tensor([int(s.table[r, c // 16]) * 16 + c % 16 for r, c in enumerate(cached)]))
        s.q.copy_(_normal(sum(cached), 4, 8, 128, dtype=BF16))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        s.check(out)


def test_attention_captured_without_new_keys(pk, cuda):
    s = Step([1, 300], [3000, 40], 8, 2, 128, 16, F16)
    want = s.run(pk).clone()
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.run(pk, key=None, value=None, slots=None, out=out)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_attention_of_a_wrong_hint(pk, cuda):
    """max_new below what a request brings: slower, not wrong."""
    s = Step([300, 1, 40], [500, 77, 0], 8, 2, 64, 16, F16)
    s.check(s.run(pk, max_new=1))


@pytest.mark.parametrize("dim", [64, 128])
def test_attention_of_a_mixed_step_captured(pk, cuda, dim):
    """New keys, chunk kernel over shares of the keys, few-row kernel beside it and the join, replayed on other data."""
    s = Step([1, 200, 3], [3000, 1500, 0], 8, 2, dim, 32, BF16)
    out = torch.empty_like(s.q)
    s.run(pk, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.run(pk, out=out)
    for seed in range(3):
        s.q.copy_(_normal(100 + seed, *s.q.shape, dtype=BF16))
        s.v.copy_(_normal(200 + seed, *s.v.shape, dtype=BF16))
        graph.replay()
        torch.cuda.synchronize()
        s.check(out)


@pytest.mark.parametrize("dim,kv", [(128, 8), (64, 8)])
@pytest.mark.parametrize("requests", [40, 300])
def test_attention_of_more_chunks_than_blocks(pk, cuda, requests, dim, kv):
    """More than 32 requests, each block of threads takes several; chunks that fill one tile of a pair, both, or neither."""
    new = [(20, 130, 9, 20, 3, 64)[i % 6] for i in range(requests)]
    cached = [(7 * i) % 200 for i in range(requests)]
    s, status = Step(new, cached, 2 * kv, kv, dim, 16, F16, seed=requests), _int([0])
    out = s.run(pk, status=status)
    assert int(status) == 0
    s.check(out)
    assert torch.equal(s.run(pk), out)


@pytest.mark.parametrize("dim,kv", [(128, 2), (64, 4)])
def test_attention_of_single_tokens_beside_chunks(pk, cuda, dim, kv):
    """The kernels for single tokens and for chunks run side by side: the same bits every time, and what each request gets
    alone."""
    new = [1] * 30 + [700, 3, 90] + [1] * 10
    cached = [100 * i for i in range(30)] + [1300, 50, 0] + [37 * i for i in range(10)]
    s = Step(new, cached, 8, kv, dim, 32, BF16, seed=3)
    want = s.run(pk).clone()
    s.check(want)
    for _ in range(10):
        assert torch.equal(s.run(pk), want)


def _one_request(tokens, heads, dim, dtype, seed):
    """Every head its own key-value head, pages of 64 in order, one request without a past."""
    pages = -(-tokens // 64)
    q, k, v = (_normal(seed + i, tokens, heads, dim, dtype=dtype) for i in range(3))
    caches = [torch.zeros(pages, 64, heads, dim, dtype=dtype, device="cuda") for _ in range(2)]
    rest = dict(block_table=_int([list(range(pages))]), starts=_int([0, tokens]), lengths=_int([tokens]),
                slots=torch.arange(tokens, device="cuda"))
    return q, k, v, lambda pk, k, v, **kw: pk.ops.paged_attention(q, *caches, key=k, value=v, **rest, **kw)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("tokens", [3, 150])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_of_keys_that_are_not_finite(pk, cuda, dim, tokens, dtype):
    """A key of NaN at another place in each head: the rows that see it are no numbers, the others as they were."""
    heads = 130 if tokens > 100 else tokens
    q, k, v, run = _one_request(tokens, heads, dim, dtype, 300)
    before = run(pk, k, v)
    bad = k.clone()
    for h in range(heads):
        bad[h, h, 5] = math.nan
    lse = torch.empty(tokens, heads, device="cuda")
    out = run(pk, bad, v, lse=lse)
    sees = torch.arange(tokens, device="cuda")[:, None] >= torch.arange(heads, device="cuda")[None]
    assert bool(out[sees].isnan().all()) and bool(lse[sees].isnan().all())
    assert torch.equal(out[~sees], before[~sees]) and bool(lse[~sees].isfinite().all())
    # plus infinity where the query's sign agrees: no number either; minus infinity: a key of no weight
    bad = k.clone()
    for h in range(heads):
        bad[h, h, 5] = math.inf
    out = run(pk, bad, v)
    up = sees & (q[:, :, 5] > 0)
    assert not bool(out[up].isfinite().any())
    assert bool(out[~up & (torch.arange(tokens, device="cuda")[:, None] > 0) & (torch.arange(heads, device="cuda")[None] > 0)].isfinite().all())


@pytest.mark.parametrize("tokens", [3, 150])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_of_largest_values_that_a_row_does_not_see(pk, cuda, dim, tokens):
    """A masked key has no weight, not a small one: the type's largest value behind a row changes nothing in it."""
    q, k, v, run = _one_request(tokens, 2, dim, BF16, 310)
    before = run(pk, k, v)
    for first in range(1, tokens, 7 if tokens > 100 else 1):
        large = v.clone()
        large[first:] = torch.finfo(BF16).max
        assert torch.equal(run(pk, k, large)[:first], before[:first]), first


@pytest.mark.parametrize("n,k", [(1000, 1024), (20000, 1024)])
def test_gemv_captured_and_under_a_cap(pk, cuda, n, k):
    codes, scales = _packed(n, k, 1, cuda)
    x, status = _normal(2, 3, k), _int([0])
    want = pk.ops.gemv_w4g128(x, codes, scales, status=status).clone()
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pk.ops.gemv_w4g128(x, codes, scales, out=out, status=status)
    graph.replay()
    assert torch.equal(out, want)
    x.mul_(2.0)                                                            # (a power of two: twice the result, to the bit)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want * 2) and int(status) == 0
    try:
        for cap in (1, 3, 50):
            pk.lib.lib.pk100_set_gemm_cta_cap(cap)
            assert torch.equal(pk.ops.gemv_w4g128(x, codes, scales), out)
    finally:
        pk.lib.lib.pk100_set_gemm_cta_cap(0)


def test_gemv_rows_of_the_wide_kernel_stay_alone(pk, cuda):
    codes, scales = _packed(16500, 1152, 4, cuda)
    x = _normal(2, 4, 1152)
    clean = pk.ops.gemv_w4g128(x, codes, scales)
    x[2, 700], x[3, 1100] = math.inf, math.nan
    got = pk.ops.gemv_w4g128(x, codes, scales)
    assert torch.equal(got[:2], clean[:2]) and torch.isnan(got[3]).all()
    assert torch.equal(pk.ops.gemv_w4g128(x[1:2], codes, scales), clean[1:2])


def test_calls_on_two_streams_at_once(pk, cuda):
    steps = [Step([1] * 8, [800 + 100 * i] * 8, 8, 2, 128, 16, F16, seed=i) for i in range(2)]
    want = [s.run(pk).clone() for s in steps]
    streams = [torch.cuda.Stream() for _ in steps]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (s, stream) in enumerate(zip(steps, streams)):
            with torch.cuda.stream(stream):
                got[i].append(s.run(pk))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])


def test_kernels_of_all_kinds_on_streams_at_once(pk, cuda):
    """Chunks of both head widths, single tokens, the wide INT4 product and the norm beside each other: tensor memory, shared
    memory and workspaces are each call's own, the bits those of a call alone."""
    codes, scales = _packed(20000, 1024, 1, cuda)
    x, g, r = _normal(2, 5, 1024), _normal(3, 1024), _normal(4, 5, 1024)
    a, b, c = Step([300, 5], [900, 3], 8, 2, 128, 32, F16, seed=1), Step([400], [0], 8, 8, 64, 16, BF16, seed=2), Step([1] * 9, [500] * 9, 8, 1, 128, 64, F16, seed=3)
    calls = [lambda: a.run(pk), lambda: b.run(pk), lambda: c.run(pk), lambda: pk.ops.gemv_w4g128(x, codes, scales), lambda: pk.ops.add_rms_norm(x, g, residual=r)[0]]
    want = [f().clone() for f in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    got = [[] for _ in calls]
    for _ in range(15):
        for i, (f, stream) in enumerate(zip(calls, streams)):
            with torch.cuda.stream(stream):
                got[i].append(f())
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(len(calls)) for o in got[i])


def test_attention_refuses(pk, cuda):
    s = Step([1], [20], 8, 2, 128, 16, F16)
    with pytest.raises(ValueError):
        s.run(pk, value=None)
    with pytest.raises(TypeError):
        pk.ops.paged_attention(s.q.float(), s.k_cache, s.v_cache, s.table, s.starts, s.lengths)
    with pytest.raises(TypeError):
        s.run(pk, key=s.k.to(BF16))
    with pytest.raises(ValueError):
        pk.ops.paged_attention(s.q, s.k_cache, s.v_cache.transpose(1, 2).contiguous().transpose(1, 2), s.table, s.starts, s.lengths)
    with pytest.raises(ValueError):
        pk.ops.paged_attention(s.q[:, :7], s.k_cache, s.v_cache, s.table, s.starts, s.lengths)
    with pytest.raises(pk.lib.Pk100Error):
        s.run(pk, workspace=torch.empty(256, dtype=torch.uint8, device=cuda))
    with pytest.raises(pk.lib.Pk100Error):
        s.run(pk, out=torch.empty(1, 8, 128, dtype=F16))


# ------------------------------------------------------------- together
def test_a_layer_over_several_steps(pk, cuda):
    """Norm, INT4 projections, plan, attention, output projection with the residual, norm in INT8 and an INT8 product,
    over a prompt and single tokens; every operator against its own inputs, the cache against the whole history."""
    L, width, heads, kv, dim, page, requests = pk.lib, 512, 8, 2, 64, 16, 3
    qkv_codes, qkv_scales = _w4(pk, (heads + 2 * kv) * dim, width, 1)
    out_codes, out_scales = _w4(pk, width, heads * dim, 2)
    up_q, up_s = pk.ops.pack_weight_rows(_normal(3, 1024, width, scale=0.02), L.PACK_S8)
    gamma = _normal(4, width, scale=0.1) + 1.0
    k_cache, v_cache = (torch.full((20, page, kv, dim), math.nan, device=cuda, dtype=F16) for _ in range(2))
    table = torch.full((requests, 8), -1, dtype=torch.int32, device=cuda)
    free = torch.randperm(20, device=cuda).int()
    cached, status = _int([0] * requests), _int([0])
    history = [[] for _ in range(requests)]
    for step, new in enumerate(([6, 1, 9], [1, 1, 1], [1, 0, 1], [4, 12, 0], [1, 1, 1])):
        tokens = sum(new)
        x = _normal(10 + step, tokens, width)
        plan = pk.ops.paged_plan(cached, _int(new), table, free, _int([free.numel()]), tokens=tokens, page_size=page, status=status)
        h, _, _ = pk.ops.add_rms_norm(x, gamma)
        qkv = pk.ops.gemv_w4g128(h, qkv_codes, qkv_scales)
        q, k, v = (t.unflatten(1, (-1, dim)) for t in qkv.split([heads * dim, kv * dim, kv * dim], 1))
        att = pk.ops.paged_attention(q, k_cache, v_cache, table, plan.starts, plan.lengths, key=k, value=v, slots=plan.slots, status=status)
        y = pk.ops.gemv_w4g128(att.flatten(1), out_codes, out_scales, residual=x)
        codes, scales, _ = pk.ops.add_rms_norm(y, gamma, mode=L.LN_S8_ROW)
        z = torch.empty(tokens, 1024, device=cuda, dtype=F16)
        pk.ops.gemm(codes, up_q, kind=L.KIND_S8, row_scales=scales, col_scales=up_s, out=z, act=L.ACT_SILU)
        assert int(status) == 0
        _, hd = R.rms_norm(x, gamma, None, 1e-5)
        _within(h, hd, (R.HALF[F16] + R.NORM_REL) * hd.abs() + R.TINY[F16])
        for got, a, weights, extra in ((qkv, h, (qkv_codes, qkv_scales), 0), (y, att.flatten(1), (out_codes, out_scales), x.double())):
            w = R.w4_weights(*weights)
            want = a.double() @ w.t() + extra
            _within(got, want, R.gemv_tolerance(a, w, want, F16))
        at = 0
        for r, n in enumerate(new):
            history[r] += [(k[at + i].clone(), v[at + i].clone()) for i in range(n)]
            if n:
                keys, values = (torch.stack([t[i] for t in history[r]]) for i in range(2))
                places = torch.arange(len(history[r]) - n, len(history[r]), device=cuda)
                want, _, spread, off = R.attention(q[at:at + n], keys, values, places, True, 0, 1 / math.sqrt(dim))
                _within(att[at:at + n], want, R.attention_tolerance(want, spread, off, values, len(history[r]), F16), f"step {step}")
            at += n
        a = codes.double() @ up_q.double().t() * scales.double()[:, None] * up_s.double()
        want = a * torch.sigmoid(a)
        _within(z, want, (R.HALF[F16] + 1e-5) * want.abs() + 1e-6)        # the GEMM's SiLU has a hardware exponential
        cached, free = plan.lengths.clone(), free[int(plan.used):]
