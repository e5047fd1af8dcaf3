"""GPU tests of what the serving operators promise about single roundings: quotients of the norm's codes, small weights and
sums of attention."""
import math

import numpy as np
import pytest
import torch

from tests import serving_reference as R
from tests.test_gpu_serving import Step

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


# ------------------------------------------------------------- norm
def _values_below(peak, dtype):
    """Every number of the type between 0.05 and the peak, the peak among them."""
    v = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    return v[(v.float() > 0.05) & (v.float() <= peak)]


@pytest.mark.parametrize("mode,dtype,peak", [("e4m3", F16, 56.5), ("int8", F16, 14.8828125), ("e4m3", BF16, 24.5), ("int8", BF16, 53.75),
                                             ("int8", F16, 63.5), ("int8", BF16, 63.5), ("e4m3", F16, 56.0)])
def test_norm_codes_are_those_of_the_quotient(pk, cuda, mode, dtype, peak):
    """Rows of +1 and -1 have a mean square of 1, so y = s * gamma exactly, and y / c = y * top / max |y|: the code is the nearest of
    that, ties to even.  A product with the rounded reciprocal of c gives other codes for some of the first four rows' values.  In
    64 bits the quotient of these numbers is half-way where the exact one is, and only there; E4M3 codes are those of its fp32 value."""
    L = pk.lib
    gamma = _values_below(peak, dtype)
    width, top = gamma.numel(), 448.0 if mode == "e4m3" else 127.0
    x = torch.ones(3, width, dtype=dtype)
    x[1] = -1
    x[2, ::2] = -1
    out, scales, _ = pk.ops.add_rms_norm(x.cuda(), gamma.cuda(), mode=L.LN_E4M3_ROW if mode == "e4m3" else L.LN_S8_ROW, eps=0.0)
    y = x.double().numpy() * gamma.double().numpy()
    c = np.float32(peak) / np.float32(top)
    product = y.astype(np.float32) * (np.float32(1) / c)
    code = lambda q: torch.from_numpy(np.rint(q) if mode == "int8" else q.astype(np.float32)).to(torch.int8 if mode == "int8" else torch.float8_e4m3fn).float()
    want = code(y * top / peak)
    assert peak in (56.0, 63.5) or not torch.equal(want, code(product))
    assert (scales.cpu() == torch.from_numpy(np.array(c))).all()
    got = (out if mode == "int8" else out.view(torch.float8_e4m3fn)).float().cpu()
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,width", [(777, 2560), (2000, 4096), (40, 96)])
def test_norm_int8_codes_are_the_nearest(pk, cuda, dtype, rows, width):
    """Rows as a model has them: every code is the nearest integer of limit * s * gamma / max |s * gamma|, which 64 bits hold."""
    gen = torch.Generator(device="cuda").manual_seed(rows)
    x, r = (torch.randn(rows, width, generator=gen, device="cuda").to(dtype) for _ in range(2))
    gamma = (torch.randn(width, generator=gen, device="cuda") * 0.1 + 1.0).to(dtype)
    out, _, s = pk.ops.add_rms_norm(x, gamma, residual=r, mode=pk.lib.LN_S8_ROW)
    y = s.double() * gamma.double()
    assert torch.equal(out.double(), torch.round(y * 127.0 / y.abs().amax(1, keepdim=True)))


def test_norm_int8_codes_beside_a_gamma_that_is_none(pk, cuda):
    x = torch.randn(5, 300, generator=torch.Generator().manual_seed(1)).half().cuda()
    gamma = torch.ones(300, dtype=F16, device="cuda")
    want, want_scales, _ = pk.ops.add_rms_norm(x[:, :299].contiguous(), gamma[:299], mode=pk.lib.LN_S8_ROW)
    gamma[299] = math.nan
    x[:, 299] = 0.5
    out, scales, _ = pk.ops.add_rms_norm(x, gamma, mode=pk.lib.LN_S8_ROW)
    assert bool((out[:, 299] == 0).all()) and torch.equal(out[:, :299], want)


@pytest.mark.parametrize("width", [40, 256, 4096, 20000])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_norm_products_beyond_the_largest_number_stay_out_of_the_maximum(pk, cuda, dtype, width):
    """Rows beside each other, some of them with infinities: theirs have y = 0 or NaN and a scale of 1, the others their own codes
    and scales to the bit."""
    L = pk.lib
    gen = torch.Generator().manual_seed(width)
    x = torch.randn(40, width, generator=gen).to(dtype).cuda()
    gamma = (torch.rand(width, generator=gen) + 0.5).to(dtype).cuda()
    bad = x.clone()
    bad[3, 7], bad[4, width - 1], bad[4, 0], bad[21, width // 2], bad[39, 5] = math.inf, -math.inf, math.inf, math.inf, math.nan
    whole = torch.tensor([r not in (3, 4, 21, 39) for r in range(40)])
    for mode in (L.LN_E4M3_ROW, L.LN_S8_ROW):
        want, want_scales, _ = pk.ops.add_rms_norm(x, gamma, mode=mode)
        out, scales, _ = pk.ops.add_rms_norm(bad, gamma, mode=mode)
        assert torch.equal(out[whole], want[whole]) and torch.equal(scales[whole], want_scales[whole])
        assert (scales[~whole] == 1.0).all()
        codes = out.float() if mode == L.LN_S8_ROW else out.view(torch.float8_e4m3fn).float()
        assert (codes[3][torch.isfinite(bad[3])] == 0).all() and (codes[21][torch.isfinite(bad[21])] == 0).all()
        if mode == L.LN_E4M3_ROW:
            assert torch.isnan(codes[3, 7]) and torch.isnan(codes[39]).all()


def test_norm_products_beyond_the_largest_number_by_gamma_alone(pk, cuda):
    """s * gamma beyond fp32 where s * rstd * gamma is not: such a y is clamped, the scale is that of the others."""
    L = pk.lib
    x = torch.full((2, 64), 1000.0, dtype=BF16, device="cuda")
    gamma = torch.ones(64, dtype=BF16, device="cuda")
    gamma[9] = 1e36
    for mode, top in ((L.LN_E4M3_ROW, 448.0), (L.LN_S8_ROW, 127.0)):
        out, scales, _ = pk.ops.add_rms_norm(x, gamma, mode=mode)
        codes = out.float() if mode == L.LN_S8_ROW else out.view(torch.float8_e4m3fn).float()
        assert (codes == top).all() and float((scales * top - 1).abs().max()) < 1e-5


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_norm_with_a_fixed_scale_multiplies_by_whatever_it_is_given(pk, cuda, dtype):
    """E4M3(y * inv_scale): an infinite factor saturates what is not zero and makes NaN of what is, NaN makes NaN."""
    x = torch.randn(3, 100, generator=torch.Generator().manual_seed(1)).to(dtype)
    x[1, ::3] = 0
    gamma = torch.ones(100, dtype=dtype)
    def codes(factor):
        out, _, _ = pk.ops.add_rms_norm(x.cuda(), gamma.cuda(), mode=pk.lib.LN_E4M3_FIXED, inv_scale=factor)
        return out.view(torch.float8_e4m3fn).float().cpu()
    want = torch.where(x == 0, math.nan, 448.0 * torch.sign(x.float()))
    assert torch.equal(codes(math.inf).nan_to_num(7.0), want.nan_to_num(7.0))
    assert torch.equal(codes(-math.inf).nan_to_num(7.0), (-want).nan_to_num(7.0))
    assert torch.isnan(codes(math.nan)).all()
    assert (codes(0.0) == 0).all()


# ------------------------------------------------------------- attention
def _one_key_and_many(kernel, dim, dtype, first, value, keys=1 << 17, far=25.5):
    """A key that scores 0, the first or the last, and `keys` of -far (base 2): of this value, and of -1.  The arguments of a call in
    which every row sees all of them, whole, and the rows' value and lse in 64 bits."""
    kv, page = 8, 256
    length = keys + 1
    pages = -(-length // page)
    k = torch.zeros(pages * page, kv, dim, dtype=dtype, device="cuda")
    v = torch.full_like(k, -1.0)
    k[:, :, 0] = -far
    at = 0 if first else keys
    k[at], v[at] = 0, value
    # as many rows as leave no keys to be shared out: a part of the keys has another largest one
    requests, new = (37, 1) if kernel == "rows" else (1, 4864)
    q = torch.zeros(requests * new, kv, dim, dtype=dtype, device="cuda")
    q[:, :, 0] = 1
    ids = torch.arange(pages, dtype=torch.int32, device="cuda")
    args = dict(query=q, key_cache=k.view(pages, page, kv, dim), value_cache=v.view(pages, page, kv, dim), block_table=ids.expand(requests, -1).contiguous(),
                starts=torch.arange(requests + 1, dtype=torch.int32, device="cuda") * new,
                lengths=torch.full((requests,), length, dtype=torch.int32, device="cuda"), causal=False, scale=math.log(2.0), max_new=new)
    rest = keys * 2.0 ** -far
    return args, (value - rest) / (1 + rest), math.log1p(rest)


@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("kernel,dim", [("rows", 64), ("rows", 128), ("chunk", 64), ("chunk", 128)])
def test_attention_of_many_small_weights(pk, cuda, kernel, dim, dtype, first):
    """2^17 keys of 2^-25.5, each less than half of fp16's smallest number, behind one whose value is 0: all of the row is theirs.
    Tolerance: half a step of every weight and of the output, and in fp16 half the smallest number, 2^-25, of each weight, which
    a factor of 2^6 at least has made smaller; 1e-5 for the exponentials, 1e-3 for what the tensor cores cut off their sums."""
    half = 2.0 ** -11 if dtype is F16 else 2.0 ** -8
    args, want, _ = _one_key_and_many(kernel, dim, dtype, first, 0.0)
    out = pk.ops.paged_attention(**args)
    tolerance = (2 * half + 1e-5 + 1e-3) * abs(want) + (2.0 ** 17 * 2.0 ** -31 if dtype is F16 else 0.0)
    assert tolerance < 0.03 * abs(want)
    assert float((out.double() - want).abs().max()) <= tolerance


@pytest.mark.parametrize("tokens", [2, 300])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_of_scores_of_millions(pk, cuda, dim, tokens):
    """fp16, the largest key of a row far above the others, scores up to 4e9: its value, but for the rounding of a weight and of
    the output."""
    k = torch.zeros(16, 32, 2, dim, dtype=F16, device="cuda")
    v = torch.randn(16, 32, 2, dim, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").half()
    flat = k.view(512, 2, dim)
    flat[:, :, 0] = torch.arange(512, device="cuda").half()[:, None]
    for large in (1.0, 300.0, 30000.0, 65504.0):
        q = torch.zeros(tokens, 4, dim, dtype=F16, device="cuda")
        q[:, :, 0] = large
        for sign in (1.0, -1.0):
            out = pk.ops.paged_attention(q, k, v, torch.arange(16, dtype=torch.int32, device="cuda")[None], torch.tensor([0, tokens], dtype=torch.int32, device="cuda"),
                                         torch.tensor([512], dtype=torch.int32, device="cuda"), causal=False, scale=128.0 * sign)
            want = v.view(512, 2, dim)[511 if sign > 0 else 0].repeat_interleave(2, 0)
            assert bool(((out.double() - want.double()).abs() <= 2 * 2.0 ** -11 * want.double().abs() + 2.0 ** -25).all()), (large, sign)


@pytest.mark.parametrize("tokens", [2, 300])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_of_a_scale_of_zero_and_of_none(pk, cuda, dim, tokens):
    """Scale 0 makes all keys alike, whatever they score (1e37 here); a scale that is no number makes rows that are none."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    v = torch.randn(12, 32, 2, dim, generator=gen, device="cuda").to(BF16)
    k = torch.zeros_like(v)
    k[..., 0] = torch.randn(12, 32, 2, generator=gen, device="cuda") * 1e18
    q = torch.zeros(tokens, 4, dim, dtype=BF16, device="cuda")
    q[..., 0] = 1e19
    lse = torch.empty(tokens, 4, device="cuda")
    rest = (k, v, torch.arange(12, dtype=torch.int32, device="cuda")[None], torch.tensor([0, tokens], dtype=torch.int32, device="cuda"),
            torch.tensor([384], dtype=torch.int32, device="cuda"))
    out = pk.ops.paged_attention(q, *rest, causal=False, scale=0.0, lse=lse)
    flat = v.view(384, 2, dim).double()
    want, spread = (t.mean(0).repeat_interleave(2, 0) for t in (flat, flat.abs()))
    # half a step of each weight and of the output; 1e-4 for the exponentials
    assert bool(((out.double() - want).abs() <= (2.0 ** -8 + 1e-4) * spread + 2.0 ** -8 * want.abs()).all())
    assert float((lse.double() - math.log(384.0)).abs().max()) <= 1.1e-4
    out = pk.ops.paged_attention(q, *rest, causal=False, scale=math.nan, lse=lse)
    assert bool(out.isnan().all()) and bool(lse.isnan().all())


@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("kernel,dim", [("rows", 64), ("rows", 128), ("chunk", 64), ("chunk", 128)])
def test_attention_sums_of_small_weights_beside_a_large_one(pk, cuda, kernel, dim, first):
    """The same rows with values of 1 and -1: sums that hold the large term have to take up the small ones.  Tolerance as above, and
    what the tensor cores may lose of the 16384 keys that they add to one sum, 2.8e-3 / 8.  lse: the scores are exact; ln 2 and
    log2(e) as factors of them, with their roundings, 26 * 2^-22, and the exponentials' 1.1e-4 of the small part; below 1e-5."""
    args, want, want_lse = _one_key_and_many(kernel, dim, F16, first, 1.0)
    lse = torch.empty(args["query"].shape[:2], device="cuda")
    out = pk.ops.paged_attention(**args, lse=lse)
    tolerance = 2.0 ** -11 * (1 + abs(want)) + 2.0 ** 17 * 2.0 ** -31 + 16384 * 2.0 ** -25.5 + 1e-5
    assert tolerance < 0.6 * abs(1 / (1 + 2.0 ** -8.5) - want)                   # what a row without the small ones is off
    assert float((out.double() - want).abs().max()) <= tolerance
    assert float((lse.double() - want_lse).abs().max()) <= 1e-5


def _repeated(keys, new, requests, dim, heads, kv, value, dtype=F16):
    """Requests over 16 pages again and again: as many keys as wanted, all of score 0 and of this value."""
    page, pages = 256, 16
    table = (torch.arange(-(-keys // page), device="cuda", dtype=torch.int32) % pages).expand(requests, -1).contiguous()
    return dict(query=torch.zeros(requests * new, heads, dim, dtype=dtype, device="cuda"), key_cache=torch.zeros(pages, page, kv, dim, dtype=dtype, device="cuda"),
                value_cache=torch.full((pages, page, kv, dim), value, dtype=dtype, device="cuda"), block_table=table,
                starts=torch.arange(requests + 1, dtype=torch.int32, device="cuda") * new,
                lengths=torch.full((requests,), keys, dtype=torch.int32, device="cuda"), causal=False, max_new=new)


@pytest.mark.parametrize("requests,new,heads", [(37, 1, 8), (1, 4864, 8), (1, 20, 16), (40, 20, 16), (3, 700, 16)])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_means_of_many_keys(pk, cuda, dim, requests, new, heads):
    """The mean of 2^19 equal values is that value: the weights are exact, the tensor cores lose up to 2^-23 of a sum for 16 keys, 1024 times
    at most, and the output is rounded."""
    for keys in (1 << 19, 70001, 8192, 8193, 16384, 16385):
        args = _repeated(keys, new, requests, dim, heads, 8, 1.7)
        value = float(args["value_cache"][0, 0, 0, 0])
        lse = torch.empty(args["query"].shape[:2], device="cuda")
        out = pk.ops.paged_attention(**args, lse=lse)
        assert float((out.double() - value).abs().max()) <= value * (2.0 ** -11 + 1024 * 2.0 ** -23 + 1e-6), keys
        assert float((lse.double() - math.log(keys)).abs().max()) <= 2e-6 * math.log(keys)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_whose_maximum_grows_over_many_keys(pk, cuda, dim, dtype):
    """Rows over 40 000 keys, two and a half sums in tensor memory, while the scores grow: what has left it is scaled down."""
    kv, heads, tokens, page, keys = 8, 16, 2400, 64, 40000
    pages = -(-keys // page)
    normal = lambda seed, *shape: torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")
    grow = torch.linspace(0.05, 3.0, pages * page, device="cuda")[:, None, None]
    k = (normal(1, pages * page, kv, dim) * grow).to(dtype)
    v, q = normal(2, pages * page, kv, dim).to(dtype), normal(3, tokens, heads, dim).to(dtype)
    lse = torch.empty(tokens, heads, device="cuda")
    out = pk.ops.paged_attention(q, k.view(pages, page, kv, dim), v.view(pages, page, kv, dim), torch.arange(pages, dtype=torch.int32, device="cuda")[None],
                                 torch.tensor([0, tokens], dtype=torch.int32, device="cuda"), torch.tensor([keys], dtype=torch.int32, device="cuda"), lse=lse)
    rows = torch.tensor([0, 1, 127, 128, 1000, 2271, 2399], device="cuda")
    want, want_lse, spread, off = R.attention(q[rows], k[:keys], v[:keys], keys - tokens + rows, True, 0, 1 / math.sqrt(dim))
    assert bool(((out[rows].double() - want).abs() <= R.attention_tolerance(want, spread, off, v, 1, dtype) + 1e-4 * spread).all())
    assert float((lse[rows].double() - want_lse).abs().max()) <= 24 * 2.0 ** -22 * off + 1e-5 * (1 + off)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_lse_of_a_row_that_one_key_dominates(pk, cuda, dim, dtype):
    """In the second block of keys, in each of its places (one a head), a key a little less than 2^8 above the first one's largest, so
    that the kernel's reference stays behind: the row's lse is that key's score and the sum's logarithm.  The exponentials are good
    to 2.9e-6, their argument and the sum to some units of 2^-22 of at most 16, the result to 2^-23 of at most 6."""
    heads, tokens, keys = 128, 40, 256
    q = torch.zeros(tokens, heads, dim, dtype=dtype, device="cuda")
    q[..., 0] = 1
    v = torch.randn(4, 64, heads, dim, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda").to(dtype)
    for large in (7.25, 7.3125, 6.625, 5.6875, 4.5):
        k = torch.zeros(4, 64, heads, dim, dtype=dtype, device="cuda")
        flat = k.view(keys, heads, dim)
        flat[:, :, 0] = -40.0
        flat[0, :, 0] = 0.0
        for h in range(heads):
            flat[128 + h, h, 0] = large
        lse = torch.empty(tokens, heads, device="cuda")
        out = pk.ops.paged_attention(q, k, v, torch.arange(4, dtype=torch.int32, device="cuda")[None], torch.tensor([0, tokens], dtype=torch.int32, device="cuda"),
                                     torch.tensor([keys], dtype=torch.int32, device="cuda"), causal=False, scale=math.log(2.0), lse=lse)
        total = 1 + 2.0 ** large + 254 * 2.0 ** -40
        assert float((lse.double() - math.log(total)).abs().max()) <= 2.9e-6 + 16 * 2.0 ** -22 + 6 * 2.0 ** -23, large
        flat_v = v.view(keys, heads, dim).double()
        picked = torch.stack([flat_v[128 + h, h] for h in range(heads)])
        want = (flat_v[0] + 2.0 ** large * picked + 2.0 ** -40 * (flat_v.sum(0) - flat_v[0] - picked)) / total
        half = 2.0 ** -11 if dtype is F16 else 2.0 ** -8
        bound = (half + 1e-5) * (flat_v[0].abs() + 2.0 ** large * picked.abs()) / total + half * want.abs() + 1e-6
        assert bool(((out.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,kv,dim", [(8, 8, 128), (16, 2, 64), (20, 4, 128)])
def test_attention_of_single_tokens_rounds_no_weight(pk, cuda, heads, kv, dim, dtype):
    """Where values cancel, a rounding of the weights would show beside the small output: there is none but the output's.  The
    weights' second numbers leave a half step of a step, and a last bit of that is set: (1 + 2) * 2 half steps of a half step."""
    s = Step([1] * 8, [0, 1, 20, 63, 64, 500, 3000, 9000], heads, kv, dim, 32, dtype, seed=11)
    s.q.mul_(0.2)
    out, at, half = s.run(pk, max_new=1), 0, R.HALF[dtype]
    for r, (n, c) in enumerate(zip(s.new, s.cached)):
        k, v = (R.paged(cache, s.table[r], c + n) for cache in (s.k_cache, s.v_cache))
        want, _, spread, off = R.attention(s.q[at:at + n], k, v, torch.arange(c, c + n, device="cuda"), True, 0, dim ** -0.5)
        score = 24 * 2.0 ** -22 * off + 1e-6                           # of an exponent: see attention_tolerance
        bound = half * want.abs() + (6 * half * half + 2 * score) * spread + R.TINY[dtype]
        assert bool(((out[at:at + n].double() - want).abs() <= bound).all()), r
        at += n


# ------------------------------------------------------------- few-row products
def test_gemv_of_more_columns_than_a_block_counts_in_32_bits(pk, cuda):
    """One block takes 1.5 M columns (12 GB of codes): its tiles times its chunks pass 2^31.  The bits are those of all blocks."""
    n, k = 1500000, 16512
    codes = torch.empty(n, k // 2, dtype=torch.uint8, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(1)
    for part in codes.split(100000):
        part.copy_(torch.randint(0, 256, part.shape, generator=gen, device="cuda", dtype=torch.uint8))
    scales = (torch.rand(k // 128, n, generator=gen, device="cuda") * 0.02 + 1e-4).half()
    x = torch.randn(2, k, generator=gen, device="cuda").half()
    want = pk.ops.gemv_w4g128(x, codes, scales, out_type=pk.lib.OUT_F32)
    out = torch.full_like(want, 7.0)
    try:
        pk.lib.lib.pk100_set_gemm_cta_cap(1)
        pk.ops.gemv_w4g128(x, codes, scales, out=out, out_type=pk.lib.OUT_F32)
    finally:
        pk.lib.lib.pk100_set_gemm_cta_cap(0)
    assert torch.equal(out, want)
    rows = torch.tensor([0, 1, 63, 64, 749999, 1372096, 1372097, 1499999], device="cuda")
    w = R.w4_weights(codes[rows], scales[:, rows])
    ref = x.double() @ w.t()
    assert bool(((out[:, rows].double() - ref).abs() <= R.gemv_tolerance(x, w, ref, torch.float32)).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("tokens,causal", [(1, True), (3, False), (150, False)])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_of_an_infinite_value(pk, cuda, dim, tokens, causal, dtype):
    """A value that is infinite makes that feature of the rows that see it infinite, of its sign, not NaN; the others stay."""
    s = Step([tokens], [90], 4, 2, dim, 32, dtype, seed=6)
    want = s.run(pk, causal=causal).clone()
    places = {(5, 0, 3): math.inf, (77, 1, 9): -math.inf, (40, 1, dim - 1): math.inf}
    for (j, h, d), value in places.items():
        s.v_cache[int(s.table[0, j // 32]), j % 32, h, d] = value
    out = s.run(pk, causal=causal)
    for (j, h, d), value in places.items():
        assert bool((out[:, 2 * h:2 * h + 2, d] == value).all()), (j, h, d)
        want[:, 2 * h:2 * h + 2, d] = value
    assert torch.equal(out, want)
