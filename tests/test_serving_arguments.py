"""Refusals of the serving operators, on the host: no GPU, nothing is launched.  Pointers are numbers that no launch sees."""
import ctypes as C

import pytest
import torch


def _norm(L, **changes):
    a = L.RmsNormArgs(type=L.TYPE_F16, mode=L.LN_S8_ROW, rows=4, width=64, input=256, ld_in=64, residual=512, ld_res=64, residual_out=512,
                      ld_res_out=64, gamma=1024, eps=1e-5, inv_scale=1.0, output=2048, ld_out=64, scales=4096)
    for name, value in changes.items():
        setattr(a, name, value)
    return L.lib.pk100_add_rms_norm(None, a)


def test_norm_refusals(pk):
    L = pk.lib
    assert L.lib.pk100_add_rms_norm(None, None) == L.ERR_NULL
    assert _norm(L, input=None) == _norm(L, gamma=None) == _norm(L, output=None) == _norm(L, scales=None) == L.ERR_NULL
    assert _norm(L, type=2) == _norm(L, mode=L.LN_S4_ROW) == _norm(L, mode=-1) == L.ERR_UNSUPPORTED
    assert _norm(L, rows=-1) == _norm(L, width=0) == _norm(L, ld_in=63) == _norm(L, ld_res=1) == _norm(L, ld_out=0) == L.ERR_SHAPE
    assert _norm(L, ld_res_out=63) == L.ERR_SHAPE
    assert _norm(L, width=32769, ld_in=40000, ld_res=40000, ld_res_out=40000, ld_out=40000) == L.ERR_LIMIT
    assert _norm(L, input=257) == _norm(L, scales=4098) == _norm(L, gamma=1025) == _norm(L, residual=513) == L.ERR_ALIGN
    assert _norm(L, mode=L.LN_F16, output=2049) == L.ERR_ALIGN
    assert _norm(L, rows=0, input=None) == L.OK


def _gemv(L, **changes):
    a = L.GemmArgs(kind=L.KIND_F16_W4G128, epilogue=L.EPI_LINEAR, m=3, n=40, k=256, a=256, lda=256, b=512, ldb=128, row_scale=1.0, alpha=1.0,
                   out=1024, ld_out=40, out_type=L.OUT_F16, b_group_scales=2048)
    for name, value in changes.items():
        setattr(a, name, value)
    return L.lib.pk100_gemv_w4g128(None, a)


def test_gemv_refusals(pk):
    L = pk.lib
    assert L.lib.pk100_gemv_w4g128(None, None) == L.ERR_NULL
    assert _gemv(L, a=None) == _gemv(L, b=None) == _gemv(L, out=None) == _gemv(L, b_group_scales=None) == L.ERR_NULL
    assert _gemv(L, kind=L.KIND_F16) == _gemv(L, epilogue=L.EPI_GLU) == _gemv(L, act=3) == _gemv(L, out_type=L.OUT_S8) == L.ERR_UNSUPPORTED
    assert _gemv(L, m=-1) == _gemv(L, n=0) == _gemv(L, k=0) == _gemv(L, k=192) == L.ERR_SHAPE
    assert _gemv(L, lda=255) == _gemv(L, lda=260) == _gemv(L, ld_out=39) == _gemv(L, residual=512, ld_res=39) == L.ERR_SHAPE
    assert _gemv(L, m=17) == L.ERR_LIMIT
    assert _gemv(L, a=264) == _gemv(L, b=520) == _gemv(L, out=1025) == _gemv(L, bias=2) == _gemv(L, out_type=L.OUT_F32, out=1026) == L.ERR_ALIGN
    assert _gemv(L, m=0, a=None) == L.OK


def _plan(L, **changes):
    a = L.PagedPlanArgs(requests=2, tokens=8, page_size=16, max_pages=4, free_capacity=9, cached=256, new_tokens=512, free_pages=1024, free_count=1280,
                        block_table=2048, starts=4096, lengths=4352, positions=4608, slots=5120, used=6144)
    for name, value in changes.items():
        setattr(a, name, value)
    return L.lib.pk100_paged_plan(None, a)


def test_plan_refusals(pk):
    L = pk.lib
    assert L.lib.pk100_paged_plan(None, None) == L.ERR_NULL
    for name in ("cached", "new_tokens", "free_count", "block_table", "starts", "lengths", "positions", "slots", "used"):
        assert _plan(L, **{name: None}) == L.ERR_NULL, name
    assert _plan(L, requests=-1) == _plan(L, tokens=-1) == _plan(L, page_size=0) == _plan(L, max_pages=0) == L.ERR_SHAPE
    assert _plan(L, requests=L.PLAN_MAX_REQUESTS + 1) == L.ERR_LIMIT
    # in place: other blocks read what one has written
    assert _plan(L, lengths=256) == _plan(L, lengths=512) == L.ERR_UNSUPPORTED
    assert _plan(L, free_capacity=-1) == L.ERR_SHAPE
    assert _plan(L, cached=258) == _plan(L, slots=5124) == _plan(L, status=2) == L.ERR_ALIGN


def test_plan_refuses_more_rows_than_it_counts(pk):
    # a warp's end of its run is at most the rows and 32 * 4 on top: in 32 bits up to 2^30 rows, not at the largest int
    L = pk.lib
    assert _plan(L, tokens=(1 << 30) + 1) == _plan(L, tokens=(1 << 31) - 1) == L.ERR_LIMIT


def _attention(L, **changes):
    a = L.PagedAttentionArgs(type=L.TYPE_BF16, tokens=6, requests=2, heads=8, kv_heads=2, head_dim=64, pages=10, page_size=16, max_pages=4,
                             query=4096, ld_query=512, key_cache=8192, value_cache=16384, page_stride=2048, token_stride=128,
                             head_stride=64, starts=256, lengths=512, block_table=1024, causal=1, window=0, scale=0.125, out=32768, ld_out=512,
                             workspace=65536, workspace_bytes=1 << 30)
    for name, value in changes.items():
        setattr(a, name, value)
    return L.lib.pk100_paged_attention(None, a)


def test_attention_refusals(pk):
    L = pk.lib
    new = dict(key=4096, ld_key=128, value=8192, ld_value=128, slots=512)
    assert L.lib.pk100_paged_attention(None, None) == L.ERR_NULL
    for name in ("query", "key_cache", "value_cache", "starts", "lengths", "block_table", "out", "workspace"):
        assert _attention(L, **{name: None}) == L.ERR_NULL, name
    assert _attention(L, **dict(new, value=None)) == _attention(L, **dict(new, slots=None)) == L.ERR_NULL
    assert _attention(L, type=7) == _attention(L, head_dim=96) == _attention(L, page_size=24) == _attention(L, page_size=512) == L.ERR_UNSUPPORTED
    assert _attention(L, tokens=-1) == _attention(L, requests=-1) == _attention(L, heads=7) == _attention(L, kv_heads=0) == L.ERR_SHAPE
    assert _attention(L, pages=0) == _attention(L, max_pages=0) == _attention(L, ld_query=511) == _attention(L, ld_out=516) == L.ERR_SHAPE
    assert _attention(L, **dict(new, ld_key=100)) == _attention(L, **dict(new, ld_value=132)) == L.ERR_SHAPE
    assert _attention(L, token_stride=60) == _attention(L, head_stride=68) == _attention(L, page_stride=4) == L.ERR_SHAPE
    assert _attention(L, page_stride=1 << 39) == L.ERR_SHAPE
    assert _attention(L, max_pages=1 << 27) == _attention(L, tokens=1 << 28) == _attention(L, requests=1 << 28) == L.ERR_LIMIT
    assert _attention(L, workspace_bytes=1000) == L.ERR_LIMIT
    assert _attention(L, query=4104) == _attention(L, key_cache=8200) == _attention(L, workspace=65552) == L.ERR_ALIGN
    assert _attention(L, **dict(new, key=4104)) == _attention(L, **dict(new, slots=516)) == _attention(L, starts=258) == L.ERR_ALIGN
    assert _attention(L, tokens=0, query=None) == _attention(L, requests=0, lengths=None) == L.OK


def test_attention_workspace_is_asked_for_in_bytes(pk):
    L = pk.lib
    a = L.PagedAttentionArgs(type=L.TYPE_F16, tokens=4, requests=2, heads=8, kv_heads=2, head_dim=128, pages=9, page_size=16, max_pages=4)
    small = L.lib.pk100_paged_attention_workspace_bytes(a)
    a.tokens, a.requests, a.max_pages = 4096, 64, 2048
    assert 0 < small < L.lib.pk100_paged_attention_workspace_bytes(a) < 1 << 28
    a.head_dim = 80
    assert L.lib.pk100_paged_attention_workspace_bytes(a) == 0
    assert C.sizeof(L.PagedAttentionArgs) % 8 == 0


def test_wrappers_refuse_tensors_of_the_host(pk):
    ops, x = pk.ops, torch.zeros(2, 128, dtype=torch.float16)
    with pytest.raises(pk.lib.Pk100Error):
        ops.add_rms_norm(x, x[0])
    with pytest.raises(pk.lib.Pk100Error):
        ops.gemv_w4g128(x, torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(1, 4, dtype=torch.float16))
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(pk.lib.Pk100Error):
        ops.paged_plan(i, i, i[:, None], i, i[:1], tokens=4, page_size=16)
    with pytest.raises(TypeError):
        ops.add_rms_norm(x.float(), x[0].float())
    with pytest.raises(ValueError):
        ops.add_rms_norm(x, x[0], mode=pk.lib.LN_S4_ROW)


class _Placed(torch.Tensor):
    """A tensor of the host that says it is on the current device: the wrapper's checks without a GPU."""
    def get_device(self):
        return 0


def _attention_call(pk, monkeypatch, kv_heads=2, **changes):
    placed = lambda *shape, dtype=torch.float16: torch.zeros(shape, dtype=dtype).as_subclass(_Placed)
    monkeypatch.setattr(pk.ops, "_device", lambda t: 0)
    args = dict(query=placed(3, 8, 64), key_cache=placed(5, 16, kv_heads, 64), value_cache=placed(5, 16, kv_heads, 64),
                block_table=placed(1, 4, dtype=torch.int32), starts=placed(2, dtype=torch.int32), lengths=placed(1, dtype=torch.int32))
    new = dict(key=placed(3, 2, 64), value=placed(3, 2, 64), slots=placed(3, dtype=torch.int64))
    args.update({name: new[name] for name in changes.pop("new", ())}, **changes)
    return pk.ops.paged_attention(**args)


@pytest.mark.parametrize("new", [("value",), ("value", "slots"), ("key",), ("key", "value"), ("key", "slots")])
def test_attention_wants_key_value_and_slots_together(pk, monkeypatch, new):
    with pytest.raises(ValueError, match="together"):
        _attention_call(pk, monkeypatch, new=new)


@pytest.mark.parametrize("kv_heads", [0, 3])
def test_attention_refuses_heads_that_do_not_divide(pk, monkeypatch, kv_heads):
    with pytest.raises(ValueError, match="evenly"):
        _attention_call(pk, monkeypatch, kv_heads=kv_heads)
