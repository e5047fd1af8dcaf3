"""torch-tensor convenience wrappers around the C ABI.

torch supplies device memory and the current stream; every computation happens
inside libpk100.so.  Tensors must be CUDA and contiguous where stated.
"""
from __future__ import annotations

import functools
import struct
from collections import namedtuple

import torch

from . import lib as L

EPS = 1e-5


# The arguments of a GEMM as bytes (native sizes and alignment): filling the structure field by field took half of
# the host time of a launch.
def _packer(args):
    packer = struct.Struct("@" + "".join({L.i32: "i", L.f32: "f", L.vp: "P", L.i64: "q"}[t] for _, t in args._fields_) + "0P")
    assert packer.size == L.C.sizeof(args)
    return packer


def _taking_bytes(name):
    function = L.lib[name]                       # (a function object of its own, with bytes as its argument)
    function.argtypes, function.restype = [L.vp, L.C.c_char_p], L.i32
    return function


_GEMM_ARGS, _gemm = _packer(L.GemmArgs), _taking_bytes("pk100_gemm")


def _ptr(t):
    return 0 if t is None else t.data_ptr()


# torch.cuda.current_stream().cuda_stream without the Stream object around it, where torch has it (a private name)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream():
    if _raw_stream is None:
        return torch.cuda.current_stream().cuda_stream
    return _raw_stream(torch.cuda.current_device())


def _need(t, dtype=None):
    if not t.is_cuda:
        raise L.Pk100Error("libpk100 operates on CUDA tensors only (there is no CPU path)")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"expected {dtype}, got {t.dtype}")
    return t


def gemm(a, b, *, kind, out, epilogue=L.EPI_LINEAR, row_scales=None, row_scale=1.0,
         col_scales=None, bias=None, act=L.ACT_NONE, residual=None, alpha=1.0, valid_rows=0,
         out_type=L.OUT_F16, out_scale=1.0, tau=0.0, keep_out=None, stats_out=None, keep_in=None,
         status=None, max_ctas=0, n=None, b_group_scales=None):
    """D = epilogue(A . B^T); see `pk100_gemm` in include/pk100.h."""
    _need(a), _need(b), _need(out)
    m, k = a.shape
    fields = (                                   # in the order of GemmArgs
        kind, epilogue, m, b.shape[0] if n is None else n, k,
        a.data_ptr(), a.stride(0), b.data_ptr(), b.stride(0),
        _ptr(row_scales), row_scale, _ptr(col_scales), _ptr(bias),
        act, _ptr(residual), 0 if residual is None else residual.stride(0), alpha, valid_rows,
        out.data_ptr(), out.stride(0), out_type, out_scale,
        tau, _ptr(keep_out), _ptr(stats_out), _ptr(keep_in),
        _ptr(status), max_ctas, _ptr(b_group_scales))
    try:
        args = _GEMM_ARGS.pack(*fields)
    except (struct.error, OverflowError):        # what only the structure's own conversions take
        args = bytes(L.GemmArgs(*fields))
    L.check(_gemm(_stream(), args), "pk100_gemm")
    return out


def layer_norm(x, gamma, beta, mode=L.LN_F16, inv_scale=0.0, seg_stride=None, valid_rows=None,
               seg_valid=None, out=None, scales=None):
    _need(x, torch.float16)
    rows = x.shape[0]
    seg_stride = rows if seg_stride is None else seg_stride
    valid_rows = seg_stride if valid_rows is None else valid_rows
    if out is None:
        out = torch.empty((rows, 1024), device=x.device,
                          dtype=torch.float16 if mode == L.LN_F16 else
                          (torch.int8 if mode in (L.LN_S8_ROW, L.LN_S4_ROW) else torch.uint8))
    if scales is None and mode in (L.LN_E4M3_ROW, L.LN_S8_ROW, L.LN_S4_ROW):
        scales = torch.empty(rows, device=x.device, dtype=torch.float32)
    L.check(L.lib.pk100_layer_norm(_stream(), _ptr(x), _ptr(gamma), _ptr(beta), _ptr(out),
                                   _ptr(scales), mode, inv_scale, rows, seg_stride, valid_rows,
                                   _ptr(seg_valid), EPS), "pk100_layer_norm")
    return out, scales


def layer_norm_pair(x, gamma, beta, next_gamma, next_beta, next_mode, next_inv_scale=0.0,
                    seg_stride=None, valid_rows=None, seg_valid=None, out=None, next_out=None,
                    next_scales=None):
    _need(x, torch.float16)
    rows = x.shape[0]
    seg_stride = rows if seg_stride is None else seg_stride
    valid_rows = seg_stride if valid_rows is None else valid_rows
    if out is None:
        out = torch.empty_like(x)
    if next_out is None:
        next_out = torch.empty((rows, 1024), device=x.device,
                               dtype=torch.float16 if next_mode == L.LN_F16 else
                               (torch.int8 if next_mode in (L.LN_S8_ROW, L.LN_S4_ROW) else torch.uint8))
    if next_scales is None and next_mode in (L.LN_E4M3_ROW, L.LN_S8_ROW, L.LN_S4_ROW):
        next_scales = torch.empty(rows, device=x.device, dtype=torch.float32)
    L.check(L.lib.pk100_layer_norm_pair(
        _stream(), _ptr(x), _ptr(gamma), _ptr(beta), _ptr(out), _ptr(next_gamma), _ptr(next_beta),
        _ptr(next_out), _ptr(next_scales), next_mode, next_inv_scale, rows, seg_stride, valid_rows,
        _ptr(seg_valid), EPS), "pk100_layer_norm_pair")
    return out, next_out, next_scales


def quantize_fp8_fixed(x, inverse_scale):
    _need(x, torch.float16)
    out = torch.empty(x.shape, device=x.device, dtype=torch.uint8)
    L.check(L.lib.pk100_quantize_fp8_fixed(_stream(), _ptr(x), _ptr(out), x.numel(), inverse_scale),
            "pk100_quantize_fp8_fixed")
    return out


def quantize_int8(x, inverse_scale):
    _need(x, torch.float16)
    out = torch.empty(x.shape, device=x.device, dtype=torch.int8)
    L.check(L.lib.pk100_quantize_int8(_stream(), _ptr(x), _ptr(out), inverse_scale, x.numel()),
            "pk100_quantize_int8")
    return out


def pack_weight_rows(w, fmt):
    """fp16 [n, k] -> (packed, scales) ; S4_G128 returns fp16 group scales [k/128, n]."""
    _need(w, torch.float16)
    n, k = w.shape
    dev = w.device
    if fmt in (L.PACK_E4M3, L.PACK_S8):
        packed = torch.empty((n, k), device=dev, dtype=torch.uint8 if fmt == L.PACK_E4M3 else torch.int8)
    else:
        packed = torch.empty((n, k // 2), device=dev, dtype=torch.uint8)
    scales = torch.empty(n, device=dev, dtype=torch.float32) if fmt != L.PACK_S4_G128 else None
    gscales = torch.empty((k // 128, n), device=dev, dtype=torch.float16) if fmt == L.PACK_S4_G128 else None
    L.check(L.lib.pk100_pack_weight_rows(_stream(), _ptr(w), n, k, w.stride(0), fmt, _ptr(packed),
                                         _ptr(scales), _ptr(gscales)), "pk100_pack_weight_rows")
    return packed, (gscales if fmt == L.PACK_S4_G128 else scales)


def dequant_w4g128(codes, group_scales):
    n, k2 = codes.shape
    out = torch.empty((n, k2 * 2), device=codes.device, dtype=torch.float16)
    L.check(L.lib.pk100_dequant_w4g128(_stream(), _ptr(codes), _ptr(group_scales), n, k2 * 2,
                                       _ptr(out)), "pk100_dequant_w4g128")
    return out


def glu_masked(e, seg_stride=None, valid_rows=None, seg_valid=None):
    _need(e, torch.float16)
    rows = e.shape[0]
    seg_stride = rows if seg_stride is None else seg_stride
    valid_rows = seg_stride if valid_rows is None else valid_rows
    out = torch.empty((rows, 1024), device=e.device, dtype=torch.float16)
    L.check(L.lib.pk100_glu_masked(_stream(), _ptr(e), _ptr(out), rows, seg_stride, valid_rows,
                                   _ptr(seg_valid)), "pk100_glu_masked")
    return out


def unpack_s4(packed):
    """Packed INT4 codes [..., n/2] (low nibble = even index) -> INT8 codes [..., n]."""
    out = torch.empty(packed.shape[:-1] + (packed.shape[-1] * 2,), dtype=torch.int8, device=packed.device)
    L.check(L.lib.pk100_unpack_s4(_stream(), _ptr(packed), _ptr(out), packed.numel()), "pk100_unpack_s4")
    return out


def prune_2of4_e4m3(dense):
    """E4M3 bytes [rows, cols] with the two smaller magnitudes of every quartet zeroed
    (the values the reference's 2:4-sparse FF2 multiplies, kernels/sm89/encoder.cu:685-713)."""
    rows, cols = dense.shape
    out = torch.empty_like(dense)
    L.check(L.lib.pk100_prune_2of4_e4m3(_stream(), _ptr(dense), _ptr(out), rows, cols), "pk100_prune_2of4_e4m3")
    return out


def compress_2of4_e4m3(dense):
    """The reference's compressed FF2 activation arena: data [rows, cols/2] + metadata [rows, cols/8], flat."""
    rows, cols = dense.shape
    out = torch.empty(rows * cols * 5 // 8, dtype=torch.uint8, device=dense.device)
    L.check(L.lib.pk100_compress_2of4_e4m3(_stream(), _ptr(dense), _ptr(out), rows, cols), "pk100_compress_2of4_e4m3")
    return out


def decompress_2of4_e4m3(flat, rows, cols):
    out = torch.empty((rows, cols), dtype=torch.uint8, device=flat.device)
    L.check(L.lib.pk100_decompress_2of4_e4m3(_stream(), _ptr(flat), _ptr(out), rows, cols),
            "pk100_decompress_2of4_e4m3")
    return out


def depthwise_bn_silu(g, wdw, bn_gamma, bn_beta, bn_mean, bn_var, quantize=False, seg_stride=None,
                      valid_rows=None, seg_valid=None):
    _need(g, torch.float16)
    rows = g.shape[0]
    seg_stride = rows if seg_stride is None else seg_stride
    valid_rows = seg_stride if valid_rows is None else valid_rows
    segments = rows // seg_stride
    out = torch.empty((rows, 1024), device=g.device, dtype=torch.uint8 if quantize else torch.float16)
    scales = torch.empty(rows, device=g.device, dtype=torch.float32) if quantize else None
    L.check(L.lib.pk100_depthwise_bn_silu(
        _stream(), _ptr(g), _ptr(wdw), _ptr(bn_gamma), _ptr(bn_beta), _ptr(bn_mean), _ptr(bn_var),
        _ptr(out), _ptr(scales), int(quantize), segments, seg_stride, valid_rows, _ptr(seg_valid),
        EPS), "pk100_depthwise_bn_silu")
    return out, scales


def local_attention(q, k, v, pos, bias_u, bias_v, seg_stride=None, valid_rows=None,
                    seg_valid=None, out=None):
    """Tensor-core local relative-position attention (the hot-path kernel)."""
    rows = q.shape[0]
    seg_stride = rows if seg_stride is None else seg_stride
    valid_rows = seg_stride if valid_rows is None else valid_rows
    if out is None:
        out = torch.empty((rows, 1024), device=q.device, dtype=torch.float16)
    L.check(L.lib.pk100_local_relpos_attention(
        _stream(), _ptr(q), q.stride(0), _ptr(k), k.stride(0), _ptr(v), v.stride(0), _ptr(pos),
        _ptr(bias_u), _ptr(bias_v), _ptr(out), out.stride(0), rows // seg_stride, seg_stride,
        valid_rows, _ptr(seg_valid)), "pk100_local_relpos_attention")
    return out


def local_attention_tcgen05(q, k, v, pos, bias_u, bias_v, seg_stride=None, valid_rows=None,
                            seg_valid=None, out=None, status=None):
    """The tcgen05 kernel (128 queries per CTA, accumulators in tensor memory); seg_stride % 128 == 0."""
    rows = q.shape[0]
    seg_stride = rows if seg_stride is None else seg_stride
    valid_rows = seg_stride if valid_rows is None else valid_rows
    if out is None:
        out = torch.empty((rows, 1024), device=q.device, dtype=torch.float16)
    L.check(L.lib.pk100_local_relpos_attention_tcgen05(
        _stream(), _ptr(q), q.stride(0), _ptr(k), k.stride(0), _ptr(v), v.stride(0), _ptr(pos),
        _ptr(bias_u), _ptr(bias_v), _ptr(out), out.stride(0), rows // seg_stride, seg_stride,
        valid_rows, _ptr(seg_valid), _ptr(status)), "pk100_local_relpos_attention_tcgen05")
    return out


def local_attention_simple(q, k, v, pos, bias_u, bias_v, seg_stride=None, valid_rows=None,
                           seg_valid=None, out=None):
    rows = q.shape[0]
    seg_stride = rows if seg_stride is None else seg_stride
    valid_rows = seg_stride if valid_rows is None else valid_rows
    if out is None:
        out = torch.empty((rows, 1024), device=q.device, dtype=torch.float16)
    L.check(L.lib.pk100_local_relpos_attention_simple(
        _stream(), _ptr(q), q.stride(0), _ptr(k), k.stride(0), _ptr(v), v.stride(0), _ptr(pos),
        _ptr(bias_u), _ptr(bias_v), _ptr(out), out.stride(0), rows // seg_stride, seg_stride,
        valid_rows, _ptr(seg_valid)), "pk100_local_relpos_attention_simple")
    return out


def pack_position_heads(p):
    out = torch.empty((8, 272, 128), device=p.device, dtype=torch.float16)
    L.check(L.lib.pk100_pack_position_heads(_stream(), _ptr(p), _ptr(out)), "pk100_pack_position_heads")
    return out


# ---- operators of a language-model layer in serving
_RMS_NORM_ARGS, _add_rms_norm = _packer(L.RmsNormArgs), _taking_bytes("pk100_add_rms_norm")
_PAGED_PLAN_ARGS, _paged_plan = _packer(L.PagedPlanArgs), _taking_bytes("pk100_paged_plan")
_PAGED_ATTENTION_ARGS, _paged_attention = _packer(L.PagedAttentionArgs), _taking_bytes("pk100_paged_attention")
_gemv_w4g128 = _taking_bytes("pk100_gemv_w4g128")
_TYPES = {torch.float16: L.TYPE_F16, torch.bfloat16: L.TYPE_BF16}


def _type(t):
    code = _TYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"expected torch.float16 or torch.bfloat16, got {t.dtype}")
    return code


_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)      # (without the look whether CUDA is up)


def _device(t):
    """The operators launch on the current device's stream: its index, which what they are given has to have."""
    return _current_device() if t.is_cuda else -2


def _refuse(name, t, shape, dtype, device):
    if t.get_device() != device:
        raise L.Pk100Error(f"{name}: libpk100 operates on tensors of the current CUDA device only (there is no CPU path)")
    if t.dtype != dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    raise ValueError(f"{name}: the elements of a row have to lie one behind the other")


# (a tensor is looked at with as few calls as its checks take: they are most of the host time of a small launch)
def _whole(name, t, shape, dtype, device):
    """Address of a contiguous tensor of this shape and type."""
    if t.dtype is not dtype or t.get_device() != device or t.shape != shape or not t.is_contiguous():
        _refuse(name, t, shape, dtype, device)
    return t.data_ptr()


def _rows(name, t, shape, dtype, device):
    """Address of [rows, width] and elements between its rows."""
    if t.dtype is not dtype or t.get_device() != device or t.shape != shape:
        _refuse(name, t, shape, dtype, device)
    if t.is_contiguous():
        return t.data_ptr(), shape[1]
    step, inner = t.stride()
    if inner != 1 and shape[1] > 1 and shape[0] > 0:
        _refuse(name, t, shape, dtype, device)
    return t.data_ptr(), step if shape[0] > 1 else shape[1]           # (a single row's stride may be anything)


def _heads(name, t, shape, dtype, device):
    """Address of [tokens, heads, head_dim] and elements between its tokens."""
    if t.dtype is not dtype or t.get_device() != device or t.shape != shape:
        _refuse(name, t, shape, dtype, device)
    tokens, heads, dim = shape
    if t.is_contiguous():
        return t.data_ptr(), heads * dim
    step, head, inner = t.stride()
    if (inner != 1 or (head != dim and heads > 1)) and tokens > 0:
        _refuse(name, t, shape, dtype, device)
    return t.data_ptr(), step if tokens > 1 else heads * dim


def _stream_of(device):
    return _stream() if _raw_stream is None else _raw_stream(device)


def _out_dtype(mode, dtype):
    return dtype if mode == L.LN_F16 else torch.int8 if mode == L.LN_S8_ROW else torch.uint8


def add_rms_norm(x, gamma, residual=None, mode=L.LN_F16, inv_scale=0.0, eps=EPS, out=None, residual_out=None, scales=None):
    """(out, scales, s): s = x + residual, out = the RMS norm of s in `mode`; see `pk100_add_rms_norm`.

    x, residual [rows, width] fp16 or bf16, rows any distance apart.  s is kept in residual_out (one of the inputs, or
    a new tensor when a residual is given) and is x itself without a residual.  scales is None for the modes without them."""
    kind, dtype, shape, device = _type(x), x.dtype, x.shape, _device(x)
    if len(shape) != 2:
        raise ValueError(f"x: expected [rows, width], got {tuple(shape)}")
    rows, width = shape
    if mode not in (L.LN_F16, L.LN_E4M3_FIXED, L.LN_E4M3_ROW, L.LN_S8_ROW):
        raise ValueError(f"add_rms_norm has no output mode {mode}")
    x_at, x_ld = (x.data_ptr(), width) if x.is_contiguous() and device >= 0 and x.get_device() == device else _rows("x", x, shape, dtype, device)
    gamma_at = _whole("gamma", gamma, (width,), dtype, device)
    out_dtype = _out_dtype(mode, dtype)
    if out is None:
        out = torch.empty(shape, device=x.device, dtype=out_dtype)
    out_at, out_ld = _rows("out", out, shape, out_dtype, device)
    res_at = res_ld = kept_at = kept_ld = scales_at = 0
    if residual is not None:
        res_at, res_ld = _rows("residual", residual, shape, dtype, device)
        if residual_out is None:
            residual_out = torch.empty(shape, device=x.device, dtype=dtype)
    if residual_out is not None:
        kept_at, kept_ld = _rows("residual_out", residual_out, shape, dtype, device)
    if mode == L.LN_E4M3_ROW or mode == L.LN_S8_ROW:
        if scales is None:
            scales = torch.empty(rows, device=x.device, dtype=torch.float32)
        scales_at = _whole("scales", scales, (rows,), torch.float32, device)
    else:
        scales = None
    rc = _add_rms_norm(_stream_of(device), _RMS_NORM_ARGS.pack(kind, mode, rows, width, x_at, x_ld, res_at, res_ld, kept_at, kept_ld, gamma_at, eps,
                                                      inv_scale, out_at, out_ld, scales_at))
    L.check(rc, "pk100_add_rms_norm")
    return out, scales, x if residual_out is None else residual_out


def gemv_w4g128(a, codes, group_scales, *, out=None, row_scales=None, row_scale=1.0, col_scales=None, bias=None, act=L.ACT_NONE,
                residual=None, alpha=1.0, valid_rows=0, out_type=L.OUT_F16, status=None):
    """D = epilogue(A . W^T) for up to 16 rows, W from `pack_weight_rows(PACK_S4_G128)`; see `pk100_gemv_w4g128`."""
    m, k = a.shape
    n, device = codes.shape[0], _device(a)
    a_at, a_ld = _rows("a", a, (m, k), torch.float16, device)
    codes_at = _whole("codes", codes, (n, k // 2), torch.uint8, device)
    groups_at = _whole("group_scales", group_scales, (k // 128, n), torch.float16, device)
    dtype = torch.float32 if out_type == L.OUT_F32 else torch.float16
    if out is None:
        out = torch.empty((m, n), device=a.device, dtype=dtype)
    out_at, out_ld = _rows("out", out, (m, n), dtype, device)
    res_at, res_ld = (0, 0) if residual is None else _rows("residual", residual, (m, n), torch.float16, device)
    rows_at = 0 if row_scales is None else _whole("row_scales", row_scales, (m,), torch.float32, device)
    cols_at = 0 if col_scales is None else _whole("col_scales", col_scales, (n,), torch.float32, device)
    bias_at = 0 if bias is None else _whole("bias", bias, (n,), torch.float32, device)
    status_at = 0 if status is None else _whole("status", status, (1,), torch.int32, device)
    rc = _gemv_w4g128(_stream_of(device), _GEMM_ARGS.pack(
        L.KIND_F16_W4G128, L.EPI_LINEAR, m, n, k, a_at, a_ld, codes_at, k // 2, rows_at, row_scale, cols_at, bias_at, act, res_at, res_ld, alpha,
        valid_rows, out_at, out_ld, out_type, 1.0, 0.0, 0, 0, 0, status_at, 0, groups_at))
    L.check(rc, "pk100_gemv_w4g128")
    return out


PagedPlan = namedtuple("PagedPlan", "starts lengths positions slots used")


def paged_plan(cached, new_tokens, block_table, free_pages, free_count, *, tokens, page_size, status=None, out=None):
    """One step's bookkeeping of a paged cache; see `pk100_paged_plan`.

    cached, new_tokens [requests], block_table [requests, max_pages] (its new pages are written), free_pages [any],
    free_count [1], all int32.  `tokens` rows of positions (int32) and slots (int64) are returned in a PagedPlan with
    starts [requests + 1], lengths [requests] and used [1]; `out`: such a tuple to write to."""
    requests, max_pages = block_table.shape
    device, i32 = _device(block_table), torch.int32
    table_at = _whole("block_table", block_table, (requests, max_pages), i32, device)
    cached_at = _whole("cached", cached, (requests,), i32, device)
    new_at = _whole("new_tokens", new_tokens, (requests,), i32, device)
    free_at = _whole("free_pages", free_pages, free_pages.shape, i32, device)
    count_at = _whole("free_count", free_count, (1,), i32, device)
    status_at = 0 if status is None else _whole("status", status, (1,), i32, device)
    if out is None:
        words = block_table.new_empty(2 * requests + 2 + tokens)
        starts, lengths, positions, used = words.split_with_sizes((requests + 1, requests, tokens, 1))
        slots = block_table.new_empty(tokens, dtype=torch.int64)
        out = PagedPlan(starts, lengths, positions, slots, used)
        at = words.data_ptr()
        starts_at, lengths_at, positions_at, used_at = at, at + 4 * (requests + 1), at + 4 * (2 * requests + 1), at + 4 * (2 * requests + 1 + tokens)
        slots_at = slots.data_ptr()
    else:
        starts_at = _whole("starts", out.starts, (requests + 1,), i32, device)
        lengths_at = _whole("lengths", out.lengths, (requests,), i32, device)
        positions_at = _whole("positions", out.positions, (tokens,), i32, device)
        slots_at = _whole("slots", out.slots, (tokens,), torch.int64, device)
        used_at = _whole("used", out.used, (1,), i32, device)
    rc = _paged_plan(_stream_of(device), _PAGED_PLAN_ARGS.pack(requests, tokens, page_size, max_pages, free_pages.shape[0], cached_at, new_at, free_at, count_at, table_at, starts_at,
                                                      lengths_at, positions_at, slots_at, used_at, status_at))
    L.check(rc, "pk100_paged_plan")
    return out


@functools.lru_cache(maxsize=1024)
def _paged_workspace(device, tokens, requests, heads, kv_heads, head_dim, page_size, max_pages):
    args = L.PagedAttentionArgs(tokens=tokens, requests=requests, heads=heads, kv_heads=kv_heads, head_dim=head_dim, pages=1, page_size=page_size,
                                max_pages=max_pages)
    return L.lib.pk100_paged_attention_workspace_bytes(args)


def paged_attention_workspace(query, key_cache, block_table):
    """Bytes that `paged_attention` needs for these tensors on the current device."""
    return _paged_workspace(torch.cuda.current_device(), query.shape[0], block_table.shape[0], query.shape[1], key_cache.shape[2],
                            query.shape[2], key_cache.shape[1], block_table.shape[1])


def paged_attention(query, key_cache, value_cache, block_table, starts, lengths, *, key=None, value=None, slots=None, causal=True,
                    window=0, scale=None, max_new=0, out=None, lse=None, workspace=None, status=None):
    """Attention of new tokens over a paged cache; see `pk100_paged_attention`.

    query [tokens, heads, head_dim] fp16 or bf16 (tokens any distance apart), caches [pages, page_size, kv_heads, head_dim]
    with any strides of the first three dimensions (the same ones in both), block_table [requests, max_pages], starts
    [requests + 1] and lengths [requests] int32.  key, value [tokens, kv_heads, head_dim] with slots [tokens] int64 are
    written to the cache first.  scale: 1 / sqrt(head_dim) by default.  workspace (uint8): allocated for the call where
    it is not given; one that is given is not used by another call at the same time."""
    kind, dtype, device, shape, i32 = _type(query), query.dtype, _device(query), query.shape, torch.int32
    tokens, heads, head_dim = shape
    pages, page_size, kv_heads, _ = cache_shape = key_cache.shape
    requests, max_pages = table_shape = block_table.shape
    query_at, query_ld = _heads("query", query, shape, dtype, device)
    strides = key_cache.stride()
    for name, t in (("key_cache", key_cache), ("value_cache", value_cache)):
        if t.dtype is not dtype or t.get_device() != device or t.shape != cache_shape or cache_shape[3] != head_dim or strides[3] != 1:
            _refuse(name, t, (pages, page_size, kv_heads, head_dim), dtype, device)
    if value_cache.stride() != strides:
        raise ValueError("key_cache and value_cache have to have the same strides")
    table_at = _whole("block_table", block_table, table_shape, i32, device)
    starts_at = _whole("starts", starts, (requests + 1,), i32, device)
    lengths_at = _whole("lengths", lengths, (requests,), i32, device)
    key_at = key_ld = value_at = value_ld = slots_at = 0
    if key is not None or value is not None:
        if key is None or value is None or slots is None:
            raise ValueError("key, value and slots are given together")
        new_shape = (tokens, kv_heads, head_dim)
        key_at, key_ld = _heads("key", key, new_shape, dtype, device)
        value_at, value_ld = _heads("value", value, new_shape, dtype, device)
        slots_at = _whole("slots", slots, (tokens,), torch.int64, device)
    if not kv_heads or heads % kv_heads:
        raise ValueError(f"{heads} query heads do not share {kv_heads} key-value heads evenly")
    if out is None:
        out = torch.empty(shape, device=query.device, dtype=dtype)
    out_at, out_ld = _heads("out", out, shape, dtype, device)
    lse_at = 0 if lse is None else _whole("lse", lse, (tokens, heads), torch.float32, device)
    status_at = 0 if status is None else _whole("status", status, (1,), i32, device)
    if workspace is None:
        need = _paged_workspace(device, tokens, requests, heads, kv_heads, head_dim, page_size, max_pages)
        workspace = block_table.new_empty(need // 4)         # (whole multiples of 256 bytes)
    else:
        need = workspace.numel()
        _whole("workspace", workspace, (need,), torch.uint8, device)
    rc = _paged_attention(_stream_of(device), _PAGED_ATTENTION_ARGS.pack(
        kind, tokens, requests, heads, kv_heads, head_dim, pages, page_size, max_pages, query_at, query_ld, key_at, key_ld, value_at, value_ld,
        slots_at, key_cache.data_ptr(), value_cache.data_ptr(), strides[0], strides[1], strides[2], starts_at, lengths_at, table_at, int(causal),
        min(window, 1 << 30), min(max_new, 1 << 30), head_dim ** -0.5 if scale is None else scale, out_at, out_ld, lse_at,
        workspace.data_ptr(), need, status_at))
    L.check(rc, "pk100_paged_attention")
    return out
