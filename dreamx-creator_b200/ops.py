"""Tensor-level wrappers over the C ABI (torch tensors in, device pointers out).

Each function validates dtype / device / layout, then calls exactly one entry
point of libsrdit_b200.so on the current CUDA stream. Nothing here computes:
there is no fallback when the library or a GPU is missing.
"""
from __future__ import annotations

import ctypes
import struct

import torch

from . import _lib

EPILOGUES = {"store": _lib.SRDIT_EPI_STORE, "gelu": _lib.SRDIT_EPI_GELU,
             "gated_res": _lib.SRDIT_EPI_GATED_RES, "res": _lib.SRDIT_EPI_RES}


class Stats:
    """Launch accounting.

    ``launches`` counts the kernels this module launched. When ``events`` is a
    list, every launch appends ``(kind, start_event, end_event, work)``, the
    events recorded on the launching stream around the launch and ``work`` its
    algorithmic FLOPs (GEMM, attention) or bytes (row kernels), so a profiling
    pass can attribute time per kernel kind. Leave it None in timed regions:
    the event records themselves cost time, and the lengths of packed sequences
    are read from the device, behind the launch (not while a graph is captured:
    ``work`` is 0 then).
    """
    launches = 0
    events = None


def _launch(name, *args, kind=None, work=0):
    ev = Stats.events
    if ev is not None:
        e0 = torch.cuda.Event(enable_timing=True)
        e1 = torch.cuda.Event(enable_timing=True)
        e0.record()
    _lib.call(name, *args)
    Stats.launches += 1
    if ev is not None:
        e1.record()
        ev.append((kind or name, e0, e1, int(work() if callable(work) else work)))


def _ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _addr(t):
    return None if t is None else t.data_ptr()


def _stream(device=None):
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _need_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise _lib.SrditError("the B200 kernels need CUDA tensors (there is no CPU path)")


def _rows(t: torch.Tensor):
    """(row stride in elements) of a 2-D row-major view with unit inner stride."""
    st = t.stride()
    if len(st) != 2 or st[1] != 1:
        raise _lib.SrditError(f"expected a 2-D row-major tensor, got shape {tuple(t.shape)} "
                              f"strides {st}")
    return st[0]


def as_rows(x, K):
    """x [..., K] as rows [M, K] that the row kernels take (unit inner stride, no row over
    another): a view where x is laid out so, else (expanded or transposed inputs) a copy."""
    rows = x.reshape(-1, K)
    st = rows.stride()
    if st[1] != 1 or (st[0] < K and rows.shape[0] > 1):
        rows = rows.clone(memory_format=torch.contiguous_format)
    return rows


def fp8_gemm(a_fp8, a_scale, w_fp8, w_scale, bias=None, out=None, *, epilogue="store",
             residual=None, gate=None, row_amax=None, status=None, v_ring=None):
    """out[M,N] = epilogue(a_fp8 @ w_fp8^T * a_scale[:,None] * w_scale[None,:] + bias).

    ``v_ring`` (STORE only): (ring [slots*frame_tokens, W] bf16, col0, frame_tokens,
    slot0, n_slots) -- columns [col0, N) go into the frame ring (output frame f
    into slot (slot0 + f) % n_slots) instead of ``out``."""
    _need_cuda(a_fp8, a_scale, w_fp8, w_scale, bias, out, residual, gate, row_amax)
    if a_fp8.dtype != torch.float8_e4m3fn or w_fp8.dtype != torch.float8_e4m3fn:
        raise _lib.SrditError("fp8_gemm operands must be float8_e4m3fn")
    M, K = a_fp8.shape
    N, K2 = w_fp8.shape
    if K != K2:
        raise _lib.SrditError(f"K mismatch {K} vs {K2}")
    if out is None:
        out = torch.empty(M, N, dtype=torch.bfloat16, device=a_fp8.device)
    for t, nm in ((a_scale, "a_scale"), (w_scale, "w_scale"), (gate, "gate"),
                  (row_amax, "row_amax")):
        if t is not None and (t.dtype != torch.float32 or not t.is_contiguous()):
            raise _lib.SrditError(f"{nm} must be contiguous float32")
    if bias is not None and (bias.dtype != torch.bfloat16 or not bias.is_contiguous()):
        raise _lib.SrditError("bias must be contiguous bf16")
    if v_ring is not None:
        if epilogue != "store":
            raise _lib.SrditError("v_ring needs the store epilogue")
        ring, col0, frame_tokens, slot0, n_slots = v_ring
        _need_cuda(ring)
        if ring.dtype != torch.bfloat16:
            raise _lib.SrditError("the V ring is bf16")
        vr = _lib.VRing(ctypes.c_void_p(ring.data_ptr()), _rows(ring), int(col0),
                        int(frame_tokens), int(slot0), int(n_slots))
        _launch("srdit_fp8_gemm_vring", _ptr(a_fp8), _ptr(a_scale), _ptr(w_fp8), _ptr(w_scale),
                _ptr(bias), _ptr(out), M, N, K, _rows(a_fp8), _rows(w_fp8), _rows(out),
                ctypes.byref(vr), _ptr(status), _stream(a_fp8.device), kind="fp8_gemm",
                work=2 * M * N * K)
        return out
    ldr = _rows(residual) if residual is not None else 0
    _launch("srdit_fp8_gemm", _ptr(a_fp8), _ptr(a_scale), _ptr(w_fp8), _ptr(w_scale),
            _ptr(bias), _ptr(out), M, N, K, _rows(a_fp8), _rows(w_fp8), _rows(out),
            EPILOGUES[epilogue], _ptr(residual), ldr, _ptr(gate), _ptr(row_amax),
            _ptr(status), _stream(a_fp8.device), kind="fp8_gemm", work=2 * M * N * K)
    return out


def quant_rowwise(x, amax=None, q=None, scale=None):
    """(e4m3 [M,K], fp32 scale [M]) of a bf16 [M,K] matrix (fp8_linear.py:93-103)."""
    _need_cuda(x, amax, q, scale)
    if x.dtype != torch.bfloat16:
        raise _lib.SrditError("quant_rowwise takes bf16")
    M, K = x.shape
    if q is None:
        q = torch.empty(M, K, dtype=torch.float8_e4m3fn, device=x.device)
    if scale is None:
        scale = torch.empty(M, dtype=torch.float32, device=x.device)
    _launch("srdit_quant_rowwise", _ptr(x), _rows(x), M, K, _ptr(amax), _ptr(q), _rows(q),
            _ptr(scale), _stream(x.device), kind="quant_rowwise",
            work=M * K * 3 + 4 * M)
    return q, scale


def ln_mod_quant(x, eps=1e-6, *, ln_weight=None, ln_bias=None, shift=None, scale=None,
                 q=None, qscale=None):
    """LayerNorm (+affine) -> bf16 -> adaLN modulate -> row-wise e4m3."""
    _need_cuda(x, ln_weight, ln_bias, shift, scale, q, qscale)
    if x.dtype != torch.bfloat16:
        raise _lib.SrditError("ln_mod_quant takes bf16")
    M, K = x.shape
    if q is None:
        q = torch.empty(M, K, dtype=torch.float8_e4m3fn, device=x.device)
    if qscale is None:
        qscale = torch.empty(M, dtype=torch.float32, device=x.device)
    _launch("srdit_ln_mod_quant", _ptr(x), _rows(x), M, K, float(eps), _ptr(ln_weight),
            _ptr(ln_bias), _ptr(shift), _ptr(scale), _ptr(q), _rows(q), _ptr(qscale),
            _stream(x.device), kind="ln_mod_quant", work=M * K * 2 + M * K + 4 * M)
    return q, qscale


def rms_rope(src, weight, eps, dst, *, frame_tokens, slot0=0, n_slots=1 << 30, cos=None,
             sin=None, grid_h=0, grid_w=0, t_offset=0, v_src=None, v_dst=None, ss=None,
             norm_width=0, t_offset_dev=None, w_offset=0, dst_grid_w=0, dst_w0=0, halo=None):
    """RMSNorm(src) * weight [-> 3-D RoPE] -> dst frame slots (+ V copy).

    ``ss`` ([M] fp32, optional): per-row sum of squares over ``norm_width``
    columns (a tensor-parallel slice's all-reduced statistic). ``t_offset_dev``
    (optional int32 [1] on the device): added to ``t_offset`` at run time.
    ``w_offset``: width position of the grid's column 0 (a strip of a wider grid).
    ``dst_grid_w`` > 0: destination frames of grid_h x dst_grid_w tokens, the
    grid's column c written to column c + ``dst_w0``. ``halo`` (a ``_lib.RopeHalo``):
    the strip's edge columns also stored into the neighbours' rings, then signalled."""
    _need_cuda(src, weight, dst, cos, sin, v_src, v_dst, ss)
    if ss is not None and (ss.dtype != torch.float32 or not ss.is_contiguous()):
        raise _lib.SrditError("ss must be contiguous float32")
    M, K = src.shape
    if cos is not None and (cos.dtype != torch.float64 or sin.dtype != torch.float64
                            or cos.shape != sin.shape or cos.shape[1] != 64
                            or not cos.is_contiguous() or not sin.is_contiguous()):
        raise _lib.SrditError("RoPE tables must be contiguous float64 [rows, 64]")
    tab_rows = cos.shape[0] if cos is not None else 0
    _launch("srdit_rms_rope", _ptr(src), _rows(src), M, K, _ptr(weight), float(eps),
            _ptr(dst), _rows(dst), int(frame_tokens), int(slot0), int(n_slots), _ptr(cos),
            _ptr(sin), int(tab_rows), int(grid_h), int(grid_w), int(t_offset), _ptr(v_src),
            _rows(v_src) if v_src is not None else 0, _ptr(v_dst),
            _rows(v_dst) if v_dst is not None else 0, _ptr(ss), int(norm_width),
            _ptr(t_offset_dev), int(w_offset), int(dst_grid_w), int(dst_w0),
            ctypes.byref(halo) if halo is not None else None,
            _stream(src.device), kind="rms_rope",
            work=M * K * 2 * (4 if v_src is not None else 2))
    return dst


DTYPES = {torch.bfloat16: _lib.SRDIT_BF16, torch.float16: _lib.SRDIT_FP16,
          torch.float32: _lib.SRDIT_FP32}
HALF_TYPES = {torch.bfloat16: _lib.SRDIT_BF16, torch.float16: _lib.SRDIT_FP16}
CODES = {torch.int8: _lib.SRDIT_Q_INT8, torch.float8_e4m3fn: _lib.SRDIT_Q_E4M3}


def _code(table, dtype, what):
    code = table.get(dtype)
    if code is None:
        raise _lib.SrditError(f"{what} takes {', '.join(map(str, table))}, got {dtype}")
    return code


def _same_device(x, *ts):
    """Every given tensor on x's device, and that the current one (kernels are launched
    on the current device). Returns the current stream's handle there."""
    dev = x.get_device()
    if dev < 0:
        _need_cuda(x)
    for t in ts:
        if t is not None and t.get_device() != dev:
            raise _lib.SrditError(f"tensors on {x.device} and {t.device}")
    if dev != torch._C._cuda_getDevice():
        raise _lib.SrditError(f"tensors on {x.device}, the current device is "
                              f"cuda:{torch.cuda.current_device()}")
    return torch._C._cuda_getCurrentRawStream(dev)


def _scales(t, n, what):
    if t.dtype != torch.float32 or t.shape != (n,) or not t.is_contiguous():
        raise _lib.SrditError(f"{what} must be contiguous float32 [{n}]")


def code_rows(M, K, dtype, device):
    """An empty [M, K] of 8-bit codes whose rows start 16 bytes apart at least, as the
    products' operands have to."""
    return torch.empty(M, (K + 15) // 16 * 16, dtype=dtype, device=device)[:, :K]


def _codes_out(x, M, K, qdtype, q, qscale):
    """The output tensors of a row quantiser of x [M, K], checked or made, and the code
    type's number."""
    if q is None:
        q = code_rows(M, K, qdtype or torch.int8, x.device)
    elif q.shape != (M, K) or (qdtype is not None and q.dtype != qdtype):
        raise _lib.SrditError(f"q {tuple(q.shape)} {q.dtype} for rows {(M, K)} to "
                              f"{qdtype or q.dtype}")
    if qscale is None:
        qscale = torch.empty(M, dtype=torch.float32, device=x.device)
    else:
        _scales(qscale, M, "qscale")
    return q, qscale, _code(CODES, q.dtype, "qdtype")


def add_rms_quant(x, weight, eps=1e-6, *, residual=None, sum_out=None, qdtype=None, q=None,
                  qscale=None):
    """RMS norm of x [+ residual], quantised per row to 8 bits in the same pass.

    x, residual [M, K] and weight [K] in one type (bf16, fp16 or fp32), K at most 32768.
    Returns (q, qscale, sum): codes [M, K] of ``qdtype`` (int8, the default, or
    float8_e4m3fn; or ``q``'s own), fp32 scales [M], and x + residual in x's type (None
    without a residual). ``sum_out`` may be x or residual, which is then updated in place.
    Without ``q`` the codes' rows are laid out as ``int8_gemm`` takes them."""
    stream = _same_device(x, weight, residual, sum_out, q, qscale)
    ldx = _rows(x)
    M, K = x.shape
    dt = _code(DTYPES, x.dtype, "add_rms_quant")
    if weight.dtype != x.dtype or weight.shape != (K,) or not weight.is_contiguous():
        raise _lib.SrditError(f"weight must be contiguous {x.dtype} [{K}]")
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise _lib.SrditError(f"residual must be {x.dtype} {tuple(x.shape)}")
        if sum_out is None:
            sum_out = torch.empty(M, K, dtype=x.dtype, device=x.device)
        elif sum_out.shape != x.shape or sum_out.dtype != x.dtype:
            raise _lib.SrditError(f"sum_out must be {x.dtype} {tuple(x.shape)}")
        ldr, lds = _rows(residual), _rows(sum_out)
    elif sum_out is not None:
        raise _lib.SrditError("sum_out without a residual")
    else:
        ldr = lds = 0
    q, qscale, code = _codes_out(x, M, K, qdtype, q, qscale)
    _launch("srdit_add_rms_quant", x.data_ptr(), ldx, M, K, dt, _addr(residual), ldr,
            weight.data_ptr(), eps, _addr(sum_out), lds, q.data_ptr(), _rows(q), code,
            qscale.data_ptr(), stream, kind="add_rms_quant",
            work=M * K * ((3 if residual is not None else 1) * x.element_size() + 1))
    return q, qscale, sum_out


def quant_rows(x, *, qdtype=None, q=None, qscale=None):
    """(codes [M, K], fp32 scales [M]) of rows of bf16, fp16 or fp32, K at most 32768: the
    row-wise quantiser for int8 codes and for the widths and types ``quant_rowwise`` does
    not take. Arguments as ``add_rms_quant``."""
    stream = _same_device(x, q, qscale)
    ldx = _rows(x)
    M, K = x.shape
    dt = _code(DTYPES, x.dtype, "quant_rows")
    q, qscale, code = _codes_out(x, M, K, qdtype, q, qscale)
    _launch("srdit_quant_rows", x.data_ptr(), ldx, M, K, dt, q.data_ptr(), _rows(q), code,
            qscale.data_ptr(), stream, kind="quant_rows", work=M * K * (x.element_size() + 1))
    return q, qscale


def int8_gemm(a_q, a_scale, w_q, w_scale, bias=None, out=None, *, out_dtype=None, status=None):
    """out[M,N] = a_q @ w_q^T * a_scale[:,None] * w_scale[None,:] + bias, the sum exact in int32.

    a_q [M, K], w_q [N, K] int8 with row pitches that are multiples of 16 (``code_rows``
    makes such), fp32 scales [M] and [N]; bias [N] in out's type: ``out_dtype`` bf16 (the
    default), fp16 or fp32, or ``out``'s own. Any M and N; K below 131072."""
    stream = _same_device(a_q, a_scale, w_q, w_scale, bias, out, status)
    if a_q.dtype != torch.int8 or w_q.dtype != torch.int8:
        raise _lib.SrditError("int8_gemm operands must be int8")
    lda, ldw = _rows(a_q), _rows(w_q)
    M, K = a_q.shape
    N, K2 = w_q.shape
    if K != K2:
        raise _lib.SrditError(f"K mismatch {K} vs {K2}")
    _scales(a_scale, M, "a_scale")
    _scales(w_scale, N, "w_scale")
    if out is None:
        out = torch.empty(M, N, dtype=out_dtype or torch.bfloat16, device=a_q.device)
    elif out.shape != (M, N) or (out_dtype is not None and out.dtype != out_dtype):
        raise _lib.SrditError(f"out {tuple(out.shape)} {out.dtype} for a product {(M, N)} in "
                              f"{out_dtype or out.dtype}")
    if bias is not None and (bias.dtype != out.dtype or bias.shape != (N,)
                             or not bias.is_contiguous()):
        raise _lib.SrditError(f"bias must be contiguous {out.dtype} [{N}]")
    _launch("srdit_int8_gemm", a_q.data_ptr(), a_scale.data_ptr(), w_q.data_ptr(),
            w_scale.data_ptr(), _addr(bias), out.data_ptr(), _code(DTYPES, out.dtype, "int8_gemm"),
            M, N, K, lda, ldw, _rows(out), _addr(status), stream, kind="int8_gemm",
            work=2 * M * N * K)
    return out


def cross_attn(q, k, v, out=None, *, kv_lens=None, key_mask=None, scale=None, status=None):
    """Attention of q [B, Lq, H, D] over an encoder's k, v [B, Lk, Hkv, D] (bf16 or fp16, unit
    stride over D, D a multiple of 8 up to 128, H a multiple of Hkv; views with other strides
    that are multiples of 8 elements are read in place). Returns out [B, Lq, H, D].

    ``kv_lens`` (int32 [B] on the device): sample b sees its first kv_lens[b] keys.
    ``key_mask`` (bool or uint8 [B, Lk]): keys that are seen. A query that sees no key gets
    zeros; what lies in the rows of unseen keys does not matter. ``scale``: D ** -0.5."""
    stream = _same_device(q, k, v, out, kv_lens, key_mask, status)
    dt = _code(HALF_TYPES, q.dtype, "cross_attn")
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape:
        raise _lib.SrditError(f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}: "
                              "[B, L, heads, D] each")
    B, Lq, H, D = q.shape
    Bk, Lk, Hkv, Dk = k.shape
    dtype = q.dtype
    if Bk != B or Dk != D or Hkv == 0 or H % Hkv or k.dtype != dtype or v.dtype != dtype:
        raise _lib.SrditError(f"q {tuple(q.shape)} {dtype} does not go with k "
                              f"{tuple(k.shape)} {k.dtype}, v {v.dtype}")
    if out is None:
        out = torch.empty(B, Lq, H, D, dtype=dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != dtype:
        raise _lib.SrditError(f"out must be {dtype} {tuple(q.shape)}")
    qs, ks, vs, os = q.stride(), k.stride(), v.stride(), out.stride()
    if not (qs[3] == ks[3] == vs[3] == os[3] == 1):
        raise _lib.SrditError(f"q, k, v, out need unit stride over D, have {qs}, {ks}, {vs}, {os}")
    lens = mask = mask_stride = 0
    if kv_lens is not None:
        if kv_lens.dtype != torch.int32 or kv_lens.shape != (B,) or not kv_lens.is_contiguous():
            raise _lib.SrditError(f"kv_lens must be contiguous int32 [{B}]")
        lens = kv_lens.data_ptr()
    if key_mask is not None:
        if key_mask.dtype not in (torch.bool, torch.uint8) or key_mask.shape != (B, Lk):
            raise _lib.SrditError(f"key_mask must be bool or uint8 {(B, Lk)}")
        if Lk > 1 and key_mask.stride(1) != 1:
            raise _lib.SrditError("key_mask needs unit stride over the keys")
        mask, mask_stride = key_mask.data_ptr(), key_mask.stride(0)
    a = _lib.CrossAttnArgs()
    fill = _lib.CROSS_ATTN_LAYOUT.pack_into
    fields = (q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), dt, B, Lq, Lk, H, Hkv, D,
              *qs[:3], *ks[:3], *vs[:3], *os[:3], lens, mask, mask_stride,
              D ** -0.5 if scale is None else scale)
    st = 0 if status is None else status.data_ptr()
    fill(a, 0, *fields, 0, 0, st)
    ref = ctypes.byref(a)
    kib = _lib.count("srdit_cross_attn_workspace", ref)
    if kib:
        ws = torch.empty(kib << 10, dtype=torch.uint8, device=q.device)
        fill(a, 0, *fields, ws.data_ptr(), kib << 10, st)
    _launch("srdit_cross_attn", ref, stream, kind="cross_attn",
            work=4 * B * Lq * H * D * Lk)
    if kib:
        Stats.launches += 1   # a second kernel joins the parts
    return out


_calls = ()   # the extension that makes a call's checks on the tensors themselves, when loaded


def _short(name, entry, *args):
    """A call by the extension's function ``name``; whether it was one (else the wrapper goes on
    with its own checks). Launches that are timed one by one go the long way."""
    global _calls
    if _calls == ():
        _calls = _lib.calls()
    if _calls is None or Stats.events is not None:
        return False
    rc = getattr(_calls, name)(*args)
    if rc is None:
        return False
    if rc:
        _lib.check(rc, entry)
    Stats.launches += 1
    return True


def _fill(layout, into, *fields):
    """Put a call's numbers into its C structure; those that its fields do not hold are refused."""
    try:
        layout.pack_into(into, 0, *fields)
    except (struct.error, OverflowError) as e:
        raise _lib.SrditError(f"sizes or numbers that the call's arguments do not hold: {e}") from None


def _int32(t, n, what):
    if t.dtype != torch.int32 or t.shape != (n,) or not t.is_contiguous():
        raise _lib.SrditError(f"{what} must be contiguous int32 [{n}]")
    return t.data_ptr()


def _pages(k_pages, v_pages, table, k_scale, v_scale, dtype):
    """The C view (``_lib.KvPages``) of a cache's pages, whose rows go to or from ``dtype``; the
    sequences, key heads and their width."""
    shape, held, ks, vs = k_pages.shape, k_pages.dtype, k_pages.stride(), v_pages.stride()
    if len(shape) != 4 or v_pages.shape != shape or v_pages.dtype != held:
        raise _lib.SrditError(f"pages {tuple(shape)} {held}, {tuple(v_pages.shape)} "
                              f"{v_pages.dtype}: [pages, page_size, kv_heads, D] of one type each")
    n, size, Hkv, D = shape
    if ks[3] != 1 or vs[3] != 1:
        raise _lib.SrditError(f"pages need unit stride over D, have {ks}, {vs}")
    entries, ts = table.shape, table.stride()
    if len(entries) != 2 or table.dtype != torch.int32 or (ts[1] != 1 and entries[1] > 1):
        raise _lib.SrditError("the page table must be int32 [sequences, pages] with unit stride")
    dt = HALF_TYPES.get(dtype)
    if dt is None:
        _code(HALF_TYPES, dtype, "rows of a cache")
    if held == dtype:
        if k_scale is not None or v_scale is not None:
            raise _lib.SrditError(f"scales for pages of {dtype}")
        code, scales, ss = _lib.SRDIT_KV_PLAIN, (0, 0), (0, 0, 0, 0, 0, 0)
    else:
        code = CODES.get(held)
        if code is None:
            _code(CODES, held, f"pages for rows of {dtype}, other than that type,")
        if k_scale is None or v_scale is None:
            raise _lib.SrditError(f"pages of {held} need k_scale and v_scale")
        rows = (n, size, Hkv)
        if (k_scale.shape != rows or v_scale.shape != rows or k_scale.dtype != torch.float32
                or v_scale.dtype != torch.float32):
            raise _lib.SrditError(f"scales must be float32 {rows}")
        scales = (k_scale.data_ptr(), v_scale.data_ptr())
        ss = k_scale.stride() + v_scale.stride()
    p = _lib.KvPages()
    B = entries[0]
    _fill(_lib.KV_PAGES_LAYOUT, p, k_pages.data_ptr(), v_pages.data_ptr(), *scales, code, dt, n, size,
          Hkv, D, *ks[:3], *vs[:3], *ss, table.data_ptr(), ts[0], entries[1], B)
    return p, B, Hkv, D


def _kv_rows(k, v, Hkv, D):
    """The tokens of packed k, v [T, Hkv, D], and the address of their strides {token, head} as the
    C entries take them, in a buffer that is to be kept."""
    shape, ks, vs = k.shape, k.stride(), v.stride()
    if v.shape != shape or len(shape) != 3 or shape[1] != Hkv or shape[2] != D or k.dtype != v.dtype:
        raise _lib.SrditError(f"k {tuple(shape)} {k.dtype}, v {tuple(v.shape)} {v.dtype}: "
                              f"[tokens, {Hkv}, {D}] of one type each")
    if ks[2] != 1 or vs[2] != 1:
        raise _lib.SrditError(f"k, v need unit stride over D, have {ks}, {vs}")
    if shape[0] > 0x7fffffff:   # (a C int)
        raise _lib.SrditError(f"{shape[0]} tokens")
    st = _lib.KvStrides(ks[0], ks[1], vs[0], vs[1])
    return shape[0], st, ctypes.addressof(st)


def _row_ends(cu, T, B):
    """The rows of B packed sequences as the kernels take them: (first, behind the last) of each."""
    if cu is None:
        return [(b * (T // B), (b + 1) * (T // B)) for b in range(B)]
    at = [min(max(x, 0), T) for x in cu.tolist()]
    return [(x, max(x, y)) for x, y in zip(at, at[1:])]


def _kv_bytes(T, B, cu, Hkv, D, rows, pages):
    """Bytes that kv_write and kv_read move: every sequence's rows, here and in the cache."""
    def work():
        if torch.cuda.is_current_stream_capturing():
            return 0
        held = D * pages.itemsize + (0 if pages == rows else 4)   # a scale with codes
        return 2 * Hkv * (D * rows.itemsize + held) * sum(y - x for x, y in _row_ends(cu, T, B))
    return work


def _attn_flops(shape, B, cu_q, keys, causal):
    """FLOPs of attention of packed sequences: 4 D for each query, head and key that it sees.
    ``keys()``: the sequences' lengths."""
    def work():
        if torch.cuda.is_current_stream_capturing():
            return 0
        (T, H, D), seen = shape, 0
        for (x, y), L in zip(_row_ends(cu_q, T, B), keys()):
            n = y - x
            if causal:   # the last of n sees L keys, each before it one less
                rows = min(n, L)
                seen += rows * L - rows * (rows - 1) // 2
            else:
                seen += n * L
        return 4 * H * D * seen
    return work


def kv_write(k, v, k_pages, v_pages, page_table, kv_lens, *, cu_q=None, k_scale=None,
             v_scale=None):
    """Write new tokens' k, v [T, Hkv, D] (bf16 or fp16) into a cache's pages.

    k_pages, v_pages [pages, page_size, Hkv, D]: of k's type, or int8 / float8_e4m3fn codes with
    float32 scales [pages, page_size, Hkv] (any strides). ``page_table`` int32 [B, width]: token
    p of sequence b lies in row p % page_size of page ``page_table[b, p // page_size]``.
    ``cu_q`` (int32 [B + 1]): sequence b's new tokens are the rows cu_q[b] to cu_q[b + 1] of k
    and v (default: T / B each); ``kv_lens`` (int32 [B]): its length with them. D a multiple of
    8 (16 for codes) up to 128, page_size 16, 32, 64 or a multiple of 128. A token whose page
    the table does not have is left out; no two tokens of a call may go to one row."""
    if _short("kv_write", "srdit_kv_write", k, v, k_pages, v_pages, page_table, kv_lens, cu_q,
              k_scale, v_scale):
        return
    stream = _same_device(k, v, k_pages, v_pages, page_table, kv_lens, cu_q, k_scale, v_scale)
    p, B, Hkv, D = _pages(k_pages, v_pages, page_table, k_scale, v_scale, k.dtype)
    T, st, at = _kv_rows(k, v, Hkv, D)
    _launch("srdit_kv_write", ctypes.byref(p), k.data_ptr(), at, v.data_ptr(), at + 16, T,
            None if cu_q is None else _int32(cu_q, B + 1, "cu_q"), _int32(kv_lens, B, "kv_lens"),
            stream, kind="kv_write", work=_kv_bytes(T, B, cu_q, Hkv, D, k.dtype, k_pages.dtype))


def kv_read(k_pages, v_pages, page_table, cu_k, k=None, v=None, *, total=None, dtype=None,
            k_scale=None, v_scale=None):
    """Read the first tokens of every sequence back: (k, v) [T, Hkv, D], sequence b's in the rows
    cu_k[b] to cu_k[b + 1] (int32 [B + 1]), codes times their scales. Without ``k`` and ``v``
    they are made, of ``total`` rows and ``dtype`` (bf16, or the pages' own). Rows behind the
    last sequence are left as they were; tokens without a page are zeros."""
    if k is None:
        if total is None or v is not None:
            raise _lib.SrditError("kv_read needs k and v, or total")
        dtype = dtype or (k_pages.dtype if k_pages.dtype in HALF_TYPES else torch.bfloat16)
        k, v = (torch.empty(total, *k_pages.shape[2:], dtype=dtype, device=k_pages.device)
                for _ in range(2))
    elif v is None or (dtype is not None and k.dtype != dtype) or (
            total is not None and k.shape[0] != total):
        raise _lib.SrditError("k and v do not go with total and dtype")
    if _short("kv_read", "srdit_kv_read", k_pages, v_pages, page_table, cu_k, k, v, k_scale,
              v_scale):
        return k, v
    stream = _same_device(k, v, k_pages, v_pages, page_table, cu_k, k_scale, v_scale)
    p, B, Hkv, D = _pages(k_pages, v_pages, page_table, k_scale, v_scale, k.dtype)
    T, st, at = _kv_rows(k, v, Hkv, D)
    _launch("srdit_kv_read", ctypes.byref(p), k.data_ptr(), at, v.data_ptr(), at + 16, T,
            _int32(cu_k, B + 1, "cu_k"), stream, kind="kv_read",
            work=_kv_bytes(T, B, cu_k, Hkv, D, k.dtype, k_pages.dtype))
    return k, v


def _seq_attn(kind, q, out, Hkv, width, B, pages, k, v, Tk, kv_strides, cu_q, cu_k, kv_lens, max_q,
              max_kv, causal, scale, status, stream, work):
    shape, dtype, qs = q.shape, q.dtype, q.stride()
    if len(shape) != 3 or shape[2] != width or Hkv == 0 or shape[1] % Hkv:
        raise _lib.SrditError(f"q {tuple(shape)} [tokens, heads, D] does not go with {Hkv} key heads "
                              f"of {width}")
    T, H, D = shape
    dt = HALF_TYPES.get(dtype)
    if dt is None:
        _code(HALF_TYPES, dtype, kind)
    if out.shape != shape or out.dtype != dtype:
        raise _lib.SrditError(f"out must be {dtype} {tuple(shape)}")
    os = out.stride()
    if qs[2] != 1 or os[2] != 1:
        raise _lib.SrditError(f"q, out need unit stride over D, have {qs}, {os}")
    a = _lib.SeqAttnArgs()
    fields = (pages, q.data_ptr(), k, v, out.data_ptr(), dt, T, Tk, B, H, Hkv, D, qs[0], qs[1],
              *kv_strides, os[0], os[1], cu_q, cu_k, kv_lens, max_q, max_kv, bool(causal),
              D ** -0.5 if scale is None else scale)
    st = 0 if status is None else status.data_ptr()
    _fill(_lib.SEQ_ATTN_LAYOUT, a, *fields, 0, 0, st)
    ref = ctypes.byref(a)
    kib = _lib.count("srdit_seq_attn_workspace", ref)
    if kib:
        ws = torch.empty(kib << 10, dtype=torch.uint8, device=q.device)
        _fill(_lib.SEQ_ATTN_LAYOUT, a, *fields, ws.data_ptr(), kib << 10, st)
    _launch("srdit_seq_attn", ref, stream, kind=kind, work=work)
    if kib:
        Stats.launches += 1   # a second kernel joins the parts
    return out


def paged_attn(q, k_pages, v_pages, page_table, kv_lens, out=None, *, cu_q=None, max_q=None,
               max_kv=None, causal=True, k_scale=None, v_scale=None, scale=None, status=None):
    """Attention of new tokens' q [T, H, D] over their sequences' cached tokens, which
    ``kv_write`` has put there, the new ones included. Returns out [T, H, D].

    Pages, table, ``kv_lens`` and ``cu_q`` as in ``kv_write``; H a multiple of the pages' heads.
    Sequence b's n new tokens are its last ones: with ``causal`` each sees the tokens up to its
    own, else all kv_lens[b] of them. One that sees none gets zeros; rows of out behind the last
    sequence are left as they were. ``max_q``: no sequence has more new tokens (default: T / B
    without ``cu_q``, else T; steps of one token each say 1); ``max_kv``: about the longest
    sequence (default: what the table holds), by which work is split. ``scale``: D ** -0.5.
    T * H at most 2^26, B * kv_heads at most 65535. Scales of values 0, or 2^-80 to 2^121 (fp16 q:
    2^100)."""
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if _short("paged_attn", "srdit_seq_attn", q, k_pages, v_pages, page_table, kv_lens, out, cu_q,
              max_q, max_kv, causal, k_scale, v_scale, scale, status):
        return out
    stream = _same_device(q, k_pages, v_pages, page_table, kv_lens, out, cu_q, k_scale, v_scale,
                          status)
    p, B, Hkv, D = _pages(k_pages, v_pages, page_table, k_scale, v_scale, q.dtype)
    if max_q is None:
        max_q = q.shape[0] if cu_q is not None or B == 0 else q.shape[0] // B
    held = p.table_width * p.page_size
    work = _attn_flops(q.shape, B, cu_q, lambda: [min(max(x, 0), held) for x in kv_lens.tolist()],
                       causal)
    return _seq_attn("paged_attn", q, out, Hkv, D, B, ctypes.addressof(p), 0, 0, 0, (0, 0, 0, 0),
                     0 if cu_q is None else _int32(cu_q, B + 1, "cu_q"), 0,
                     _int32(kv_lens, B, "kv_lens"), max_q,
                     0 if max_kv is None else max_kv, causal, scale, status, stream, work)


def packed_attn(q, k, v, cu_q, out=None, *, cu_k=None, causal=True, scale=None, status=None):
    """Attention of whole packed sequences: q [T, H, D] (bf16 or fp16) over k, v [Tk, Hkv, D],
    sequence b's rows being cu_q[b] to cu_q[b + 1] of q (int32 [B + 1] on the device) and, with
    ``cu_k``, cu_k[b] to cu_k[b + 1] of k and v (default: cu_q). Returns out [T, H, D].

    With ``causal`` a sequence's queries are its last tokens: query i of n sees the keys up to
    L - n + i of its L. Views whose strides are multiples of 8 are read in place (k and v of one
    projection side by side). A query that sees no key gets zeros; rows of out behind the last
    sequence are left as they were. ``scale``: D ** -0.5."""
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if _short("packed_attn", "srdit_seq_attn", q, k, v, cu_q, out, cu_k, causal, scale, status):
        return out
    stream = _same_device(q, k, v, cu_q, out, cu_k, status)
    shape, ks, vs = k.shape, k.stride(), v.stride()
    if (len(shape) != 3 or v.shape != shape or k.dtype != q.dtype or v.dtype != q.dtype
            or ks[2] != 1 or vs[2] != 1):
        raise _lib.SrditError(f"k {tuple(shape)} {k.dtype} {ks}, v {tuple(v.shape)} {v.dtype} {vs}: "
                              f"[tokens, kv_heads, D] of {q.dtype} with unit stride over D")
    B = cu_q.numel() - 1
    if B < 0 or (cu_k is None and shape[0] != q.shape[0]):
        raise _lib.SrditError(f"{B} sequences; without cu_k k and v have q's {q.shape[0]} rows")
    ends = cu_q if cu_k is None else cu_k
    work = _attn_flops(q.shape, B, cu_q, lambda: [y - x for x, y in _row_ends(ends, shape[0], B)],
                       causal)
    return _seq_attn("packed_attn", q, out, shape[1], shape[2], B, 0, k.data_ptr(), v.data_ptr(),
                     shape[0], (ks[0], ks[1], vs[0], vs[1]), _int32(cu_q, B + 1, "cu_q"),
                     0 if cu_k is None else _int32(cu_k, B + 1, "cu_k"), 0, 0, 0, causal, scale,
                     status, stream, work)


def row_reduce(x, op, out=None):
    """Per-row sum of squares (op "sumsq") or max |x| (op "absmax") of a bf16 [M, K]."""
    _need_cuda(x, out)
    if x.dtype != torch.bfloat16:
        raise _lib.SrditError("row_reduce takes bf16")
    M, K = x.shape
    if out is None:
        out = torch.empty(M, dtype=torch.float32, device=x.device)
    code = {"sumsq": _lib.SRDIT_ROW_SUMSQ, "absmax": _lib.SRDIT_ROW_ABSMAX}[op]
    _launch("srdit_row_reduce", _ptr(x), _rows(x), M, K, code, _ptr(out), _stream(x.device),
            kind="row_reduce", work=M * K * 2 + 4 * M)
    return out


def residual(x, parts, bias=None, gate=None):
    """x = bf16(x + bf16(sum(parts) + bias) [* gate]) in place; parts [S, M, N] or [M, N]."""
    _need_cuda(x, parts, bias, gate)
    p3 = parts if parts.dim() == 3 else parts.unsqueeze(0)
    if p3.dtype != torch.bfloat16 or p3.stride(2) != 1:
        raise _lib.SrditError("residual parts must be bf16 with unit inner stride")
    S, M, N = p3.shape
    if x.shape != (M, N):
        raise _lib.SrditError(f"x {tuple(x.shape)} vs parts {tuple(p3.shape)}")
    if gate is not None and (gate.dtype != torch.float32 or not gate.is_contiguous()):
        raise _lib.SrditError("gate must be contiguous float32")
    _launch("srdit_residual", _ptr(x), _rows(x), M, N, _ptr(p3), S, p3.stride(0), p3.stride(1),
            _ptr(bias), _ptr(gate), _stream(x.device), kind="residual",
            work=M * N * 2 * (S + 2))
    return x


def winattn_plan(params_host: torch.Tensor, p_stride: int, anchor_mode: int):
    """Tiling of a window plan (int32 [n_w, p_stride] rows on the host)."""
    p = params_host.contiguous()
    if p.dtype != torch.int32 or p.device.type != "cpu":
        raise _lib.SrditError("params rows must be a CPU int32 tensor")
    t = _lib.WinattnTiling()
    _lib.call("srdit_winattn_plan", ctypes.c_void_p(p.data_ptr()), p.shape[0], int(p_stride),
              int(anchor_mode), ctypes.byref(t))
    return t


def winattn(q, k_hr, v_hr, out, *, params_dev, n_w, p_stride, anchor_mode, geom, tiling,
            k_anchor=None, v_anchor=None, status=None, flops=0):
    """One window-attention launch (see include/srdit_b200.h, srdit_winattn_fwd).
    ``flops``: the launch's visible-pair FLOPs, for launch accounting only."""
    _need_cuda(q, k_hr, v_hr, out, params_dev, k_anchor, v_anchor)
    for t in (q, k_hr, v_hr, out, k_anchor, v_anchor):
        if t is not None and t.dtype != torch.bfloat16:
            raise _lib.SrditError("window attention takes bf16 q/k/v")
    _launch("srdit_winattn_fwd", _ptr(q), _ptr(k_hr), _ptr(v_hr), _ptr(k_anchor),
            _ptr(v_anchor), _ptr(out), _ptr(params_dev), int(n_w), int(p_stride),
            int(anchor_mode), ctypes.byref(geom), ctypes.byref(tiling), _ptr(status),
            _stream(q.device), kind="winattn", work=flops)
    return out


# --------------------------------------------------------------------------- tensor parallel
def peer_ptrs(ptrs):
    """ctypes table of per-rank device addresses (ints)."""
    t = _lib.PeerPtrs()
    for i, v in enumerate(ptrs):
        t.p[i] = int(v)
    return t


def fp8_gemm_ctas(M, N):
    return _lib.count("srdit_fp8_gemm_ctas", int(M), int(N))


def fp8_gemm_tp(a_fp8, a_scale, w_fp8, w_scale, bias=None, out=None, *, tp, epilogue="store",
                row_amax=None, status=None):
    """srdit_fp8_gemm_tp: ``tp`` is a filled ``_lib.TpGemm``; epilogue "peer" stores the
    partial into the owners' receive slots (``out`` unused)."""
    _need_cuda(a_fp8, a_scale, w_fp8, w_scale, bias, out, row_amax)
    M, K = a_fp8.shape
    N = w_fp8.shape[0]
    code = {"store": _lib.SRDIT_EPI_STORE, "gelu": _lib.SRDIT_EPI_GELU,
            "peer": _lib.SRDIT_EPI_PEER}[epilogue]
    ldo = _rows(out) if out is not None else 0
    _launch("srdit_fp8_gemm_tp", _ptr(a_fp8), _ptr(a_scale), _ptr(w_fp8), _ptr(w_scale),
            _ptr(bias), _ptr(out), M, N, K, _rows(a_fp8), _rows(w_fp8), ldo, code,
            _ptr(row_amax), ctypes.byref(tp), _ptr(status), _stream(a_fp8.device),
            kind="fp8_gemm", work=2 * M * N * K)
    return out


def residual_tp(x, parts, *, bias=None, gate=None, flags, expected, status=None):
    """srdit_residual_tp over the receive buffer ``parts`` [S, M, N]."""
    _need_cuda(x, parts, bias, gate)
    S, M, N = parts.shape
    _launch("srdit_residual_tp", _ptr(x), _rows(x), M, N, _ptr(parts), S, parts.stride(0),
            parts.stride(1), _ptr(bias), _ptr(gate), ctypes.c_void_p(int(flags)),
            int(expected) & 0xffffffff, _ptr(status), _stream(x.device), kind="residual",
            work=M * N * 2 * (S + 2))
    return x


def tp_allreduce(t, op, *, slots, flags, rank, world, epoch, status=None):
    """In-place all-reduce (op "sum" / "max") of a contiguous fp32 vector through peer memory."""
    _need_cuda(t)
    if t.dtype != torch.float32 or not t.is_contiguous():
        raise _lib.SrditError("tp_allreduce takes a contiguous float32 vector")
    code = {"sum": _lib.SRDIT_RED_SUM, "max": _lib.SRDIT_RED_MAX}[op]
    _launch("srdit_tp_allreduce", _ptr(t), _ptr(t), t.numel(), code, ctypes.byref(slots),
            ctypes.byref(flags), int(rank), int(world), int(epoch) & 0xffffffff, _ptr(status),
            _stream(t.device), kind="allreduce", work=t.numel() * 4 * world)
    return t


def conv3x3(x, weight, bias, *, frames_per_clip, n_src=1, replicate=True, residual=None,
            res_scale=1.0, relu=False, shuffle=1, out=None, status=None):
    """srdit_conv3x3 of channels-last frames x [F, H, W, cin] bf16 (cin a multiple of
    64) with ``weight`` [cout, n_src * 9 * cin] bf16 (``conv_weight`` builds it) and
    fp32 ``bias`` [cout]; returns out [F, H, W, cout], or [F, r H, r W, cout / r^2]
    with ``shuffle`` = r."""
    _need_cuda(x, weight, bias, residual, out, status)
    if x.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16 or bias.dtype != torch.float32:
        raise _lib.SrditError("conv3x3 takes bf16 frames and weights and fp32 bias")
    if x.dim() != 4 or not x.is_contiguous() or not weight.is_contiguous():
        raise _lib.SrditError("conv3x3 takes contiguous [F, H, W, C] frames")
    F, H, W, cin = x.shape
    cout = weight.shape[0]
    if weight.shape[1] != n_src * 9 * cin or bias.shape != (cout,):
        raise _lib.SrditError(f"weight {tuple(weight.shape)} / bias {tuple(bias.shape)} do not "
                              f"match {n_src} source(s) of {cin} channels")
    r = int(shuffle)
    shape = (F, H, W, cout) if r == 1 else (F, r * H, r * W, cout // (r * r))
    if out is None:
        out = torch.empty(shape, dtype=torch.bfloat16, device=x.device)
    elif tuple(out.shape) != shape or not out.is_contiguous() or out.dtype != torch.bfloat16:
        raise _lib.SrditError(f"out must be a contiguous bf16 {shape}")
    if residual is not None and (tuple(residual.shape) != (F, H, W, cout)
                                 or not residual.is_contiguous()
                                 or residual.dtype != torch.bfloat16):
        raise _lib.SrditError(f"residual must be a contiguous bf16 {(F, H, W, cout)}")
    _launch("srdit_conv3x3", _ptr(x), F, int(frames_per_clip), H, W, cin, int(n_src),
            int(bool(replicate)), _ptr(weight), _ptr(bias), cout, _ptr(residual),
            float(res_scale), int(bool(relu)), r, _ptr(out), _ptr(status), _stream(x.device),
            kind="conv3x3", work=2 * F * H * W * cout * n_src * 9 * cin)
    return out


def conv3d(x, weight, bias, *, kt=1, kh=3, residual=None, res_scale=1.0, relu=False,
           shuffle=1, shuffle_t=1, up2_phase=-1, dup=None, out=None, status=None):
    """srdit_conv3d: x [in_frames, H, W, cin] bf16 (the causal history of kt - 1
    frames first), ``weight`` [cout, kt * kh * kh * cin] bf16 (``conv3d_weight``),
    fp32 ``bias``; returns out [in_frames - kt + 1, H, W, cout] (shuffled shapes
    as the header states; with ``up2_phase`` >= 0 the caller passes ``out`` of
    the upsampled size, of which this launch writes one sub-pixel). ``dup`` =
    (block input [frames, H, W, cin], ft, shift): a phase launch's DupUp3D
    residual, gathered in the epilogue."""
    _need_cuda(x, weight, bias, residual, out, status)
    if x.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16 or bias.dtype != torch.float32:
        raise _lib.SrditError("conv3d takes bf16 frames and weights and fp32 bias")
    if x.dim() != 4 or not x.is_contiguous() or not weight.is_contiguous():
        raise _lib.SrditError("conv3d takes contiguous [F, H, W, C] frames")
    Fi, H, W, cin = x.shape
    Fo = Fi - kt + 1
    cout = weight.shape[0]
    if weight.shape[1] != kt * kh * kh * cin or bias.shape != (cout,):
        raise _lib.SrditError(f"weight {tuple(weight.shape)} / bias {tuple(bias.shape)} do not "
                              f"match a {kt}x{kh}x{kh} conv of {cin} channels")
    r, st = int(shuffle), int(shuffle_t)
    if up2_phase >= 0:
        shape = (Fo, 2 * H, 2 * W, cout)
        if out is None:
            raise _lib.SrditError("an up2_phase launch writes into a given out")
    else:
        shape = (Fo * st, r * H, r * W, cout // (r * r * st))
    if out is None:
        out = torch.empty(shape, dtype=torch.bfloat16, device=x.device)
    elif tuple(out.shape) != shape or not out.is_contiguous() or out.dtype != torch.bfloat16:
        raise _lib.SrditError(f"out must be a contiguous bf16 {shape}")
    if residual is not None and (tuple(residual.shape) != tuple(out.shape)
                                 or not residual.is_contiguous()
                                 or residual.dtype != torch.bfloat16):
        raise _lib.SrditError(f"residual must be a contiguous bf16 {tuple(out.shape)}")
    a = _lib.Conv3dArgs()
    a.x, a.in_frames, a.out_frames, a.H, a.W, a.cin = x.data_ptr(), Fi, Fo, H, W, cin
    a.kt, a.kh, a.weight, a.bias, a.cout = kt, kh, weight.data_ptr(), bias.data_ptr(), cout
    a.residual = residual.data_ptr() if residual is not None else None
    a.res_scale, a.relu, a.shuffle, a.shuffle_t = float(res_scale), int(bool(relu)), r, st
    a.up2_phase, a.out = int(up2_phase), out.data_ptr()
    if dup is not None:
        xd, ft, shift = dup
        _need_cuda(xd)
        if (xd.dim() != 4 or tuple(xd.shape[1:3]) != (H, W) or not xd.is_contiguous()
                or xd.dtype != torch.bfloat16):
            raise _lib.SrditError(f"the DupUp3D source must be contiguous bf16 [frames, {H}, "
                                  f"{W}, cin], got {tuple(xd.shape)}")
        reps = cout * 4 * ft // xd.shape[3]
        du = _lib.DupUp(ctypes.c_void_p(xd.data_ptr()), xd.shape[0], xd.shape[3], int(ft),
                        int(reps), int(shift))
        a.dup = ctypes.pointer(du)
    a.status = status.data_ptr() if status is not None else None
    _launch("srdit_conv3d", ctypes.byref(a), _stream(x.device), kind="conv3d",
            work=2 * Fo * H * W * cout * kt * kh * kh * cin)
    return out


def conv3d_weight(w, *, cin_pad=None):
    """A Conv3d weight [cout, cin, kt, kh, kw] (or Conv2d [cout, cin, kh, kw]) as
    srdit_conv3d's K-major [cout, kt * kh * kw * cin_pad] bf16 matrix (column
    ((dt * kh + ky) * kw + kx) * cin_pad + c; channels past cin zero)."""
    if w.dim() == 4:
        w = w[:, :, None]
    cout, cin, kt, kh, kw = w.shape
    cin_pad = cin if cin_pad is None else int(cin_pad)
    t = w.detach().to(torch.float32).permute(0, 2, 3, 4, 1)
    if cin_pad != cin:
        t = torch.nn.functional.pad(t, (0, cin_pad - cin))
    return t.reshape(cout, kt * kh * kw * cin_pad).to(torch.bfloat16).contiguous()


def rms_silu(x, gamma, *, silu=True, out=None):
    """srdit_rms_silu over the channels of [..., C] bf16 frames (WanVAE RMS_norm, then
    SiLU); ``out`` may be x or a same-shaped view of another buffer."""
    _need_cuda(x, gamma, out)
    if (x.dtype != torch.bfloat16 or gamma.dtype != torch.bfloat16 or not x.is_contiguous()
            or not gamma.is_contiguous()):
        raise _lib.SrditError("rms_silu takes contiguous bf16 frames and a contiguous bf16 gamma")
    C = x.shape[-1]
    if gamma.numel() != C:
        raise _lib.SrditError(f"gamma of {gamma.numel()} for {C} channels")
    if out is None:
        out = torch.empty_like(x)
    elif out.shape != x.shape or not out.is_contiguous() or out.dtype != torch.bfloat16:
        raise _lib.SrditError("out must be a contiguous bf16 tensor of x's shape")
    P = x.numel() // C
    _launch("srdit_rms_silu", _ptr(x), P, C, _ptr(gamma), int(bool(silu)),
            _ptr(out), _stream(x.device), kind="rms_silu", work=4 * x.numel())
    return out


def conv_weight(w, *, n_src=1, cin_pad=None, shuffle=1):
    """An nn.Conv2d weight [cout, n_src * cin, 3, 3] as srdit_conv3x3's K-major
    [cout, n_src * 9 * cin_pad] bf16 matrix (column (s * 9 + ky * 3 + kx) * cin_pad
    + c; channels past cin zero). With ``shuffle`` = r the rows are reordered
    so that row g * cg + c holds output channel c * r^2 + g -- PixelShuffle(r)'s
    channel for sub-pixel g -- as the kernel's shuffled store expects."""
    cout, cin_all, kh, kw = w.shape
    if (kh, kw) != (3, 3) or cin_all % n_src:
        raise _lib.SrditError(f"not a 3x3 conv weight of {n_src} source(s): {tuple(w.shape)}")
    cin = cin_all // n_src
    cin_pad = cin if cin_pad is None else int(cin_pad)
    t = w.detach().to(torch.float32).reshape(cout, n_src, cin, 3, 3).permute(0, 1, 3, 4, 2)
    if cin_pad != cin:
        t = torch.nn.functional.pad(t, (0, cin_pad - cin))
    t = t.reshape(cout, n_src * 9 * cin_pad)
    r = int(shuffle)
    if r > 1:
        cg = cout // (r * r)
        t = t.reshape(cg, r * r, -1).transpose(0, 1).reshape(cout, -1)
    return t.to(torch.bfloat16).contiguous()


def conv_bias(b, *, shuffle=1):
    """The conv's bias [cout] as fp32, in ``conv_weight``'s row order."""
    t = b.detach().to(torch.float32)
    r = int(shuffle)
    if r > 1:
        t = t.reshape(-1, r * r).t().reshape(-1)
    return t.contiguous()


def wait_counters(counters: int, mask: int, expected: int, *, status=None, device=None):
    """srdit_wait_counters: the stream waits (bounded) until the uint32 counters at
    device address ``counters`` selected by ``mask`` reach ``expected``."""
    _need_cuda(status)
    _launch("srdit_wait_counters", ctypes.c_void_p(int(counters)), int(mask) & 0xffffffff,
            int(expected) & 0xffffffff, _ptr(status), _stream(device), kind="wait")


def ln_mod_quant_tp(x, eps=1e-6, *, ln_weight=None, ln_bias=None, shift=None, scale=None,
                    q_rows, s_rows, flags, done, rank, world, ldq):
    """srdit_ln_mod_quant_tp: this rank's LN-modulate-quant rows stored into every
    rank's gather buffer (``q_rows`` / ``s_rows`` peer tables), then ``flags``
    signalled; ``done`` is a zeroed uint32 tensor of this rank."""
    _need_cuda(x, ln_weight, ln_bias, shift, scale, done)
    if x.dtype != torch.bfloat16:
        raise _lib.SrditError("ln_mod_quant takes bf16")
    M, K = x.shape
    _launch("srdit_ln_mod_quant_tp", _ptr(x), _rows(x), M, K, float(eps), _ptr(ln_weight),
            _ptr(ln_bias), _ptr(shift), _ptr(scale), int(ldq), ctypes.byref(q_rows),
            ctypes.byref(s_rows), ctypes.byref(flags), _ptr(done), int(rank), int(world),
            _stream(x.device), kind="ln_mod_quant", work=M * K * 2 + (M * K + 4 * M) * world)


def tp_push(src, dst, src2, dst2, *, flags, rank, world, stream=None):
    """srdit_tp_push: copy-engine pushes of src (and src2) to every other rank's
    dst / dst2 addresses (``peer_ptrs`` tables), then signal ``flags``."""
    _need_cuda(src, src2)
    st = ctypes.c_void_p((stream or torch.cuda.current_stream(src.device)).cuda_stream)
    _lib.call("srdit_tp_push", _ptr(src), ctypes.byref(dst), src.numel() * src.element_size(),
              _ptr(src2), ctypes.byref(dst2) if dst2 is not None else None,
              (src2.numel() * src2.element_size()) if src2 is not None else 0,
              ctypes.byref(flags), int(rank), int(world), st)
    Stats.launches += 1


def ipc_handle(t):
    """(64-byte CUDA IPC handle, byte offset) of the allocation holding tensor ``t``."""
    h = ctypes.create_string_buffer(64)
    off = ctypes.c_ulonglong(0)
    _lib.call("srdit_ipc_handle", _ptr(t), h, ctypes.byref(off))
    return bytes(h.raw), int(off.value)


def ipc_open(handle: bytes) -> int:
    """Map a peer's allocation; returns its base address in this process."""
    buf = ctypes.create_string_buffer(handle, 64)
    ptr = ctypes.c_void_p()
    _lib.call("srdit_ipc_open", buf, ctypes.byref(ptr))
    return int(ptr.value)


def ipc_close(addr: int) -> None:
    _lib.call("srdit_ipc_close", ctypes.c_void_p(addr))
