"""Tensor-level wrappers of the libmi355q kernels.

Each function validates shapes, allocates outputs and workspaces with the
torch caching allocator on the inputs' device, and launches on torch's
current stream.  All tensors must live on a ROCm GPU; there is no CPU path.
"""
from __future__ import annotations

import ctypes as C
import functools

import torch

from . import _lib as L


def _dt(t: torch.Tensor) -> int:
    if t.dtype == torch.bfloat16:
        return L.BF16
    if t.dtype == torch.float32:
        return L.F32
    raise TypeError(f"unsupported dtype {t.dtype} (bf16 or fp32)")


def _ws(nbytes: int, device) -> torch.Tensor | None:
    if nbytes == 0:
        return None
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


# ---------------------------------------------------------------- Hessian
_HESS_DT = {torch.bfloat16: L.BF16, torch.float16: L.F16, torch.float32: L.F32}


def _hessian_input(x: torch.Tensor) -> torch.Tensor:
    """x as a row-major 2-D matrix of a type the Hessian kernels take: bf16 and
    fp16 as they are (16-byte aligned rows, a multiple of 8 features), any
    other floating type - and 16-bit inputs whose width is not a multiple
    of 8 - converted to fp32, as the reference converts every input
    (gptq_quantize.py:93)."""
    if not x.dtype.is_floating_point:
        raise TypeError(f"hessian input must be a floating-point tensor, got {x.dtype}")
    if x.dim() != 2 or x.stride(1) != 1:
        x = x.reshape(-1, x.shape[-1]).contiguous()
    if x.dtype not in _HESS_DT or (x.dtype != torch.float32 and x.shape[1] % 8):
        x = x.to(torch.float32)
    if x.dtype != torch.float32 and (x.data_ptr() % 16 or x.stride(0) % 8):
        x = x.contiguous()
    return x


def hessian_syrk_(H: torch.Tensor, x: torch.Tensor, alpha: float = 2.0, beta: float = 1.0) -> torch.Tensor:
    """H[i, j] = beta * H[i, j] + alpha * sum_t x[t, i] x[t, j] for i <= j, in
    place (beta == 1: H += ...).

    ``x`` is [tokens, d] (row stride may exceed d) bf16 or fp16 (16-bit MFMA,
    exact products) or fp32 (six products of three bf16 planes, small ones on
    the fp32 MFMA); other floating types are converted to fp32.  H is fp32
    [d, d].
    """
    L.require_gpu(H, x)
    x = _hessian_input(x)
    n, d = x.shape
    if H.dtype != torch.float32 or H.shape != (d, d) or H.stride(1) != 1:
        raise ValueError(f"H must be fp32 [{d}, {d}] row-major, got {tuple(H.shape)} {H.dtype}")
    lib = L.lib()
    dt = _HESS_DT[x.dtype]
    try:
        ws = _ws(lib.mi355q_hessian_syrk_workspace_size(n, d, dt), x.device)
    except torch.cuda.OutOfMemoryError:
        if dt != L.F32:
            raise
        ws = None   # no room for the planes (up to about 1 GiB): the fp32 product needs none
    L.check(lib.mi355q_hessian_syrk(x.data_ptr(), dt, n, d, x.stride(0), H.data_ptr(), H.stride(0), C.c_float(alpha),
                                    C.c_float(beta), L.ptr(ws), 0 if ws is None else ws.numel(), L.stream_of(x)))
    return H


def hessian_syrk_segments_(H: torch.Tensor, xs, alpha: float = 2.0, beta: float = 1.0) -> torch.Tensor:
    """``hessian_syrk_`` over the rows of several [n_k, d] tensors at once:
    H = beta * H + alpha * sum_k X_k^T X_k (upper triangle, in place), the
    sum a single call over their concatenation forms (segments of
    multiples of 32 rows: bit for bit) without the concatenation.  16-bit
    segments sharing one dtype and row stride run in one launch per 64
    segments; others take one ``hessian_syrk_`` per segment."""
    xs = [_hessian_input(x) for x in xs]
    if len(xs) == 1:
        return hessian_syrk_(H, xs[0], alpha=alpha, beta=beta)
    L.require_gpu(H, *xs)
    d = H.shape[-1]
    if any(x.shape[1] != d for x in xs):
        raise ValueError(f"every segment needs {d} columns, got {[tuple(x.shape) for x in xs]}")
    if H.dtype != torch.float32 or H.shape != (d, d) or H.stride(1) != 1:
        raise ValueError(f"H must be fp32 [{d}, {d}] row-major, got {tuple(H.shape)} {H.dtype}")
    dts = {x.dtype for x in xs}
    ldx = {x.stride(0) for x in xs if x.shape[0] > 0}
    if len(dts) != 1 or len(ldx) > 1 or xs[0].dtype == torch.float32 or any(x.device != H.device for x in xs):
        b = beta
        for x in xs:
            if x.shape[0] > 0 or x is xs[-1]:
                hessian_syrk_(H, x, alpha=alpha, beta=b)
                b = 1.0
        return H
    lib = L.lib()
    dt = _HESS_DT[xs[0].dtype]
    n = len(xs)
    ptrs = (C.c_void_p * n)(*[x.data_ptr() for x in xs])
    rows = (C.c_int64 * n)(*[x.shape[0] for x in xs])
    ws = _ws(lib.mi355q_hessian_syrk_segments_workspace_size(rows, n, d, dt), H.device)
    L.check(lib.mi355q_hessian_syrk_segments(ptrs, rows, n, dt, d, ldx.pop() if ldx else d, H.data_ptr(), H.stride(0),
                                             C.c_float(alpha), C.c_float(beta), L.ptr(ws),
                                             0 if ws is None else ws.numel(), L.stream_of(xs[0])))
    return H


def hessian_grouped_syrk_(H: torch.Tensor, x: torch.Tensor, rows: torch.Tensor | None, offsets,
                          alpha: float = 2.0, beta: float = 1.0) -> torch.Tensor:
    """Per-group upper-triangle syrk: H[e] = beta * H[e] + alpha * X_e^T X_e
    where X_e are the rows ``x[rows[offsets[e]:offsets[e+1]]]`` (``rows``
    None: the rows ``x[offsets[e]:offsets[e+1]]``).  H is [E, d, d] fp32;
    ``offsets`` a list or an int64 tensor of E + 1 non-decreasing entries.
    ``beta`` is 1 (add) or 0: H's upper triangle is written without being
    read (a freshly allocated H need not be zeroed; groups without rows get
    zeros).  bf16 and fp16 ``x`` take one grouped launch whose work table is
    built on the device; other types are converted to fp32 and each group's
    rows take the dense fp32 product."""
    if beta not in (0.0, 1.0):
        raise ValueError("beta must be 0 or 1")
    L.require_gpu(H, x)
    if isinstance(offsets, torch.Tensor):
        off_dev = offsets.to(device=x.device, dtype=torch.int64).contiguous()
        E = off_dev.numel() - 1
        off_list = None
    else:
        off_list = [int(o) for o in offsets]
        E = len(off_list) - 1
        if any(b < a for a, b in zip(off_list, off_list[1:])) or (off_list and off_list[0] < 0):
            raise ValueError("offsets must be non-negative and non-decreasing")
        off_dev = None
    x = _hessian_input(x)
    n_x, d = x.shape
    n_rows = n_x if rows is None else rows.numel()
    if off_list is not None and off_list[-1] > n_rows:
        raise ValueError(f"offsets end at {off_list[-1]} > {n_rows} rows")
    if H.shape != (E, d, d) or H.dtype != torch.float32 or not H.is_contiguous():
        raise ValueError(f"H must be contiguous fp32 [{E}, {d}, {d}]")
    if x.dtype == torch.float32:
        offs = off_list if off_list is not None else off_dev.tolist()
        for e in range(E):
            if offs[e + 1] > offs[e]:
                xe = x[offs[e]:offs[e + 1]] if rows is None else x[rows[offs[e]:offs[e + 1]].long()]
                if beta == 0.0:
                    H[e].zero_()
                hessian_syrk_(H[e], xe, alpha=alpha)
            elif beta == 0.0:
                H[e].zero_()
        return H
    if rows is not None:
        L.require_gpu(rows)
        rows = rows.to(torch.int32).contiguous()
    if off_dev is None:
        off_dev = torch.tensor(off_list, dtype=torch.int64).to(x.device, non_blocking=True)
    lib = L.lib()
    ws = _ws(lib.mi355q_hessian_grouped_syrk_workspace_size(n_rows, E, d), x.device)
    L.check(lib.mi355q_hessian_grouped_syrk(x.data_ptr(), _HESS_DT[x.dtype], n_x, x.stride(0), d,
                                            None if rows is None else rows.data_ptr(), n_rows, off_dev.data_ptr(),
                                            E, H.data_ptr(), d * d, C.c_float(alpha), C.c_float(beta), L.ptr(ws),
                                            0 if ws is None else ws.numel(), L.stream_of(x)))
    return H


def symmetrize_upper_(H: torch.Tensor) -> torch.Tensor:
    """Copy the upper triangle onto the lower one, in place."""
    L.require_gpu(H)
    d = H.shape[0]
    L.call("mi355q_symmetrize_upper", H.data_ptr(), d, H.stride(0), L.stream_of(H))
    return H


# ---------------------------------------------------------------- GPTQ pieces
def _row_major_square(H: torch.Tensor) -> torch.Tensor:
    """H as a row-major fp32 square matrix (rows may be padded): the kernels
    read H[i][j] at i * ldh + j."""
    if H.dim() != 2 or H.shape[0] != H.shape[1] or H.dtype != torch.float32:
        raise ValueError(f"H must be a square fp32 matrix, got {tuple(H.shape)} {H.dtype}")
    return H if H.stride(1) == 1 and H.stride(0) >= H.shape[1] else H.contiguous()


def gptq_hinv(H: torch.Tensor, perm: torch.Tensor | None, num_samples: float, percdamp: float):
    """Upper Cholesky factor of inverse(damped H / num_samples).

    Returns (hinv [d, d] fp32, dead [d] int32, positive_definite: bool).
    Synchronises once to read the status flag.
    """
    L.require_gpu(H)
    H = _row_major_square(H)
    d = H.shape[0]
    dev = H.device
    hinv = torch.empty((d, d), dtype=torch.float32, device=dev)
    dead = torch.empty(d, dtype=torch.int32, device=dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    lib = L.lib()
    ws = _ws(lib.mi355q_gptq_hinv_workspace_size(d), dev)
    p = None if perm is None else perm.to(torch.int32).contiguous()
    L.check(lib.mi355q_gptq_hinv(H.data_ptr(), H.stride(0), d, L.ptr(p), C.c_float(num_samples),
                                 C.c_float(percdamp), hinv.data_ptr(), dead.data_ptr(), status.data_ptr(),
                                 ws.data_ptr(), ws.numel(), L.stream_of(H)))
    st = int(status.item())
    L.check_hinv_status([st])
    return hinv, dead, st == 0


def gptq_hinv_rtn(H: torch.Tensor, perm: torch.Tensor | None, num_samples: float, percdamp: float):
    """``gptq_hinv`` without a host synchronisation: a Hessian that is not
    positive definite gets hinv = identity on the device (the reference's
    round-to-nearest fallback).  Returns (hinv, dead, status [1] int32 on the
    device, 0 = positive definite)."""
    L.require_gpu(H)
    H = _row_major_square(H)
    d = H.shape[0]
    dev = H.device
    hinv = torch.empty((d, d), dtype=torch.float32, device=dev)
    dead = torch.empty(d, dtype=torch.int32, device=dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    lib = L.lib()
    ws = _ws(lib.mi355q_gptq_hinv_workspace_size(d), dev)
    p = None if perm is None else perm.to(torch.int32).contiguous()
    L.check(lib.mi355q_gptq_hinv(H.data_ptr(), H.stride(0), d, L.ptr(p), C.c_float(num_samples),
                                 C.c_float(percdamp), hinv.data_ptr(), dead.data_ptr(), status.data_ptr(),
                                 ws.data_ptr(), ws.numel(), L.stream_of(H)))
    L.call("mi355q_gptq_hinv_fallback", hinv.data_ptr(), d, d * d, 1, status.data_ptr(), L.stream_of(H))
    return hinv, dead, status


def gptq_load_weight(w: torch.Tensor, perm=None, dead=None) -> torch.Tensor:
    L.require_gpu(w)
    rows, cols = w.shape
    out = torch.empty((rows, cols), dtype=torch.float32, device=w.device)
    p = None if perm is None else perm.to(torch.int32).contiguous()
    dd = None if dead is None else dead.to(torch.int32).contiguous()
    L.call("mi355q_gptq_load_weight", w.data_ptr(), _dt(w), rows, cols, w.stride(0), L.ptr(p), L.ptr(dd),
           out.data_ptr(), L.stream_of(w))
    return out


STRATEGY_CODE = {"tensor": L.TENSOR, "channel": L.CHANNEL, "group": L.GROUP, "tensor_group": L.GROUP,
                 "block": L.BLOCK, "token": L.TOKEN}


QTYPE = {"int": L.QTYPE_INT, "fp8": L.QTYPE_FP8_E4M3, "fp4": L.QTYPE_FP4_E2M1, "mxfp4_ct": L.QTYPE_MXFP4_CT,
         "mxfp4_ocp": L.QTYPE_MXFP4_OCP}


def gptq_sweep_(w_work: torch.Tensor, hinv: torch.Tensor, scale: torch.Tensor, zero_point, strategy: str,
                g_idx: torch.Tensor | None, qmin: float, qmax: float, dequant_bf16: bool,
                blocksize: int = 128, block_h: int = 1, qtype: str = "int",
                global_scale: torch.Tensor | None = None):
    """In-place GPTQ column sweep.  Returns (codes int8 [rows, cols], losses
    fp32 [rows]); ``qtype`` int / fp8 / fp4 (codes: integers, e4m3 bits, e2m1
    codes), ``global_scale`` (fp32 [1]) divides the scales (tensor groups)."""
    L.require_gpu(w_work, hinv, scale)
    rows, cols = w_work.shape
    if hinv.shape != (cols, cols) or hinv.dtype != torch.float32:
        raise ValueError(f"hinv must be fp32 [{cols}, {cols}], got {tuple(hinv.shape)} {hinv.dtype}")
    s = scale.to(torch.float32).contiguous()
    if s.dim() == 1:
        s = s.reshape(-1, 1)
    z = None if zero_point is None else \
        zero_point.to(device=w_work.device, dtype=torch.float32).reshape(s.shape).contiguous()
    return gptq_sweep_batched_(w_work.unsqueeze(0), hinv.unsqueeze(0), s.unsqueeze(0),
                               None if z is None else z.unsqueeze(0), strategy, g_idx, qmin, qmax, dequant_bf16,
                               blocksize, block_h, qtype, global_scale, _unbatch=True)


def gptq_store_weight(w_work: torch.Tensor, invperm, out_dtype: torch.dtype, codes=None):
    rows, cols = w_work.shape
    out = torch.empty((rows, cols), dtype=out_dtype, device=w_work.device)
    ip = None if invperm is None else invperm.to(torch.int32).contiguous()
    cout = None if codes is None else torch.empty_like(codes)
    L.call("mi355q_gptq_store_weight", w_work.data_ptr(), rows, cols, L.ptr(ip), out.data_ptr(), _dt(out),
           out.stride(0), L.ptr(codes), L.ptr(cout), L.stream_of(w_work))
    return out, cout


# ---------------------------------------------------------------- batched GPTQ
def gptq_hinv_batched(H: torch.Tensor, perm: torch.Tensor | None, num_samples: torch.Tensor, percdamp: float,
                      sync: bool = True):
    """``gptq_hinv`` for a stack H [B, d, d] of same-order Hessians (perm [B, d]
    or None, num_samples [B]).  Returns (hinv [B, d, d], dead [B, d], ok
    [B] bool tensor on the host); synchronises once.  With ``sync=False``:
    no synchronisation, members that are not positive definite get
    hinv = identity on the device, and the third value is the status [B]
    int32 device tensor (0 = positive definite)."""
    L.require_gpu(H)
    if H.dim() != 3 or H.shape[1] != H.shape[2] or H.dtype != torch.float32:
        raise ValueError(f"H must be a stack of square fp32 matrices, got {tuple(H.shape)} {H.dtype}")
    if H.stride(2) != 1 or H.stride(1) < H.shape[2] or H.stride(0) < H.stride(1) * H.shape[1]:
        H = H.contiguous()
    B, d, _ = H.shape
    dev = H.device
    hinv = torch.empty((B, d, d), dtype=torch.float32, device=dev)
    dead = torch.empty((B, d), dtype=torch.int32, device=dev)
    status = torch.zeros(B, dtype=torch.int32, device=dev)
    ns = num_samples.to(device=dev, dtype=torch.float32).reshape(B).contiguous()
    lib = L.lib()
    ws = _ws(lib.mi355q_gptq_hinv_workspace_size(d) * B, dev)
    p = None if perm is None else perm.to(torch.int32).reshape(B, d).contiguous()
    L.check(lib.mi355q_gptq_hinv_batched(H.data_ptr(), H.stride(1), H.stride(0), d, B, L.ptr(p),
                                         0 if p is None else d, ns.data_ptr(), C.c_float(percdamp),
                                         hinv.data_ptr(), d * d, dead.data_ptr(), status.data_ptr(),
                                         ws.data_ptr(), ws.numel(), L.stream_of(H)))
    if not sync:
        L.call("mi355q_gptq_hinv_fallback", hinv.data_ptr(), d, d * d, B, status.data_ptr(), L.stream_of(H))
        return hinv, dead, status
    st = status.cpu()
    L.check_hinv_status(st.tolist())
    return hinv, dead, st == 0


def gptq_load_weight_batched(w: torch.Tensor, perm=None, dead=None) -> torch.Tensor:
    L.require_gpu(w)
    B, rows, cols = w.shape
    out = torch.empty((B, rows, cols), dtype=torch.float32, device=w.device)
    p = None if perm is None else perm.to(torch.int32).reshape(B, cols).contiguous()
    dd = None if dead is None else dead.to(torch.int32).reshape(B, cols).contiguous()
    L.call("mi355q_gptq_load_weight_batched", w.data_ptr(), _dt(w), rows, cols, w.stride(1), w.stride(0), B,
           L.ptr(p), 0 if p is None else cols, L.ptr(dd), out.data_ptr(), L.stream_of(w))
    return out


def gptq_sweep_batched_(w_work: torch.Tensor, hinv: torch.Tensor, scale: torch.Tensor, zero_point, strategy: str,
                        g_idx: torch.Tensor | None, qmin: float, qmax: float, dequant_bf16: bool,
                        blocksize: int = 128, block_h: int = 1, qtype: str = "int",
                        global_scale: torch.Tensor | None = None, _unbatch: bool = False):
    """``gptq_sweep_`` over a batch: w_work [B, rows, cols], hinv [B, cols, cols],
    scale / zero_point [B, rows or 1, groups], g_idx [B, cols] or [cols] (shared),
    global_scale [B] (or one value for all)."""
    L.require_gpu(w_work, hinv, scale)
    B, rows, cols = w_work.shape
    dev = w_work.device
    if hinv.shape != (B, cols, cols) or hinv.dtype != torch.float32:
        raise ValueError(f"hinv must be fp32 [{B}, {cols}, {cols}], got {tuple(hinv.shape)} {hinv.dtype}")
    if hinv.stride(2) != 1 or hinv.stride(1) != cols:
        hinv = hinv.contiguous()   # row-major matrices, any batch stride
    s = scale.to(torch.float32).reshape(B, -1, scale.shape[-1] if scale.dim() == 3 else 1).contiguous()
    z = None if zero_point is None else zero_point.to(device=dev, dtype=torch.float32).reshape(s.shape).contiguous()
    gi = None if g_idx is None else g_idx.to(device=dev, dtype=torch.int32).contiguous()
    gs = None
    if global_scale is not None:
        gs = global_scale.to(device=dev, dtype=torch.float32).reshape(-1)
        gs = (gs.expand(B) if gs.numel() == 1 else gs).contiguous()
    codes = torch.empty((B, rows, cols), dtype=torch.int8, device=dev)
    losses = torch.zeros((B, rows), dtype=torch.float32, device=dev)
    lib = L.lib()
    ws = _ws(lib.mi355q_gptq_sweep_workspace_size(rows, cols, blocksize) * B, dev)
    L.check(lib.mi355q_gptq_sweep_typed_batched(
        w_work.data_ptr(), rows, cols, B, hinv.data_ptr(), hinv.stride(0), s.data_ptr(), L.ptr(z), s.stride(1),
        s.stride(0), L.ptr(gi), 0 if gi is None or gi.dim() == 1 else gi.stride(0), STRATEGY_CODE[strategy],
        block_h, QTYPE[qtype], C.c_float(qmin), C.c_float(qmax), L.ptr(gs), 1 if dequant_bf16 else 0, blocksize,
        codes.data_ptr(), losses.data_ptr(), ws.data_ptr(), ws.numel(), L.stream_of(w_work)))
    if _unbatch:
        return codes[0], losses[0]
    return codes, losses


def gptq_store_weight_batched(w_work: torch.Tensor, invperm, out_dtype: torch.dtype, codes=None):
    B, rows, cols = w_work.shape
    out = torch.empty((B, rows, cols), dtype=out_dtype, device=w_work.device)
    ip = None if invperm is None else invperm.to(torch.int32).reshape(B, cols).contiguous()
    cout = None if codes is None else torch.empty_like(codes)
    L.call("mi355q_gptq_store_weight_batched", w_work.data_ptr(), rows, cols, B, L.ptr(ip),
           0 if ip is None else cols, out.data_ptr(), _dt(out), out.stride(1), out.stride(0), L.ptr(codes),
           L.ptr(cout), L.stream_of(w_work))
    return out, cout


# ---------------------------------------------------------------- observers
def observe_minmax(x: torch.Tensor, strategy: str, group_size: int | None = None,
                   block_structure=None, dtype: torch.dtype = torch.float32):
    """Min/max statistics of a 2-D tensor per strategy, as fp32 tensors or,
    of a bf16 tensor, with ``dtype`` bf16.

    Shapes: tensor -> [1]; channel/token -> [rows, 1]; group ->
    [rows, cols / group]; block -> [ceil(rows/bh), ceil(cols/bw)].
    """
    L.require_gpu(x)
    if x.dim() != 2:
        raise ValueError("observe_minmax expects a 2-D tensor")
    if x.stride(1) != 1:
        x = x.contiguous()
    rows, cols = x.shape
    bh = bw = 1
    if strategy == "tensor":
        shape = (1,)
    elif strategy in ("channel", "token"):
        shape = (rows, 1)
    elif strategy in ("group", "tensor_group"):
        if not group_size or cols % group_size:
            raise ValueError(f"columns ({cols}) must be divisible by group_size ({group_size})")
        shape = (rows, cols // group_size)
    elif strategy == "block":
        bh, bw = block_structure
        shape = (-(-rows // bh), -(-cols // bw))
    else:
        raise ValueError(f"unknown strategy {strategy}")
    out = torch.bfloat16 if dtype == x.dtype == torch.bfloat16 and strategy != "tensor" else torch.float32
    mn = torch.empty(shape, dtype=out, device=x.device)
    mx = torch.empty(shape, dtype=out, device=x.device)
    L.call("mi355q_observe_minmax_typed", x.data_ptr(), _dt(x), rows, cols, x.stride(0), STRATEGY_CODE[strategy],
           group_size or 0, bh, bw, mn.data_ptr(), mx.data_ptr(), _dt(mn), L.stream_of(x))
    return (mn, mx) if out == dtype else (mn.to(dtype), mx.to(dtype))


def calculate_qparams(mn: torch.Tensor, mx: torch.Tensor, qmin: float, qmax: float, symmetric: bool,
                      scale_dtype: torch.dtype, strict: bool = False, out_dtype: torch.dtype = torch.float32,
                      zp_dtype: torch.dtype = torch.float32):
    """Scale / zero-point from min/max statistics (outputs holding
    ``scale_dtype`` values, stored as ``out_dtype``, and integer zero-points,
    stored as ``zp_dtype``)."""
    L.require_gpu(mn, mx)
    if mn.dtype != mx.dtype or mn.dtype != torch.bfloat16:
        mn, mx = mn.to(torch.float32), mx.to(torch.float32)
    mn, mx = mn.contiguous(), mx.contiguous()
    # the kernel stores bf16 / fp32 scales and int8 / fp32 zero points
    st = out_dtype if out_dtype in (torch.bfloat16, torch.float32) else torch.float32
    zt = zp_dtype if zp_dtype == torch.int8 and qmin >= -128 and qmax <= 127 else torch.float32
    scale = torch.empty_like(mn, dtype=st)
    zp = torch.empty_like(mn, dtype=zt)
    L.call("mi355q_calculate_qparams_typed", mn.data_ptr(), mx.data_ptr(), _dt(mn), mn.numel(), qmin, qmax,
           1 if symmetric else 0, 1 if strict else 0, L.BF16 if scale_dtype == torch.bfloat16 else L.F32,
           scale.data_ptr(), _dt(scale), zp.data_ptr(), 1 if zt == torch.int8 else 0, L.stream_of(mn))
    return scale if st == out_dtype else scale.to(out_dtype), zp if zt == zp_dtype else zp.to(zp_dtype)


MX_RULES = {"ct": L.MX_RULE_CT, "ocp": L.MX_RULE_OCP}


def mx_scales(mn: torch.Tensor, mx: torch.Tensor, rule: str = "ct"):
    """(e8m0 uint8, 2^(e-127) fp32) per group from min/max statistics."""
    L.require_gpu(mn, mx)
    mn = mn.to(torch.float32).contiguous()
    mx = mx.to(torch.float32).contiguous()
    e8 = torch.empty(mn.shape, dtype=torch.uint8, device=mn.device)
    sc = torch.empty_like(mn)
    L.call("mi355q_mx_scales", mn.data_ptr(), mx.data_ptr(), mn.numel(), MX_RULES[rule], e8.data_ptr(),
           sc.data_ptr(), L.stream_of(mn))
    return e8, sc


def nvfp4_qparams(mn: torch.Tensor, mx: torch.Tensor, stats_dtype: torch.dtype):
    """NVFP4 tensor-group qparams from group min / max statistics: (global
    scale fp32 [1], group scales as float8_e4m3fn shaped like ``mn``)."""
    L.require_gpu(mn, mx)
    mn = mn.to(torch.float32).contiguous()
    mx = mx.to(torch.float32).contiguous()
    gs = torch.empty(1, dtype=torch.float32, device=mn.device)
    bits = torch.empty(mn.shape, dtype=torch.uint8, device=mn.device)
    L.call("mi355q_nvfp4_qparams", mn.data_ptr(), mx.data_ptr(), mn.numel(),
           L.BF16 if stats_dtype == torch.bfloat16 else L.F32, gs.data_ptr(), None, bits.data_ptr(), L.stream_of(mn))
    return gs, bits.view(torch.float8_e4m3fn)


# ---------------------------------------------------------------- quantize / pack
def quantize_int(x: torch.Tensor, scale: torch.Tensor, zero_point, strategy: str, num_bits: int,
                 group_size: int | None = None, g_idx=None, block_structure=None,
                 div_dtype: torch.dtype | None = None) -> torch.Tensor:
    """Integer codes (int8) of ``x`` with CT quantize arithmetic."""
    L.require_gpu(x, scale)
    if x.stride(1) != 1:
        x = x.contiguous()
    rows, cols = x.shape
    s = (scale if scale.dtype == torch.bfloat16 else scale.to(torch.float32)).contiguous()
    s2 = s.reshape(-1, 1) if s.dim() < 2 else s
    z = None
    if zero_point is not None:
        zt = torch.int8 if zero_point.dtype == torch.int8 else torch.float32
        z = zero_point.to(device=x.device, dtype=zt).reshape(s2.shape).contiguous()
    gi = None if g_idx is None else g_idx.to(device=x.device, dtype=torch.int32).contiguous()
    bh, bw = block_structure if block_structure else (1, 1)
    if div_dtype is None:
        div_dtype = torch.promote_types(x.dtype, scale.dtype)
    out = torch.empty((rows, cols), dtype=torch.int8, device=x.device)
    L.call("mi355q_quantize_int_typed", x.data_ptr(), _dt(x), rows, cols, x.stride(0), s2.data_ptr(), _dt(s2),
           L.ptr(z), 1 if z is not None and z.dtype == torch.int8 else 0, s2.stride(0), L.ptr(gi), STRATEGY_CODE[strategy], group_size or 0, bh, bw, num_bits,
           L.BF16 if div_dtype == torch.bfloat16 else L.F32, out.data_ptr(), L.stream_of(x))
    return out


def pack_int4_int32(codes: torch.Tensor) -> torch.Tensor:
    L.require_gpu(codes)
    codes = codes.contiguous()
    rows, cols = codes.shape
    out = torch.empty((rows, cols // 8), dtype=torch.int32, device=codes.device)
    L.call("mi355q_pack_int4_int32", codes.data_ptr(), rows, cols, out.data_ptr(), L.stream_of(codes))
    return out


def observe_mse(x: torch.Tensor, cell_rows: int, cell_cols: int, mn: torch.Tensor, mx: torch.Tensor, qmin: float,
                qmax: float, symmetric: bool, total_steps: int, patience: int, grid: float, norm: float,
                importance: torch.Tensor | None = None, imatrix: bool = False, qtype: str = "int"):
    """MSE grid search over the cells of x (``mi355q_observe_mse``, or with
    ``imatrix`` ``mi355q_observe_imatrix_mse`` weighted by ``importance``
    [cols]) on the integer grid or, with ``qtype="fp8"``, the fp8 e4m3 grid:
    returns the chosen (min, max) per cell as fp32 tensors shaped like
    ``mn``."""
    L.require_gpu(x, mn, mx, importance)
    if x.dim() != 2 or x.stride(1) != 1:
        x = x.reshape(-1, x.shape[-1]).contiguous()
    rows, cols = x.shape
    mn32, mx32 = mn.to(torch.float32).contiguous(), mx.to(torch.float32).contiguous()
    out_mn, out_mx = torch.empty_like(mn32), torch.empty_like(mx32)
    lib = L.lib()
    ws = _ws(lib.mi355q_observe_mse_workspace_size(rows, cols, cell_rows, cell_cols, total_steps), x.device)
    common = (x.data_ptr(), _dt(x), rows, cols, x.stride(0), cell_rows, cell_cols, C.c_float(qmin), C.c_float(qmax),
              1 if symmetric else 0, QTYPE[qtype], int(total_steps), int(patience), C.c_double(grid), C.c_float(norm))
    tail = (mn32.data_ptr(), mx32.data_ptr(), out_mn.data_ptr(), out_mx.data_ptr(), L.ptr(ws),
            0 if ws is None else ws.numel(), L.stream_of(x))
    if imatrix:
        imp = None if importance is None else importance.to(torch.float32).contiguous()
        if imp is not None and imp.numel() != cols:
            raise ValueError(f"importance must have {cols} entries, got {imp.numel()}")
        L.check(lib.mi355q_observe_imatrix_mse(*common, L.ptr(imp), *tail))
    else:
        L.check(lib.mi355q_observe_mse(*common, *tail))
    return out_mn, out_mx


def column_sumsq_(x: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
    """out[c] += sum over rows of x[:, c]^2 (fp32 accumulation), in place."""
    L.require_gpu(x, out)
    if x.dim() != 2 or x.stride(1) != 1:
        x = x.reshape(-1, x.shape[-1]).contiguous()
    if x.dtype not in (torch.bfloat16, torch.float32):
        x = x.to(torch.float32)
    rows, cols = x.shape
    if out.dtype != torch.float32 or out.numel() != cols or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous fp32 vector of {cols}")
    lib = L.lib()
    ws = _ws(lib.mi355q_column_sumsq_workspace_size(rows, cols), x.device)
    L.check(lib.mi355q_column_sumsq(x.data_ptr() if rows else None, _dt(x), rows, cols, x.stride(0), out.data_ptr(),
                                    L.ptr(ws), 0 if ws is None else ws.numel(), L.stream_of(x)))
    return out


def pack_int32(codes: torch.Tensor, num_bits: int) -> torch.Tensor:
    """CT pack_to_int32 layout for 2-, 4- or 8-bit codes (rows padded with 0)."""
    L.require_gpu(codes)
    codes = codes.contiguous()
    rows, cols = codes.shape
    pf = 32 // num_bits
    out = torch.empty((rows, -(-cols // pf)), dtype=torch.int32, device=codes.device)
    L.call("mi355q_pack_int32", codes.data_ptr(), rows, cols, int(num_bits), out.data_ptr(), L.stream_of(codes))
    return out


def pack_int4_int8(codes: torch.Tensor) -> torch.Tensor:
    L.require_gpu(codes)
    if codes.dim() != 2:
        raise ValueError(f"Expected 2D tensor, but got {codes.dim()}D")
    rows, cols = codes.shape
    if cols % 2:
        raise ValueError(f"Expected even number of columns for int4 packing, but got shape {tuple(codes.shape)}")
    codes = codes.contiguous()
    out = torch.empty((rows, cols // 2), dtype=torch.int8, device=codes.device)
    L.call("mi355q_pack_int4_int8", codes.data_ptr(), rows, cols, out.data_ptr(), L.stream_of(codes))
    return out


def mxfp4_quantize_pack(x: torch.Tensor, rule: str = "ct", out=None):
    """bf16 [rows, cols] -> (codes uint8 [rows, cols/2], e8m0 uint8 [rows, cols/32])."""
    L.require_gpu(x)
    if x.dtype != torch.bfloat16:
        raise TypeError("MXFP4 quantize expects bf16 input")
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    if x.stride(1) != 1 or x.stride(0) % 8 or x.data_ptr() % 16:
        x = x.contiguous()
    rows, cols = x.shape
    if cols % 32:
        raise ValueError(f"MXFP4 needs the last dim divisible by 32, got {cols}")
    if out is None:
        codes = torch.empty((rows, cols // 2), dtype=torch.uint8, device=x.device)
        scales = torch.empty((rows, cols // 32), dtype=torch.uint8, device=x.device)
    else:
        codes, scales = out
    L.call("mi355q_mxfp4_quantize_pack", x.data_ptr(), rows, cols, x.stride(0), MX_RULES[rule],
           codes.data_ptr(), scales.data_ptr(), L.stream_of(x))
    return codes, scales


def mxfp4_dequantize(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    L.require_gpu(codes, scales)
    rows, half = codes.shape
    out = torch.empty((rows, half * 2), dtype=torch.bfloat16, device=codes.device)
    L.call("mi355q_mxfp4_dequantize", codes.contiguous().data_ptr(), scales.contiguous().data_ptr(), rows,
           half * 2, out.data_ptr(), L.stream_of(codes))
    return out


def quantize_fp8(x: torch.Tensor, scale: torch.Tensor, strategy: str, group_size: int | None = None,
                 div_dtype: torch.dtype | None = None) -> torch.Tensor:
    """float8_e4m3fn codes (as a float8 tensor) with CT quantize arithmetic."""
    L.require_gpu(x, scale)
    if x.stride(1) != 1:
        x = x.contiguous()
    rows, cols = x.shape
    s = scale.to(torch.float32).contiguous()
    s2 = s.reshape(-1, 1) if s.dim() < 2 else s
    if div_dtype is None:
        div_dtype = torch.promote_types(x.dtype, scale.dtype)
    out = torch.empty((rows, cols), dtype=torch.uint8, device=x.device)
    L.call("mi355q_quantize_fp8", x.data_ptr(), _dt(x), rows, cols, x.stride(0), s2.data_ptr(), s2.stride(0),
           STRATEGY_CODE[strategy], group_size or 0, L.BF16 if div_dtype == torch.bfloat16 else L.F32,
           out.data_ptr(), L.stream_of(x))
    return out.view(torch.float8_e4m3fn)


def fp4_quantize_pack(x: torch.Tensor, scale: torch.Tensor, group_size: int,
                      global_scale: torch.Tensor | None = None) -> torch.Tensor:
    """e2m1 codes of x / (scale / global_scale) per column group, two per byte
    (even column in the low nibble): uint8 [rows, cols / 2] (the NVFP4
    ``weight_packed`` tensor)."""
    L.require_gpu(x, scale)
    if x.dtype not in (torch.bfloat16, torch.float32):
        x = x.float()
    if x.stride(1) != 1:
        x = x.contiguous()
    rows, cols = x.shape
    s = scale.to(torch.float32).reshape(rows, -1).contiguous()
    gs = None if global_scale is None else \
        global_scale.to(device=x.device, dtype=torch.float32).reshape(1).contiguous()
    out = torch.empty((rows, cols // 2), dtype=torch.uint8, device=x.device)
    L.call("mi355q_fp4_quantize_pack", x.data_ptr(), _dt(x), rows, cols, x.stride(0), s.data_ptr(), s.stride(0),
           group_size, L.ptr(gs), out.data_ptr(), L.stream_of(x))
    return out


def quantize_int8_per_token(x: torch.Tensor):
    """Dynamic per-token int8: (codes int8 [rows, cols], scale bf16 [rows, 1])."""
    L.require_gpu(x)
    if x.dtype != torch.bfloat16:
        raise TypeError("per-token int8 expects bf16 activations")
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    if x.stride(1) != 1:
        x = x.contiguous()
    rows, cols = x.shape
    codes = torch.empty((rows, cols), dtype=torch.int8, device=x.device)
    scale = torch.empty((rows, 1), dtype=torch.bfloat16, device=x.device)
    L.call("mi355q_quantize_int8_per_token", x.data_ptr(), rows, cols, x.stride(0), codes.data_ptr(),
           scale.data_ptr(), L.stream_of(x))
    return codes, scale


# ---------------------------------------------------------------- block-scaled fp8
FP8_GROUP = 128     # columns per activation scale, rows and columns per weight scale
_FP8_DT = {torch.bfloat16: L.BF16, torch.float16: L.F16, torch.float32: L.F32}
_FP8_SCALES = {torch.float32: L.SCALE_F32, torch.float8_e8m0fnu: L.SCALE_E8M0}
_FP8_F32, _FP8_E8M0 = (torch.float32,), (torch.float8_e8m0fnu,)


# These calls take a few microseconds on the device at serving sizes, so the
# checks are written to cost little: each attribute of an operand is read once (a
# tensor's shape or strides cost 0.1 us a look), and the workspace sizes, which
# depend on the shape alone, are looked up.
def _rows_2d(t: torch.Tensor, cols: int):
    """t with contiguous rows that do not overlap, and their pitch.
    (``contiguous()`` would return a single row as it is, whatever its
    pitch.)"""
    pitch, step = t.stride()
    if step == 1 and pitch >= cols:
        return t, pitch
    return t.clone(memory_format=torch.contiguous_format), cols


def _rows_16(t: torch.Tensor, cols: int, width: int):
    """``_rows_2d``, and copied if its rows are a multiple of ``width``
    elements (16 bytes) but do not lie on 16-byte boundaries: the product
    kernels load such rows in whole chunks."""
    pitch, step = t.stride()
    if step == 1 and pitch >= cols and (cols % width or (pitch % width == 0 and t.data_ptr() % 16 == 0)):
        return t, pitch
    return t.clone(memory_format=torch.contiguous_format), cols


def _fp8_source(x: torch.Tensor, what: str):
    """x as a 2-D matrix with contiguous rows of bf16, fp16 or fp32: (x, its
    rows, columns and pitch, its type's number)."""
    if not x.is_cuda:
        L.require_gpu(x)
    kind = _FP8_DT.get(x.dtype)
    if kind is None:
        raise TypeError(f"{what} must be bf16, fp16 or fp32, got {x.dtype}")
    shape = x.shape
    if len(shape) != 2 or shape[1] == 0:
        raise ValueError(f"{what} must be a 2-D matrix with columns, got {tuple(shape)}")
    rows, cols = shape
    x, pitch = _rows_2d(x, cols)
    return x, rows, cols, pitch, kind


def _fp8_matrix(codes: torch.Tensor, scales: torch.Tensor, what: str, blocks: bool, scale_dtypes):
    """A checked fp8 matrix, e4m3 codes and scales: (codes, their rows,
    columns and pitch, scales, their pitch)."""
    if not (codes.is_cuda and scales.is_cuda):
        L.require_gpu(codes, scales)
    shape = codes.shape
    if codes.dtype != torch.float8_e4m3fn or len(shape) != 2 or shape[1] == 0:
        raise TypeError(f"{what} must be a 2-D float8_e4m3fn matrix with columns, got {tuple(shape)} {codes.dtype}")
    rows, cols = shape
    groups = -(-cols // FP8_GROUP)
    want = (-(-rows // FP8_GROUP) if blocks else rows, groups)
    if scales.dtype not in scale_dtypes:
        raise TypeError(f"{what} scales must be {' or '.join(str(d) for d in scale_dtypes)}, got {scales.dtype}")
    if scales.shape != want:
        raise ValueError(f"{what} of {(rows, cols)} takes scales of {want}, got {tuple(scales.shape)}")
    codes, pitch = _rows_16(codes, cols, 16)
    scales, scale_pitch = _rows_2d(scales, groups)
    return codes, rows, cols, pitch, scales, scale_pitch


def _fp8_gradient(dy: torch.Tensor, rows: int | None, cols: int | None):
    """A checked output gradient of these sizes (None: any): (dy, its rows,
    columns and pitch)."""
    if not dy.is_cuda:
        L.require_gpu(dy)
    if dy.dtype != torch.bfloat16:
        raise TypeError(f"the output gradient must be bf16, got {dy.dtype}")
    shape = dy.shape
    if len(shape) != 2 or (rows is not None and shape[0] != rows) or (shape[1] != cols if cols else shape[1] == 0):
        raise ValueError(f"the output gradient must be [{'rows' if rows is None else rows}, {cols or 'out'}], got "
                         f"{tuple(shape)}")
    dy, pitch = _rows_16(dy, shape[1], 8)
    return dy, shape[0], shape[1], pitch


def _several_devices(*operands) -> ValueError:
    return ValueError("operands on several devices: " + " and ".join(str(t.device) for t in operands if t is not None))


@functools.lru_cache(maxsize=4096)
def _fp8_workspace(query: str, rows: int, out: int, cols: int) -> int:
    return getattr(L.lib(), query)(rows, out, cols)


def _fp8_scratch(query: str, rows: int, out: int, cols: int, like: torch.Tensor):
    """(workspace or None to keep alive over the call, its address, its bytes)"""
    n = _fp8_workspace(query, rows, out, cols)
    if n == 0:
        return None, None, 0
    ws = like.new_empty(n, dtype=torch.uint8)
    return ws, ws.data_ptr(), n


def fp8_quantize_groups(x: torch.Tensor, scale_dtype: torch.dtype = torch.float32):
    """x [rows, cols] as float8_e4m3fn codes and one scale per row and 128
    columns: (codes [rows, cols], scales [rows, ceil(cols / 128)]).

    ``scale_dtype`` float32: max |x| / 448; float8_e8m0fnu: the least power
    of two not below it, with which the codes are also the 8-bit checkpoint
    that ``fp8_block_grad_weight`` reads.  A group holding an infinity or a
    NaN becomes NaN as a whole."""
    x, rows, cols, pitch, kind = _fp8_source(x, "x")
    scale_kind = _FP8_SCALES.get(scale_dtype)
    if scale_kind is None:
        raise TypeError(f"scale_dtype must be float32 or float8_e8m0fnu, got {scale_dtype}")
    groups = -(-cols // FP8_GROUP)
    codes = x.new_empty((rows, cols), dtype=torch.float8_e4m3fn)
    scales = x.new_empty((rows, groups), dtype=scale_dtype)
    rc = L.lib().mi355q_fp8_quantize_groups(x.data_ptr(), kind, rows, cols, pitch, codes.data_ptr(), cols,
                                            scales.data_ptr(), scale_kind, groups, L.stream_of(x))
    if rc:
        L.check(rc)
    return codes, scales


def fp8_quantize_blocks(w: torch.Tensor):
    """w [rows, cols] as float8_e4m3fn codes and one fp32 scale (max |w| /
    448) per 128 x 128 block: (codes [rows, cols], scales [ceil(rows / 128),
    ceil(cols / 128)]).  A block holding an infinity or a NaN becomes NaN as a
    whole."""
    w, rows, cols, pitch, kind = _fp8_source(w, "w")
    groups = -(-cols // FP8_GROUP)
    codes = w.new_empty((rows, cols), dtype=torch.float8_e4m3fn)
    scales = w.new_empty((-(-rows // FP8_GROUP), groups), dtype=torch.float32)
    rc = L.lib().mi355q_fp8_quantize_blocks(w.data_ptr(), kind, rows, cols, pitch, codes.data_ptr(), cols,
                                            scales.data_ptr(), groups, L.stream_of(w))
    if rc:
        L.check(rc)
    return codes, scales


def fp8_block_matmul(x: torch.Tensor, x_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor,
                     bias: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """y = X W^T (+ bias) [rows, out] of two fp8 matrices: x [rows, cols] with
    scales per row and 128 columns (float32 or float8_e8m0fnu,
    ``fp8_quantize_groups``), w [out, cols] with float32 scales per 128 x 128
    block (``fp8_quantize_blocks``, or an FP8_BLOCK checkpoint's
    ``weight_scale`` in fp32).  Sums in fp32, rounded once to ``out_dtype``
    (bf16, fp16 or fp32).  ``bias`` [out] is bf16, fp16 or fp32.

    Views whose rows lie 2^22 or more elements apart, codes or x_scales, are right but
    slow above 32 rows, and in the gradients: about 30 times on large products.  Make them
    contiguous first."""
    x, rows, cols, x_pitch, x_scales, xs_pitch = _fp8_matrix(x, x_scales, "x", False, _FP8_SCALES)
    w, out, w_cols, w_pitch, w_scales, ws_pitch = _fp8_matrix(w, w_scales, "w", True, _FP8_F32)
    if w_cols != cols or out == 0:
        raise ValueError(f"x [{rows}, {cols}] does not multiply w {tuple(w.shape)}")
    kind = _FP8_DT.get(out_dtype)
    if kind is None:
        raise TypeError(f"out_dtype must be bf16, fp16 or fp32, got {out_dtype}")
    here = x.get_device()
    bias_ptr, bias_kind = None, 0
    if bias is not None:
        if not bias.is_cuda:
            L.require_gpu(bias)
        bias_kind = _FP8_DT.get(bias.dtype)
        if bias_kind is None:
            raise TypeError(f"bias must be bf16, fp16 or fp32, got {bias.dtype}")
        if bias.shape != (out,):
            raise ValueError(f"bias must be [{out}], got {tuple(bias.shape)}")
        bias = bias.contiguous()
        bias_ptr = bias.data_ptr()
        if bias.get_device() != here:
            raise _several_devices(x, bias)
    if w.get_device() != here or x_scales.get_device() != here or w_scales.get_device() != here:
        raise _several_devices(x, x_scales, w, w_scales)
    y = x.new_empty((rows, out), dtype=out_dtype)
    ws, ws_ptr, ws_bytes = _fp8_scratch("mi355q_fp8_block_matmul_workspace_size", rows, out, cols, x)
    rc = L.lib().mi355q_fp8_block_matmul(
        x.data_ptr(), x_pitch, x_scales.data_ptr(), _FP8_SCALES[x_scales.dtype], xs_pitch, w.data_ptr(), w_pitch,
        w_scales.data_ptr(), ws_pitch, bias_ptr, bias_kind, y.data_ptr(), kind, out, rows, out, cols, ws_ptr, ws_bytes,
        L.stream_of(x))
    if rc:
        L.check(rc)
    return y


def fp8_block_grad_input(dy: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor) -> torch.Tensor:
    """dX = dY W [rows, cols] in bf16: the input gradient of
    ``fp8_block_matmul`` (dy bf16 [rows, out], w as in the forward product;
    the weight's values enter exactly, sums in fp32)."""
    w, out, cols, w_pitch, w_scales, ws_pitch = _fp8_matrix(w, w_scales, "w", True, _FP8_F32)
    if out == 0:
        raise ValueError("w has no rows")
    dy, rows, _, pitch = _fp8_gradient(dy, None, out)
    here = dy.get_device()
    if w.get_device() != here or w_scales.get_device() != here:
        raise _several_devices(dy, w, w_scales)
    dx = dy.new_empty((rows, cols))
    ws, ws_ptr, ws_bytes = _fp8_scratch("mi355q_fp8_block_grad_input_workspace_size", rows, out, cols, dy)
    rc = L.lib().mi355q_fp8_block_grad_input(dy.data_ptr(), pitch, w.data_ptr(), w_pitch, w_scales.data_ptr(),
                                             ws_pitch, dx.data_ptr(), cols, rows, out, cols, ws_ptr, ws_bytes,
                                             L.stream_of(dy))
    if rc:
        L.check(rc)
    return dx


def fp8_block_grad_weight(dy: torch.Tensor, x: torch.Tensor, x_scales: torch.Tensor,
                          out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """dW = dY^T X [out, cols]: the weight gradient of ``fp8_block_matmul``
    from the 8-bit checkpoint of its input (``fp8_quantize_groups`` with
    ``scale_dtype=torch.float8_e8m0fnu``; the checkpoint's values enter
    exactly).  dy bf16 [rows, out]; sums in fp32, rounded once to
    ``out_dtype`` (bf16, fp16 or fp32).  Zeros when there are no rows."""
    x, rows, cols, x_pitch, x_scales, xs_pitch = _fp8_matrix(x, x_scales, "x", False, _FP8_E8M0)
    dy, _, out, pitch = _fp8_gradient(dy, rows, None)
    kind = _FP8_DT.get(out_dtype)
    if kind is None:
        raise TypeError(f"out_dtype must be bf16, fp16 or fp32, got {out_dtype}")
    here = dy.get_device()
    if x.get_device() != here or x_scales.get_device() != here:
        raise _several_devices(dy, x, x_scales)
    dw = dy.new_empty((out, cols), dtype=out_dtype)
    ws, ws_ptr, ws_bytes = _fp8_scratch("mi355q_fp8_block_grad_weight_workspace_size", rows, out, cols, dy)
    rc = L.lib().mi355q_fp8_block_grad_weight(dy.data_ptr(), pitch, x.data_ptr(), x_pitch, x_scales.data_ptr(),
                                              xs_pitch, dw.data_ptr(), kind, cols, rows, out, cols, ws_ptr, ws_bytes,
                                              L.stream_of(dy))
    if rc:
        L.check(rc)
    return dw


def fp8_silu_mul(gate_up: torch.Tensor, save: bool = True):
    """h = silu(gate) * up of gate_up [rows, 2 n] (gate in the first n
    columns) as an fp8 matrix with e8m0 scales: (h codes [rows, n], h scales
    [rows, ceil(n / 128)]).  With ``save`` also gate and up in 8 bits for the
    backward pass: (..., saved codes [rows, 2 n], saved scales [rows, 2
    ceil(n / 128)]), gate's groups before up's."""
    x, rows, both, pitch, kind = _fp8_source(gate_up, "gate_up")
    if both % 2:
        raise ValueError(f"gate_up must hold gate and up side by side, got {both} columns")
    cols = both // 2
    groups = -(-cols // FP8_GROUP)
    h = x.new_empty((rows, cols), dtype=torch.float8_e4m3fn)
    hs = x.new_empty((rows, groups), dtype=torch.float8_e8m0fnu)
    kept = x.new_empty((rows, 2 * cols), dtype=torch.float8_e4m3fn) if save else None
    ks = x.new_empty((rows, 2 * groups), dtype=torch.float8_e8m0fnu) if save else None
    rc = L.lib().mi355q_fp8_silu_mul(x.data_ptr(), kind, rows, cols, pitch, h.data_ptr(), cols, hs.data_ptr(),
                                     kept.data_ptr() if save else None, 2 * cols,
                                     ks.data_ptr() if save else None, L.stream_of(x))
    if rc:
        L.check(rc)
    return (h, hs, kept, ks) if save else (h, hs)


def fp8_silu_mul_backward(dh: torch.Tensor, saved: torch.Tensor, saved_scales: torch.Tensor) -> torch.Tensor:
    """The gradient [rows, 2 n] of ``fp8_silu_mul``'s input, in dh's type,
    from dh [rows, n] (bf16, fp16 or fp32) and what the forward pass saved."""
    dh, rows, cols, pitch, kind = _fp8_source(dh, "dh")
    if not (saved.is_cuda and saved_scales.is_cuda):
        L.require_gpu(saved, saved_scales)
    groups = -(-cols // FP8_GROUP)
    if saved.dtype != torch.float8_e4m3fn or saved_scales.dtype != torch.float8_e8m0fnu:
        raise TypeError(f"saved codes and scales must be float8_e4m3fn and float8_e8m0fnu, got {saved.dtype} and "
                        f"{saved_scales.dtype}")
    if saved.shape != (rows, 2 * cols) or saved_scales.shape != (rows, 2 * groups):
        raise ValueError(f"dh of {(rows, cols)} takes saved codes of {(rows, 2 * cols)} and scales of "
                         f"{(rows, 2 * groups)}, got {tuple(saved.shape)} and {tuple(saved_scales.shape)}")
    here = dh.get_device()
    if saved.get_device() != here or saved_scales.get_device() != here:
        raise _several_devices(dh, saved, saved_scales)
    saved, saved_pitch = _rows_2d(saved, 2 * cols)
    saved_scales, ss_pitch = _rows_2d(saved_scales, 2 * groups)
    dx = dh.new_empty((rows, 2 * cols))
    rc = L.lib().mi355q_fp8_silu_mul_backward(dh.data_ptr(), kind, rows, cols, pitch, saved.data_ptr(), saved_pitch,
                                              saved_scales.data_ptr(), ss_pitch, dx.data_ptr(), 2 * cols,
                                              L.stream_of(dh))
    if rc:
        L.check(rc)
    return dx


# ---------------------------------------------------------------- tokens by expert
_MOE_DT = _FP8_DT
MOE_MAX_EXPERTS = 2040      # of a plan


@functools.lru_cache(maxsize=4096)
def _moe_workspace(tokens: int, top: int, num_experts: int) -> int:
    return L.lib().mi355q_moe_plan_workspace_size(tokens, top, num_experts)


def moe_plan(top_k_index: torch.Tensor, num_experts: int):
    """The order of tokens by expert of ``top_k_index`` [tokens, top] (int32 or
    int64): (rows int32 [tokens * top], slots int32 [tokens, top], offsets int64
    [num_experts + 1]).

    Pairs (token, choice) are ordered by expert, then choice, then token;
    ``slots`` is the place of each, ``rows`` the token at each place and
    ``offsets`` the first place of each expert.  Pairs whose id is outside [0,
    num_experts) - padding - come last, from ``offsets[-1]`` on."""
    L.require_gpu(top_k_index)
    bits = {torch.int32: 32, torch.int64: 64}.get(top_k_index.dtype)
    if bits is None:
        raise TypeError(f"top_k_index must be int32 or int64, got {top_k_index.dtype}")
    if num_experts <= 0:
        raise ValueError(f"num_experts must be positive, got {num_experts}")
    if top_k_index.dim() != 2 or top_k_index.shape[1] == 0:
        raise ValueError(f"top_k_index must be [tokens, top], got {tuple(top_k_index.shape)}")
    tokens, top = top_k_index.shape
    ids, pitch = _rows_2d(top_k_index, top)
    rows = ids.new_empty(tokens * top, dtype=torch.int32)
    slots = ids.new_empty((tokens, top), dtype=torch.int32)
    offsets = ids.new_empty(num_experts + 1, dtype=torch.int64)
    lib = L.lib()
    need = _moe_workspace(tokens, top, num_experts)
    ws = ids.new_empty(need, dtype=torch.uint8) if need else None
    rc = lib.mi355q_moe_plan(ids.data_ptr(), bits, tokens, top, pitch, num_experts, rows.data_ptr(), slots.data_ptr(),
                             offsets.data_ptr(), None if ws is None else ws.data_ptr(), need, L.stream_of(ids))
    if rc:
        L.check(rc)
    return rows, slots, offsets


def _moe_places(slots: torch.Tensor, offsets: torch.Tensor, like: torch.Tensor):
    """Checked slots and offsets: (slots, tokens, top, the address of offsets'
    last entry)."""
    if not (slots.is_cuda and offsets.is_cuda):
        L.require_gpu(slots, offsets)
    if slots.dtype != torch.int32 or slots.dim() != 2 or slots.shape[1] == 0:
        raise TypeError(f"slots must be int32 [tokens, top], got {tuple(slots.shape)} {slots.dtype}")
    if offsets.dtype != torch.int64 or offsets.dim() != 1 or offsets.shape[0] < 2:
        raise TypeError(f"offsets must be int64 [experts + 1], got {tuple(offsets.shape)} {offsets.dtype}")
    if slots.device != like.device or offsets.device != like.device:
        raise _several_devices(like, slots, offsets)
    return slots.contiguous(), *slots.shape, offsets.data_ptr() + 8 * (offsets.shape[0] - 1) * offsets.stride(0)


def _moe_weights(weights: torch.Tensor, slots: torch.Tensor):
    if not weights.is_cuda:
        L.require_gpu(weights)
    if weights.dtype not in _MOE_DT:
        raise TypeError(f"weights must be bf16, fp16 or fp32, got {weights.dtype}")
    if weights.shape != slots.shape:
        raise ValueError(f"slots of {tuple(slots.shape)} take weights of the same shape, got {tuple(weights.shape)}")
    if weights.device != slots.device:
        raise _several_devices(slots, weights)
    return weights.contiguous(), _MOE_DT[weights.dtype]


def moe_sort(x: torch.Tensor, slots: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """x [tokens, cols] (bf16, fp16 or fp32) in the order of the experts:
    out[slots[t, k]] = x[t], [tokens * top, cols]; zeros from ``offsets[-1]``
    on."""
    x, rows, cols, pitch, kind = _fp8_source(x, "x")
    slots, tokens, top, end = _moe_places(slots, offsets, x)
    if rows != tokens:
        raise ValueError(f"slots of {tuple(slots.shape)} take x of {tokens} rows, got {rows}")
    y = x.new_empty((tokens * top, cols))
    L.check(L.lib().mi355q_moe_sort(x.data_ptr(), kind, tokens, top, cols, pitch, slots.data_ptr(), end, y.data_ptr(),
                                    cols, L.stream_of(x)))
    return y


def moe_combine(x: torch.Tensor, weights: torch.Tensor | None, slots: torch.Tensor,
                offsets: torch.Tensor) -> torch.Tensor:
    """The experts' rows x [tokens * top, cols] back at their tokens: out[t] =
    sum over k of weights[t, k] * x[slots[t, k]] (``weights`` None: ones), fp32
    sums in the order of k, rounded once to x's type.  Places from
    ``offsets[-1]`` on take no part, whatever x holds there."""
    x, rows, cols, pitch, kind = _fp8_source(x, "x")
    slots, tokens, top, end = _moe_places(slots, offsets, x)
    if rows != tokens * top:
        raise ValueError(f"slots of {tuple(slots.shape)} take x of {tokens * top} rows, got {rows}")
    w_ptr, w_kind = None, 0
    if weights is not None:
        weights, w_kind = _moe_weights(weights, slots)
        w_ptr = weights.data_ptr()
    y = x.new_empty((tokens, cols))
    L.check(L.lib().mi355q_moe_combine(x.data_ptr(), kind, tokens, top, cols, pitch, w_ptr, w_kind, slots.data_ptr(),
                                       end, y.data_ptr(), cols, L.stream_of(x)))
    return y


def moe_combine_backward(dy: torch.Tensor, x: torch.Tensor | None, weights: torch.Tensor, slots: torch.Tensor,
                         offsets: torch.Tensor, need_x: bool = True, need_weights: bool = True):
    """The gradients of ``moe_combine`` for dy [tokens, cols]: (dx [tokens *
    top, cols] in dy's type or None, dweights [tokens, top] in the weights'
    type or None).  ``x`` is read for dweights only.  Zeros at places from
    ``offsets[-1]`` on."""
    dy, rows, cols, pitch, kind = _fp8_source(dy, "dy")
    slots, tokens, top, end = _moe_places(slots, offsets, dy)
    if rows != tokens:
        raise ValueError(f"slots of {tuple(slots.shape)} take dy of {tokens} rows, got {rows}")
    weights, w_kind = _moe_weights(weights, slots)
    x_ptr, x_pitch = None, 0
    if need_weights:
        if x is None:
            raise ValueError("the weights' gradient takes x")
        x, n, x_cols, x_pitch, x_kind = _fp8_source(x, "x")
        if (n, x_cols, x_kind) != (tokens * top, cols, kind):
            raise ValueError(f"dy of {tuple(dy.shape)} {dy.dtype} takes x of {(tokens * top, cols)} in its type, got "
                             f"{tuple(x.shape)} {x.dtype}")
        if x.device != dy.device:
            raise _several_devices(dy, x)
        x_ptr = x.data_ptr()
    dx = dy.new_empty((tokens * top, cols)) if need_x else None
    dw = torch.empty_like(weights) if need_weights else None
    L.check(L.lib().mi355q_moe_combine_backward(dy.data_ptr(), kind, tokens, top, cols, pitch, x_ptr, x_pitch,
                                                weights.data_ptr(), w_kind, slots.data_ptr(), end, L.ptr(dx), cols,
                                                L.ptr(dw), L.stream_of(dy)))
    return dx, dw


# ---------------------------------------------------------------- 4-bit weights
_W4_DT = {torch.bfloat16: L.BF16, torch.float16: L.F16}


def _w4_operand(t: torch.Tensor, shape, dtypes, what: str, lead: int):
    """A checked part of a 4-bit weight with contiguous rows: (t, its pitch, the
    stride of its experts); ``lead`` 1: [experts, ...]."""
    if not t.is_cuda:
        L.require_gpu(t)
    if t.dtype not in dtypes:
        raise TypeError(f"{what} must be {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what} must be {tuple(shape)}, got {tuple(t.shape)}")
    rows, cols = shape[-2], shape[-1]
    strides = t.stride()
    if strides[-1] != 1 and cols > 1 or strides[-2] < cols and rows > 1:
        t = t.clone(memory_format=torch.contiguous_format)
        strides = t.stride()
    return t, strides[-2] if rows > 1 else cols, strides[0] if lead else 0


@functools.lru_cache(maxsize=4096)
def _w4_workspace(in_place: bool, n_x: int, rows: int, experts: int, out: int, cols: int, fmt: int, group: int) -> int:
    lib = L.lib()
    query = lib.mi355q_w4a16_matmul_workspace_size_in_place if in_place else lib.mi355q_w4a16_matmul_workspace_size
    return query(n_x, rows, experts, out, cols, fmt, group)


def _w4_matmul(x, index, offsets, experts, n_rows, weight_packed, weight_scale, weight_zero_point, group_size, bias,
               gated, out_dtype):
    if not x.is_cuda:
        L.require_gpu(x)
    kind = _W4_DT.get(x.dtype)
    if kind is None:
        raise TypeError(f"x must be bf16 or fp16, got {x.dtype}")
    if x.dim() != 2 or x.shape[1] == 0:
        raise ValueError(f"x must be a 2-D matrix with columns, got {tuple(x.shape)}")
    n_x, cols = x.shape
    if cols < 8:                  # the kernels read x in chunks of 8: zeros behind it
        if group_size is None or group_size >= cols:
            group_size = 32       # one group
        x, cols = torch.nn.functional.pad(x, (0, 8 - cols)), 8
    x, pitch = _rows_2d(x, cols)
    lead = 0 if experts is None else 1
    if weight_packed.dim() != 2 + lead:
        raise ValueError(f"weight_packed must be {'[experts, out, ...]' if lead else '[out, ...]'}, got "
                         f"{tuple(weight_packed.shape)}")
    out = weight_packed.shape[-2]
    first = (experts,) if lead else ()
    mx = weight_packed.dtype == torch.uint8
    if out == 0:
        raise ValueError("weight_packed has no rows")
    if gated and out % 2:
        raise ValueError(f"a gated weight holds gate and up, got {out} rows")
    if mx:
        if cols % 32:
            raise ValueError(f"MXFP4 weights take whole groups of 32 columns, got {cols}")
        if weight_zero_point is not None:
            raise ValueError("MXFP4 weights have no zero points")
        group, groups = 32, cols // 32
        w, ldw, stride_w = _w4_operand(weight_packed, (*first, out, cols // 2), (torch.uint8,), "weight_packed", lead)
        s, lds, stride_s = _w4_operand(weight_scale, (*first, out, groups), (torch.uint8, torch.float8_e8m0fnu),
                                       "weight_scale", lead)
        s_kind = L.BF16
    else:
        group = cols if group_size is None else group_size
        if group <= 0 or not (group in (32, 64) or group % 128 == 0 or group >= cols):
            raise ValueError(f"group_size must be 32, 64, a multiple of 128 or all columns (None), got {group_size}")
        groups = -(-cols // group)
        w, ldw, stride_w = _w4_operand(weight_packed, (*first, out, -(-cols // 8)), (torch.int32,), "weight_packed",
                                       lead)
        ldw, stride_w = 4 * ldw, 4 * stride_w
        s, lds, stride_s = _w4_operand(weight_scale, (*first, out, groups), tuple(_FP8_DT), "weight_scale", lead)
        s_kind = _FP8_DT[s.dtype]
    wide = (cols // 2 if mx else -(-cols // 8) * 4)
    if wide % 16 == 0 and (ldw % 16 or stride_w % 16 or w.data_ptr() % 16):
        # rows of whole 16-byte chunks that do not lie on 16-byte boundaries
        w = w.clone(memory_format=torch.contiguous_format)
        ldw, stride_w = wide, out * wide
    here, z_ptr, ldz, stride_z, b_ptr, b_kind = x.get_device(), None, 0, 0, None, 0
    z = b = None
    if weight_zero_point is not None:
        z, ldz, stride_z = _w4_operand(weight_zero_point, (*first, -(-out // 8), groups), (torch.int32,),
                                       "weight_zero_point", lead)
        z_ptr = z.data_ptr()
    if bias is not None:
        if not bias.is_cuda:
            L.require_gpu(bias)
        b_kind = _FP8_DT.get(bias.dtype)
        if b_kind is None:
            raise TypeError(f"bias must be bf16, fp16 or fp32, got {bias.dtype}")
        if bias.shape != (out,):
            raise ValueError(f"bias must be [{out}], got {tuple(bias.shape)}")
        b = bias.contiguous()
        b_ptr = b.data_ptr()
    if any(t is not None and t.get_device() != here for t in (w, s, z, b, index, offsets)):
        raise _several_devices(x, w, s, z, b, index, offsets)
    out_dtype = x.dtype if out_dtype is None else out_dtype
    y_kind = _FP8_DT.get(out_dtype)
    if y_kind is None:
        raise TypeError(f"out_dtype must be bf16, fp16 or fp32, got {out_dtype}")
    width = out // 2 if gated else out
    y = x.new_empty((n_rows, width), dtype=out_dtype)
    fmt = L.W4_MXFP4 if mx else L.W4_INT4
    in_place = pitch % 8 == 0 and x.data_ptr() % 16 == 0
    ws_bytes = _w4_workspace(in_place, n_x, n_rows, experts or 1, out, cols, fmt, group)
    ws = x.new_empty(ws_bytes, dtype=torch.uint8) if ws_bytes else None
    ws_ptr = None if ws is None else ws.data_ptr()
    rc = L.lib().mi355q_w4a16_matmul(
        x.data_ptr(), kind, n_x, pitch, None if index is None else index.data_ptr(),
        None if offsets is None else offsets.data_ptr(), experts or 1, w.data_ptr(), fmt, ldw,
        stride_w, s.data_ptr(), s_kind, lds, stride_s, z_ptr, ldz, stride_z, group, b_ptr, b_kind, int(gated),
        y.data_ptr(), y_kind, width, n_rows, out, cols, ws_ptr, ws_bytes, L.stream_of(x))
    if rc:
        L.check(rc)
    return y


def w4a16_matmul(x: torch.Tensor, weight_packed: torch.Tensor, weight_scale: torch.Tensor,
                 weight_zero_point: torch.Tensor | None = None, group_size: int | None = 128,
                 bias: torch.Tensor | None = None, gated: bool = False,
                 out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """y = x W^T (+ bias) [rows, out] of 16-bit activations x [rows, cols] (bf16
    or fp16) and a 4-bit weight as a compressed checkpoint holds it:

    * ``pack-quantized``: ``weight_packed`` int32 [out, ceil(cols / 8)],
      ``weight_scale`` [out, ceil(cols / group_size)] in bf16, fp16 or fp32,
      ``weight_zero_point`` int32 [ceil(out / 8), groups] or None (symmetric);
      ``group_size`` 32, 64, a multiple of 128, or None (channel);
    * ``mxfp4-pack-quantized``: ``weight_packed`` uint8 [out, cols / 2],
      ``weight_scale`` uint8 (or float8_e8m0fnu) [out, cols / 32]; cols % 32 == 0.

    ``gated``: the weight holds gate's rows and then up's, and y [rows, out /
    2] = silu(gate) * up.  Sums in fp32, rounded once to ``out_dtype`` (x's
    type, or bf16, fp16, fp32).  No gradients.  A row of x that holds an infinity may
    come out as NaN throughout, as one with a NaN does."""
    return _w4_matmul(x, None, None, None, x.shape[0], weight_packed, weight_scale, weight_zero_point, group_size,
                      bias, gated, out_dtype)


def w4a16_experts_matmul(x: torch.Tensor, rows: torch.Tensor | None, offsets: torch.Tensor,
                         weight_packed: torch.Tensor, weight_scale: torch.Tensor,
                         weight_zero_point: torch.Tensor | None = None, group_size: int | None = 128,
                         gated: bool = False, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``w4a16_matmul`` for rows grouped by expert, with the experts' weights
    stacked ([experts, ...] each): row i of y, offsets[e] <= i < offsets[e +
    1], is x[rows[i]] times expert e's weight (``rows`` int32, as ``moe_plan``
    gives them, or None: x[i]).  ``offsets`` int64 [experts + 1], ascending, stays on
    the device: the call waits for nothing.  Rows before offsets[0] (of experts
    that others hold) and from offsets[-1] on are zeros."""
    if not offsets.is_cuda:
        L.require_gpu(offsets)
    if offsets.dtype != torch.int64 or offsets.dim() != 1 or offsets.shape[0] < 2:
        raise TypeError(f"offsets must be int64 [experts + 1], got {tuple(offsets.shape)} {offsets.dtype}")
    if rows is not None:
        if not rows.is_cuda:
            L.require_gpu(rows)
        if rows.dtype != torch.int32 or rows.dim() != 1:
            raise TypeError(f"rows must be int32 and 1-D, got {tuple(rows.shape)} {rows.dtype}")
        rows = rows.contiguous()
    return _w4_matmul(x, rows, offsets.contiguous(), offsets.shape[0] - 1,
                      x.shape[0] if rows is None else rows.shape[0], weight_packed, weight_scale, weight_zero_point,
                      group_size, None, gated, out_dtype)


# ---------------------------------------------------------------- SparseGPT
def sparsegpt_base_mask(w_work: torch.Tensor):
    """(mask uint8 [rows, cols] = w_work == 0, count int32 [1] on the device)."""
    L.require_gpu(w_work)
    rows, cols = w_work.shape
    mask = torch.empty((rows, cols), dtype=torch.uint8, device=w_work.device)
    count = torch.empty(1, dtype=torch.int32, device=w_work.device)
    L.call("mi355q_sparsegpt_base_mask", w_work.data_ptr(), rows, cols, mask.data_ptr(), count.data_ptr(),
           L.stream_of(w_work))
    return mask, count


def sparsegpt_sweep_(w_work: torch.Tensor, hinv: torch.Tensor, sparsity: float, prune_n: int, prune_m: int,
                     blocksize: int = 128, mask: torch.Tensor | None = None) -> torch.Tensor:
    """In-place SparseGPT sweep of w_work (fp32 [rows, cols]) with the upper
    factor hinv.  ``mask`` (uint8, from ``sparsegpt_base_mask``) preserves the
    entries it holds.  Returns the per-row losses fp32 [rows]."""
    L.require_gpu(w_work, hinv, mask)
    rows, cols = w_work.shape
    if hinv.shape != (cols, cols) or hinv.dtype != torch.float32 or not hinv.is_contiguous():
        raise ValueError(f"hinv must be a contiguous fp32 [{cols}, {cols}] matrix")
    if mask is not None and (mask.shape != (rows, cols) or mask.dtype != torch.uint8 or not mask.is_contiguous()):
        raise ValueError("mask must be a contiguous uint8 matrix shaped like w_work")
    losses = torch.zeros(rows, dtype=torch.float32, device=w_work.device)
    lib = L.lib()
    ws = _ws(lib.mi355q_sparsegpt_workspace_size(rows, cols, blocksize), w_work.device)
    L.check(lib.mi355q_sparsegpt_sweep(w_work.data_ptr(), rows, cols, hinv.data_ptr(), C.c_double(sparsity),
                                       int(prune_n), int(prune_m), blocksize, L.ptr(mask), losses.data_ptr(),
                                       ws.data_ptr(), ws.numel(), L.stream_of(w_work)))
    return losses
