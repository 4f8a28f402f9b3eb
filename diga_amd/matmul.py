"""Token rows in 8 bits and the matrix products on them (no reference counterpart; csrc/rowquant.hip, csrc/matmul.hip).

An 8-bit row is e4m3 (torch.float8_e4m3fn) with one fp32 scale per 128 columns, value = q * scale; a weight matrix [N, K] has one
scale per 128 x 128 block.  One gated block of an encoder, dense or by expert:

    q, s, h = rms_norm_fp8(x, norm_w, residual)                       # h = x + residual, normalised, in 8 bits
    up      = matmul_fp8(q, s, up_w, up_s)                            # [.., 2 N]: gate | up
    q, s    = silu_mul_fp8(up)
    y       = matmul_fp8(q, s, down_w, down_s)

    up      = grouped_matmul_fp8(q, s, up_w, up_s, offsets, rows)     # up_w [E, 2 N, K]; rows: token of every slot, by expert

Everything is enqueued on the current stream of the tensors' device, allocates through torch and can be captured into a graph.
Scales of rows come back as a [rows, blocks] view whose rows lie side by side in memory (stride 1), the layout the products read
fastest; any strides are accepted.  A call that would write a result over its own operands is refused, but for a norm's residual_out on x
or the residual.  There is no CPU path and no backward pass: tensors are taken detached.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version as _written      # a tensor written in place: a backward that saved it has to notice

from ._lib import DigaError, check, load

try:
    from . import _calls
except ImportError as e:
    raise DigaError(f"diga_amd/_calls.so: {e}: build it with `python -c 'import __graft_entry__ as g; g.build()'` (or `make -C diga_amd/csrc`)") from e

# Every function first hands its call to _calls (csrc/calls.cpp), which takes the ordinary ones: plain tensors on the current GPU of
# the documented types, shapes and layouts.  It returns None for anything else; what follows checks, explains and takes the rest.
_BOUND = ("diga_rms_norm_fp8", "diga_silu_mul_fp8", "diga_quantize_fp8", "diga_matmul_fp8", "diga_grouped_matmul_fp8", "diga_grouped_matmul",
          "diga_last_error_string")
_calls.bind(*(ctypes.cast(getattr(load(), name), ctypes.c_void_p).value for name in _BOUND), DigaError)

BLOCK = 128
E4M3 = torch.float8_e4m3fn
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_HALVES = {torch.bfloat16: 0, torch.float16: 1}
_E4M3 = {E4M3: 0}
_stream_of = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice
_empty, _strided = torch.empty, torch.empty_strided


class _Entry:
    """An entry point of the library, looked up at its first call and called on the current stream of device `index` (the stream is
    appended as the last argument)."""

    __slots__ = ("name", "fn")

    def __init__(self, name):
        self.name, self.fn = name, None

    def __call__(self, index, *args):
        fn = self.fn
        if fn is None:
            fn = self.fn = getattr(load(), self.name)
        if index == _current_device():
            rc = fn(*args, _stream_of(index))
        else:
            with torch.cuda.device(index):
                rc = fn(*args, _stream_of(index))
        if rc < 0:
            check(rc, self.name)


_rms_norm, _silu_mul, _quantize = _Entry("diga_rms_norm_fp8"), _Entry("diga_silu_mul_fp8"), _Entry("diga_quantize_fp8")
_matmul, _grouped_fp8, _grouped = _Entry("diga_matmul_fp8"), _Entry("diga_grouped_matmul_fp8"), _Entry("diga_grouped_matmul")
_matmul_f32, _grouped_fp8_f32 = _Entry("diga_matmul_fp8_f32"), _Entry("diga_grouped_matmul_fp8_f32")


def _device(who, *tensors):
    """Index of the one GPU all of `tensors` are on (None = an argument that was not given)."""
    index = tensors[0].get_device()
    if index < 0:
        raise DigaError(f"{who}: tensors must be on the GPU: there is no CPU fallback")
    tangents = forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled()      # (no tensor has one outside a level)
    for t in tensors:
        if t is not None:
            if t.get_device() != index:
                raise DigaError(f"{who}: tensors on {t.device} and {tensors[0].device}")
            if t.is_neg():
                raise DigaError(f"{who}: a tensor's values are held negated: pass its resolve_neg()")
            if t.requires_grad and torch.is_grad_enabled():
                raise DigaError(f"{who} has no backward pass: call it under torch.no_grad() or on detached tensors")
            if tangents and forward_ad.unpack_dual(t).tangent is not None:
                raise DigaError(f"{who} has no derivative: a tensor carries a tangent, which would be dropped: pass it without")
    return index


def _counts(who, what, n):
    """The entry points take columns, weight rows and groups as 32-bit integers, which ctypes would cut off without a word."""
    if n >= 1 << 31:
        raise DigaError(f"{who}: {n} {what} are more than 2^31 - 1")


def _rows(who, name, t, dtypes):
    """A matrix whose columns are adjacent, of one of `dtypes` -> (rows, columns, row stride)."""
    if t.dim() == 2:
        m, n = t.shape
        ld, step = t.stride()
        if n and (step == 1 or n == 1):
            if t.dtype in dtypes:
                _counts(who, f"columns of {name}", n)
                return m, n, ld
            raise DigaError(f"{who}: {name} is {t.dtype}, not one of {', '.join(str(d) for d in dtypes)}")
    raise DigaError(f"{who}: {name} must be a matrix with adjacent columns, got {tuple(t.shape)} with strides {t.stride()}")


def _plain(who, name, t, dtype, shape):
    if t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
        raise DigaError(f"{who}: {name} must be contiguous {dtype} {tuple(shape)}, got {t.dtype} {tuple(t.shape)} with strides {t.stride()}")


def _operand(who, name, t, rows, cols, ld, piece):
    """Row stride of a product's operand.  The kernels read rows in pieces of 16 bytes (`piece` elements): a row that ends inside one
    needs the rest of the piece to be there."""
    whole = cols if cols % piece == 0 else (cols // piece + 1) * piece
    if whole != cols and rows:
        end = t.storage_offset() + sum((n - 1) * s for n, s in zip(t.shape[:-1], t.stride())) + whole
        if end * t.element_size() > t.untyped_storage().nbytes():
            raise DigaError(f"{who}: rows of {name} end inside 16 bytes ({cols} columns) and its storage ends with the last one: allocate "
                            f"rows of {whole} columns and take [..., :{cols}]")
    return ld if rows > 1 else whole


def _check_out(who, out, m, n, dtype):
    if dtype not in _TYPES:
        raise DigaError(f"{who}: outputs are {', '.join(str(d) for d in _TYPES)}, not {dtype}")
    if out is not None and (out.dtype is not dtype or out.shape != (m, n) or (n > 1 and out.stride(1) != 1)):
        raise DigaError(f"{who}: out must be {dtype} ({m}, {n}) with adjacent columns, got {out.dtype} {tuple(out.shape)} with strides {out.stride()}")


def _empty_rows(m, n, device):
    """e4m3 [m, n] in rows that start at multiples of 16 bytes, its scales [m, blocks] with adjacent rows, and their row strides."""
    ldq = -(-n // 16) * 16
    q = _empty((m, ldq), dtype=E4M3, device=device)
    if ldq != n:
        q = q[:, :n]
    return q, ldq, _strided((m, -(-n // BLOCK)), (1, m), dtype=torch.float32, device=device)


def rms_norm_fp8(x, weight, residual=None, eps=1e-6, residual_out=None):
    """h = x (+ residual); h * rsqrt(mean(h^2) + eps) * weight in 8 bits.

    x [M, N] bf16 / fp16 / fp32; residual like x; weight [N] of any of these types.  -> (q e4m3 [M, N], scale fp32
    [M, ceil(N / 128)], h): h is the sum in x's type, written to residual_out where that is given (it may be x or residual), and
    None without a residual.  The norm is taken from the unrounded fp32 sum."""
    done = _calls.rms_norm(x, weight, residual, eps, residual_out)
    if done is not None:
        return done
    who = "rms_norm_fp8"
    m, n, ldx = _rows(who, "x", x, _TYPES)
    dtype = x.dtype
    if weight.dtype not in _TYPES:
        raise DigaError(f"{who}: weight is {weight.dtype}")
    _plain(who, "weight", weight, weight.dtype, (n,))
    if residual is not None:
        if residual.shape != x.shape or residual.dtype is not dtype:
            raise DigaError(f"{who}: residual {residual.dtype} {tuple(residual.shape)} is not like x {x.dtype} {tuple(x.shape)}")
        ldr = _rows(who, "residual", residual, _TYPES)[2]
        _check_out(who, residual_out, m, n, dtype)
        index = _device(who, x, weight, residual, residual_out)
        if residual_out is None:
            residual_out = torch.empty_like(residual)
        r, h, ldh = residual.data_ptr(), residual_out.data_ptr(), residual_out.stride(0)
    elif residual_out is not None:
        raise DigaError(f"{who}: residual_out without a residual")
    else:
        index = _device(who, x, weight)
        r, h, ldr, ldh = None, None, 0, 0
    q, ldq, s = _empty_rows(m, n, x.device)
    _rms_norm(index, x.data_ptr(), ldx, r, ldr, _TYPES[dtype], weight.data_ptr(), _TYPES[weight.dtype], eps, m, n, q.data_ptr(), ldq,
              s.data_ptr(), 1, m, h, ldh)
    if h is not None:
        _written(residual_out)
    return q, s, residual_out


def silu_mul_fp8(x):
    """silu(gate) * up in 8 bits, x [M, 2 N] = [gate | up] bf16 / fp16 / fp32 -> (q e4m3 [M, N], scale fp32 [M, ceil(N / 128)])."""
    done = _calls.silu_mul(x)
    if done is not None:
        return done
    who = "silu_mul_fp8"
    m, n, ldx = _rows(who, "x", x, _TYPES)
    if n % 2:
        raise DigaError(f"{who}: x has {n} columns, not a gate and an up half")
    n //= 2
    index = _device(who, x)
    q, ldq, s = _empty_rows(m, n, x.device)
    _silu_mul(index, x.data_ptr(), ldx, _TYPES[x.dtype], m, n, q.data_ptr(), ldq, s.data_ptr(), 1, m)
    return q, s


def quantize_fp8(x):
    """x [M, N] bf16 / fp16 / fp32 in 8 bits -> (q e4m3 [M, N], scale fp32 [M, ceil(N / 128)])."""
    done = _calls.quantize(x)
    if done is not None:
        return done
    who = "quantize_fp8"
    m, n, ldx = _rows(who, "x", x, _TYPES)
    index = _device(who, x)
    q, ldq, s = _empty_rows(m, n, x.device)
    _quantize(index, x.data_ptr(), ldx, _TYPES[x.dtype], m, n, q.data_ptr(), ldq, s.data_ptr(), 1, m)
    return q, s


def quantize_weight_fp8(w):
    """Weight matrices [..., N, K] of finite values in 8 bits -> (q e4m3 [..., N, K], scale fp32 [..., ceil(N/128), ceil(K/128)]), the
    scale being max(max|w|, 2^-100) / 448 of a 128 x 128 block.  One-off work at load time, on the weights' own device."""
    if w.dim() < 2 or not w.is_floating_point() or 0 in w.shape:
        raise DigaError(f"quantize_weight_fp8: expected weights [..., N, K], got {w.dtype} {tuple(w.shape)}")
    w = w.detach()
    n, k = w.shape[-2:]
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    p = torch.nn.functional.pad(w.float(), (0, kb * BLOCK - k, 0, nb * BLOCK - n)).view(*w.shape[:-2], nb, BLOCK, kb, BLOCK)
    s = p.abs().amax((-3, -1)).clamp_min(2.0 ** -100) / 448
    q = torch.zeros(*w.shape[:-1], -(-k // 16) * 16, dtype=E4M3, device=w.device)[..., :k]
    q.copy_((p / s[..., :, None, :, None]).reshape(*w.shape[:-2], nb * BLOCK, kb * BLOCK)[..., :n, :k])
    return q, s


def _check_scales(who, xs, ws, m, k, lead):
    kb = -(-k // BLOCK)
    if xs.dtype is not torch.float32 or xs.shape != (m, kb):
        raise DigaError(f"{who}: the rows' scales must be float32 ({m}, {kb}), got {xs.dtype} {tuple(xs.shape)}")
    _plain(who, "the weights' scales", ws, torch.float32, (*lead, kb))
    return xs.stride()


def _check_wide(who, out_dtype, x):
    if out_dtype is torch.float32 and not x.is_cuda:
        raise DigaError(f"{who}: float32 outputs are summed from 16-bit operands on the GPU: there is no CPU fallback")


def _fp8_entry(out_dtype, halves, f32):
    """The entry point for outputs of out_dtype, and its argument that says which."""
    return (f32, ()) if out_dtype is torch.float32 else (halves, (_HALVES[out_dtype],))


def matmul_fp8(xq, xs, wq, ws, out_dtype=torch.bfloat16, out=None):
    """x @ w.T of 8-bit rows and weights: xq e4m3 [M, K] with xs fp32 [M, ceil(K / 128)], wq e4m3 [N, K] with ws fp32
    [ceil(N / 128), ceil(K / 128)] -> [M, N] of out_dtype (bf16 / fp16 / fp32), fp32 sums over the blocks, rounded once.  Rows of xq and wq start
    at multiples of 16 bytes.  For fp32 the products are summed in 32 bits too, at half the matrix rate."""
    done = _calls.matmul(xq, xs, wq, ws, out_dtype, out)
    if done is not None:
        return done
    who = "matmul_fp8"
    m, k, ldx = _rows(who, "xq", xq, _E4M3)
    n, kw, ldw = _rows(who, "wq", wq, _E4M3)
    if k != kw or n == 0:
        raise DigaError(f"{who}: xq {tuple(xq.shape)} and wq {tuple(wq.shape)} do not fit")
    _counts(who, "rows of wq", n)
    sm, sb = _check_scales(who, xs, ws, m, k, (-(-n // BLOCK),))
    ldx, ldw = _operand(who, "xq", xq, m, k, ldx, 16), _operand(who, "wq", wq, n, k, ldw, 16)
    _check_out(who, out, m, n, out_dtype)
    _check_wide(who, out_dtype, xq)
    index = _device(who, xq, xs, wq, ws, out)
    given = out is not None
    if not given:
        out = _empty((m, n), dtype=out_dtype, device=xq.device)
    entry, kind = _fp8_entry(out_dtype, _matmul, _matmul_f32)
    entry(index, xq.data_ptr(), ldx, xs.data_ptr(), sm, sb, wq.data_ptr(), ldw, ws.data_ptr(), out.data_ptr(), *kind, out.stride(0), m, n, k)
    if given:
        _written(out)
    return out


def _groups(who, x, w, offsets, rows, dtypes, piece):
    xr, k, ldx = _rows(who, "x", x, dtypes)
    if w.dim() != 3 or w.dtype is not x.dtype or w.shape[2] != k or 0 in w.shape or (k > 1 and w.stride(2) != 1):
        raise DigaError(f"{who}: weights must be {x.dtype} (experts, N, {k}) with adjacent columns, got {w.dtype} {tuple(w.shape)} with strides {w.stride()}")
    e, n, _ = w.shape
    _counts(who, "weight rows", n)
    _counts(who, "weight matrices", e)
    _plain(who, "offsets", offsets, torch.int32, (e + 1,))
    t = xr
    if rows is not None:
        t = rows.numel()
        _plain(who, "rows", rows, torch.int32, (t,))
    we, ldw, _ = w.stride()
    return xr, k, e, n, t, we, _operand(who, "x", x, xr, k, ldx, piece), _operand(who, "the weights", w, n, k, ldw, piece)


def grouped_matmul_fp8(xq, xs, wq, ws, offsets, rows=None, out_dtype=torch.bfloat16, out=None):
    """matmul_fp8 with a weight matrix per expert: wq e4m3 [E, N, K], ws fp32 [E, ceil(N / 128), ceil(K / 128)].  Rows
    offsets[e] <= t < offsets[e + 1] (int32 [E + 1] on the GPU, E at most 4096) of the result [T, N] are expert e's; groups may be empty.  rows (int32 [T])
    gathers: row t takes row rows[t] of xq (at most 4 GiB), an index outside it a row of zeros; without it T = M.  Rows outside all
    groups are left as they are in `out`, and hold anything in a result allocated here."""
    done = _calls.grouped(xq, xs, wq, ws, offsets, rows, out_dtype, out)
    if done is not None:
        return done
    who = "grouped_matmul_fp8"
    xr, k, e, n, t, we, ldx, ldw = _groups(who, xq, wq, offsets, rows, _E4M3, 16)
    sm, sb = _check_scales(who, xs, ws, xr, k, (e, -(-n // BLOCK)))
    _check_out(who, out, t, n, out_dtype)
    _check_wide(who, out_dtype, xq)
    index = _device(who, xq, xs, wq, ws, offsets, rows, out)
    given = out is not None
    if not given:
        out = _empty((t, n), dtype=out_dtype, device=xq.device)
    entry, kind = _fp8_entry(out_dtype, _grouped_fp8, _grouped_fp8_f32)
    entry(index, xq.data_ptr(), ldx, xr, xs.data_ptr(), sm, sb, rows.data_ptr() if rows is not None else None, wq.data_ptr(), ldw,
          we, ws.data_ptr(), offsets.data_ptr(), e, out.data_ptr(), *kind, out.stride(0), t, n, k)
    if given:
        _written(out)
    return out


def grouped_matmul(x, w, offsets, rows=None, out_dtype=None, out=None):
    """The same on bf16 or fp16 rows x [M, K] and weights w [E, N, K], without scales -> [T, N] of out_dtype (x's type unless given)."""
    out_dtype = out_dtype or x.dtype
    done = _calls.grouped(x, None, w, None, offsets, rows, out_dtype, out)
    if done is not None:
        return done
    who = "grouped_matmul"
    xr, k, e, n, t, we, ldx, ldw = _groups(who, x, w, offsets, rows, _HALVES, 8)
    _check_out(who, out, t, n, out_dtype)
    index = _device(who, x, w, offsets, rows, out)
    given = out is not None
    if not given:
        out = _empty((t, n), dtype=out_dtype, device=x.device)
    _grouped(index, x.data_ptr(), ldx, xr, _HALVES[x.dtype], rows.data_ptr() if rows is not None else None, w.data_ptr(), ldw, we,
             offsets.data_ptr(), e, out.data_ptr(), _TYPES[out_dtype], out.stride(0), t, n, k)
    if given:
        _written(out)
    return out
