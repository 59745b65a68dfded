"""Operators of a dense block on the device: 8-bit linear layers, group norm with an activation, dropout.

Functions on device tensors like onto_vae_amd.stats: the arithmetic is in libontovae_hip.so (ontovae_quantize_rows,
ontovae_int8_matmul, ontovae_group_norm_act, ontovae_dropout of include/ontovae_hip.h), torch allocates the buffers, there is no CPU
path.  Forward and backward are explicit calls, no autograd graph is recorded (group_norm_act, dropout and int8_linear warn where an x that
requires grad comes in with grad mode on: the graph ends there; inside a torch.autograd.Function, under torch.no_grad() or on
x.detach() they do not).  Tensors are float32, bfloat16 or float16, channels
last ([..., C]); every sum and statistic is held in 32 bits and each output is rounded once.  Work is queued on the
current stream of the tensors' device, which need not be the current device.

The reference has no counterpart: its blocks are torch's Linear, BatchNorm1d, Dropout and ReLU (onto_vae/modules.py:43-64, 116-133).
The models use these operators through set_precision('int8') and VAE(norm='group', input_drop=...).
"""
import contextlib
import math
import warnings

import torch

from . import _lib
from .stats import _need_gpu

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}
I32_MAX = 2 ** 31 - 1


_SAME = contextlib.nullcontext()


def _gpu(t, what):
    if not t.is_cuda:
        _need_gpu(t, what)


def _no_graph(x, what):
    if x.requires_grad and torch.is_grad_enabled():
        warnings.warn(f"{what} records no autograd graph: its result does not require grad though x does", stacklevel=3)


def _on(device):
    """The tensors' device as the current one (entering torch's guard only when it changes something)."""
    return _SAME if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _p(t):
    return None if t is None else t.data_ptr()


def _stream(device):
    return torch._C._cuda_getCurrentRawStream(device.index)


def _workspace(nbytes, device):
    """(buffer, address, bytes): torch's device allocations are 512-byte aligned, the library asks for 256."""
    if nbytes <= 0:
        return None, None, 0
    buf = torch.empty(nbytes, dtype=torch.uint8, device=device)
    return buf, buf.data_ptr(), nbytes


def _dtype(t, what):
    if t.dtype not in DTYPES:
        raise ValueError(f"{what}: float32, bfloat16 or float16 expected, got {t.dtype}")
    return DTYPES[t.dtype]


def _matrix(x, what):
    """[..., C] as a 2-D view with unit inner stride (copied only when its strides leave no other way)."""
    if x.dim() < 1:
        raise ValueError(f"{what}: at least one dimension expected")
    m = x if x.dim() == 2 else x.reshape(math.prod(x.shape[:-1]), x.shape[-1])
    R, Cn = m.shape
    if R > I32_MAX or Cn > I32_MAX:
        raise ValueError(f"{what}: a dimension of {tuple(m.shape)} exceeds {I32_MAX}")
    ld, inner = m.stride()
    if inner != 1 and Cn > 1 or ld < Cn and R > 1:
        m = m.contiguous()
        ld = Cn
    return m, max(ld, Cn)


def _rows(rows, x, what):
    if rows is None:
        return None
    if rows.dim() != 1 or rows.dtype not in (torch.int32, torch.int64) or rows.device != x.device:
        raise ValueError(f"{what}: rows must be an int32 or int64 vector on {x.device}")
    if x.dim() != 2:
        raise ValueError(f"{what}: rows select from a 2-D matrix")
    if rows.dtype == torch.int64:          # an index outside int32 stays outside the matrix
        rows = rows.clamp(-1, I32_MAX)
    return rows.to(torch.int32).contiguous()


def _vector(t, n, device, what, dtypes=(torch.float32,)):
    if t is None:
        return None
    if t.dim() != 1 or t.shape[0] != n or t.dtype not in dtypes or t.device != device:
        raise ValueError(f"{what} must be {' / '.join(str(d).split('.')[-1] for d in dtypes)} [{n}] on {device}")
    return t.contiguous()


def _u64(v, what):
    v = int(v)
    if not 0 <= v < 2 ** 64:
        raise ValueError(f"{what} must be in [0, 2^64)")
    return v


# ---------------------------------------------------------------- 8-bit linear layers
def quantize_rows(x, rows=None):
    """(q, scale): the rows of a [..., K] tensor (of the rows x[rows] of a matrix) in 8 bits, scale = max|row| * (1 / 127) in float32 and
    q = x / scale rounded to the nearest integer, ties to even.  q has shape [..., K] and a row stride padded with zeros to a
    multiple of 64, the layout int8_matmul reads fastest.  A row that holds an infinity or a NaN (or a row index outside x) gets
    the scale NaN."""
    _gpu(x, "quantize_rows")
    dt = _dtype(x, "quantize_rows")
    rows = _rows(rows, x, "quantize_rows")
    xm, ld = _matrix(x, "quantize_rows")
    K = xm.shape[1]
    M = xm.shape[0] if rows is None else rows.shape[0]
    lead = tuple(x.shape[:-1]) if rows is None else (M,)
    ldq = max((K + 63) // 64 * 64, 64)
    if ldq % 1024 == 0:          # rows a multiple of 1024 bytes apart meet in the same memory channels
        ldq += 128
    with _on(x.device):
        q = torch.empty(M, ldq, dtype=torch.int8, device=x.device)
        scale = torch.empty(M, dtype=torch.float32, device=x.device)
        _lib.check(_lib.lib().ontovae_quantize_rows(_p(xm), dt, ld, _p(rows), xm.shape[0], M, K, _p(q), ldq, _p(scale), _stream(x.device)),
                   "quantize_rows")
    qk = q[:, :K]
    return (qk if len(lead) == 1 else qk.view(*lead, K) if M else q.new_empty(*lead, K)), scale.view(lead)


def int8_matmul(a, a_scale, b, b_scale, bias=None, dtype=torch.float32):
    """y [..., N] = (a [..., K] . b [N, K]^T) a_scale[..., None] b_scale + bias: int8 operands with one float32 scale per row of each
    (quantize_rows), the sum over K (at most 131071) exact, bias float32 [N], y rounded once to `dtype`."""
    _gpu(a, "int8_matmul")
    if a.dtype != torch.int8 or b.dtype != torch.int8 or b.dim() != 2 or a.dim() < 1 or a.shape[-1] != b.shape[1] or a.device != b.device:
        raise ValueError("int8_matmul: int8 a [..., K] and b [N, K] on one device expected")
    if dtype not in DTYPES:
        raise ValueError(f"int8_matmul: dtype must be float32, bfloat16 or float16, got {dtype}")
    am, lda = _matrix(a, "int8_matmul")
    bm, ldb = _matrix(b, "int8_matmul")
    M, K, N = am.shape[0], am.shape[1], bm.shape[0]
    lead = tuple(a.shape[:-1])
    if tuple(a_scale.shape) != lead:
        raise ValueError(f"int8_matmul: a_scale must have shape {lead}, got {tuple(a_scale.shape)}")
    sa = _vector(a_scale.reshape(-1), M, a.device, "int8_matmul: a_scale")
    sb = _vector(b_scale, N, a.device, "int8_matmul: b_scale")
    bias = _vector(bias, N, a.device, "int8_matmul: bias")
    L = _lib.lib()
    with _on(a.device):
        y = torch.empty(*lead, N, dtype=dtype, device=a.device)
        keep, ws, nbytes = _workspace(L.ontovae_int8_matmul_workspace_bytes(M, N, K), a.device)
        _lib.check(L.ontovae_int8_matmul(_p(am), lda, _p(sa), _p(bm), ldb, _p(sb), _p(bias), M, N, K, _p(y), DTYPES[dtype], N,
                                         ws, nbytes, _stream(a.device)), "int8_matmul")
    return y


def int8_linear(x, weight, weight_scale, bias=None, rows=None, dtype=None):
    """x weight^T + bias with an 8-bit weight [N, K] (quantize_rows of the layer's float weight, done once) and the rows of x (of
    x[rows]) quantised on the way: one scale per token and per output channel.  dtype: that of y, x's by default."""
    _gpu(x, "int8_linear")
    _no_graph(x, "int8_linear")
    dt = _dtype(x, "int8_linear")
    if dtype is None:
        dtype = x.dtype
    elif dtype not in DTYPES:
        raise ValueError(f"int8_linear: dtype must be float32, bfloat16 or float16, got {dtype}")
    rows = _rows(rows, x, "int8_linear")
    if weight.dtype != torch.int8 or weight.dim() != 2 or weight.device != x.device or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError("int8_linear: x [..., K] and int8 weight [N, K] on one device expected")
    xm, ld = _matrix(x, "int8_linear")
    wm, ldw = _matrix(weight, "int8_linear")
    K, N = xm.shape[1], wm.shape[0]
    M = xm.shape[0] if rows is None else rows.shape[0]
    sw = _vector(weight_scale, N, x.device, "int8_linear: weight_scale")
    bias = _vector(bias, N, x.device, "int8_linear: bias")
    L = _lib.lib()
    with _on(x.device):
        y = torch.empty((*x.shape[:-1], N) if rows is None else (M, N), dtype=dtype, device=x.device)
        keep, ws, nbytes = _workspace(L.ontovae_int8_linear_workspace_bytes(M, N, K), x.device)
        _lib.check(L.ontovae_int8_linear(_p(xm), dt, ld, _p(rows), xm.shape[0], _p(wm), ldw, _p(sw), _p(bias), M, N, K, _p(y), DTYPES[dtype], N,
                                         ws, nbytes, _stream(x.device)), "int8_linear")
    return y


# ---------------------------------------------------------------- group norm with an activation
def _gn_args(x, groups, weight, bias, act, drop, seed, offset, what):
    _gpu(x, what)
    dt = _dtype(x, what)
    shape = x.shape
    if len(shape) < 2:
        raise ValueError(f"{what}: x must be [N, ..., C], channels last")
    N, S, Cn = shape[0], math.prod(shape[1:-1]) if len(shape) > 2 else 1, shape[-1]
    if max(N, S, Cn) > I32_MAX:
        raise ValueError(f"{what}: a dimension of {tuple(shape)} exceeds {I32_MAX}")
    groups, drop = int(groups), float(drop)
    if groups < 1 or Cn % groups or Cn < groups:
        raise ValueError(f"{what}: {groups} groups do not divide {Cn} channels")
    if act not in ACTIVATIONS:
        raise ValueError(f"{what}: act must be one of {sorted(ACTIVATIONS)}, got {act!r}")
    if not 0.0 <= drop <= 1.0:
        raise ValueError(f"{what}: drop = {drop} outside [0, 1]")
    wdt = 0
    if weight is not None or bias is not None:
        both = (torch.float32, x.dtype)
        weight, bias = _vector(weight, Cn, x.device, f"{what}: weight", both), _vector(bias, Cn, x.device, f"{what}: bias", both)
        if weight is not None and bias is not None and weight.dtype != bias.dtype:
            raise ValueError(f"{what}: weight and bias must share one type")
        wdt = DTYPES[(bias if weight is None else weight).dtype]
    return dt, N, S, Cn, groups, weight, bias, wdt, ACTIVATIONS[act], drop, _u64(seed, f"{what}: seed"), _u64(offset, f"{what}: offset")


def group_norm_act(x, groups, weight=None, bias=None, eps=1e-5, act="none", drop=0.0, seed=0, offset=0):
    """(y, mean, rstd): group norm of x [N, ..., C] over each sample's C / groups neighbouring channels and all inner positions,
    then weight and bias ([C], float32 or x's type), then the activation ('none', 'relu', 'silu', 'gelu'), then dropout with
    probability `drop` (masked as `dropout` masks y: same seed and offset, same mask).  mean, rstd: float32 [N, groups], for
    group_norm_act_backward."""
    dt, N, S, Cn, groups, weight, bias, wdt, a, drop, seed, offset = _gn_args(x, groups, weight, bias, act, drop, seed, offset, "group_norm_act")
    _no_graph(x, "group_norm_act")
    if not float(eps) >= 0.0:
        raise ValueError(f"group_norm_act: eps = {eps}")
    x = x.contiguous()
    L = _lib.lib()
    with _on(x.device):
        y = torch.empty_like(x)
        mean, rstd = torch.empty(2, N, groups, dtype=torch.float32, device=x.device).unbind()
        if N == 0 or S == 0:          # no rows to take statistics of
            return y, mean.zero_(), rstd.zero_()
        keep, ws, nbytes = _workspace(L.ontovae_group_norm_act_workspace_bytes(dt, N, S, Cn, groups, 0), x.device)
        _lib.check(L.ontovae_group_norm_act(_p(x), dt, N, S, Cn, groups, _p(weight), _p(bias), wdt, float(eps), a, drop, seed,
                                            offset, _p(y), _p(mean), _p(rstd), ws, nbytes, _stream(x.device)), "group_norm_act")
    return y, mean, rstd


def group_norm_act_backward(dy, x, mean, rstd, groups, weight=None, bias=None, act="none", drop=0.0, seed=0, offset=0, eps=None):
    """(dx, dweight, dbias) of group_norm_act with the mean and rstd it returned and the same further arguments.  dweight and dbias
    are float32 sums, None where the parameter is None; eps is part of rstd and accepted so that the arguments can be passed on."""
    dt, N, S, Cn, groups, weight, bias, wdt, a, drop, seed, offset = _gn_args(x, groups, weight, bias, act, drop, seed, offset,
                                                                              "group_norm_act_backward")
    if dy.shape != x.shape or dy.dtype != x.dtype or dy.device != x.device:
        raise ValueError("group_norm_act_backward: dy must match x in shape, type and device")
    for t, n in ((mean, "mean"), (rstd, "rstd")):
        if t.shape != (N, groups) or t.dtype != torch.float32 or t.device != x.device:
            raise ValueError(f"group_norm_act_backward: {n} must be float32 [{N}, {groups}] on {x.device}")
    dy, x, mean, rstd = dy.contiguous(), x.contiguous(), mean.contiguous(), rstd.contiguous()
    L = _lib.lib()
    with _on(x.device):
        dx = torch.empty_like(x)
        dw, db = torch.empty(2, Cn, dtype=torch.float32, device=x.device).unbind()
        dw, db = dw if weight is not None else None, db if bias is not None else None
        if N == 0 or S == 0:
            return dx, dw.zero_() if dw is not None else None, db.zero_() if db is not None else None
        keep, ws, nbytes = _workspace(L.ontovae_group_norm_act_workspace_bytes(dt, N, S, Cn, groups, 1), x.device)
        _lib.check(L.ontovae_group_norm_act_backward(_p(dy), _p(x), dt, N, S, Cn, groups, _p(weight), _p(bias), wdt, _p(mean),
                                                     _p(rstd), a, drop, seed, offset, _p(dx), _p(dw), _p(db), ws, nbytes,
                                                     _stream(x.device)), "group_norm_act_backward")
    return dx, dw, db


# ---------------------------------------------------------------- dropout
def dropout(x, p, seed, offset=0, rows=None):
    """Inverted dropout of a [..., C] tensor (of the rows x[rows] of a matrix): each element is 0 with probability p, else divided
    by 1 - p.  The mask is a function of (seed, offset, row, channel) alone -- Philox4x32-10, 16 bits an element, so p is taken to
    the nearest 2^-16 -- and is never stored; use another offset for each draw.  A non-finite element in a dropped place gives 0."""
    _gpu(x, "dropout")
    _no_graph(x, "dropout")
    dt = _dtype(x, "dropout")
    if not 0.0 <= float(p) <= 1.0:
        raise ValueError(f"dropout: p = {p} outside [0, 1]")
    seed, offset = _u64(seed, "dropout: seed"), _u64(offset, "dropout: offset")
    rows = _rows(rows, x, "dropout")
    xm, ld = _matrix(x, "dropout")
    R = xm.shape[0] if rows is None else rows.shape[0]
    with _on(x.device):
        y = torch.empty(x.shape if rows is None else (R, xm.shape[1]), dtype=x.dtype, device=x.device)
        _lib.check(_lib.lib().ontovae_dropout(_p(xm), dt, ld, _p(rows), xm.shape[0], R, xm.shape[1], float(p), seed, offset, _p(y),
                                              _stream(x.device)), "dropout")
    return y


def dropout_backward(dy, p, seed, offset=0):
    """The gradient of dropout(x, p, seed, offset) with respect to x (of x[rows] where rows were given): the same mask and factor on dy."""
    return dropout(dy, p, seed, offset)
