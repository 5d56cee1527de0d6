"""Products of grouped rows and 4-bit tables; reached through ``extension``.

No counterpart upstream.  They carry ``project`` (one matrix for all rows) and
``routing_cuda`` (each query against the leaves of its own router) on to matrices per group
with any number of rows, their gradients, and tables held in four bits a value.  Checks,
errors (``RuntimeError``) and streams follow :mod:`pilotann_b200.extension`.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _C

MAX_GROUPS = 1024
MAX_WIDTH = 65536

_DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_FLOATS = tuple(_DTYPE)
_INT64 = (torch.int64,)
_METHOD = {"mxfp4": 0, "nvfp4": 1}
_BLOCK = {"mxfp4": 32, "nvfp4": 16}


def _require(cond: bool, what: str) -> None:
    if not cond:
        raise RuntimeError(f"Expected {what} to be true, but got false.")


def _check(name: str, x, dim, dtypes) -> None:
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if x.dim() != dim:
        raise RuntimeError(f"{name} must be of dim {dim}")
    if x.dtype not in dtypes:
        raise RuntimeError(f"{name} must be type of {' or '.join(map(str, dtypes))}")


def _row_stride(name: str, x: torch.Tensor) -> int:
    """Elements from row to row: rows may be part of wider ones, their values are contiguous."""
    if x.is_contiguous():
        return x.size(1)
    if x.stride(1) != 1 or x.stride(0) < x.size(1):
        raise RuntimeError(f"{name} custom kernel requires contiguous rows")
    return x.stride(0)


def _contiguous(name: str, x: torch.Tensor) -> None:
    if not x.is_contiguous():
        raise RuntimeError(f"{name} custom kernel requires contiguous tensor")


def _same_device(a: torch.Tensor, name: str, x: torch.Tensor) -> None:
    if x.device != a.device:
        raise RuntimeError(f"{name} must be on {a.device}, got {x.device}")


# The calls of a small batch are as long as their Python side: the raw handle instead of a Stream
# object saves 2 us of 10, checks that stop at the first look at sound arguments 2 to 3.
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice
_empty = torch.empty


def _call(device: torch.device, fn, *args) -> None:
    """``fn(*args, stream)`` on the tensors' device and its current stream."""
    index = device.index
    if _current_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _raw_stream(index))
    if rc:
        _C.check(rc)


# ---- rows by group -----------------------------------------------------------------
def group_rows(router: torch.Tensor, n_groups: int):
    """Rows in the order of the group each was sent to (``routing_cuda``'s first result):
    ``(order int64 [B], offsets int64 [n_groups + 1])``.  ``order[offsets[g]:offsets[g + 1]]``
    are the rows of group ``g``, ascending.  Rows whose id is not in ``[0, n_groups)`` come
    last, behind ``offsets[n_groups]``.  ``x[order]`` is what :func:`project_grouped` takes;
    ``y.new_empty(y.shape).index_copy_(0, order, y)`` brings its result back."""
    _check("router", router, 1, _INT64)
    _contiguous("router", router)
    if not 1 <= n_groups <= MAX_GROUPS:
        _require(False, f"1 <= n_groups <= {MAX_GROUPS}")
    rows, dev = router.size(0), router.device
    order = torch.empty_like(router)
    offsets = _empty(n_groups + 1, dtype=torch.int64, device=dev)
    L = _C.lib()
    need = L.pa_group_rows_workspace_bytes(rows, n_groups)
    ws = _empty(need, dtype=torch.uint8, device=dev) if need else None
    _call(dev, L.pa_group_rows, order.data_ptr(), offsets.data_ptr(), router.data_ptr(), rows,
          n_groups, 0 if ws is None else ws.data_ptr())
    return order, offsets


# ---- a matrix per group --------------------------------------------------------------
def _grouped_checks(query, VT, offsets) -> None:
    try:
        if (query.is_cuda and VT.is_cuda and offsets.is_cuda and query.dtype in _DTYPE
                and VT.dtype is query.dtype and offsets.dtype is torch.int64
                and query.device == VT.device == offsets.device
                and VT.is_contiguous() and offsets.is_contiguous()):
            n_groups, d_out, d = VT.shape
            if (query.size(1) == d and query.dim() == 2 and offsets.shape == (n_groups + 1,)
                    and 1 <= n_groups <= MAX_GROUPS and 1 <= d_out <= MAX_WIDTH
                    and 1 <= d <= MAX_WIDTH):
                return
    except (AttributeError, IndexError, ValueError):
        pass
    _check("query", query, 2, _FLOATS)
    _check("VT", VT, 3, (query.dtype,))
    _check("offsets", offsets, 1, _INT64)
    _contiguous("VT", VT)
    _contiguous("offsets", offsets)
    _same_device(query, "VT", VT)
    _same_device(query, "offsets", offsets)
    _require(VT.size(2) == query.size(1), "VT.size(2) == query.size(1)")
    _require(1 <= VT.size(0) <= MAX_GROUPS, f"1 <= VT.size(0) <= {MAX_GROUPS}")
    _require(offsets.size(0) == VT.size(0) + 1, "offsets.size(0) == VT.size(0) + 1")
    _require(1 <= VT.size(1) <= MAX_WIDTH and 1 <= VT.size(2) <= MAX_WIDTH,
             f"1 <= d, d_out <= {MAX_WIDTH}")


def _grouped_forward(query, VT, offsets):
    rows, d = query.shape
    n_groups, d_out, _ = VT.shape
    dev, dtype = query.device, _DTYPE[query.dtype]
    L = _C.lib()
    q, w, ld = query.data_ptr(), VT.data_ptr(), _row_stride("query", query)
    need = 0 if dtype == 0 or ((q | w) % 16 == 0 and (d | ld) % 8 == 0) else \
        L.pa_project_grouped_workspace_bytes(q, w, rows, n_groups, d, d_out, ld, dtype)
    ws = _empty(need, dtype=torch.uint8, device=dev) if need else None
    out = _empty(rows, d_out, dtype=query.dtype, device=dev)
    _call(dev, L.pa_project_grouped, out.data_ptr(), q, w, offsets.data_ptr(), rows, n_groups, d,
          d_out, ld, d_out, dtype, 0 if ws is None else ws.data_ptr())
    return out


def _grouped_backward(grad, query, VT, offsets, want_query, want_VT):
    rows, d = query.shape
    n_groups, d_out, _ = VT.shape
    dev, dtype = query.device, _DTYPE[query.dtype]
    L = _C.lib()
    y, q, w = grad.data_ptr(), query.data_ptr(), VT.data_ptr()
    ldy, ldq = _row_stride("grad", grad), _row_stride("query", query)
    need = 0 if dtype == 0 or ((y | q | w) % 16 == 0 and (d | ldy | ldq) % 8 == 0) else \
        L.pa_project_grouped_backward_workspace_bytes(y, q, w, rows, n_groups, d, d_out, ldy, ldq,
                                                      dtype, want_query, want_VT)
    ws = _empty(need, dtype=torch.uint8, device=dev) if need else None
    dq = _empty(rows, d, dtype=query.dtype, device=dev) if want_query else None
    dw = torch.empty_like(VT) if want_VT else None
    _call(dev, L.pa_project_grouped_backward, 0 if dq is None else dq.data_ptr(),
          0 if dw is None else dw.data_ptr(), y, q, w, offsets.data_ptr(), rows, n_groups, d, d_out,
          ldy, ldq, d, dtype, 0 if ws is None else ws.data_ptr())
    return dq, dw


def _no_tangent(name: str, *tensors) -> None:
    """Inside a ``forward_ad.dual_level``: a tangent would be dropped without a word."""
    if forward_ad._current_level < 0:
        return
    for x in tensors:
        if isinstance(x, torch.Tensor) and forward_ad.unpack_dual(x).tangent is not None:
            raise RuntimeError(f"{name} has no forward-mode derivative")


class _ProjectGrouped(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, VT, offsets):
        ctx.save_for_backward(query, VT, offsets)
        return _grouped_forward(query, VT, offsets)

    @staticmethod
    def backward(ctx, grad):
        if torch.is_grad_enabled():       # create_graph: the gradients have none themselves
            raise RuntimeError("project_grouped can be differentiated only once")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("project_grouped is not differentiated in a stream capture: call "
                               "project_grouped_backward")
        query, VT, offsets = ctx.saved_tensors
        if not grad.is_contiguous() and (grad.stride(1) != 1 or grad.stride(0) < grad.size(1)):
            grad = grad.contiguous()      # an expanded gradient, as of a sum
        dq, dw = _grouped_backward(grad, query, VT, offsets, *ctx.needs_input_grad[:2])
        return dq, dw, None


def project_grouped(query: torch.Tensor, VT: torch.Tensor, offsets: torch.Tensor):
    """Every row times the matrix of its group: ``out[i] = query[i] @ VT[g].T`` for
    ``offsets[g] <= i < offsets[g + 1]``; ``query`` is ``[rows, d]`` (rows of a wider tensor
    will do), ``VT`` ``[n_groups, d_out, d]``, ``offsets`` int64 ``[n_groups + 1]`` ascending
    within ``[0, rows]`` (:func:`group_rows` makes them).  float32, bfloat16 or float16, sums
    in float32, result rounded once to the type of ``query``.  Groups may be empty; rows that
    belong to no group give zeros and get no gradient.  ``offsets`` stay on the device and are
    read there: values that do not ascend give unspecified rows, never an access outside the
    tensors.

    Differentiable in ``query`` and ``VT``, once and in reverse mode (a forward-mode tangent is
    refused); not while the stream is being captured into a CUDA
    graph: autograd runs a leaf's accumulation on the stream of the oldest live graph of that
    leaf, and where that is an eager one the capture breaks, or the process.  In a capture
    call this under ``torch.no_grad()`` and :func:`project_grouped_backward` for the
    gradients."""
    _grouped_checks(query, VT, offsets)
    _row_stride("query", query)
    _no_tangent("project_grouped", query, VT)
    if torch.is_grad_enabled() and (query.requires_grad or VT.requires_grad):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("project_grouped records no gradient in a stream capture: call it "
                               "under torch.no_grad(), and project_grouped_backward")
        return _ProjectGrouped.apply(query, VT, offsets)
    return _grouped_forward(query, VT, offsets)


def project_grouped_backward(grad: torch.Tensor, query: torch.Tensor, VT: torch.Tensor,
                             offsets: torch.Tensor, want_query: bool = True,
                             want_VT: bool = True):
    """Gradients of :func:`project_grouped`: ``(grad_query [rows, d], grad_VT [n_groups,
    d_out, d])``, ``None`` for one that is not wanted.  ``grad_query[i] = grad[i] @ VT[g]``,
    ``grad_VT[g] = grad[g's rows].T @ query[g's rows]`` (zeros for a group without rows).  They
    have no gradient themselves."""
    _grouped_checks(query, VT, offsets)
    _no_tangent("project_grouped_backward", grad, query, VT)
    _check("grad", grad, 2, (query.dtype,))
    _same_device(query, "grad", grad)
    _require(tuple(grad.shape) == (query.size(0), VT.size(1)), "grad.shape == (rows, d_out)")
    return _grouped_backward(grad, query, VT, offsets, want_query, want_VT)


# ---- 4-bit tables -----------------------------------------------------------------------
class Fp4Table:
    """Vectors held in four bits a value: what :func:`quantize_fp4` returns.

    ``codes`` uint8 ``[..., P / 2]`` with ``P`` = ``d`` rounded up to a multiple of 32: E2M1,
    two a byte, the even value in the low half, zero codes behind ``d``; ``scales`` uint8
    ``[..., P / 32]`` (``mxfp4``: E8M0) or ``[..., P / 16]`` (``nvfp4``: E4M3); ``row_scale``
    float32 ``[...]`` for ``nvfp4``, else ``None``.  ``...`` is ``[rows]``, or ``[n_groups,
    d_out]`` for a table per group.  The parts are plain tensors: save and load them as such."""

    __slots__ = ("codes", "scales", "row_scale", "d", "method")

    def __init__(self, codes, scales, row_scale, d: int, method: str):
        if method not in _METHOD:
            raise RuntimeError(f"unknown 4-bit method {method!r}: mxfp4 or nvfp4")
        _require(1 <= d <= MAX_WIDTH, f"1 <= d <= {MAX_WIDTH}")
        dim = codes.dim() if isinstance(codes, torch.Tensor) else 2
        _require(dim in (2, 3), "codes.dim() in (2, 3)")
        _check("codes", codes, dim, (torch.uint8,))
        _check("scales", scales, dim, (torch.uint8,))
        _contiguous("codes", codes)
        _contiguous("scales", scales)
        padded = -(-d // 32) * 32
        _require(codes.size(-1) == padded // 2, "codes.size(-1) == d padded to 32 / 2")
        _require(tuple(scales.shape) == (*codes.shape[:-1], padded // _BLOCK[method]),
                 "scales.shape == (*codes.shape[:-1], d padded to 32 / block)")
        _require((row_scale is not None) == (method == "nvfp4"), "row_scale given for nvfp4 only")
        if row_scale is not None:
            _check("row_scale", row_scale, dim - 1, (torch.float32,))
            _contiguous("row_scale", row_scale)
            _require(row_scale.shape == codes.shape[:-1], "row_scale.shape == codes.shape[:-1]")
            _same_device(codes, "row_scale", row_scale)
        _same_device(codes, "scales", scales)
        _require(codes.data_ptr() % 16 == 0, "codes 16-byte aligned")
        self.codes, self.scales, self.row_scale = codes, scales, row_scale
        self.d, self.method = d, method

    @property
    def shape(self):
        return torch.Size((*self.codes.shape[:-1], self.d))

    @property
    def device(self):
        return self.codes.device

    def nbytes(self) -> int:
        return sum(x.numel() * x.element_size() for x in
                   (self.codes, self.scales, self.row_scale) if x is not None)


def quantize_fp4(x: torch.Tensor, method: str = "mxfp4") -> Fp4Table:
    """``x`` (``[rows, d]``, rows of a wider tensor will do, or contiguous ``[n_groups, d_out,
    d]``; float32, bfloat16 or float16) in four bits a value.

    ``mxfp4``: blocks of 32 values, scale ``2 ** (floor(log2 max|v|) - 2)``; ``nvfp4``: blocks
    of 16, scale ``max|v| / (6 s)`` in E4M3 times the row's power of two ``s``, the least with
    ``max|v| <= 6 * 448 s``.  Values go to the nearest code, ties to the even one, above 6 to
    6.  A block (``mxfp4``) or row (``nvfp4``) with NaN or infinity becomes NaN as a whole.  Equal
    values give equal codes whatever their type.  Codes have no gradient, whether or not ``x`` wants one."""
    if method not in _METHOD:
        raise RuntimeError(f"unknown 4-bit method {method!r}: mxfp4 or nvfp4")
    dim = x.dim() if isinstance(x, torch.Tensor) else 2
    if dim not in (2, 3):
        _require(False, "x.dim() in (2, 3)")
    _check("x", x, dim, _FLOATS)
    d, dev = x.size(-1), x.device
    if not 1 <= d <= MAX_WIDTH:
        _require(False, f"1 <= d <= {MAX_WIDTH}")
    width, blocks = (d + 31) // 32 * 16, (d + 31) // 32 * (32 // _BLOCK[method])
    row_scale = None
    if dim == 2:
        rows, ld = x.size(0), _row_stride("x", x)
        codes = _empty(rows, width, dtype=torch.uint8, device=dev)
        scales = _empty(rows, blocks, dtype=torch.uint8, device=dev)
    else:
        _contiguous("x", x)
        rows, ld = x.size(0) * x.size(1), d
        codes = _empty(x.size(0), x.size(1), width, dtype=torch.uint8, device=dev)
        scales = _empty(x.size(0), x.size(1), blocks, dtype=torch.uint8, device=dev)
    if method == "nvfp4":
        row_scale = _empty(x.shape[:-1], dtype=torch.float32, device=dev)
    _call(dev, _C.lib().pa_quantize_fp4, codes.data_ptr(), scales.data_ptr(),
          0 if row_scale is None else row_scale.data_ptr(), x.data_ptr(), rows, d, ld,
          _DTYPE[x.dtype], _METHOD[method])
    table = Fp4Table.__new__(Fp4Table)       # parts made here need no checks
    table.codes, table.scales, table.row_scale = codes, scales, row_scale
    table.d, table.method = d, method
    return table


def dequantize_fp4(table: Fp4Table) -> torch.Tensor:
    """What the codes stand for, float32 of ``table.shape``."""
    if not isinstance(table, Fp4Table):
        raise RuntimeError("table must be an Fp4Table")
    codes, row_scale, dev = table.codes, table.row_scale, table.codes.device
    shape = codes.shape
    if len(shape) == 2:
        rows = shape[0]
        out = _empty(rows, table.d, dtype=torch.float32, device=dev)
    else:
        rows = shape[0] * shape[1]
        out = _empty(shape[0], shape[1], table.d, dtype=torch.float32, device=dev)
    _call(dev, _C.lib().pa_dequantize_fp4, out.data_ptr(), codes.data_ptr(),
          table.scales.data_ptr(), 0 if row_scale is None else row_scale.data_ptr(), rows,
          table.d, _METHOD[table.method])
    return out


def project_fp4(query, table: Fp4Table, offsets: torch.Tensor | None = None,
                dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Scores of queries against a 4-bit table: ``out[i, n] = sum_k q[i, k] t[n, k]``, ``q``
    being the query quantised by the table's method in the same call (or an :class:`Fp4Table`
    of rows), sums in float32, result rounded once to ``dtype``.  With ``offsets`` the table is
    ``[n_groups, d_out, d]`` and every row meets the table of its group, as in
    :func:`project_grouped`; rows of no group give zeros.  The scores have no gradient, whether or
    not ``query`` wants one."""
    if not isinstance(table, Fp4Table):
        raise RuntimeError("table must be an Fp4Table")
    if dtype not in _DTYPE:
        raise RuntimeError(f"dtype must be one of {' or '.join(map(str, _DTYPE))}")
    codes, d, method = table.codes, table.d, table.method
    dev = codes.device
    if offsets is None:
        _require(codes.dim() == 2, "table of [rows, d] without offsets")
        n_groups, d_out = 1, codes.size(0)
    else:
        _require(codes.dim() == 3, "table of [n_groups, d_out, d] with offsets")
        _check("offsets", offsets, 1, _INT64)
        _contiguous("offsets", offsets)
        _same_device(codes, "offsets", offsets)
        n_groups, d_out = codes.size(0), codes.size(1)
        _require(1 <= n_groups <= MAX_GROUPS, f"1 <= n_groups <= {MAX_GROUPS}")
        _require(offsets.size(0) == n_groups + 1, "offsets.size(0) == n_groups + 1")
    L = _C.lib()
    padded = -(-d // 32) * 32
    if isinstance(query, Fp4Table):
        _require(query.codes.dim() == 2, "query of [rows, d]")
        _require(query.method == method, "query.method == table.method")
        _require(query.d == d, "query.size(1) == table.d")
        _same_device(codes, "query", query.codes)
        rows = query.codes.size(0)
        q = (query.codes.data_ptr(), query.scales.data_ptr(),
             0 if query.row_scale is None else query.row_scale.data_ptr())
    else:
        _check("query", query, 2, _FLOATS)
        if query.size(1) != d:
            _require(False, "query.size(1) == table.d")
        _same_device(codes, "query", query)
        rows = query.size(0)
        ld = _row_stride("query", query)
        # scratch: codes, row scales, block scales of the quantised queries
        width = padded // 2 + 4 + padded // _BLOCK[method]
        ws = _empty(rows * width, dtype=torch.uint8, device=dev)
        at = ws.data_ptr()
        q = (at, at + rows * (padded // 2 + 4), at + rows * (padded // 2))
        _call(dev, L.pa_quantize_fp4, q[0], q[1], q[2] if method == "nvfp4" else 0,
              query.data_ptr(), rows, d, ld, _DTYPE[query.dtype], _METHOD[method])
    out = _empty(rows, d_out, dtype=dtype, device=dev)
    _call(dev, L.pa_project_fp4, out.data_ptr(), *q, codes.data_ptr(), table.scales.data_ptr(),
          0 if table.row_scale is None else table.row_scale.data_ptr(),
          0 if offsets is None else offsets.data_ptr(), rows, n_groups, d, d_out, _DTYPE[dtype],
          _METHOD[method])
    return out
