"""The learned head in front of the search: operators that train the rows `DeviceIndex` serves, and serve them in 8 bits.

  rms_norm / rms_norm_grads          a tower's last norm, with the residual's addition, and its gradients
  catalogue_cross_entropy(_grads)    softmax cross entropy of query rows over ALL item rows, with gradients, logits never stored
  rms_norm_q8 / quantize_rows_q8     rows as int8 codes with one scale each (queries on their way out of the tower; the catalogue)
  matmul_q8                          scores (or a layer) from two sets of 8-bit rows

Everything takes and returns device tensors on their own device, runs on its current stream, never synchronises and may be captured into a
hipGraph.  `rms_norm` and `catalogue_cross_entropy` take part in autograd where an input requires a gradient; the `_grads` functions return
the gradients directly and keep nothing (what a resident training step calls, and the simple form to capture: torch's own accumulators of leaf
gradients belong to the stream that made them, so a captured `backward()` needs leaves of which no graph from outside the capture is alive).
Forward-mode derivatives are not offered: a dual tensor raises NotImplementedError.  The reference trains in DGL / PyTorch (hwer/gcn_ncf.py:126-327:
out of scope here); what it hands to the search are rows (hwer/gcn_ncf.py:431,447-456).

Errors: wrong shapes, types or devices raise before anything is launched (ValueError / TypeError; HwerNativeError from the library).  Values are
never checked on the host (that would wait for the GPU): a target that names no class makes its loss NaN."""
from __future__ import annotations

import contextlib
from typing import Optional

import torch
import torch.autograd.forward_ad as _forward_ad

from . import native

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_MAX_WIDTH = (1 << 31) - (1 << 14)      # of a norm's rows
_MAX_CODES = 131071                     # of a row of the 8-bit product: 128 * 128 times as many stay below 2^31
_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}
# A call on a single row is a few microseconds of GPU time: what the host does per call is kept short (addresses as plain integers, the device switched
# only where it is another one, the raw stream handle).
_stream_of = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
_STAY = contextlib.nullcontext()
_Tensor = torch.Tensor


def P(t):
    return None if t is None else t.data_ptr()


def _on(t):
    """Context in which `t`'s device is the current one."""
    return _STAY if t.get_device() == torch.cuda.current_device() else native.device_guard(t.device)


def _stream(t):
    return _stream_of(t.get_device())


def _like(t, dtype=None):
    """An empty contiguous tensor of t's shape (two thirds of `new_empty`'s time)."""
    return torch.empty_like(t, dtype=dtype, memory_format=torch.contiguous_format)


def _wants_grad(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and getattr(t, "requires_grad", False):      # (anything else than a tensor is refused by the checks)
                return True
    return False


def _refuse_grad(what, *tensors):
    if _wants_grad(*tensors):
        raise NotImplementedError("%s has no gradient, and an operand requires one: call it under torch.no_grad(), or with detached operands" % what)


def _check_rows(name, t, dtypes=_DTYPES, dim=2):
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s: a device tensor is needed, got %s" % (name, type(t).__name__))
    if t.dtype not in dtypes:
        raise TypeError("%s: unsupported type %s" % (name, t.dtype))
    if dim is not None and t.dim() != dim:
        raise ValueError("%s: %d dimensions needed, got shape %s" % (name, dim, tuple(t.shape)))


def _check_device(t, *others):
    if _forward_ad._current_level >= 0:
        for o in (t,) + others:
            if isinstance(o, _Tensor) and _forward_ad.unpack_dual(o).tangent is not None:
                raise NotImplementedError("the learned head's operators have no forward-mode derivative: got a dual tensor")
    index = t.get_device()
    if index < 0:
        raise native.HwerNativeError("hwer (MI355X build) needs device tensors: got one on %s; there is no CPU fallback for this path" % t.device)
    for o in others:
        if o is not None:
            if not isinstance(o, _Tensor):
                raise TypeError("a device tensor is needed, got %s" % type(o).__name__)
            if o.get_device() != index:
                raise ValueError("operands on two devices: %s and %s" % (t.device, o.device))


def _rows(t):
    """(tensor, row stride) of 2-d rows whose elements are contiguous; anything else (a transposed view, a broadcast row) is copied."""
    if t.is_contiguous():
        return t, t.shape[1]
    (n, d), (row, one) = t.shape, t.stride()
    if (one == 1 or d == 1) and (row >= d or n <= 1):
        return t, max(row, d)
    return t.contiguous(), d


def _flat(t):
    """... of rows along the last dimension of any number of leading ones"""
    if t.is_contiguous():
        return t, t.shape[-1]
    return _rows(t if t.dim() == 2 else t.reshape(-1, t.shape[-1]))


def _is_vector(t, n):
    return t.dim() == 1 and t.shape[0] == n


def _weight(weight, x):
    if weight is None:
        return None, 0
    if weight.dtype is not torch.float32 and weight.dtype is not x.dtype:
        raise TypeError("weight: float32 or the rows' type (%s), got %s" % (x.dtype, weight.dtype))
    if not _is_vector(weight, x.shape[-1]):
        raise ValueError("weight: shape (%d,) needed, got %s" % (x.shape[-1], tuple(weight.shape)))
    return (weight if weight.is_contiguous() else weight.contiguous()), _DTYPES[weight.dtype]


def _norm_checks(x, weight, residual, eps, dy=None):
    _check_rows("x", x, dim=None)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x: rows of at least one element needed, got shape %s" % (tuple(x.shape),))
    if x.shape[-1] > _MAX_WIDTH:
        raise ValueError("x: rows of at most %d elements, got %d" % (_MAX_WIDTH, x.shape[-1]))
    _check_device(x, weight, residual, dy)
    if residual is not None and (residual.dtype != x.dtype or residual.shape != x.shape):
        raise ValueError("residual: shape and type of x needed (%s %s), got %s %s" % (tuple(x.shape), x.dtype, tuple(residual.shape), residual.dtype))
    if not 0.0 <= float(eps) < float("inf"):
        raise ValueError("eps must be finite and not negative")


# ---------------------------------------------------------------------------------------------------------------- root-mean-square norm
def _norm_forward(x, weight, residual, eps):
    w, wt = _weight(weight, x)
    xr, ldx = _flat(x)
    rr, ldr = _flat(residual) if residual is not None else (None, 0)
    d = x.shape[-1]
    n = x.numel() // d
    with _on(x):
        y = _like(x)
        h = _like(x) if residual is not None else None
        native.check(native.lib().hwer_rms_norm(P(xr), ldx, P(rr), ldr, P(w), wt, n, d, _DTYPES[x.dtype], eps, P(y), d, P(h), d, _stream(x)), "rms_norm")
    return y, h


def rms_norm_grads(dy, h, weight=None, eps: float = 1e-6, dh=None):
    """Gradients of `rms_norm`: -> (dx, dweight).  dx is the gradient of x and of the residual alike; dweight is None without a weight.
    h: what the norm was taken of (the second result of `rms_norm` with a residual, x without one).  dh: the gradient that reaches h by other ways."""
    return _norm_backward(dy, h, weight, eps, dh, weight is not None)


def _norm_backward(dy, h, weight, eps, dh, want_dw):
    _check_rows("dy", dy, dim=None)
    _norm_checks(h, weight, dh, eps, dy)
    if dy.shape != h.shape or dy.dtype != h.dtype:
        raise ValueError("dy: shape and type of h needed")
    w, wt = _weight(weight, h)
    (hr, ldh), (gr, ldg) = _flat(h), _flat(dy)
    ar, lda = _flat(dh) if dh is not None else (None, 0)
    d = h.shape[-1]
    n = h.numel() // d
    lib = native.lib()
    with _on(h):
        dx = _like(h)
        dw = torch.empty_like(w) if want_dw else None
        nbytes = lib.hwer_rms_norm_backward_workspace_bytes(n, d) if want_dw else 0
        ws = h.new_empty(nbytes, dtype=torch.uint8) if want_dw else None
        native.check(lib.hwer_rms_norm_backward(P(gr), ldg, P(hr), ldh, P(w), wt, P(ar), lda, n, d, _DTYPES[h.dtype], eps, P(dx), d, P(dw), P(ws), nbytes,
                                                _stream(h)), "rms_norm_backward")
    return dx, dw


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, h = _norm_forward(x, weight, residual, eps)
        ctx.save_for_backward(x if h is None else h, weight)
        ctx.eps, ctx.two = eps, h is not None
        ctx.set_materialize_grads(False)
        return y if h is None else (y, h)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh=None):
        h, weight = ctx.saved_tensors
        if dy is None:       # only h was used further
            return dh, None if weight is None or not ctx.needs_input_grad[1] else torch.zeros_like(weight), dh if ctx.two else None, None
        dx, dw = _norm_backward(dy, h, weight, ctx.eps, dh, ctx.needs_input_grad[1])
        return dx if ctx.needs_input_grad[0] else None, dw, dx if ctx.two and ctx.needs_input_grad[2] else None, None


def rms_norm(x, weight=None, residual=None, eps: float = 1e-6):
    """y = h * weight / sqrt(mean(h^2, last dimension) + eps) with h = x, or h = x + residual rounded to their type: -> y, or (y, h) with a residual.
    x: float32 / float16 / bfloat16, any number of leading dimensions; weight: (d,) float32 or x's type, None = ones.  Squares are summed in float32:
    |h| below 1.8e19 / sqrt(d), and with eps below 1e-28 a row's largest above 1e-14."""
    _norm_checks(x, weight, residual, eps)
    eps = float(eps)
    if _wants_grad(x, weight, residual):
        return _RmsNorm.apply(x, weight, residual, eps)
    y, h = _norm_forward(x, weight, residual, eps)
    return y if h is None else (y, h)


def _codes(x, weight, residual, eps, norm):
    w, wt = _weight(weight, x)
    xr, ldx = _flat(x)
    rr, ldr = _flat(residual) if residual is not None else (None, 0)
    d = x.shape[-1]
    n = x.numel() // d
    with _on(x):
        q = _like(x, torch.int8)
        scale = x.new_empty(n, dtype=torch.float32)
        h = _like(x) if residual is not None else None
        native.check(native.lib().hwer_rms_norm_q8(P(xr), ldx, P(rr), ldr, P(w), wt, n, d, _DTYPES[x.dtype], norm, eps, P(q), d, P(scale), P(h), d,
                                                   _stream(x)), "rms_norm_q8")
    if x.dim() != 2:
        scale = scale.view(x.shape[:-1])
    return (q, scale) if h is None else (q, scale, h)


def rms_norm_q8(x, weight=None, residual=None, eps: float = 1e-6):
    """`rms_norm` whose y comes as int8 codes and one float32 scale for each row: -> (codes, scales) or (codes, scales, h).  y = codes * scale to half a
    step, max|y| / 254.  No gradient, of h neither (codes are for serving): an operand that requires one raises where gradients are enabled."""
    _norm_checks(x, weight, residual, eps)
    _refuse_grad("rms_norm_q8", x, weight, residual)
    return _codes(x, weight, residual, float(eps), 1)


def quantize_rows_q8(x):
    """Rows as int8 codes and one float32 scale each, x = codes * scale to half a step: -> (codes, scales).  What a catalogue is stored as for `matmul_q8`.
    No gradient: rows that require one (a trained table) raise where gradients are enabled."""
    _norm_checks(x, None, None, 0.0)
    _refuse_grad("quantize_rows_q8", x)
    return _codes(x, None, None, 0.0, 0)


# ---------------------------------------------------------------------------------------------------------------- 8-bit product
def _check_vector(name, t, n):
    if t is None:
        raise TypeError("%s: a device tensor is needed, got None" % name)
    if t.dtype is not torch.float32 or not _is_vector(t, n):
        raise ValueError("%s: float32 of shape (%d,) needed, got %s %s" % (name, n, t.dtype, tuple(t.shape)))


def matmul_q8(a, a_scale, b, b_scale, bias=None, out_dtype=torch.float32):
    """out = (a @ b.T) * a_scale[:, None] * b_scale (+ bias): a (m, k) and b (n, k) int8 codes, a_scale (m,), b_scale (n,), bias (n,) float32;
    out (m, n) float32 / float16 / bfloat16.  The integer sums are exact (k <= 131 071).  No gradient: scales or a bias that
    require one raise where gradients are enabled."""
    _check_rows("a", a, (torch.int8,))
    _check_rows("b", b, (torch.int8,))
    _check_device(a, b, a_scale, b_scale, bias)
    _refuse_grad("matmul_q8", a_scale, b_scale, bias)
    if a.shape[1] != b.shape[1]:
        raise ValueError("rows of %d against rows of %d codes" % (a.shape[1], b.shape[1]))
    if a.shape[1] > _MAX_CODES:
        raise ValueError("rows of at most %d codes, got %d" % (_MAX_CODES, a.shape[1]))
    if out_dtype not in _DTYPES:
        raise TypeError("out_dtype: float32, float16 or bfloat16, got %s" % out_dtype)
    (m, k), n = a.shape, b.shape[0]
    _check_vector("a_scale", a_scale, m)
    _check_vector("b_scale", b_scale, n)
    if bias is not None:
        _check_vector("bias", bias, n)
    (ar, lda), (br, ldb) = _rows(a), _rows(b)
    sa, sb, bi = a_scale.contiguous(), b_scale.contiguous(), None if bias is None else bias.contiguous()
    with _on(a):
        out = torch.empty_strided((m, n), (n, 1), dtype=out_dtype, device=a.device)
        native.check(native.lib().hwer_matmul_q8(P(ar), lda, P(sa), P(br), ldb, P(sb), P(bi), m, n, k, P(out), n, _DTYPES[out_dtype], _stream(a)), "matmul_q8")
    return out


# ---------------------------------------------------------------------------------------------------------------- cross entropy over the catalogue
class _CeCall:
    """Checked operands of one call, and its two launches."""

    def __init__(self, queries, table, targets, scale, bias, reduction):
        _check_rows("queries", queries)
        _check_rows("table", table)
        if table.dtype != queries.dtype or table.shape[1] != queries.shape[1]:
            raise ValueError("table: rows of the queries' width and type needed (%d %s), got %s %s" % (queries.shape[1], queries.dtype, tuple(table.shape), table.dtype))
        if targets is None:
            raise TypeError("targets: a device tensor is needed, got None")
        _check_device(queries, table, targets, bias)
        if targets.dtype not in (torch.int64, torch.int32) or not _is_vector(targets, queries.shape[0]):
            raise ValueError("targets: int64 or int32 of shape (%d,) needed, got %s %s" % (queries.shape[0], targets.dtype, tuple(targets.shape)))
        if bias is not None:
            _check_vector("bias", bias, table.shape[0])
        if reduction not in _REDUCTIONS:
            raise ValueError("reduction: one of %s, got %r" % (sorted(_REDUCTIONS), reduction))
        self.scale = float(scale)
        if not 0.0 < self.scale < float("inf"):
            raise ValueError("scale must be positive and finite")
        self.lib = native.lib()
        self.n, self.d = queries.shape
        self.v = table.shape[0]
        if self.v < 1 or not 1 <= self.d <= self.lib.hwer_catalogue_ce_max_dim():
            raise ValueError("table: at least one row of 1..%d elements needed, got shape %s" % (self.lib.hwer_catalogue_ce_max_dim(), tuple(table.shape)))
        self.q, self.ldq = _rows(queries)
        self.e, self.lde = _rows(table)
        self.targets, self.b = targets, None if bias is None else bias.contiguous()
        self.code, self.reduction = _DTYPES[queries.dtype], _REDUCTIONS[reduction]

    def on(self):
        """Context of the call's device; work that is enqueued belongs in it."""
        return _on(self.q)

    def operands(self):
        t = self.targets
        self.t = t if t.dtype is torch.int64 and t.is_contiguous() else t.to(torch.int64).contiguous()
        return P(self.q), self.ldq, P(self.e), self.lde, P(self.b), P(self.t), self.n, self.v, self.d, self.code, self.scale, self.reduction

    def workspace(self, gradients):
        lib = self.lib
        # (with a bias the table is laid out anew: rows that it takes out may hold anything)
        in_place = self.b is None and lib.hwer_catalogue_ce_reads_in_place(P(self.e), self.lde, self.d, self.code)
        nbytes = lib.hwer_catalogue_ce_workspace_bytes(self.n, self.v, self.d, self.code, lib.hwer_catalogue_ce_reads_in_place(P(self.q), self.ldq, self.d, self.code),
                                                       in_place, gradients)
        return self.q.new_empty(nbytes, dtype=torch.uint8), nbytes

    def forward(self, want_mean):
        new = lambda *shape: self.q.new_empty(shape, dtype=torch.float32)  # noqa: E731
        ws, nbytes = self.workspace(want_mean)
        self.rows, self.state, self.counted, loss = new(self.n), new(self.n, 4), new(), new()
        self.mean = new(self.n, self.d) if want_mean else None
        native.check(self.lib.hwer_catalogue_ce(*self.operands(), P(self.rows), P(self.state), P(loss), P(self.counted), P(self.mean), P(ws), nbytes, _stream(self.q)),
                     "catalogue_cross_entropy")
        return self.rows if self.reduction == 0 else loss

    def backward(self, grad, want_q, want_e, want_b):
        ws, nbytes = self.workspace(True)
        dq = _like(self.q) if want_q else None
        de = _like(self.e) if want_e or want_b else None
        db = _like(self.b) if want_b else None
        native.check(self.lib.hwer_catalogue_ce_backward(*self.operands(), P(grad), P(self.state), P(self.counted), P(self.mean), P(dq), self.d, P(de), self.d, P(db),
                                                         P(ws), nbytes, _stream(self.q)), "catalogue_cross_entropy(backward)")
        return dq, de if want_e else None, db

    def gradients(self):
        ws, nbytes = self.workspace(True)
        loss, dq, de = self.q.new_empty((), dtype=torch.float32), _like(self.q), _like(self.e)
        db = None if self.b is None else _like(self.b)
        native.check(self.lib.hwer_catalogue_ce_grads(*self.operands(), P(loss), P(dq), self.d, P(de), self.d, P(db), P(ws), nbytes, _stream(self.q)),
                     "catalogue_cross_entropy_grads")
        return (loss, dq, de) if db is None else (loss, dq, de, db)


class _CatalogueCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, queries, table, bias, targets, scale, reduction):
        call = _CeCall(queries, table, targets, scale, bias, reduction)
        with call.on():
            loss = call.forward(bool(ctx.needs_input_grad[0]))
        ctx.save_for_backward(queries, table, bias, targets, call.state, call.counted, call.mean)
        ctx.args = (scale, reduction)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        queries, table, bias, targets, state, counted, mean = ctx.saved_tensors
        call = _CeCall(queries, table, targets, ctx.args[0], bias, ctx.args[1])
        call.state, call.counted, call.mean = state, counted, mean
        want = ctx.needs_input_grad
        with call.on():
            dq, de, db = call.backward(grad.float().contiguous(), want[0], want[1], want[2])
        return dq, de, db, None, None, None


def catalogue_cross_entropy(queries, table, targets, scale: float = 1.0, bias: Optional[torch.Tensor] = None, reduction: str = "mean"):
    """Softmax cross entropy over the whole catalogue: logits scale * queries @ table.T + bias, target = row of `table`; -> the loss (float32; with
    reduction "none" one for each row).  Logits are never in memory; gradients for queries, table and bias through autograd.

    queries (n, d), table (v, d): float32 / float16 / bfloat16 of one type, 1 <= d <= 256.  targets (n,): -1 = the row does not count (an unknown
    node, as everywhere in this package; padding); any other value outside the table makes its loss NaN.  scale > 0, a number: 1 / temperature (a learned
    one belongs on the queries).  bias (v,) float32,
    e.g. a correction for popularity; -inf takes a row out of the catalogue.  Rows that do not count or are taken out may hold anything, NaN and
    infinities included; their gradients are zero.  A target that is taken out: a loss of +inf, and the gradients as if its row were zeros.  float32 products keep 2^-22 of an element and 2^-40 of its operand's largest one;
    float16 and float32 rows' gradients keep a probability's 2^-40 of the largest (of the largest upstream gradient, with one for each row).  "mean" divides by the counted rows and is 0 without any."""
    if _wants_grad(scale):
        raise NotImplementedError("scale has no gradient here: multiply the queries by a learned temperature, or pass a number")
    if _wants_grad(queries, table, bias):
        return _CatalogueCrossEntropy.apply(queries, table, bias, targets, scale, reduction)
    call = _CeCall(queries, table, targets, scale, bias, reduction)
    with call.on():
        return call.forward(False)


def catalogue_cross_entropy_grads(queries, table, targets, scale: float = 1.0, bias: Optional[torch.Tensor] = None, reduction: str = "mean"):
    """The loss of `catalogue_cross_entropy` ("mean" or "sum") and its gradients in one go, without autograd: -> (loss, dqueries, dtable), and with a
    bias (loss, dqueries, dtable, dbias).  float32 operands are laid out for the matrix instructions once for both directions."""
    if reduction == "none":
        raise ValueError("reduction: \"mean\" or \"sum\" (gradients of which loss?)")
    call = _CeCall(queries, table, targets, scale, bias, reduction)
    with call.on():
        return call.gradients()
