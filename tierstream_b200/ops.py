"""The operators an engine runs beside the streamed units, on torch tensors: the router's selection (route), the gated
feed-forward block of the units in their slots (ffn), and the matrix product with its epilogue (linear), each with its
backward pass. Every function is one call of the C ABI (include/tierstream/tsb.h has the formulas, limits and what is
rounded where) on torch's current stream of the tensors' device; outputs and scratch come from torch's allocator, so a
call may be captured into a CUDA graph. Gradients are explicit functions: nothing is recorded for autograd.

Tensors are bfloat16 or float16 (logits float32 too), two-dimensional, with any stride between rows and stride 1 inside
them; an argument that does not fit raises ValueError, a call the library refuses raises abi.TsError.
"""
import ctypes as C

import torch

from . import abi

ACTIVATIONS = {"none": abi.TSB_ACT_NONE, "silu": abi.TSB_ACT_SILU, "gelu": abi.TSB_ACT_GELU,
               "gelu_tanh": abi.TSB_ACT_GELU_TANH, "relu": abi.TSB_ACT_RELU}
_HALF = {torch.bfloat16: abi.TSB_BF16, torch.float16: abi.TSB_F16}
_ANY = {**_HALF, torch.float32: abi.TSB_F32}


def _act(name):
    try:
        return ACTIVATIONS[name]
    except KeyError:
        raise ValueError("unknown activation %r: one of %s" % (name, ", ".join(ACTIVATIONS))) from None


def _mat(name, t, rows, cols, like):
    """A [rows][cols] matrix of like's type on like's device: (address, elements between rows)."""
    if t.dtype != like.dtype or t.device != like.device:
        raise ValueError("%s: %s on %s is wanted, got %s on %s" % (name, like.dtype, like.device, t.dtype, t.device))
    if t.dim() != 2 or t.shape[0] != rows or t.shape[1] != cols:
        raise ValueError("%s: shape %s is wanted, got %s" % (name, (rows, cols), tuple(t.shape)))
    s0, s1 = t.stride()
    if cols > 1 and s1 != 1:
        raise ValueError("%s: the elements of a row must be adjacent" % name)
    if rows > 1 and s0 < cols:
        raise ValueError("%s: rows overlap" % name)
    return t.data_ptr(), s0 if rows > 1 else max(s0, cols)


def _flat(name, t, shape, dtype, device):
    """A contiguous tensor of the given shape: its address."""
    if t.dtype != dtype or t.device != device or t.shape != shape or not t.is_contiguous():
        raise ValueError("%s: a contiguous %s of shape %s on %s is wanted, got %s %s on %s" %
                         (name, dtype, tuple(shape), device, t.dtype, tuple(t.shape), t.device))
    return t.data_ptr()


def _first(name, t, types):
    if t.dtype not in types:
        raise ValueError("%s: %s is not served (%s)" % (name, t.dtype, ", ".join(str(d) for d in types)))
    if t.dim() != 2:
        raise ValueError("%s: two dimensions are wanted, got %s" % (name, tuple(t.shape)))
    if not t.is_cuda:
        raise ValueError("%s: a CUDA tensor is wanted" % name)
    return types[t.dtype]


def _call(fn, args, device, size=None):
    """Runs one entry point on the current stream of `device` with scratch of the size it asks for."""
    if torch.cuda.current_device() != device.index:
        with torch.cuda.device(device):
            return _call(fn, args, device, size)
    args.stream = torch.cuda.current_stream().cuda_stream
    scratch = None
    n = size(C.byref(args)) if size else 0
    if n:
        scratch = torch.empty(n + 256, dtype=torch.uint8, device=device)
        args.workspace = (scratch.data_ptr() + 255) & ~255
        args.workspace_bytes = n
    abi.check(fn(C.byref(args)))


def linear(x, w, bias=None, residual=None, act="none", pre=None, out=None):
    """act(x w^T + bias) + residual: x [rows][k], w [n][k], bias [n], residual [rows][n]. pre: a [rows][n] tensor that
    receives x w^T + bias for linear_backward. out: where to write (may be the residual)."""
    lib = abi.load()
    dt = _first("x", x, _HALF)
    rows, k = x.shape
    n = w.shape[0]
    a = abi.tsb_linear_args(C.sizeof(abi.tsb_linear_args), dt, _act(act), 0, rows, n, k)
    a.x, a.ldx = _mat("x", x, rows, k, x)
    a.w, a.ldw = _mat("w", w, n, k, x)
    if bias is not None:
        a.bias = _flat("bias", bias, (n,), x.dtype, x.device)
    if residual is not None:
        a.residual, a.ldr = _mat("residual", residual, rows, n, x)
    if pre is not None:
        a.pre, a.ldp = _mat("pre", pre, rows, n, x)
    if out is None:
        out = torch.empty((rows, n), dtype=x.dtype, device=x.device)
    a.y, a.ldy = _mat("out", out, rows, n, x)
    _call(lib.tsb_linear, a, x.device, lib.tsb_linear_workspace)
    return out


def linear_backward(dy, x, w, act="none", pre=None, need=("x", "w", "bias")):
    """(dx, dw, dbias) of linear() from dy [rows][n]; None for what `need` does not name. pre: what the forward pass
    wrote there (needed unless act is "none"). The residual's gradient is dy."""
    lib = abi.load()
    dt = _first("dy", dy, _HALF)
    rows, n = dy.shape
    k = x.shape[1]
    a = abi.tsb_linear_grad_args(C.sizeof(abi.tsb_linear_grad_args), dt, _act(act), 0, rows, n, k)
    a.dy, a.lddy = _mat("dy", dy, rows, n, dy)
    a.x, a.ldx = _mat("x", x, rows, k, dy)
    a.w, a.ldw = _mat("w", w, n, k, dy)
    if act != "none":
        if pre is None:
            raise ValueError("pre: an activation's slope needs it")
        a.pre, a.ldp = _mat("pre", pre, rows, n, dy)
    dx = dw = db = None
    if "x" in need:
        dx = torch.empty((rows, k), dtype=dy.dtype, device=dy.device)
        a.dx, a.lddx = dx.data_ptr(), k
    if "w" in need:
        dw = torch.empty((n, k), dtype=dy.dtype, device=dy.device)
        a.dw, a.lddw = dw.data_ptr(), k
    if "bias" in need:
        db = torch.empty(n, dtype=dy.dtype, device=dy.device)
        a.db = db.data_ptr()
    _call(lib.tsb_linear_backward, a, dy.device, lib.tsb_linear_backward_workspace)
    return dx, dw, db


def route(logits, top, norm=True):
    """(ids int32 [rows][top], weights float32 [rows][top]): the `top` largest logits of each row, the lowest expert
    first among equal ones; weights by softmax over the chosen (norm) or over the whole row. -inf and NaN are never
    chosen: a row with fewer than `top` others ends in ids -1 with weight 0."""
    lib = abi.load()
    dt = _first("logits", logits, _ANY)
    rows, experts = logits.shape
    p, ld = _mat("logits", logits, rows, experts, logits)
    ids = torch.empty((rows, top), dtype=torch.int32, device=logits.device)
    weights = torch.empty((rows, top), dtype=torch.float32, device=logits.device)

    def go():
        abi.check(lib.tsb_route(dt, p, ld, rows, experts, top, 1 if norm else 0, ids.data_ptr(), weights.data_ptr(),
                                torch.cuda.current_stream().cuda_stream))
    _on(logits.device, go)
    return ids, weights


def _on(device, go):
    if torch.cuda.current_device() == device.index:
        go()
    else:
        with torch.cuda.device(device):
            go()


def route_backward(dweights, logits, ids, weights, norm=True):
    """dlogits [rows][experts] (logits' type) of route() from dweights [rows][top] and the ids and weights it gave."""
    lib = abi.load()
    dt = _first("logits", logits, _ANY)
    wt = _first("dweights", dweights, _ANY)
    rows, experts = logits.shape
    top = ids.shape[1]
    p, ld = _mat("logits", logits, rows, experts, logits)
    d = _flat("dweights", dweights, (rows, top), dweights.dtype, logits.device)
    i = _flat("ids", ids, (rows, top), torch.int32, logits.device)
    w = _flat("weights", weights, (rows, top), torch.float32, logits.device)
    out = torch.empty((rows, experts), dtype=logits.dtype, device=logits.device)

    def go():
        abi.check(lib.tsb_route_backward(dt, wt, d, p, ld, i, w, rows, experts, top, 1 if norm else 0, out.data_ptr(),
                                         experts, torch.cuda.current_stream().cuda_stream))
    _on(logits.device, go)
    return out


class Units:
    """Where a layer's units live: gate and up [slots][ffn][hidden], down [slots][hidden][ffn] (any stride between
    slots), and slot_of [units] int32 on the device, read when the kernels run (None: unit u in slot u). A unit whose
    slot is outside the arrays is not there: its rows contribute nothing."""

    def __init__(self, gate, up, down, slot_of=None):
        _first("gate", gate[:, 0] if gate.dim() == 3 else gate, _HALF)
        slots, ffn, hidden = gate.shape
        self.dtype, self.device, self.hidden, self.ffn = gate.dtype, gate.device, hidden, ffn
        self.n_units = slots if slot_of is None else slot_of.numel()
        self.keep = (gate, up, down, slot_of)  # the tensors behind the addresses
        s = abi.tsb_units(C.sizeof(abi.tsb_units), self.n_units, slots)
        for i, (name, t, shape) in enumerate((("gate", gate, (slots, ffn, hidden)), ("up", up, (slots, ffn, hidden)),
                                              ("down", down, (slots, hidden, ffn)))):
            if t.dtype != gate.dtype or t.device != gate.device or t.shape != shape:
                raise ValueError("%s: %s of shape %s on %s is wanted" % (name, gate.dtype, shape, gate.device))
            if t.stride()[1:] != (shape[2], 1) or (slots > 1 and t.stride(0) < ffn * hidden):
                raise ValueError("%s: a slot's matrix must be contiguous, and slots apart" % name)
            s.part[i] = t.data_ptr()
            s.stride[i] = t.stride(0) * 2
        if slot_of is not None:
            s.slot_of = _flat("slot_of", slot_of, (self.n_units,), torch.int32, gate.device)
        self.struct = s

    @classmethod
    def of_context(cls, ctx, g, n_units, hidden, ffn, dtype=torch.bfloat16, device=None):
        """Gated layer g of a runtime.DgContext whose units are gate, up and down parts of this type: valid between
        ss_dg_enqueue_wait(g) and the token's end, for the context's life."""
        self = cls.__new__(cls)
        if dtype not in _HALF:
            raise ValueError("%s is not served" % dtype)
        self.dtype, self.hidden, self.ffn, self.n_units = dtype, hidden, ffn, n_units
        self.device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self.keep, self.struct = (ctx,), abi.tsb_units()
        v = ctx.view()
        abi.check(abi.load().tsb_units_from_view(C.byref(v), g, n_units, hidden * ffn * 2, C.byref(self.struct)))
        return self

    @classmethod
    def of_table(cls, table, n_units, hidden, ffn, dtype=torch.bfloat16, device=None):
        """A layer acquired in host forward mode: `table` the device address of its n_units unit addresses
        (ss_layer_view.table_dev), each unit gate, up and down back to back. Valid until the layer's release."""
        self = cls.__new__(cls)
        if dtype not in _HALF:
            raise ValueError("%s is not served" % dtype)
        self.dtype, self.hidden, self.ffn, self.n_units = dtype, hidden, ffn, n_units
        self.device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self.keep = ()
        s = self.struct = abi.tsb_units(C.sizeof(abi.tsb_units), n_units, 0)
        s.table = table
        for i in range(3):
            s.stride[i] = i * hidden * ffn * 2
        return self


def _ffn_args(struct, x, ids, weights, units, act):
    dt = _first("x", x, _HALF)
    rows, hidden = x.shape
    if ids.dim() != 2:
        raise ValueError("ids: two dimensions are wanted, got %s" % (tuple(ids.shape),))
    top = ids.shape[1]
    if units.dtype != x.dtype or units.hidden != hidden or units.device != x.device:
        raise ValueError("units: %s with hidden %d on %s is wanted" % (x.dtype, hidden, x.device))
    a = struct(C.sizeof(struct), dt, _act(act), top, rows, hidden, units.ffn)
    a.x, a.ldx = _mat("x", x, rows, hidden, x)
    a.ids = _flat("ids", ids, (rows, top), torch.int32, x.device)
    a.weights = _flat("weights", weights, (rows, top), torch.float32, x.device)
    a.units = C.addressof(units.struct)
    return a


def ffn(x, ids, weights, units, act="silu", residual=None, out=None):
    """residual + sum over k of weights[t][k] x the gated block of unit ids[t][k]: x [rows][hidden], ids int32 and
    weights float32 [rows][top]. An id outside the units (-1: a padded row) contributes nothing. out: where to write
    (may be the residual)."""
    lib = abi.load()
    a = _ffn_args(abi.tsb_ffn_args, x, ids, weights, units, act)
    rows, hidden = x.shape
    if residual is not None:
        a.residual, a.ldr = _mat("residual", residual, rows, hidden, x)
    if out is None:
        out = torch.empty((rows, hidden), dtype=x.dtype, device=x.device)
    a.y, a.ldy = _mat("out", out, rows, hidden, x)
    _call(lib.tsb_ffn, a, x.device, lib.tsb_ffn_workspace)
    return out


def ffn_backward(dy, x, ids, weights, units, act="silu", need=("x", "weights", "units")):
    """The gradients of ffn() from dy [rows][hidden] as a dict: dx, dweights [rows][top], and dgate, dup, ddown by unit
    (zeros for a unit without rows); None for what `need` ("x", "weights", "units") does not name. All of x's type."""
    lib = abi.load()
    a = _ffn_args(abi.tsb_ffn_grad_args, x, ids, weights, units, act)
    rows, hidden = x.shape
    a.dy, a.lddy = _mat("dy", dy, rows, hidden, x)
    like = dict(dtype=x.dtype, device=x.device)
    g = dict.fromkeys(("dx", "dweights", "dgate", "dup", "ddown"))
    if "x" in need:
        g["dx"] = torch.empty((rows, hidden), **like)
        a.dx, a.lddx = g["dx"].data_ptr(), hidden
    if "weights" in need:
        g["dweights"] = torch.empty(tuple(ids.shape), **like)
        a.dweights = g["dweights"].data_ptr()
    if "units" in need:
        g["dgate"] = torch.empty((units.n_units, units.ffn, hidden), **like)
        g["dup"] = torch.empty((units.n_units, units.ffn, hidden), **like)
        g["ddown"] = torch.empty((units.n_units, hidden, units.ffn), **like)
        a.dgate, a.dup, a.ddown = (g[k].data_ptr() for k in ("dgate", "dup", "ddown"))
    _call(lib.tsb_ffn_backward, a, x.device, lib.tsb_ffn_backward_workspace)
    return g
