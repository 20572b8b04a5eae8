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
HALF = {torch.bfloat16: abi.TSB_BF16, torch.float16: abi.TSB_F16}
_ANY = {**HALF, torch.float32: abi.TSB_F32}
_LINEAR, _LINEAR_GRAD = C.sizeof(abi.tsb_linear_args), C.sizeof(abi.tsb_linear_grad_args)
_FFN, _FFN_GRAD, _UNITS = C.sizeof(abi.tsb_ffn_args), C.sizeof(abi.tsb_ffn_grad_args), C.sizeof(abi.tsb_units)
# the current stream's handle; torch.cuda.current_stream() builds an object around it, which costs 4 us a call
_raw_stream = torch._C._cuda_getCurrentRawStream


def _act(name):
    try:
        return ACTIVATIONS[name]
    except KeyError:
        raise ValueError("unknown activation %r: one of %s" % (name, ", ".join(ACTIVATIONS))) from None


def _first(name, t, types):
    """The type code and the device of an operator's first matrix."""
    dt = types.get(t.dtype)
    if dt is None:
        raise ValueError("%s: %s is not served (%s)" % (name, t.dtype, ", ".join(str(d) for d in types)))
    if t.dim() != 2:
        raise ValueError("%s: two dimensions are wanted, got %s" % (name, tuple(t.shape)))
    if not t.is_cuda:
        raise ValueError("%s: a CUDA tensor is wanted" % name)
    return dt, t.get_device()


def _mat(name, t, rows, cols, dtype, dev):
    """A [rows][cols] matrix of that type on that device: (address, elements between rows)."""
    if t.dtype is not dtype or t.get_device() != dev:
        raise ValueError("%s: %s on cuda:%d is wanted, got %s on %s" % (name, dtype, dev, t.dtype, t.device))
    if t.shape != (rows, cols):
        raise ValueError("%s: shape %s is wanted, got %s" % (name, (rows, cols), tuple(t.shape)))
    if t.is_contiguous():
        return t.data_ptr(), cols
    s0, s1 = t.stride()
    if cols > 1 and s1 != 1:
        raise ValueError("%s: the elements of a row must be adjacent" % name)
    if rows > 1 and s0 < cols:
        raise ValueError("%s: rows overlap" % name)
    return t.data_ptr(), s0 if rows > 1 else cols


def _flat(name, t, shape, dtype, dev):
    """A contiguous tensor of the given shape: its address."""
    if t.dtype is not dtype or t.get_device() != dev or t.shape != shape or not t.is_contiguous():
        raise ValueError("%s: a contiguous %s of shape %s on cuda:%d is wanted, got %s %s on %s" %
                         (name, dtype, tuple(shape), dev, t.dtype, tuple(t.shape), t.device))
    return t.data_ptr()


def _apart(name, out, *inputs):
    """Refuses an output that shares memory with an input (its residual apart, element by element)."""
    def span(t):
        n = sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1 if t.numel() else 0
        return t.data_ptr(), t.data_ptr() + n * t.element_size()
    lo, hi = span(out)
    for t in inputs:
        a, b = span(t)
        if a < hi and lo < b:
            raise ValueError("%s: overlaps an input" % name)


def _call(fn, args, dev, size=None):
    """Runs one entry point on the current stream of device `dev` with scratch of the size it asks for."""
    if torch.cuda.current_device() != dev:
        with torch.cuda.device(dev):
            return _call(fn, args, dev, size)
    args.stream = _raw_stream(dev)
    ref = C.byref(args)
    n = size(ref) if size else 0
    if n:
        scratch = torch.empty(n + 256, dtype=torch.uint8, device="cuda")
        args.workspace = (scratch.data_ptr() + 255) & ~255
        args.workspace_bytes = n
    st = fn(ref)
    if st:
        abi.check(st)


def linear(x, w, bias=None, residual=None, act="none", pre=None, out=None):
    """act(x w^T + bias) + residual: x [rows][k], w [n][k], bias [n], residual [rows][n]. pre: a [rows][n] tensor that
    receives x w^T + bias for linear_backward. out: where to write (may be the residual)."""
    lib = abi.load()
    dt, dev = _first("x", x, HALF)
    (rows, k), n, t = x.shape, w.shape[0], x.dtype
    px, ldx = _mat("x", x, rows, k, t, dev)
    pw, ldw = _mat("w", w, n, k, t, dev)
    pb = pr = pp = None
    ldr = ldp = 0
    if bias is not None:
        pb = _flat("bias", bias, (n,), t, dev)
    if residual is not None:
        pr, ldr = _mat("residual", residual, rows, n, t, dev)
    if pre is not None:
        pp, ldp = _mat("pre", pre, rows, n, t, dev)
        _apart("pre", pre, x, w)
    if out is None:
        out = x.new_empty((rows, n))
    else:
        _apart("out", out, x, w)
    py, ldy = _mat("out", out, rows, n, t, dev)
    a = abi.tsb_linear_args(_LINEAR, dt, _act(act), 0, rows, n, k, px, ldx, pw, ldw, pb, pr, ldr, py, ldy, pp, ldp)
    _call(lib.tsb_linear, a, dev, lib.tsb_linear_workspace)
    return out


def linear_backward(dy, x, w, act="none", pre=None, need=("x", "w", "bias")):
    """(dx, dw, dbias) of linear() from dy [rows][n]; None for what `need` does not name. pre: what the forward pass
    wrote there (needed unless act is "none"). The residual's gradient is dy."""
    lib = abi.load()
    dt, dev = _first("dy", dy, HALF)
    (rows, n), t = dy.shape, dy.dtype
    if x.dim() != 2:
        raise ValueError("x: two dimensions are wanted, got %s" % (tuple(x.shape),))
    k = x.shape[1]
    a = abi.tsb_linear_grad_args(_LINEAR_GRAD, dt, _act(act), 0, rows, n, k)
    a.dy, a.lddy = _mat("dy", dy, rows, n, t, dev)
    a.x, a.ldx = _mat("x", x, rows, k, t, dev)
    a.w, a.ldw = _mat("w", w, n, k, t, dev)
    if act != "none":
        if pre is None:
            raise ValueError("pre: an activation's slope needs it")
        a.pre, a.ldp = _mat("pre", pre, rows, n, t, dev)
    dx = dw = db = None
    if "x" in need:
        dx = dy.new_empty((rows, k))
        a.dx, a.lddx = dx.data_ptr(), k
    if "w" in need:
        dw = dy.new_empty((n, k))
        a.dw, a.lddw = dw.data_ptr(), k
    if "bias" in need:
        db = dy.new_empty((n,))
        a.db = db.data_ptr()
    _call(lib.tsb_linear_backward, a, dev, lib.tsb_linear_backward_workspace)
    return dx, dw, db


def _route_call(dev, fn, *args):
    if torch.cuda.current_device() != dev:
        with torch.cuda.device(dev):
            return _route_call(dev, fn, *args)
    st = fn(*args, _raw_stream(dev))
    if st:
        abi.check(st)


def route(logits, top, norm=True):
    """(ids int32 [rows][top], weights float32 [rows][top]): the `top` largest logits of each row, the lowest expert
    first among equal ones; weights by softmax over the chosen (norm) or over the whole row. -inf and NaN are never
    chosen: a row with fewer than `top` others ends in ids -1 with weight 0."""
    lib = abi.load()
    dt, dev = _first("logits", logits, _ANY)
    rows, experts = logits.shape
    p, ld = _mat("logits", logits, rows, experts, logits.dtype, dev)
    if not 1 <= top <= min(32, experts):
        raise ValueError("top: must be in [1, 32] and at most the experts, got %d" % top)
    ids = logits.new_empty((rows, top), dtype=torch.int32)
    weights = logits.new_empty((rows, top), dtype=torch.float32)
    _route_call(dev, lib.tsb_route, dt, p, ld, rows, experts, top, 1 if norm else 0, ids.data_ptr(),
                weights.data_ptr())
    return ids, weights


def route_backward(dweights, logits, ids, weights, norm=True):
    """dlogits [rows][experts] (logits' type) of route() from dweights [rows][top] and the ids and weights it gave."""
    lib = abi.load()
    dt, dev = _first("logits", logits, _ANY)
    wt, _ = _first("dweights", dweights, _ANY)
    rows, experts = logits.shape
    shape = dweights.shape
    p, ld = _mat("logits", logits, rows, experts, logits.dtype, dev)
    if shape[0] != rows:
        raise ValueError("dweights: %d rows are wanted, got %d" % (rows, shape[0]))
    d = _flat("dweights", dweights, shape, dweights.dtype, dev)
    i = _flat("ids", ids, shape, torch.int32, dev)
    w = _flat("weights", weights, shape, torch.float32, dev)
    out = logits.new_empty((rows, experts))
    _route_call(dev, lib.tsb_route_backward, dt, wt, d, p, ld, i, w, rows, experts, shape[1], 1 if norm else 0,
                out.data_ptr(), experts)
    return out


class Units:
    """Where a layer's units live: gate and up [slots][ffn][hidden], down [slots][hidden][ffn] (any stride between
    slots), and slot_of [units] int32 on the device, read when the kernels run (None: unit u in slot u). A unit whose
    slot is outside the arrays is not there: its rows contribute nothing."""

    def __init__(self, gate, up, down, slot_of=None):
        if gate.dim() != 3 or gate.dtype not in HALF or not gate.is_cuda:
            raise ValueError("gate: [slots][ffn][hidden] of bfloat16 or float16 on a CUDA device is wanted, got %s %s on "
                             "%s" % (gate.dtype, tuple(gate.shape), gate.device))
        slots, ffn, hidden = gate.shape
        t, dev = gate.dtype, gate.get_device()
        self.dtype, self.dev, self.hidden, self.ffn = t, dev, hidden, ffn
        self.n_units = n = slots if slot_of is None else slot_of.numel()
        self.keep = (gate, up, down, slot_of)  # the tensors behind the addresses
        self.struct = s = abi.tsb_units(_UNITS, n, slots)
        for i, (m, shape) in enumerate(((gate, (slots, ffn, hidden)), (up, (slots, ffn, hidden)),
                                        (down, (slots, hidden, ffn)))):
            if m.dtype is not t or m.get_device() != dev or m.shape != shape:
                raise ValueError("%s: %s of shape %s on cuda:%d is wanted, got %s %s on %s" %
                                 (("gate", "up", "down")[i], t, shape, dev, m.dtype, tuple(m.shape), m.device))
            s0, s1, s2 = m.stride()
            if not m.is_contiguous() and (s1 != shape[2] or s2 != 1 or (slots > 1 and s0 < ffn * hidden)):
                raise ValueError("%s: a slot's matrix must be contiguous, and slots apart" % ("gate", "up", "down")[i])
            s.part[i] = m.data_ptr()
            s.stride[i] = s0 * 2
        if slot_of is not None:
            s.slot_of = _flat("slot_of", slot_of, (n,), torch.int32, dev)

    @classmethod
    def of_context(cls, ctx, g, n_units, hidden, ffn, dtype=torch.bfloat16, device=None):
        """Gated layer g of a runtime.DgContext whose units are gate, up and down parts of this type: valid between
        ss_dg_enqueue_wait(g) and the token's end, for the context's life."""
        self = cls.__new__(cls)
        if dtype not in HALF:
            raise ValueError("%s is not served" % dtype)
        self.dtype, self.hidden, self.ffn, self.n_units = dtype, hidden, ffn, n_units
        self.dev = torch.cuda.current_device() if device is None else torch.device(device).index
        self.keep, self.struct = (ctx,), abi.tsb_units()
        v = ctx.view()
        abi.check(abi.load().tsb_units_from_view(C.byref(v), g, n_units, hidden * ffn * 2, C.byref(self.struct)))
        return self

    @classmethod
    def of_table(cls, table, n_units, hidden, ffn, dtype=torch.bfloat16, device=None):
        """A layer acquired in host forward mode: `table` the device address of its n_units unit addresses
        (ss_layer_view.table_dev), each unit gate, up and down back to back. Valid until the layer's release."""
        self = cls.__new__(cls)
        if dtype not in HALF:
            raise ValueError("%s is not served" % dtype)
        self.dtype, self.hidden, self.ffn, self.n_units = dtype, hidden, ffn, n_units
        self.dev = torch.cuda.current_device() if device is None else torch.device(device).index
        self.keep = ()
        s = self.struct = abi.tsb_units(C.sizeof(abi.tsb_units), n_units, 0)
        s.table = table
        for i in range(3):
            s.stride[i] = i * hidden * ffn * 2
        return self


def _ffn_args(struct, size, x, ids, weights, units, act):
    dt, dev = _first("x", x, HALF)
    rows, hidden = x.shape
    if ids.dim() != 2:
        raise ValueError("ids: two dimensions are wanted, got %s" % (tuple(ids.shape),))
    shape = (rows, ids.shape[1])
    if units.dtype is not x.dtype or units.hidden != hidden or units.dev != dev:
        raise ValueError("units: %s with hidden %d on cuda:%d is wanted" % (x.dtype, hidden, dev))
    px, ldx = _mat("x", x, rows, hidden, x.dtype, dev)
    pi = _flat("ids", ids, shape, torch.int32, dev)
    pw = _flat("weights", weights, shape, torch.float32, dev)
    pu = C.addressof(units.struct)
    if struct is abi.tsb_ffn_args:
        a = struct(size, dt, _act(act), shape[1], rows, hidden, units.ffn, px, ldx, pi, pw, pu)
    else:
        a = struct(size, dt, _act(act), shape[1], rows, hidden, units.ffn, None, 0, px, ldx, pi, pw, pu)
    return a, dev


def ffn(x, ids, weights, units, act="silu", residual=None, out=None):
    """residual + sum over k of weights[t][k] x the gated block of unit ids[t][k]: x [rows][hidden], ids int32 and
    weights float32 [rows][top]. An id outside the units (-1: a padded row) contributes nothing. out: where to write
    (may be the residual)."""
    lib = abi.load()
    a, dev = _ffn_args(abi.tsb_ffn_args, _FFN, x, ids, weights, units, act)
    rows, hidden = x.shape
    if residual is not None:
        a.residual, a.ldr = _mat("residual", residual, rows, hidden, x.dtype, dev)
    if out is None:
        out = x.new_empty((rows, hidden))
    elif out.data_ptr() != x.data_ptr() or residual is not x:  # (in place on x as its own residual: x is read first)
        _apart("out", out, x)
    a.y, a.ldy = _mat("out", out, rows, hidden, x.dtype, dev)
    _call(lib.tsb_ffn, a, dev, lib.tsb_ffn_workspace)
    return out


def ffn_backward(dy, x, ids, weights, units, act="silu", need=("x", "weights", "units")):
    """The gradients of ffn() from dy [rows][hidden] as a dict: dx, dweights [rows][top], and dgate, dup, ddown by unit
    (zeros for a unit without rows); None for what `need` ("x", "weights", "units") does not name. All of x's type."""
    lib = abi.load()
    a, dev = _ffn_args(abi.tsb_ffn_grad_args, _FFN_GRAD, x, ids, weights, units, act)
    rows, hidden = x.shape
    a.dy, a.lddy = _mat("dy", dy, rows, hidden, x.dtype, dev)
    g = dict.fromkeys(("dx", "dweights", "dgate", "dup", "ddown"))
    if "x" in need:
        g["dx"] = x.new_empty((rows, hidden))
        a.dx, a.lddx = g["dx"].data_ptr(), hidden
    if "weights" in need:
        g["dweights"] = x.new_empty(tuple(ids.shape))
        a.dweights = g["dweights"].data_ptr()
    if "units" in need:
        g["dgate"] = x.new_empty((units.n_units, units.ffn, hidden))
        g["dup"] = x.new_empty((units.n_units, units.ffn, hidden))
        g["ddown"] = x.new_empty((units.n_units, hidden, units.ffn))
        a.dgate, a.dup, a.ddown = (g[k].data_ptr() for k in ("dgate", "dup", "ddown"))
    _call(lib.tsb_ffn_backward, a, dev, lib.tsb_ffn_backward_workspace)
    return g
