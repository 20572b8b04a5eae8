"""The operators an engine runs beside the streamed units, on torch tensors: the router's selection (route), the gated
feed-forward block of the units in their slots (ffn), and the matrix product with its epilogue (linear), each with its
backward pass. Every function is one call of the C ABI (include/tierstream/tsb.h has the formulas, limits and what is
rounded where) on torch's current stream of the tensors' device; outputs and scratch come from torch's allocator, so a
call may be captured into a CUDA graph. Gradients are explicit functions: nothing is recorded for autograd.

Tensors are bfloat16 or float16 (logits float32 too), two-dimensional, with any stride between rows and stride 1 inside
them; a tensor that does not fit raises ValueError, a call the library refuses raises abi.TsError.
"""
import ctypes as C

import torch

from . import abi

abi.load()  # (what _torch_ops links; raises when it is not built)
from . import _torch_ops as _ops  # noqa: E402

_ops.set_error(abi.TsError)

ACTIVATIONS = {"none": abi.TSB_ACT_NONE, "silu": abi.TSB_ACT_SILU, "gelu": abi.TSB_ACT_GELU,
               "gelu_tanh": abi.TSB_ACT_GELU_TANH, "relu": abi.TSB_ACT_RELU}
HALF = {torch.bfloat16: abi.TSB_BF16, torch.float16: abi.TSB_F16}


def _act(name):
    try:
        return ACTIVATIONS[name]
    except KeyError:
        raise ValueError("unknown activation %r: one of %s" % (name, ", ".join(ACTIVATIONS))) from None


def linear(x, w, bias=None, residual=None, act="none", pre=None, out=None):
    """act(x w^T + bias) + residual: x [rows][k], w [n][k], bias [n], residual [rows][n]. pre: a [rows][n] tensor that
    receives x w^T + bias for linear_backward. out: where to write (may be the residual)."""
    return _ops.linear(x, w, bias, residual, _act(act), pre, out)


def linear_backward(dy, x, w, act="none", pre=None, need=("x", "w", "bias")):
    """(dx, dw, dbias) of linear() from dy [rows][n]; None for what `need` does not name. pre: what the forward pass
    wrote there (needed unless act is "none"). The residual's gradient is dy."""
    return _ops.linear_backward(dy, x, w, _act(act), pre, "x" in need, "w" in need, "bias" in need)


def route(logits, top, norm=True):
    """(ids int32 [rows][top], weights float32 [rows][top]): the `top` largest logits of each row, the lowest expert
    first among equal ones; weights by softmax over the chosen (norm) or over the whole row. -inf and NaN are never
    chosen: a row with fewer than `top` others ends in ids -1 with weight 0."""
    return _ops.route(logits, top, norm)


def route_backward(dweights, logits, ids, weights, norm=True):
    """dlogits [rows][experts] (logits' type) of route() from dweights [rows][top] and the ids and weights it gave."""
    return _ops.route_backward(dweights, logits, ids, weights, norm)


class Units:
    """Where a layer's units live: gate and up [slots][ffn][hidden], down [slots][hidden][ffn] (any stride between
    slots), and slot_of [units] int32 on the device, read when the kernels run (None: unit u in slot u). A unit whose
    slot is outside the arrays is not there: its rows contribute nothing."""

    def __init__(self, gate, up, down, slot_of=None):
        self.struct = abi.tsb_units()
        self.addr = C.addressof(self.struct)
        self.n_units, self.ffn, self.hidden = _ops.units(self.addr, gate, up, down, slot_of)
        self.dtype, self.dev = gate.dtype, gate.get_device()
        self.keep = (gate, up, down, slot_of)  # the tensors behind the addresses

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
        self.addr = C.addressof(self.struct)
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
        self.addr = C.addressof(s)
        s.table = table
        for i in range(3):
            s.stride[i] = i * hidden * ffn * 2
        return self


    def check(self, x):
        if self.dtype is not x.dtype or self.dev != x.get_device() or x.dim() != 2 or self.hidden != x.shape[1]:
            raise ValueError("units: %s with hidden %d on cuda:%d; x is %s %s on %s" %
                             (self.dtype, self.hidden, self.dev, x.dtype, tuple(x.shape), x.device))


def ffn(x, ids, weights, units, act="silu", residual=None, out=None):
    """residual + sum over k of weights[t][k] x the gated block of unit ids[t][k]: x [rows][hidden], ids int32 and
    weights float32 [rows][top]. An id outside the units (-1: a padded row) contributes nothing. out: where to write
    (may be the residual, x itself among them)."""
    units.check(x)
    return _ops.ffn(x, ids, weights, units.addr, units.ffn, _act(act), residual, out)


def ffn_backward(dy, x, ids, weights, units, act="silu", need=("x", "weights", "units")):
    """The gradients of ffn() from dy [rows][hidden] as a dict: dx, dweights [rows][top], and dgate, dup, ddown by unit
    (zeros for a unit without rows); None for what `need` ("x", "weights", "units") does not name. All of x's type."""
    units.check(x)
    return dict(zip(("dx", "dweights", "dgate", "dup", "ddown"),
                    _ops.ffn_backward(dy, x, ids, weights, units.addr, units.n_units, units.ffn, _act(act), "x" in need,
                                      "weights" in need, "units" in need)))
