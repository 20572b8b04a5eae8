"""The operators' argument checks (tsb_linear, tsb_route, tsb_ffn and their backward passes), which come before any
device work: each refusal names its reason, a workspace question about refused arguments answers 0, and a view without
gate, up and down parts gives no units. No GPU."""
import ctypes as C

import pytest

from tierstream_b200 import abi

BUF = (C.c_char * 4096)()
P = (C.addressof(BUF) + 255) & ~255  # never read: every call here is refused or empty


def linear(**kw):
    a = abi.tsb_linear_args(C.sizeof(abi.tsb_linear_args), abi.TSB_BF16, abi.TSB_ACT_NONE, 0, 2, 3, 4, x=P, ldx=4, w=P,
                            ldw=4, y=P, ldy=3)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def linear_back(**kw):
    a = abi.tsb_linear_grad_args(C.sizeof(abi.tsb_linear_grad_args), abi.TSB_BF16, abi.TSB_ACT_NONE, 0, 2, 3, 4, dy=P,
                                 lddy=3, x=P, ldx=4, w=P, ldw=4, dx=P, lddx=4, dw=P, lddw=4, db=P)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def units(**kw):
    u = abi.tsb_units(C.sizeof(abi.tsb_units), 4, 5)
    for i in range(3):
        u.part[i], u.stride[i] = P, 64
    for k, v in kw.items():
        setattr(u, k, v)
    return u


def ffn(u=None, struct=abi.tsb_ffn_args, **kw):
    u = units() if u is None else u
    a = struct(C.sizeof(struct), abi.TSB_BF16, abi.TSB_ACT_SILU, 2, 3, 8, 8, x=P, ldx=8, ids=P, weights=P,
               units=C.addressof(u))
    a._keep = u
    if struct is abi.tsb_ffn_args:
        a.y, a.ldy = P, 8
    else:
        a.dy, a.lddy, a.dx, a.lddx = P, 8, P, 8
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def ffn_back(u=None, **kw):
    return ffn(u, abi.tsb_ffn_grad_args, **kw)


def refused(lib, fn, a, text):
    assert getattr(lib, fn)(C.byref(a)) == abi.SS_E_INVALID
    assert text.encode() in lib.ss_last_error(), lib.ss_last_error()
    assert fn.encode() in lib.ss_last_error()


@pytest.mark.parametrize("kw,text", [
    (dict(struct_size=8), "short argument struct"), (dict(dtype=abi.TSB_F32), "dtype"), (dict(act=9), "activation"),
    (dict(n=0), "n and k"), (dict(k=0), "n and k"), (dict(k=1 << 22), "n and k"), (dict(rows=1 << 28), "rows"),
    (dict(x=None), "null"), (dict(w=None), "null"), (dict(y=None), "null"), (dict(ldx=3), "leading dimension"),
    (dict(ldw=3), "leading dimension"), (dict(ldy=2), "leading dimension"),
    (dict(residual=P, ldr=2), "leading dimension"), (dict(pre=P, ldp=2), "leading dimension")])
def test_linear_refusals(lib, kw, text):
    refused(lib, "tsb_linear", linear(**kw), text)
    assert lib.tsb_linear_workspace(C.byref(linear(**kw))) == 0


@pytest.mark.parametrize("kw,text", [
    (dict(struct_size=8), "short argument struct"), (dict(dtype=7), "dtype"), (dict(act=5), "activation"),
    (dict(n=0), "n and k"), (dict(rows=1 << 28), "rows"), (dict(dy=None), "null"), (dict(x=None), "null"),
    (dict(w=None), "null"), (dict(act=abi.TSB_ACT_SILU), "pre"), (dict(lddy=2), "leading dimension"),
    (dict(lddx=3), "leading dimension"), (dict(lddw=3), "leading dimension"),
    (dict(act=abi.TSB_ACT_SILU, pre=P, ldp=1), "leading dimension"), (dict(), "workspace")])
def test_linear_backward_refusals(lib, kw, text):
    refused(lib, "tsb_linear_backward", linear_back(**kw), text)


def test_workspaces_are_asked_for_and_checked(lib):
    a = linear_back(act=abi.TSB_ACT_SILU, pre=P, ldp=3)
    n = lib.tsb_linear_backward_workspace(C.byref(a))
    assert n > 0
    a.workspace, a.workspace_bytes = P, n - 1
    refused(lib, "tsb_linear_backward", a, "smaller")
    a.workspace, a.workspace_bytes = P + 16, n
    refused(lib, "tsb_linear_backward", a, "256-byte")
    for fn, make in (("tsb_ffn", ffn), ("tsb_ffn_backward", ffn_back)):
        a = make()
        n = getattr(lib, fn + "_workspace")(C.byref(a))
        assert n > 0
        refused(lib, fn, a, "smaller")
        a.workspace, a.workspace_bytes = P + 16, n
        refused(lib, fn, a, "256-byte")


@pytest.mark.parametrize("fn,make", [("tsb_ffn", ffn), ("tsb_ffn_backward", ffn_back)])
@pytest.mark.parametrize("kw,text", [
    (dict(struct_size=8), "short argument struct"), (dict(dtype=abi.TSB_F32), "dtype"), (dict(act=9), "activation"),
    (dict(hidden=0), "hidden and ffn"), (dict(ffn=1 << 22), "hidden and ffn"), (dict(top=0), "top"),
    (dict(top=65), "top"), (dict(rows=1 << 28), "rows"), (dict(units=None), "units"), (dict(x=None), "null"),
    (dict(ids=None), "null"), (dict(weights=None), "null"), (dict(ldx=7), "leading dimension")])
def test_ffn_refusals(lib, fn, make, kw, text):
    refused(lib, fn, make(**kw), text)
    assert getattr(lib, fn + "_workspace")(C.byref(make(**kw))) == 0


@pytest.mark.parametrize("fn,make", [("tsb_ffn", ffn), ("tsb_ffn_backward", ffn_back)])
@pytest.mark.parametrize("kw,text", [(dict(struct_size=8), "units struct"), (dict(n_units=0), "n_units"),
                                     (dict(n_units=70000), "n_units"), (dict(n_slots=0), "no parts")])
def test_units_refusals(lib, fn, make, kw, text):
    refused(lib, fn, make(units(**kw)), text)


def test_units_need_their_parts_and_whole_elements(lib):
    u = units()
    u.part[1] = None
    refused(lib, "tsb_ffn", ffn(u), "no parts")
    u = units()
    u.stride[2] = 63
    refused(lib, "tsb_ffn", ffn(u), "whole elements")
    refused(lib, "tsb_ffn_backward", ffn_back(dgate=P), "go together")
    refused(lib, "tsb_ffn", ffn(ldy=7), "leading dimension")
    refused(lib, "tsb_ffn", ffn(y=None), "null")
    refused(lib, "tsb_ffn_backward", ffn_back(dy=None), "null")


@pytest.mark.parametrize("args,text", [
    ((3, P, 8, 1, 8, 2, 1, P, P), "dtype"), ((0, P, 8, 1, 0, 1, 1, P, P), "experts"),
    ((0, P, 2000, 1, 1025, 2, 1, P, P), "experts"), ((0, P, 8, 1, 8, 0, 1, P, P), "top"),
    ((0, P, 8, 1, 8, 9, 1, P, P), "top"), ((0, P, 64, 1, 64, 33, 1, P, P), "top"), ((0, None, 8, 1, 8, 2, 1, P, P), "null"),
    ((0, P, 8, 1, 8, 2, 1, None, P), "null"), ((0, P, 7, 1, 8, 2, 1, P, P), "leading dimension"),
    ((0, P, 8, 1 << 28, 8, 2, 1, P, P), "rows")])
def test_route_refusals(lib, args, text):
    assert lib.tsb_route(*args, None) == abi.SS_E_INVALID
    assert text.encode() in lib.ss_last_error()
    dt, z, ld, rows, experts, top, norm, ids, w = args
    assert lib.tsb_route_backward(dt, 2, P, z, ld, ids, w, rows, experts, top, 0, P, 8, None) == abi.SS_E_INVALID
    assert text.encode() in lib.ss_last_error()


def test_pointers_on_whole_elements(lib):
    refused(lib, "tsb_linear", linear(x=P + 1), "whole element")
    refused(lib, "tsb_linear", linear(bias=P + 1), "whole element")
    refused(lib, "tsb_linear_backward", linear_back(dy=P + 1), "whole element")
    refused(lib, "tsb_ffn", ffn(x=P + 1), "whole element")
    refused(lib, "tsb_ffn", ffn(ids=P + 2), "whole element")
    refused(lib, "tsb_ffn_backward", ffn_back(dweights=P + 1), "whole element")
    for kw in (dict(slot_of=P + 2), dict(table=P + 4), dict(absent_err=P + 1)):
        refused(lib, "tsb_ffn", ffn(units(**kw)), "whole element")
    assert lib.tsb_route(abi.TSB_F32, P + 2, 8, 1, 8, 2, 1, P, P, None) == abi.SS_E_INVALID
    assert lib.tsb_route(abi.TSB_BF16, P, 8, 1, 8, 2, 1, P + 2, P, None) == abi.SS_E_INVALID
    assert lib.tsb_route_backward(0, 2, P + 2, P, 8, P, P, 1, 8, 2, 1, P, 8, None) == abi.SS_E_INVALID


def test_no_rows_is_no_work(lib):
    """rows = 0 needs no workspace, no pointers and no device."""
    a = linear(rows=0, x=None, w=None, y=None)
    assert lib.tsb_linear_workspace(C.byref(a)) == 0 and lib.tsb_linear(C.byref(a)) == abi.SS_OK
    a = linear_back(rows=0, dw=None, db=None)
    assert lib.tsb_linear_backward_workspace(C.byref(a)) == 0 and lib.tsb_linear_backward(C.byref(a)) == abi.SS_OK
    a = ffn(rows=0, x=None, y=None)
    assert lib.tsb_ffn_workspace(C.byref(a)) == 0 and lib.tsb_ffn(C.byref(a)) == abi.SS_OK
    a = ffn_back(rows=0, x=None)
    assert lib.tsb_ffn_backward_workspace(C.byref(a)) == 0 and lib.tsb_ffn_backward(C.byref(a)) == abi.SS_OK
    assert lib.tsb_route(0, None, 8, 0, 8, 2, 1, None, None, None) == abi.SS_OK


def test_units_from_a_view(lib):
    v = abi.ss_dg_device_view(C.sizeof(abi.ss_dg_device_view), 1, 3, 3, 9, 10, P, P, P)
    for i in range(3):
        v.parts[i].base, v.parts[i].stride, v.parts[i].bytes = P + 256 * i, 512, 128
    u = abi.tsb_units()
    assert lib.tsb_units_from_view(C.byref(v), 2, 7, 128, C.byref(u)) == abi.SS_OK
    assert (u.n_units, u.n_slots, u.slot_of, u.unit_base, u.abort) == (7, 10, P, P + 8, P)
    assert [u.part[i] for i in range(3)] == [P, P + 256, P + 512] and list(u.stride) == [512] * 3
    assert lib.tsb_units_from_view(C.byref(v), 3, 7, 128, C.byref(u)) == abi.SS_E_INVALID
    assert lib.tsb_units_from_view(C.byref(v), 0, 7, 129, C.byref(u)) == abi.SS_E_INVALID
    v.n_parts = 2
    assert lib.tsb_units_from_view(C.byref(v), 0, 7, 128, C.byref(u)) == abi.SS_E_INVALID
    assert lib.tsb_units_from_view(None, 0, 7, 128, C.byref(u)) == abi.SS_E_INVALID


def test_struct_layouts_match_the_header():
    """The ctypes structs of the operators have the header's sizes and offsets."""
    import os
    import subprocess
    import tempfile
    root = os.path.dirname(os.path.dirname(os.path.abspath(abi.__file__)))
    structs = [abi.tsb_linear_args, abi.tsb_linear_grad_args, abi.tsb_units, abi.tsb_ffn_args, abi.tsb_ffn_grad_args]
    src = ["#include <stdio.h>", "#include <stddef.h>", '#include "tierstream/tsb.h"', "int main(void) {"]
    for s in structs:
        src.append('printf("%%zu\\n", sizeof(%s));' % s.__name__)
        src += ['printf("%%zu\\n", offsetof(%s, %s));' % (s.__name__, f[0]) for f in s._fields_]
    with tempfile.TemporaryDirectory() as d:
        c = os.path.join(d, "l.c")
        open(c, "w").write("\n".join(src + ["return 0; }"]))
        subprocess.run(["gcc", "-std=c11", "-I", os.path.join(root, "include"), c, "-o", os.path.join(d, "l")],
                       check=True)
        got = [int(x) for x in subprocess.run([os.path.join(d, "l")], capture_output=True, check=True).stdout.split()]
    want = []
    for s in structs:
        want.append(C.sizeof(s))
        want += [getattr(s, f[0]).offset for f in s._fields_]
    assert got == want


def test_tensors_that_do_not_fit_are_refused_on_the_host():
    """ops.py's checks of types, shapes, strides and devices raise ValueError naming the tensor, before any device work."""
    torch = pytest.importorskip("torch")
    from tierstream_b200 import ops
    x = torch.zeros((4, 16), dtype=torch.bfloat16)
    w = torch.zeros((8, 16), dtype=torch.bfloat16)
    g, d = torch.zeros((3, 8, 16), dtype=torch.bfloat16), torch.zeros((3, 16, 8), dtype=torch.bfloat16)
    i, p = torch.zeros((4, 2), dtype=torch.int32), torch.zeros((4, 2))
    y = torch.zeros((4, 8), dtype=torch.bfloat16)
    for call, text in (
            (lambda: ops.linear(x.float(), w), "x: Float is not served"), (lambda: ops.linear(x, w), "CUDA tensors"),
            (lambda: ops.linear(g, w), "x: two dimensions"), (lambda: ops.linear(x, 3), "w: a tensor is wanted"),
            (lambda: ops.linear(x, w.half()), "w: BFloat16 on the CPU is wanted, got Half"),
            (lambda: ops.linear(x, w[:, :8]), r"w: shape \[8, 16\] is wanted, got \[8, 8\]"),
            (lambda: ops.linear(x.T.contiguous().T, w), "x: the elements of a row must be adjacent"),
            (lambda: ops.linear(x[:1].expand(4, 16), w), "x: rows overlap"), (lambda: ops.linear(x, x[0]), "w: two dim"),
            (lambda: ops.linear(x, w, bias=x), r"bias: a contiguous BFloat16 of shape \[8\]"),
            (lambda: ops.linear(x, w, residual=x), "residual: shape"), (lambda: ops.linear(x, w, pre=x), "pre: shape"),
            (lambda: ops.linear(x, w, act="tanh"), "unknown activation"),
            (lambda: ops.linear_backward(x.double(), x, x), "dy: Double is not served"),
            (lambda: ops.linear_backward(y, x, w), "CUDA tensors"), (lambda: ops.linear_backward(y, x, x), "w: shape"),
            (lambda: ops.linear_backward(y, x[0], w), "x: two dimensions"),
            (lambda: ops.linear_backward(y, x, w, act="silu"), "pre: an activation"),
            (lambda: ops.route(x.double(), 2), "logits: Double"), (lambda: ops.route(g, 2), "logits: two dimensions"),
            (lambda: ops.route(x, 2), "CUDA tensors"), (lambda: ops.route(x, 17), "top: must be"),
            (lambda: ops.route(x, 0), "top: must be"), (lambda: ops.route_backward(p, x, i, p), "CUDA tensors"),
            (lambda: ops.route_backward(p, x, p, p), "ids: a contiguous Int"),
            (lambda: ops.route_backward(p[:2], x, i, p), "dweights: 4 rows"),
            (lambda: ops.Units(g, g, d), "CUDA tensors"), (lambda: ops.Units(g, g, g), "down: BFloat16 of shape"),
            (lambda: ops.Units(x, x, x), "gate: .slots"), (lambda: ops.Units(g.double(), g, d), "gate: Double"),
            (lambda: ops.Units(None, g, d), "gate: a tensor"), (lambda: ops.Units(g, g[:, :, ::2], d), "up: BFloat16"),
            (lambda: ops.Units(g, g.mT.contiguous().mT, d), "up: a slot's matrix must be contiguous"),
            (lambda: ops.Units(g, g, d, p), "slot_of: a contiguous Int")):
        with pytest.raises(ValueError, match=text):
            call()
