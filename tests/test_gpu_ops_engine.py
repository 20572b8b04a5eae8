"""The operators as an engine uses them with the streamed units: a stack of mixture-of-experts layers decodes over a
device-gated context (router logits, selection, export and wait of the chosen ids, gated block of the units in their
slots) whose units are mostly outside the slots, and a host-mode layer's units are found by address. Checked against 64-bit
forms that read the units from the model file's bytes."""
import ctypes as C
import os

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tierstream_b200 import abi, harness, ops, runtime, synth  # noqa: E402

T = torch.bfloat16
U16 = torch.finfo(T).eps / 2


def write_model(name, layers, units, hidden, ffn, seed):
    """A model file of normal weights: per unit gate, up [ffn][hidden] and down [hidden][ffn]; and the units."""
    size = hidden * ffn * 2
    m = synth.Model(os.path.join(harness.model_dir(), name), layers, units, (size,) * 3, seed=seed, with_hash=False)
    g = torch.Generator().manual_seed(seed)
    w = torch.randn((layers, units, 3, hidden * ffn), generator=g)
    w[:, :, :2] *= hidden ** -0.5
    w[:, :, 2] *= ffn ** -0.5
    w = w.to(T)
    with open(m.path, "wb") as f:
        f.write(w.view(torch.int16).numpy().tobytes())
    parts = (w[:, :, 0].view(layers, units, ffn, hidden), w[:, :, 1].view(layers, units, ffn, hidden),
             w[:, :, 2].view(layers, units, hidden, ffn))
    return m, [p.cuda() for p in parts]


def layer(x, ids, weights, gate, up, down):
    """x + sum of weighted blocks in 64 bits from a 16-bit x, and its tolerance: one rounding of the result, one of the
    block's middle, sums in 32 bits (2^-22 (K + 64) of the absolute sums)."""
    xd = x.double()
    s = 2.0 ** -22 * (gate.shape[1] + gate.shape[2] + 64)
    y, tol = xd.clone(), s * xd.abs()
    for r in range(x.shape[0]):
        for k in range(ids.shape[1]):
            a, b, c = (m[int(ids[r, k])].double() for m in (gate, up, down))
            g, u = a @ xd[r], b @ xd[r]
            h = g * torch.sigmoid(g) * u
            w = float(weights[r, k])
            y[r] += w * (c @ h)
            tol[r] += w * (c.abs() @ (U16 * h.abs() + 2.4 * s * (a.abs() @ xd[r].abs()) * (b.abs() @ xd[r].abs())))
    return y, U16 * y.abs() + tol


@pytest.mark.parametrize("rows,top", [(1, 2), (3, 2), (1, 1), (6, 4)])
def test_layers_decode_over_the_slot_cache(rows, top):
    """Per token, layer by layer: the ids and weights the stack chose, each layer's output against its 64-bit form, and the
    stack's own output against the same operators on the units' arrays, bit for bit."""
    layers, units, hidden, ffn = 3, 8, 256, 192
    m, parts = write_model("tsb-ops-%d-%d.bin" % (rows, top), layers, units, hidden, ffn, 5)
    g = torch.Generator(device="cuda").manual_seed(1)
    routers = (torch.randn((layers, units, hidden), generator=g, device="cuda") * hidden ** -0.5 * 2).to(T)
    run = harness.DgLayers(m, hidden, ffn, routers, rows=rows, top=top, residents_per_layer=2)
    try:
        un = [ops.Units(*(p[L] for p in parts)) for L in range(layers)]
        for t in range(8):
            x = torch.randn((rows, hidden), generator=g, device="cuda").to(T)
            out = run.step(x)
            for L in range(layers):
                logits = ops.linear(x, routers[L])
                ids, w = ops.route(logits, top)
                assert torch.equal(run.ids[L], ids) and torch.equal(run.weights[L], w), (t, L)
                want, tol = layer(x, ids, w, *(p[L] for p in parts))
                y = ops.ffn(x, ids, w, un[L], residual=x)
                err = (y.double() - want).abs()
                assert bool((err <= tol).all()), (t, L, float((err / tol).max()))
                x = y
            assert torch.equal(out, x), t
        st = run.ctx.stats()
        assert st["tokens"] == 8 and st["misses"] > 0 and st["fetched"] > 0
        assert abi.load().tsb_ops_timeouts() == 0
    finally:
        run.close()
        os.unlink(m.path)


def test_units_of_a_context_between_tokens():
    """ops.Units.of_context reads the slot table when the kernels run: resident units compute, absent ones are left out
    and reported in the context's word."""
    layers, units, hidden, ffn = 2, 6, 128, 64
    m, parts = write_model("tsb-ops-view.bin", layers, units, hidden, ffn, 9)
    routers = torch.zeros((layers, units, hidden), dtype=T, device="cuda")
    run = harness.DgLayers(m, hidden, ffn, routers, residents_per_layer=3)
    try:
        table = run.ctx.table(layers * units).reshape(layers, units)
        there = [int(u) for u in np.flatnonzero(table[1] >= 0)]
        gone = [int(u) for u in np.flatnonzero(table[1] < 0)]
        assert there and gone
        un = ops.Units.of_context(run.ctx, 1, units, hidden, ffn)
        word = torch.zeros(1, dtype=torch.int32, device="cuda")
        un.struct.absent_err = word.data_ptr()  # (the context's own word would fail its next token)
        x = torch.randn((2, hidden), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").to(T)
        ids = torch.tensor([[there[0], there[-1]], [there[0], gone[0]]], dtype=torch.int32, device="cuda")
        w = torch.tensor([[0.75, 0.25], [0.5, 0.5]], device="cuda")
        y = ops.ffn(x, ids, w, un, residual=x)
        assert word.item() == 1
        only = w.clone()
        only[1, 1] = 0.0
        want, tol = layer(x, ids, only, *(p[1] for p in parts))
        assert bool(((y.double() - want).abs() <= tol).all())
    finally:
        run.close()
        os.unlink(m.path)


def test_host_mode_units_by_address():
    """Host forward mode: an acquired layer's units, in persistent and ring slots, found through ss_layer_view.table_dev."""
    layers, units, hidden, ffn = 2, 6, 128, 192
    m, parts = write_model("tsb-ops-host.bin", layers, units, hidden, ffn, 11)
    tiers = ([abi.SS_TIER_RESIDENT] * 2 + [abi.SS_TIER_PINNED] * (units - 2)) * layers
    b = abi.budget_defaults()
    b.device_bytes, b.margin_gib, b.margin_fraction = 1 << 30, 1.0 / 1024, 0.0
    b.ring_slots, b.dynamic_slots_per_layer, b.host_pinned_bytes = 4, 2, 1 << 30
    o = abi.options_defaults()
    o.forward_mode, o.pin_planned = abi.SS_FORWARD_HOST, 0
    desc = runtime.Desc(m.desc(order="ranked"))
    ctx = runtime.HostContext(desc, runtime.Plan(desc, b, tiers=tiers), o)
    s = torch.cuda.Stream()
    g = torch.Generator(device="cuda").manual_seed(3)
    try:
        for rows in (1, 5, 40):
            x = torch.randn((rows, hidden), generator=g, device="cuda").to(T)
            ctx.begin()
            for L in range(layers):
                routed = [1, 3, 4]
                ids = torch.tensor([[routed[(r + k) % 3] for k in range(2)] for r in range(rows)], dtype=torch.int32,
                                   device="cuda")
                w = torch.rand((rows, 2), generator=g, device="cuda")
                s.wait_stream(torch.cuda.current_stream())
                ctx.routes(L, routed)
                v = ctx.acquire(L, s.cuda_stream)
                un = ops.Units.of_table(C.cast(v.table_dev, C.c_void_p).value, units, hidden, ffn)
                with torch.cuda.stream(s):
                    y = ops.ffn(x, ids, w, un, residual=x)
                ctx.release(L, s.cuda_stream)
                s.synchronize()
                want, tol = layer(x, ids, w, *(p[L] for p in parts))
                assert bool(((y.double() - want).abs() <= tol).all()), (rows, L)
            ctx.end()
    finally:
        ctx.close()
        os.unlink(m.path)
