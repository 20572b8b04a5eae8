"""The operators (ops.linear, ops.route, ops.ffn and their backward passes) against plain 64-bit forms, at the sizes,
strides and masks where they can go wrong.

Tolerances, elementwise: u |y| for the one rounding of the result (u = finfo.eps / 2, relative), u times the sum of
absolute products for every factor that is rounded to 16 bits between two products, and S = 2^-22 (K + 64) times the sums
of absolute products for sums of K terms held in 32 bits (each addition off by at most 2^-23 of a partial sum that the
absolute products bound, twice that to spare, and as much again for the library functions' few ulp)."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tierstream_b200 import abi, ops  # noqa: E402

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
ACTS = ["none", "silu", "gelu", "gelu_tanh", "relu"]


def slope(z, act):
    """f(z) and f'(z) in 64 bits."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    if act == "silu":
        p = torch.sigmoid(z)
        return z * p, p * (1 + z * (1 - p))
    if act == "gelu":
        p = 0.5 * (1 + torch.erf(z / math.sqrt(2)))
        return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (z + 0.044715 * z ** 3))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)


def close(got, want, tol, what=""):
    assert got.shape == want.shape
    err = (got.double() - want).abs()
    tiny = torch.finfo(got.dtype).smallest_normal
    bad = ~(err <= tol + tiny)
    assert not bad.any(), "%s: %d of %d off, worst %.3g over its tolerance" % (
        what, int(bad.sum()), bad.numel(), float((err / (tol + tiny)).nan_to_num(math.inf).max()))


def half(t):
    return torch.finfo(t).eps / 2


def fp32(k):
    return 2.0 ** -22 * (k + 64)


def rand(g, *shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def wide(t, extra, shift=0):
    """The same matrix with `extra` elements between its rows, `shift` elements into its storage."""
    rows, cols = t.shape
    b = torch.full((rows * (cols + extra) + shift + 64,), float("nan"), dtype=t.dtype, device=t.device)
    v = b[shift:shift + rows * (cols + extra)].view(rows, cols + extra)[:, :cols]
    v.copy_(t)
    return v


# ---- linear ----
LINEAR = [(1, 8, 64), (1, 1, 1), (1, 128, 4096), (2, 24, 40), (3, 1000, 520), (5, 129, 264), (7, 16, 8), (8, 512, 1024),
          (9, 40, 2056), (15, 264, 512), (16, 72, 136), (17, 256, 64), (31, 136, 392), (33, 520, 200), (64, 128, 64),
          (65, 1, 513), (70, 257, 255), (127, 264, 264), (128, 256, 128), (129, 136, 72), (200, 33, 31),
          (300, 776, 1032), (513, 512, 512), (12, 1001, 4096), (40, 2055, 1024), (100, 129, 8192), (250, 1000, 2048),
          (300, 333, 4096), (600, 1001, 512), (1100, 2056, 264)]


@pytest.mark.parametrize("rows,n,k", LINEAR)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_linear(rows, n, k, dtype):
    t = TYPES[dtype]
    g = gen(rows * 7919 + n * 31 + k)
    act = ACTS[(rows + n + k) % 5]
    x, w = rand(g, rows, k, dtype=t), rand(g, n, k, dtype=t, scale=k ** -0.5)
    bias = rand(g, n, dtype=t) if (rows + k) % 2 else None
    res = rand(g, rows, n, dtype=t) if (n + k) % 3 else None
    pre = torch.empty((rows, n), dtype=t, device="cuda")
    y = ops.linear(x, w, bias=bias, residual=res, act=act, pre=pre)
    z = x.double() @ w.double().T
    mag = x.double().abs() @ w.double().abs().T
    if bias is not None:
        z, mag = z + bias.double(), mag + bias.double().abs()
    want = slope(z, act)[0]
    rmag = mag if res is None else mag + res.double().abs()
    if res is not None:
        want = want + res.double()
    close(pre, z, half(t) * z.abs() + fp32(k) * mag, "pre")
    close(y, want, half(t) * want.abs() + 1.2 * fp32(k) * rmag, "y")  # every slope is below 1.2
    again = ops.linear(x, w, bias=bias, residual=res, act=act)
    assert torch.equal(again, y)


@pytest.mark.parametrize("rows", [1, 6, 40, 200])
@pytest.mark.parametrize("extra,shift", [(8, 0), (1, 0), (0, 1), (24, 8), (3, 5)])
def test_linear_strides(rows, extra, shift):
    """Rows apart, matrices off 16 bytes, and an output between other columns that stay as they were."""
    g = gen(rows + extra)
    n, k = 152, 328
    x, w, res = (rand(g, r, c, dtype=torch.bfloat16) for r, c in ((rows, k), (n, k), (rows, n)))
    plain = ops.linear(x, w, residual=res, act="silu")
    buf = torch.full((rows, n + extra + shift + 3), 7.0, dtype=torch.bfloat16, device="cuda")
    out = buf[:, shift:shift + n]
    ops.linear(wide(x, extra, shift), wide(w, extra, shift), residual=wide(res, extra, shift), act="silu", out=out)
    z = x.double() @ w.double().T
    want = slope(z, "silu")[0] + res.double()
    mag = x.double().abs() @ w.double().abs().T + res.double().abs()
    close(out, want, half(torch.bfloat16) * want.abs() + 1.2 * fp32(k) * mag)
    close(plain, want, half(torch.bfloat16) * want.abs() + 1.2 * fp32(k) * mag)
    assert (buf[:, :shift] == 7).all() and (buf[:, shift + n:] == 7).all()


def test_linear_in_place_residual_and_nan_rows():
    """The output may be the residual; a row of NaN stays in its own row."""
    g = gen(5)
    for rows in (3, 150):
        x, w = rand(g, rows, 256, dtype=torch.float16), rand(g, 64, 256, dtype=torch.float16, scale=0.06)
        res = rand(g, rows, 64, dtype=torch.float16)
        want = ops.linear(x, w, residual=res, act="gelu")
        y = res.clone()
        ops.linear(x, w, residual=y, act="gelu", out=y)
        assert torch.equal(y, want)
        x[1, 3] = float("nan")
        y = ops.linear(x, w, residual=res, act="gelu")
        assert torch.isnan(y[1]).all()
        keep = [r for r in range(rows) if r != 1]
        assert torch.equal(y[keep], want[keep])


def test_linear_largest_and_no_rows():
    """A product whose output has more than 2^31 bytes between its first and last element; no rows."""
    g = gen(9)
    x, w = rand(g, 70000, 64, dtype=torch.bfloat16), rand(g, 64, 64, dtype=torch.bfloat16)
    out = torch.empty((70000, 20000), dtype=torch.bfloat16, device="cuda")[:, 19000:19064]
    ops.linear(x, w, out=out)
    rows = torch.tensor([0, 1, 35000, 69998, 69999], device="cuda")
    z = x[rows].double() @ w.double().T
    mag = x[rows].double().abs() @ w.double().abs().T
    close(out[rows], z, half(torch.bfloat16) * z.abs() + fp32(64) * mag)
    assert ops.linear(x[:0], w).shape == (0, 64)


BACK = [(1, 8, 64), (2, 3, 5), (7, 129, 264), (9, 2048, 1024), (70, 4096, 264), (260, 1024, 2056), (1000, 512, 1032), (16, 72, 136), (64, 128, 64), (100, 257, 255), (129, 136, 520),
        (300, 776, 264), (513, 512, 256)]


@pytest.mark.parametrize("rows,n,k", BACK)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_linear_backward(rows, n, k, dtype):
    t = TYPES[dtype]
    g = gen(rows * 13 + n + k)
    act = ACTS[(rows + n) % 5]
    dy, x, w = rand(g, rows, n, dtype=t), rand(g, rows, k, dtype=t), rand(g, n, k, dtype=t, scale=k ** -0.5)
    pre = rand(g, rows, n, dtype=t, scale=2.0)
    dx, dw, db = ops.linear_backward(dy, x, w, act=act, pre=pre)
    dz = dy.double() * slope(pre.double(), act)[1]
    dmag = 1.2 * dy.double().abs()
    u = half(t)
    mid = u if act != "none" else 0.0  # dz is rounded between the products
    for name, got, want, mag, K in (("dx", dx, dz @ w.double(), dmag @ w.double().abs(), n),
                                    ("dw", dw, dz.T @ x.double(), dmag.T @ x.double().abs(), rows)):
        close(got, want, u * want.abs() + (mid + fp32(K) + 2.0 ** -20) * mag, name)
    close(db, dz.sum(0), u * dz.sum(0).abs() + (fp32(rows) + 2.0 ** -20) * dmag.sum(0), "db")
    a, b, c = ops.linear_backward(dy, x, w, act=act, pre=pre, need=("w",))
    assert a is None and c is None and torch.equal(b, dw)


@pytest.mark.parametrize("rows,n,k", [(2049, 300, 136), (2500, 64, 64), (5000, 200, 136), (3001, 40, 1003),
                                      (4100, 129, 261), (33000, 8, 8), (6007, 1, 3), (2113, 128, 1024)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_linear_backward_in_parts(rows, n, k, dtype):
    """A small matrix and many rows: dw's sum over the rows runs in parts."""
    test_linear_backward(rows, n, k, dtype)


def test_linear_backward_without_rows():
    w = torch.ones((5, 8), dtype=torch.float16, device="cuda")
    dx, dw, db = ops.linear_backward(w[:0, :5], w[:0], w)
    assert dx.shape == (0, 8) and not dw.any() and not db.any() and dw.shape == (5, 8)


@pytest.mark.parametrize("act", ACTS)
def test_slopes_far_out(act):
    """Values whose squares pass 32 bits, where the slopes end at 0 or 1: linear's backward pass and ffn's. (At 50 the
    exponential is off by 60 ulp at most, 2^-17 of it.)"""
    t = torch.bfloat16
    far = torch.tensor([50.0, 1e4, 1e13, 1e19, 1e25, 3e38], device="cuda")
    z = torch.cat([far, -far, torch.zeros(2, device="cuda")]).to(t)[None]
    dy = torch.ones_like(z)
    x, w = torch.ones((1, 8), dtype=t, device="cuda"), torch.zeros((z.shape[1], 8), dtype=t, device="cuda")
    db = ops.linear_backward(dy, x, w, act=act, pre=z)[2]
    want = slope(z[0].double(), act)[1]
    close(db, want, (half(t) + 2.0 ** -16) * want.abs())
    hidden, ffn, rows = 64, 40, 3
    g = gen(23)
    x = torch.full((rows, hidden), 1e10, dtype=t, device="cuda")
    gate = torch.full((1, ffn, hidden), 1e10, dtype=t, device="cuda")
    gate[:, ::2] *= -1
    up = torch.full((1, ffn, hidden), 1e-12, dtype=t, device="cuda")
    down, dy = rand(g, 1, hidden, ffn, dtype=t), rand(g, rows, hidden, dtype=t)
    ids, weights = torch.zeros((rows, 1), dtype=torch.int32, device="cuda"), torch.ones((rows, 1), device="cuda")
    for d in (64, 60):  # (60: the path for rows off 16 bytes)
        parts = gate[:, :, :d].contiguous(), up[:, :, :d].contiguous(), down[:, :d].contiguous()
        got = ops.ffn_backward(dy[:, :d], x[:, :d], ids, weights, ops.Units(*parts), act=act, need=("x",))["dx"]
        # g is +-6e21 or so: with slope s, dx = (dh u s) gate + (dh act(g)) up, both of moderate size next to 1e10
        dh = dy[:, :d].double() @ parts[2][0].double()
        gz, u = x[:, :d].double() @ parts[0][0].double().T, x[:, :d].double() @ parts[1][0].double().T
        f, s = slope(gz, act)
        terms = (dh * u * s, parts[0][0].double()), (dh * f, parts[1][0].double())
        want = sum(a @ b for a, b in terms)
        mag = sum(a.abs() @ b.abs() for a, b in terms)
        dmag = dy[:, :d].double().abs() @ parts[2][0].double().abs()
        dmag = sum((dmag * c.abs()) @ b.abs() for c, b in ((u * s, terms[0][1]), (f, terms[1][1])))
        close(got, want, half(t) * (want.abs() + mag) + 3 * fp32(d + ffn) * (mag + dmag), act)


def test_linear_gradient_by_differences():
    """The gradients of sum(dy * y) against central differences of the 64-bit form, along random directions."""
    g = gen(21)
    t = torch.float16
    x, w, b, dy = (rand(g, *s, dtype=t, scale=c) for s, c in (((40, 72), 1.0), ((56, 72), 0.12), ((56,), 1.0),
                                                               ((40, 56), 1.0)))
    pre = torch.empty((40, 56), dtype=t, device="cuda")
    ops.linear(x, w, bias=b, act="gelu_tanh", pre=pre)
    grads = ops.linear_backward(dy, x, w, act="gelu_tanh", pre=pre)

    def loss(x, w, b):
        return (dy.double() * slope(x @ w.T + b, "gelu_tanh")[0]).sum()
    base = [v.double() for v in (x, w, b)]
    for i, grad in enumerate(grads):
        for seed in range(3):
            d = torch.randn(base[i].shape, generator=gen(100 + seed), device="cuda", dtype=torch.float64)
            h = 1e-4
            up, down = list(base), list(base)
            up[i], down[i] = base[i] + h * d, base[i] - h * d
            want = float((loss(*up) - loss(*down)) / (2 * h))
            got = float((grad.double() * d).sum())
            # each gradient's entries are off by about 2 u of their size with random signs; u again for pre's rounding
            assert abs(got - want) <= 16 * half(t) * float((grad.double() * d).norm()) + 1e-6 * abs(want)


# ---- route ----
def plain_route(z, top, norm):
    z = z.double()
    z = torch.where(torch.isnan(z), -math.inf, z)
    z = z.clamp(max=torch.finfo(torch.float32).max)
    v, i = torch.sort(z, dim=1, descending=True, stable=True)
    v, i = v[:, :top], i[:, :top]
    shut = v == -math.inf
    m = torch.where(shut[:, :1], 0, v[:, :1])
    p = torch.where(shut, 0, torch.exp(v - m))
    s = p.sum(1, keepdim=True) if norm else torch.exp(z - m).sum(1, keepdim=True)
    return torch.where(shut, -1, i).to(torch.int32), torch.where(shut, 0, p / s)


ROUTE = [(1, 1, 1), (1, 8, 2), (3, 8, 8), (5, 31, 7), (9, 32, 32), (2, 33, 3), (17, 64, 6), (4, 100, 10), (33, 128, 8),
         (7, 256, 8), (2, 300, 32), (1000, 160, 6), (6, 512, 16), (3, 1000, 20), (5, 1024, 32)]


@pytest.mark.parametrize("rows,experts,top", ROUTE)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_route(rows, experts, top, dtype):
    for norm in (True, False):
        z = rand(gen(rows + experts), rows, experts, dtype=dtype, scale=2.0)  # 16-bit logits: many are equal
        ids, w = ops.route(z, top, norm=norm)
        want_ids, want = plain_route(z, top, norm)
        assert torch.equal(ids, want_ids)
        # a few ulp for expf, the division and a sum of at most 1024 positive terms by lanes
        close(w, want, (2.0 ** -20) * want)


def test_route_masks_ties_and_odd_values():
    z = torch.zeros((7, 40), device="cuda")
    z[0, ::2] = -0.0  # equal to +0: the lowest expert first
    z[1] = -math.inf
    z[2, 5:] = -math.inf
    z[3, 3] = math.nan
    z[3, 7] = math.inf
    z[4] = math.nan
    z[5] = torch.finfo(torch.float32).min  # the lowest finite value is not a mask
    z[6, 10], z[6, 20] = math.inf, math.inf
    for norm in (True, False):
        ids, w = ops.route(z, 8, norm=norm)
        want_ids, want = plain_route(z, 8, norm)
        assert torch.equal(ids, want_ids)
        close(w, want, 2.0 ** -20 * want)
    assert ids[1].tolist() == [-1] * 8 and not w[1].any() and ids[2].tolist() == [0, 1, 2, 3, 4, -1, -1, -1]
    assert ids[0].tolist() == list(range(8)) and ids[5].tolist() == list(range(8))
    wide_z = torch.full((7, 64), 9.0, device="cuda")
    wide_z[:, 3:43] = z
    ids2, w2 = ops.route(wide_z[:, 3:43], 8, norm=False)
    assert torch.equal(ids2, ids) and torch.equal(w2, w)
    assert ops.route(z[:0], 3)[0].shape == (0, 3)


@pytest.mark.parametrize("experts,apart", [(1024, 32), (1001, 32), (512, 32), (257, 16), (96, 32), (1024, 1)])
def test_route_with_the_largest_far_apart(experts, apart):
    """The largest logits at equal distances (one lane's, a few lanes'), among equal, rising, falling and negative ones."""
    j = torch.arange(experts, device="cuda")
    on = j % apart == 5 % apart
    rows = [torch.where(on, 2.0, 1.0), torch.where(on, 3.0 + j / 64, 1.0), torch.where(on, 99.0 - j / 64, j / 1e4),
            torch.where(on, -1.0 - j % 3, -8.0), torch.where(on, (j // apart % 2).float(), -0.0),
            torch.where(on, 2.0, -math.inf), torch.zeros(experts, device="cuda")]
    z = torch.stack([r.float() for r in rows])
    top = min(32, experts)
    for t in (torch.float32, torch.float16):
        for norm in (True, False):
            ids, w = ops.route(z.to(t), top, norm=norm)
            want_ids, want = plain_route(z.to(t), top, norm)
            assert torch.equal(ids, want_ids)
            close(w, want, 2.0 ** -20 * want)


@pytest.mark.parametrize("rows,experts,top", ROUTE)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_route_backward(rows, experts, top, dtype):
    """Against autograd through the 64-bit softmax, masked experts among them."""
    g = gen(experts)
    z = rand(g, rows, experts, dtype=dtype, scale=2.0)
    z.masked_fill_(torch.rand((rows, experts), generator=g, device="cuda") < 0.2, -math.inf)
    for norm in (True, False):
        ids, w = ops.route(z, top, norm=norm)
        dw = torch.randn((rows, top), generator=g, device="cuda").to(torch.bfloat16 if norm else torch.float32)
        got = ops.route_backward(dw, z, ids, w, norm=norm)
        leaf = z.double().masked_fill(z == -math.inf, -1e4).requires_grad_(True)
        there = ids >= 0
        v = torch.where(there, leaf.gather(1, ids.long().clamp(min=0)), -1e9)
        over = torch.logsumexp(v if norm else leaf, 1, keepdim=True)
        p = torch.where(there, torch.exp(v - over), 0)
        want, = torch.autograd.grad((p * dw.double()).sum(), leaf)
        full = torch.exp(leaf.detach() - over.detach()).clamp(max=1)
        mag = full * (dw.double().abs().amax(1, keepdim=True) * 2)  # p (|dw| + sum |dw| p)
        close(got, want, half(dtype) * want.abs() + 2.0 ** -19 * mag)


# ---- the gated feed-forward block ----
def problem(seed, rows, hidden, ffn, units, top, t, holes=0.0, skew=0.0):
    """x, ids, weights and units in slots of no order; `holes` of the ids are outside the units, `skew` of the rows go
    to unit 0."""
    g = gen(seed)
    s = units + 2
    gate, up = (rand(g, s, ffn, hidden, dtype=t, scale=hidden ** -0.5) for _ in range(2))
    down = rand(g, s, hidden, ffn, dtype=t, scale=ffn ** -0.5)
    slot_of = torch.randperm(s, generator=g, device="cuda")[:units].to(torch.int32)
    x = rand(g, rows, hidden, dtype=t)
    ids = torch.argsort(torch.rand((rows, units), generator=g, device="cuda"), dim=1)[:, :top].to(torch.int32)
    if ids.shape[1] < top:  # more choices than units: the same unit twice
        ids = torch.randint(0, units, (rows, top), generator=g, device="cuda", dtype=torch.int32)
    ids = torch.where(torch.rand((rows, 1), generator=g, device="cuda") < skew, torch.zeros_like(ids), ids)
    out = torch.rand((rows, top), generator=g, device="cuda")
    ids = torch.where(out < holes / 2, -1, torch.where(out < holes, units + 5, ids)).to(torch.int32).contiguous()
    w = torch.rand((rows, top), generator=g, device="cuda")
    return x, ids, w, ops.Units(gate, up, down, slot_of), (gate, up, down, slot_of)


def plain_ffn(x, ids, w, parts, act, res=None):
    """y, and the tolerance of one that rounds act(g) u once and sums in 32 bits."""
    gate, up, down, slot_of = parts
    u = half(x.dtype)
    hidden, ffn = x.shape[1], gate.shape[1]
    s = fp32(hidden + ffn)
    xd = x.double()
    y, tol = torch.zeros_like(xd), torch.zeros_like(xd)
    if res is not None:
        y += res.double()
        tol += s * res.double().abs()
    for e in range(slot_of.numel()):
        slot = int(slot_of[e])
        r, k = torch.nonzero(ids == e, as_tuple=True)
        if not r.numel() or not 0 <= slot < gate.shape[0]:
            continue
        a, b, c = gate[slot].double(), up[slot].double(), down[slot].double()
        gg, uu = xd[r] @ a.T, xd[r] @ b.T
        ga, ua = xd[r].abs() @ a.abs().T, xd[r].abs() @ b.abs().T
        h = slope(gg, act)[0] * uu
        wk = w[r, k].double()[:, None]
        y.index_add_(0, r, wk * (h @ c.T))
        tol.index_add_(0, r, wk * ((u * h.abs() + 2.4 * s * ga * ua) @ c.abs().T))
    return y, u * y.abs() + tol


FFN = [(1, 8, 8, 1, 1), (1, 64, 128, 4, 2), (1, 512, 1408, 8, 2), (2, 72, 40, 3, 3), (4, 128, 64, 16, 2),
       (5, 33, 17, 4, 2), (7, 264, 520, 8, 4), (16, 256, 136, 2, 2), (24, 128, 192, 64, 8), (33, 100, 60, 5, 2),
       (65, 512, 256, 4, 1), (130, 264, 392, 3, 2), (200, 128, 256, 2, 5), (300, 256, 512, 40, 6), (700, 136, 264, 7, 3),
       (1500, 64, 72, 3, 2), (1200, 136, 264, 1, 1), (2100, 128, 72, 2, 1), (33, 72, 2056, 2, 1)]


@pytest.mark.parametrize("rows,hidden,ffn,units,top", FFN)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_ffn(rows, hidden, ffn, units, top, dtype):
    t = TYPES[dtype]
    act = ACTS[(rows + hidden) % 5]
    x, ids, w, un, parts = problem(rows + ffn, rows, hidden, ffn, units, top, t, holes=0.2 if rows % 2 else 0.0)
    res = rand(gen(1), rows, hidden, dtype=t) if rows % 3 else None
    y = ops.ffn(x, ids, w, un, act=act, residual=res)
    want, tol = plain_ffn(x, ids, w, parts, act, res)
    close(y, want, tol)
    assert torch.equal(ops.ffn(x, ids, w, un, act=act, residual=res), y)


@pytest.mark.parametrize("rows,hidden,ffn,units,top", [
    (65, 1024, 1032, 4, 1), (130, 1032, 264, 3, 2), (200, 1288, 264, 2, 5), (333, 520, 264, 9, 2), (515, 392, 520, 5, 1),
    (1500, 72, 328, 3, 2), (1201, 136, 520, 1, 1), (2100, 264, 136, 2, 1), (90, 2056, 72, 1, 6)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_ffn_long(rows, hidden, ffn, units, top, dtype):
    """More rows by units than are worth streaming."""
    test_ffn(rows, hidden, ffn, units, top, dtype)


@pytest.mark.parametrize("rows,hidden,ffn", [(3, 64, 136), (40, 128, 264), (400, 256, 264)])
def test_ffn_uneven_groups_and_empty_rows(rows, hidden, ffn):
    """Most rows in one unit, some units without rows, rows whose every id is outside, strided x, residual and y."""
    t = torch.bfloat16
    x, ids, w, un, parts = problem(3, rows, hidden, ffn, 9, 3, t, holes=0.1, skew=0.7)
    ids[0] = -1
    ids[rows - 1] = 2 ** 31 - 1
    x[0] = float("nan")  # a padded row's garbage
    w[0] = float("inf")
    res = rand(gen(2), rows, hidden, dtype=t)
    buf = torch.full((rows, hidden + 24), 5.0, dtype=t, device="cuda")
    y = ops.ffn(wide(x, 16), ids, w, un, residual=wide(res, 8), out=buf[:, 8:8 + hidden])
    want, tol = plain_ffn(x, ids, w, parts, "silu", res)
    assert torch.equal(y[0], res[0]) and torch.equal(y[rows - 1], res[rows - 1])
    close(y[1:], want[1:], tol[1:])
    assert (buf[:, :8] == 5).all() and (buf[:, 8 + hidden:] == 5).all()
    none = ops.ffn(x, torch.full_like(ids, -1), w, un)
    assert not none.any()


@pytest.mark.parametrize("rows", [2, 300])
def test_ffn_units_that_are_not_there(rows):
    """A slot outside the arrays leaves its rows out and sets the word; an abort leaves all out; a zero address too."""
    x, ids, w, un, parts = problem(8, rows, 128, 136, 6, 2, torch.float16)
    gate, up, down, slot_of = parts
    ids[0, 0] = 4
    slot_of = slot_of.clone()
    slot_of[4] = -1
    un = ops.Units(gate, up, down, slot_of)
    word = torch.zeros(2, dtype=torch.int32, device="cuda")
    un.struct.absent_err = word.data_ptr()
    y = ops.ffn(x, ids, w, un)
    want, tol = plain_ffn(x, ids, w, (gate, up, down, slot_of), "silu")
    close(y, want, tol)
    assert word.tolist() == [1, 0]
    g = ops.ffn_backward(x, x, ids, w, un)
    assert not g["dgate"][4].any() and not g["ddown"][4].any() and not g["dweights"][ids == 4].any()
    word[1] = 1
    un.struct.abort = word.data_ptr() + 4
    assert not ops.ffn(x, ids, w, un).any()
    # the same units found by address
    size = 128 * 136 * 2
    blob = torch.cat([torch.cat([gate[s].reshape(-1), up[s].reshape(-1), down[s].reshape(-1)])[None]
                      for s in range(gate.shape[0])])
    table = torch.tensor([blob.data_ptr() + 3 * size * int(s) if s >= 0 else 0 for s in slot_of], dtype=torch.int64,
                         device="cuda")
    t = ops.Units.of_table(table.data_ptr(), 6, 128, 136, dtype=torch.float16)
    close(ops.ffn(x, ids, w, t), want, tol)


@pytest.mark.parametrize("rows", [2500, 4000])
def test_ffn_units_that_are_not_there_in_long_groups(rows):
    test_ffn_units_that_are_not_there(rows)


def plain_back(dy, x, ids, w, parts, act):
    """Gradients and tolerances: dg, du and w act(g) u rounded once, sums in 32 bits."""
    gate, up, down, slot_of = parts
    u = half(x.dtype)
    hidden, ffn, units = x.shape[1], gate.shape[1], slot_of.numel()
    s = fp32(hidden + ffn) + 2.0 ** -20
    xd, yd = x.double(), dy.double()
    z = {"dx": torch.zeros_like(xd), "dweights": torch.zeros(ids.shape, dtype=torch.float64, device="cuda"),
         "dgate": torch.zeros((units, ffn, hidden), dtype=torch.float64, device="cuda")}
    z["dup"], z["ddown"] = torch.zeros_like(z["dgate"]), torch.zeros_like(z["dgate"]).mT.contiguous()
    tol = {n: torch.zeros_like(v) for n, v in z.items()}
    for e in range(units):
        slot = int(slot_of[e])
        r, k = torch.nonzero(ids == e, as_tuple=True)
        if not r.numel() or not 0 <= slot < gate.shape[0]:
            continue
        a, b, c = gate[slot].double(), up[slot].double(), down[slot].double()
        gg, uu, dh = xd[r] @ a.T, xd[r] @ b.T, yd[r] @ c
        ga, ua, da = xd[r].abs() @ a.abs().T, xd[r].abs() @ b.abs().T, yd[r].abs() @ c.abs()
        f, df = slope(gg, act)
        wk = w[r, k].double()[:, None]
        dg, du, hw = wk * dh * uu * df, wk * dh * f, wk * f * uu
        # 32-bit errors of g, u and dh: at most S of their absolute sums each, through slopes below 1.2 and a second
        # derivative below 1.2
        eg, eu, eh = 1.2 * s * wk * da * ua * (3 + ga), 3.6 * s * wk * da * ga, 3.6 * s * wk * ga * ua
        z["dx"].index_add_(0, r, dg @ a + du @ b)
        tol["dx"].index_add_(0, r, (u * dg.abs() + 2 * eg) @ a.abs() + (u * du.abs() + 2 * eu) @ b.abs())
        z["dweights"][r, k] = (dh * f * uu).sum(1)
        tol["dweights"][r, k] = (6 * s * da * ga * ua).sum(1)
        z["dgate"][e], z["dup"][e], z["ddown"][e] = dg.T @ xd[r], du.T @ xd[r], yd[r].T @ hw
        n = r.numel()
        tol["dgate"][e] = (u * dg.abs() + 2 * eg + fp32(n) * dg.abs()).T @ xd[r].abs()
        tol["dup"][e] = (u * du.abs() + 2 * eu + fp32(n) * du.abs()).T @ xd[r].abs()
        tol["ddown"][e] = yd[r].abs().T @ (u * hw.abs() + 2 * eh + fp32(n) * hw.abs())
    return z, {n: u * z[n].abs() + tol[n] for n in z}


@pytest.mark.parametrize("rows,hidden,ffn,units,top", FFN)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_ffn_backward(rows, hidden, ffn, units, top, dtype):
    t = TYPES[dtype]
    act = ACTS[(rows + hidden) % 5]
    x, ids, w, un, parts = problem(rows + ffn, rows, hidden, ffn, units, top, t, holes=0.2 if rows % 2 else 0.0)
    dy = rand(gen(4), rows, hidden, dtype=t)
    got = ops.ffn_backward(dy, x, ids, w, un, act=act)
    want, tol = plain_back(dy, x, ids, w, parts, act)
    for n in want:
        close(got[n], want[n], tol[n], n)
    some = ops.ffn_backward(dy, x, ids, w, un, act=act, need=("x", "weights"))
    assert torch.equal(some["dx"], got["dx"]) and torch.equal(some["dweights"], got["dweights"])
    assert some["dgate"] is None and some["dup"] is None and some["ddown"] is None


def test_ffn_backward_padded_rows_and_none():
    """Padded rows full of NaN leave every gradient as if they were absent; no rows zero the units' gradients."""
    x, ids, w, un, parts = problem(6, 90, 128, 192, 5, 2, torch.bfloat16)
    dy = rand(gen(4), 90, 128, dtype=torch.bfloat16)
    want = ops.ffn_backward(dy[:70], x[:70], ids[:70].contiguous(), w[:70].contiguous(), un)
    ids[70:] = -1
    x[70:], dy[70:], w[70:] = math.nan, math.inf, math.nan
    got = ops.ffn_backward(dy, x, ids, w, un)
    assert torch.equal(got["dx"][:70], want["dx"]) and not got["dx"][70:].any()
    assert torch.equal(got["dweights"][:70], want["dweights"]) and not got["dweights"][70:].any()
    for n in ("dgate", "dup", "ddown"):
        assert torch.equal(got[n], want[n])
    g = ops.ffn_backward(dy[:0], x[:0], ids[:0], w[:0], un)
    assert g["dx"].shape == (0, 128) and not g["dgate"].any() and not g["dup"].any() and not g["ddown"].any()


def test_ffn_gradient_by_differences():
    t = torch.float16
    x, ids, w, un, parts = problem(31, 60, 64, 72, 4, 2, t)
    gate, up, down, slot_of = parts
    dy = rand(gen(4), 60, 64, dtype=t)
    got = ops.ffn_backward(dy, x, ids, w, un, act="gelu")
    at = slot_of.long()

    def loss(v):
        y = torch.zeros((60, 64), dtype=torch.float64, device="cuda")
        for e in range(4):
            r, k = torch.nonzero(ids == e, as_tuple=True)
            h = slope(v["dx"][r] @ v["dgate"][e].T, "gelu")[0] * (v["dx"][r] @ v["dup"][e].T)
            y.index_add_(0, r, v["dweights"][r, k][:, None] * (h @ v["ddown"][e].T))
        return (dy.double() * y).sum()
    base = {"dx": x.double(), "dweights": w.double(), "dgate": gate[at].double(), "dup": up[at].double(),
            "ddown": down[at].double()}
    for n in base:
        for seed in range(2):
            d = torch.randn(base[n].shape, generator=gen(50 + seed), device="cuda", dtype=torch.float64)
            h = 1e-4
            want = float((loss({**base, n: base[n] + h * d}) - loss({**base, n: base[n] - h * d})) / (2 * h))
            g = got[n].double() * d
            # entries off by about 2 u of their size with random signs (the result's rounding and one before it)
            assert abs(float(g.sum()) - want) <= 16 * half(t) * float(g.norm()) + 1e-6 * abs(want), n


@pytest.mark.parametrize("rows", [2, 40, 1100])
def test_ffn_units_far_apart(rows):
    """Slots more than 2^32 bytes apart, in one allocation: forward and backward find the unit in the last one."""
    t, hidden, ffn = torch.bfloat16, 128, 72
    g = gen(17)
    size = hidden * ffn
    apart = (1 << 31) + 256  # elements between slots: 4 GiB and 512 bytes
    buf = torch.empty(apart * 2 + 3 * size, dtype=t, device="cuda")
    gate, up = (torch.as_strided(buf, (3, ffn, hidden), (apart, hidden, 1), o) for o in (0, size))
    down = torch.as_strided(buf, (3, hidden, ffn), (apart, ffn, 1), 2 * size)
    for m, k in ((gate, hidden), (up, hidden), (down, ffn)):
        m.copy_(rand(g, *m.shape, dtype=t, scale=k ** -0.5))
    slot_of = torch.tensor([2, 0], dtype=torch.int32, device="cuda")
    x, dy = rand(g, rows, hidden, dtype=t), rand(g, rows, hidden, dtype=t)
    ids = torch.zeros((rows, 1), dtype=torch.int32, device="cuda")
    ids[0] = 1
    w = torch.rand((rows, 1), generator=g, device="cuda")
    parts = (gate, up, down, slot_of)
    un = ops.Units(*parts)
    want, tol = plain_ffn(x, ids, w, parts, "silu")
    close(ops.ffn(x, ids, w, un), want, tol)
    got = ops.ffn_backward(dy, x, ids, w, un)
    want, tol = plain_back(dy, x, ids, w, parts, "silu")
    for n in want:
        close(got[n], want[n], tol[n], n)


# ---- streams, graphs, and the operators together ----
def test_on_another_stream_and_captured():
    """A layer (logits, route, block with its residual) on a side stream, captured into two graphs that are replayed with
    new inputs in between and at the same time, equals the eager calls bit for bit."""
    t = torch.bfloat16
    for rows in (1, 6, 200):
        x, _, _, un, parts = problem(rows, rows, 256, 264, 8, 2, t)
        wr = rand(gen(1), 8, 256, dtype=t, scale=0.06)

        def layer(x):
            ids, w = ops.route(ops.linear(x, wr), 2)
            return ops.ffn(x, ids, w, un, residual=x)
        xs = [x.clone(), x.flip(0).contiguous()]
        side = [torch.cuda.Stream() for _ in range(2)]
        graphs, outs = [], []
        for s, xi in zip(side, xs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                layer(xi)
            s.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                outs.append(layer(xi))
            graphs.append(g)
        for step in range(3):
            news = [rand(gen(77 + step + 10 * i), rows, 256, dtype=t) for i in range(2)]
            for xi, new in zip(xs, news):
                xi.copy_(new)
            torch.cuda.synchronize()
            for s, g in zip(side, graphs):
                with torch.cuda.stream(s):
                    g.replay()
            torch.cuda.synchronize()
            for out, new in zip(outs, news):
                assert torch.equal(out, layer(new))


def test_captured_behind_copies_and_fills():
    """A captured call right behind a fill and a copy of its inputs sees them; one in place on x as its own residual."""
    t = torch.bfloat16
    x, ids, w, un, parts = problem(4, 40, 128, 136, 5, 2, t)
    src = x.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        want = ops.ffn(src, ids, w, un, residual=src)
        lin = ops.linear(torch.zeros_like(src), parts[0][0])
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    y = torch.empty_like(x)
    with torch.cuda.graph(g, stream=s):
        y.zero_()
        z = ops.linear(y, parts[0][0])
        x.copy_(src)
        ops.ffn(x, ids, w, un, residual=x, out=x)
    for _ in range(3):
        x.fill_(9.0)
        y.fill_(9.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            g.replay()
        s.synchronize()
        assert torch.equal(x, want) and torch.equal(z, lin)


def test_ops_from_two_threads():
    """Two threads on streams of their own, the same units and different inputs: each gets its own results."""
    import threading
    t = torch.bfloat16
    jobs = []
    for k, rows in enumerate((3, 170)):
        x, ids, w, un, _ = problem(40 + k, rows, 256, 264, 6, 2, t)
        jobs.append((x, ids, w, un, ops.ffn(x, ids, w, un, residual=x), []))
    torch.cuda.synchronize()

    def work(x, ids, w, un, want, bad):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            got = [ops.ffn(x, ids, w, un, residual=x) for _ in range(40)]
        s.synchronize()
        bad += [i for i, y in enumerate(got) if not torch.equal(y, want)]
    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert all(not j[-1] for j in jobs)


def test_backward_captured():
    t = torch.bfloat16
    x, ids, w, un, parts = problem(5, 150, 128, 264, 6, 2, t)
    dy = rand(gen(4), 150, 128, dtype=t)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        want = ops.ffn_backward(dy, x, ids, w, un)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        got = ops.ffn_backward(dy, x, ids, w, un)
    for _ in range(2):
        for v in got.values():
            v.fill_(3.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            g.replay()
        s.synchronize()
        for n in want:
            assert torch.equal(got[n], want[n]), n


def test_a_layer_forward_and_backward():
    """Logits, route and block in a row and back: the gradient of x through all three against differences of the 64-bit
    layer whose ids are held."""
    t = torch.float16
    rows, hidden, ffn, units, top = 50, 64, 136, 6, 2
    x, _, _, un, parts = problem(2, rows, hidden, ffn, units, top, t)
    wr = rand(gen(9), units, hidden, dtype=t, scale=0.12)
    dy = rand(gen(10), rows, hidden, dtype=t)
    z = ops.linear(x, wr)
    ids, w = ops.route(z, top)
    ops.ffn(x, ids, w, un, residual=x)
    g = ops.ffn_backward(dy, x, ids, w, un, need=("x", "weights"))
    dz = ops.route_backward(g["dweights"], z, ids, w)
    dxr, _, _ = ops.linear_backward(dz, x, wr, need=("x",))
    got = dy.double() + g["dx"].double() + dxr.double()
    gate, up, down, slot_of = parts

    def loss(xd):
        v = (xd @ wr.double().T).gather(1, ids.long())
        p = torch.softmax(v, 1)
        y = xd.clone()
        for e in range(units):
            r, k = torch.nonzero(ids == e, as_tuple=True)
            s = int(slot_of[e])
            h = slope(xd[r] @ gate[s].double().T, "silu")[0] * (xd[r] @ up[s].double().T)
            y = y.index_add(0, r, p[r, k][:, None] * (h @ down[s].double().T))
        return (dy.double() * y).sum()
    for seed in range(3):
        d = torch.randn((rows, hidden), generator=gen(60 + seed), device="cuda", dtype=torch.float64)
        h = 1e-4
        want = float((loss(x.double() + h * d) - loss(x.double() - h * d)) / (2 * h))
        # logits rounded to 16 bits move the weights by 2 u of them; then as above, three operators' roundings
        assert abs(float((got * d).sum()) - want) <= 64 * half(t) * float((got * d).norm())


@pytest.mark.parametrize("rows", [3, 40, 300])
def test_outputs_beside_inputs(rows):
    """Outputs in other columns of the inputs' buffer are served, outputs that share elements with an input refused."""
    t, n, k = torch.bfloat16, 64, 72
    g = gen(rows)
    buf = rand(g, rows, 2 * n + k + 16, dtype=t)
    x, out, pre = buf[:, 8:8 + k], buf[:, 8 + k:8 + k + n], buf[:, 8 + k + n:8 + k + 2 * n]
    w, bias = rand(g, n, k, dtype=t), rand(g, n, dtype=t)
    edges = buf[:, :8].clone(), buf[:, -8:].clone()
    want_pre = torch.empty((rows, n), dtype=t, device="cuda")
    want = ops.linear(x.clone(), w, bias=bias, act="gelu", pre=want_pre)
    ops.linear(x, w, bias=bias, act="gelu", pre=pre, out=out)
    assert torch.equal(out, want) and torch.equal(pre, want_pre)
    assert torch.equal(buf[:, :8], edges[0]) and torch.equal(buf[:, -8:], edges[1])
    res = rand(g, rows, n, dtype=t)
    flat = rand(g, rows * n, dtype=t)
    for bad in (lambda: ops.linear(x, w, out=buf[:, k:k + n]), lambda: ops.linear(x, w, pre=buf[:, k:k + n]),
                lambda: ops.linear(x, w, out=out, pre=buf[:, 9 + k:9 + k + n]), lambda: ops.linear(x, w, residual=res, pre=res),
                lambda: ops.linear(x, w, bias=flat[:n], out=flat.view(rows, n)),
                lambda: ops.linear(x, w, bias=flat[-n:], pre=flat.view(rows, n))):
        with pytest.raises(ValueError):
            bad()
    ids, p = torch.zeros((rows, 1), dtype=torch.int32, device="cuda"), torch.ones((rows, 1), device="cuda")
    un = ops.Units(*(rand(g, 1, a, b, dtype=t) for a, b in ((24, k), (24, k), (k, 24))))
    big = torch.zeros((rows, k), dtype=t, device="cuda")
    with pytest.raises(ValueError):
        ops.ffn(x, big.view(torch.int32).view(-1)[:rows].view(rows, 1), p, un, out=big)
    assert torch.equal(ops.ffn(x, ids, p, un, out=big), ops.ffn(x.clone(), ids, p, un))


def test_refusals_on_tensors():
    t = torch.bfloat16
    x = torch.zeros((4, 16), dtype=t, device="cuda")
    w = torch.zeros((8, 16), dtype=t, device="cuda")
    ids = torch.zeros((4, 2), dtype=torch.int32, device="cuda")
    p = torch.zeros((4, 2), device="cuda")
    un = ops.Units(torch.zeros((3, 8, 16), dtype=t, device="cuda"), torch.zeros((3, 8, 16), dtype=t, device="cuda"),
                   torch.zeros((3, 16, 8), dtype=t, device="cuda"))
    for bad in (lambda: ops.linear(x.float(), w), lambda: ops.linear(x, w.half()), lambda: ops.linear(x, w[:, :8]),
                lambda: ops.linear(x.T.contiguous().T, w), lambda: ops.linear(x, w.cpu()),
                lambda: ops.linear(x, w, act="tanh"), lambda: ops.linear(x, w, bias=x),
                lambda: ops.linear(x[:1].expand(4, 16), w), lambda: ops.linear(x[0], w),
                lambda: ops.linear(x, w, residual=x), lambda: ops.linear_backward(x, x, w),
                lambda: ops.linear_backward(x[:, :8], x, w, act="silu"), lambda: ops.route(x.double(), 2),
                lambda: ops.ffn(x, ids.long(), p, un), lambda: ops.ffn(x, ids, p.half(), un),
                lambda: ops.ffn(x[:, :8], ids, p, un), lambda: ops.ffn(x.half(), ids, p, un),
                lambda: ops.ffn(x, ids.T, p, un),
                lambda: ops.Units(un.keep[0], un.keep[1], un.keep[1]),
                lambda: ops.Units(un.keep[0], un.keep[1], un.keep[2], ids.float()), lambda: ops.route(x, 17),
                lambda: ops.route(x, 0), lambda: ops.linear(x, torch.zeros((16, 16), dtype=t, device="cuda"), out=x),
                lambda: ops.ffn(x, ids, p, un, out=x), lambda: ops.ffn(x, ids, p, un, residual=x, out=x[:2]),
                lambda: ops.route_backward(p, x[:2], ids, p),
                lambda: ops.linear(x[:, :8], w[:, :8], residual=w[:4, :8], out=w[1:5, :8]),
                lambda: ops.ffn(x[:2], ids[:2], p[:2], un, residual=x[1:3], out=x[2:4])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(abi.TsError):  # the library's own refusals
        ops.ffn(x, torch.zeros((4, 65), dtype=torch.int32, device="cuda"), torch.zeros((4, 65), device="cuda"), un)
