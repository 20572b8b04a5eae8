"""Per-kernel rates through the C ABI, each timed with CUDA events on the launching stream after warm-up, with inputs
larger than L2: the land kernel (K1: one tsb_land launch per repetition) for pinned host -> HBM, HBM -> pinned host
and HBM -> HBM, the move kernel (K4: one tsb_move launch, HBM -> HBM, `--kernel move`), and the device xxh64 (K3: tsb_xxh64_units) for one unit alone (its serial chain) and for many
units at once (aggregate). Also the small cases the committed ncu summaries were captured on. The operators of ops.py
(linear, route, ffn; --back: their backward passes) are timed the same way, one call a repetition.

    python -m tierstream_b200.kernel_bench land --dir h2d --part-bytes 33030144 --parts 15
    python -m tierstream_b200.kernel_bench xxh64 --units 296 --part-bytes 12582912
    python -m tierstream_b200.kernel_bench ffn --rows 24 --hidden 4096 --ffn 1536 --units 128 --top 8
"""
import argparse
import ctypes as C
import json

import torch

from . import abi, ops


def _events(stream, fn, reps, warmup):
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for _ in range(warmup):
        fn()
    stream.synchronize()
    times = []
    for _ in range(reps):
        a.record(stream)
        fn()
        b.record(stream)
        b.synchronize()
        times.append(a.elapsed_time(b))
    return times


def land(direction, part_bytes, parts, reps, warmup, kernel="land"):
    """One tsb_land launch (or tsb_move, HBM -> HBM through shared memory) of `parts` copies of part_bytes each (at
    most 384), grid chosen by the library."""
    assert 1 <= parts <= 384
    total = part_bytes * parts
    dev = torch.empty(total, dtype=torch.uint8, device="cuda")
    other = (torch.empty(total, dtype=torch.uint8).pin_memory() if direction in ("h2d", "d2h")
             else torch.empty(total, dtype=torch.uint8, device="cuda"))
    src, dst = {"h2d": (other, dev), "d2h": (dev, other), "d2d": (other, dev)}[direction]
    sp = (C.c_void_p * parts)(*[src.data_ptr() + i * part_bytes for i in range(parts)])
    dp = (C.c_void_p * parts)(*[dst.data_ptr() + i * part_bytes for i in range(parts)])
    by = (C.c_uint64 * parts)(*([part_bytes] * parts))
    s = torch.cuda.Stream()
    lib = abi.load()

    fn = lib.tsb_move if kernel == "move" else lib.tsb_land

    def once():
        abi.check(fn(sp, dp, by, parts, None, None, None, 0, None, 0, None, 0, s.cuda_stream))

    t = _events(s, once, reps, warmup)
    ms = sorted(t)[len(t) // 2]
    if kernel == "move":
        assert lib.tsb_move_timeouts() == 0
        assert torch.equal(dst[:1 << 20], src[:1 << 20]) and torch.equal(dst[-(1 << 20):], src[-(1 << 20):])
    return {"kernel": kernel, "dir": direction, "part_bytes": part_bytes, "parts": parts, "bytes": total,
            "ms_median": round(ms, 4), "gbs": round(total / ms / 1e6, 2),
            "hbm_traffic_gbs": round(total * (2 if direction == "d2d" else 1) / ms / 1e6, 2)}


def xxh64(units, part_bytes, n_parts, reps, warmup):
    """tsb_xxh64_units over `units` units of n_parts spans of part_bytes each, all in HBM."""
    unit_bytes = part_bytes * n_parts
    data = torch.empty(units * unit_bytes, dtype=torch.uint8, device="cuda")
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    data.random_(0, 256, generator=g)
    spans = (C.c_void_p * (4 * units))()
    sb = (C.c_uint64 * (4 * units))()
    ns = (C.c_uint32 * units)(*([n_parts] * units))
    for i in range(units):
        for p in range(n_parts):
            spans[4 * i + p] = data.data_ptr() + i * unit_bytes + p * part_bytes
            sb[4 * i + p] = part_bytes
    scratch = torch.empty(units * 72 // 8 + 1, dtype=torch.int64, device="cuda")
    out = torch.empty(units, dtype=torch.int64, device="cuda")
    s = torch.cuda.Stream()
    lib = abi.load()

    def once():
        # tsb_xxh64_units returns after its kernel ran; the events bracket the upload and the kernel
        abi.check(lib.tsb_xxh64_units(spans, sb, ns, units, scratch.data_ptr(), None, out.data_ptr(), None,
                                      s.cuda_stream))

    t = _events(s, once, reps, warmup)
    ms = sorted(t)[len(t) // 2]
    total = units * unit_bytes
    return {"kernel": "xxh64", "units": units, "unit_bytes": unit_bytes, "bytes": total, "ms_median": round(ms, 4),
            "gbs": round(total / ms / 1e6, 2), "per_unit_gbs": round(unit_bytes / ms / 1e6, 3)}


def operator(name, rows, hidden, ffn, units, top, reps, warmup, back):
    """One of the operators (ops.linear [rows][hidden] x [ffn][hidden], ops.route, ops.ffn) or its backward pass, bf16,
    rotating over three inputs; bytes and flops as the operator cannot do without, units met counted."""
    t = torch.bfloat16
    s = torch.cuda.current_stream()
    sets = []
    for _ in range(3):
        x, dy = torch.randn((rows, hidden), device="cuda", dtype=t), torch.randn((rows, hidden), device="cuda", dtype=t)
        logits = torch.randn((rows, units), device="cuda")
        ids, w = ops.route(logits, top)
        sets.append((x, dy, logits, ids, w, torch.randn((rows, ffn), device="cuda", dtype=t)))
    met = sum(int(torch.unique(v[3]).numel()) for v in sets) / 3
    if name == "linear":
        ws = [torch.randn((ffn, hidden), device="cuda", dtype=t) for _ in range(3)]
        calls = [(lambda v=v, m=m: ops.linear_backward(v[5], v[0], m)) if back else (lambda v=v, m=m: ops.linear(v[0], m))
                 for v, m in zip(sets, ws)]
        nbytes = 2 * (rows * hidden + ffn * hidden + rows * ffn) + back * 2 * (rows * hidden + ffn * hidden)
        flops = 2 * rows * hidden * ffn * (2 if back else 1)
    elif name == "route":
        calls = [(lambda v=v: ops.route_backward(v[4], v[2], v[3], v[4])) if back else (lambda v=v: ops.route(v[2], top))
                 for v in sets]
        nbytes, flops = rows * (4 * units * (1 + back) + 8 * top), 4 * rows * units
    else:
        gate, up = (torch.randn((units, ffn, hidden), device="cuda", dtype=t) * hidden ** -0.5 for _ in range(2))
        un = ops.Units(gate, up, torch.randn((units, hidden, ffn), device="cuda", dtype=t) * ffn ** -0.5)
        calls = [(lambda v=v: ops.ffn_backward(v[1], v[0], v[3], v[4], un)) if back
                 else (lambda v=v: ops.ffn(v[0], v[3], v[4], un)) for v in sets]
        nbytes = 2 * (3 * met * hidden * ffn + 2 * rows * hidden) + back * 2 * (3 * units * hidden * ffn + rows * hidden)
        flops = rows * top * hidden * ffn * (16 if back else 6)
    turn = iter(range(1 << 30))
    times = sorted(_events(s, lambda: calls[next(turn) % 3](), reps, warmup))
    ms = times[len(times) // 2]
    return {"kernel": name + ("_backward" if back else ""), "rows": rows, "hidden": hidden, "ffn": ffn, "units": units,
            "top": top, "ms_median": round(ms, 4), "gbs": round(nbytes / ms / 1e6, 2),
            "tflops": round(flops / ms / 1e9, 2)}


def main():
    ap = argparse.ArgumentParser()
    sub = ap.add_subparsers(dest="what", required=True)
    a1 = sub.add_parser("land")
    a1.add_argument("--dir", default="h2d", choices=["h2d", "d2h", "d2d"])
    a1.add_argument("--part-bytes", type=int, default=33030144)
    a1.add_argument("--parts", type=int, default=15)
    a1.add_argument("--kernel", default="land", choices=["land", "move"],
                    help="move: tsb_move (HBM -> HBM through shared memory by TMA bulk copies; --dir d2d only)")
    a2 = sub.add_parser("xxh64")
    a2.add_argument("--units", type=int, default=296)
    a2.add_argument("--part-bytes", type=int, default=12582912)
    a2.add_argument("--n-parts", type=int, default=3)
    a3 = [sub.add_parser(n, help="the operator ops.%s (--back: its backward pass)" % n) for n in ("linear", "route", "ffn")]
    for p in a3:
        p.add_argument("--rows", type=int, default=1)
        p.add_argument("--hidden", type=int, default=4096)
        p.add_argument("--ffn", type=int, default=14336)
        p.add_argument("--units", type=int, default=8)
        p.add_argument("--top", type=int, default=2)
        p.add_argument("--back", action="store_true")
    for p in (a1, a2, *a3):
        p.add_argument("--reps", type=int, default=10)
        p.add_argument("--warmup", type=int, default=3)
    a = ap.parse_args()
    if a.what == "land":
        assert a.kernel == "land" or a.dir == "d2d", "the move kernel copies HBM -> HBM only"
        r = land(a.dir, a.part_bytes, a.parts, a.reps, a.warmup, a.kernel)
    elif a.what in ("linear", "route", "ffn"):
        r = operator(a.what, a.rows, a.hidden, a.ffn, a.units, a.top, a.reps, a.warmup, a.back)
    else:
        r = xxh64(a.units, a.part_bytes, a.n_parts, a.reps, a.warmup)
    print(json.dumps(r), flush=True)


if __name__ == "__main__":
    main()
