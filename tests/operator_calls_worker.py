"""Subprocess body of tests/test_gpu_operator_calls.py: torch and the backend in one process share a HIP runtime only where torch comes first, which a test process that has loaded the backend cannot
arrange.  Runs every check, printing its name before it and what came of it behind it."""
import importlib.util
import os
import sys
import traceback

import torch

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, REPO)

CASES = [
    {"kind": "store", "width": 96, "rows": 300, "taken": 17},
    {"kind": "convert", "width": 1024, "rows": 2000, "taken": 2000},
    {"kind": "read", "width": 1024, "rows": 900, "taken": 700},
    {"kind": "product", "width": 1056, "out": 1001, "cols": 1},
    {"kind": "product", "width": 2048, "out": 4096, "cols": 700},
    {"kind": "experts", "width": 256, "out": 333, "experts": 5, "used": 2, "tokens": 3, "shared": False},
    {"kind": "experts", "width": 512, "out": 1024, "experts": 8, "used": 3, "tokens": 500, "shared": True},
]


def name_of(case):
    return "-".join(str(v) for v in case.values())


def operators():
    spec = importlib.util.spec_from_file_location("operator_calls", os.path.join(REPO, "perf", "operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def close(a, b, case):
    """rows equal; products: f32 sums of 2 K products on one side and K on the other, each as far from the true sum as mx_ref.check derives in the 2-norm (sqrt(2 K) + 1 roundings of 2^-24)"""
    if case["kind"] in ("store", "convert", "read"):
        return torch.equal(a, b)
    return float((a.double() - b.double()).norm() / b.double().norm()) <= 2.0**-24 * 2 * ((2 * case["width"]) ** 0.5 + 1)


def result_is_read_at_once(ops, case):
    """a call's result, filled by torch just before it and read by torch just behind it"""
    ops.own = False
    want = ops.run(ops.prepare(case, 5)).clone()
    ops.own = True
    s = ops.prepare(case, 5)
    out = ops.run(s)
    torch.cuda.synchronize()
    for _ in range(5):
        out.fill_(float("nan"))
        got = ops.run(s).clone()
        assert close(got, want, case)


def call_waits(ops, case):
    """torch still fills and reads the last result, behind other work of its stream, when the next call comes"""
    ops.own = True
    a = ops.prepare(case, 7)
    first = ops.run(a).clone()
    torch.cuda.synchronize()
    out = ops.run(a)
    torch.cuda._sleep(20_000_000)  # (some 10 ms of the stream's time)
    out.fill_(3.0)
    kept = out.clone()
    again = ops.run(a).clone()
    torch.cuda.synchronize()
    assert bool((kept == 3.0).all()) and torch.equal(again, first)


def inputs_changed(ops, case):
    """a call takes what the state's tensors hold and which tensors they are when it comes: written anew in place behind other work of torch's stream, and exchanged for others"""
    ops.own = False
    plain = [ops.prepare(case, seed) for seed in (11, 12)]
    names = [k for k, v in plain[0].items() if isinstance(v, torch.Tensor)]
    given = [{k: p[k].clone() for k in names} for p in plain]
    want = [ops.run(p).clone() for p in plain]
    stored = [p.get("table") for p in plain]
    ops.own = True
    s = ops.prepare(case, 11)
    got = [ops.run(s).clone()]
    torch.cuda._sleep(5_000_000)
    for k in names:
        s[k].copy_(given[1][k])
    got.append(ops.run(s).clone())
    for k in names:
        s[k] = given[0][k]
    got.append(ops.run(s).clone())
    for g, w in zip(got, (want[0], want[1], want[0])):
        assert close(g, w, case)
    if case["kind"] == "store":
        assert torch.equal(s["table"], stored[0])  # (the rows are in the state's own table)


CHECKS = {f.__name__ + ":" + name_of(c): (f, c) for f in (result_is_read_at_once, inputs_changed) for c in CASES} | {"call_waits:" + name_of(c): (call_waits, c) for c in CASES if c["kind"] != "store"}


def main():
    ops = operators()
    for name, (check, case) in CHECKS.items():
        print("CHECK", name, flush=True)
        try:
            check(ops, case)
            print("OK", name, flush=True)
        except Exception:
            traceback.print_exc(file=sys.stdout)
            torch.cuda.synchronize()  # (a device that is gone ends the process here)


if __name__ == "__main__":
    main()
    sys.stdout.flush()
    os._exit(0)
