"""A context on the stream of the library that owns the operands (torch here): calls in order with that library's work without a
synchronization between them, eager and captured into its graphs.  A program of its own, which tests/test_gpu_stream.py starts:
the library and torch share one HIP runtime only in a process that imports torch first.  Prints a line for every check that
passed."""
import importlib.util
import os
import random
import sys

import numpy as np
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [ROOT, os.path.join(ROOT, "tests")]

from hodu_amd import ffi  # noqa: E402
import seq_util as S  # noqa: E402


class Prompt:
    """attention over three packed prompts, operands and result in torch's memory"""

    def __init__(self, ctx, lens=(300, 7, 513), hq=4, hk=2, d=64, seed=0):
        self.ctx, t = ctx, sum(lens)
        gen = torch.Generator().manual_seed(seed)
        self.host = [torch.randn(t, h, d, generator=gen).to(torch.bfloat16) for h in (hq, hk, hk)]
        self.q, self.k, self.v = (torch.zeros_like(x, device="cuda") for x in self.host)
        self.source = [x.cuda() for x in self.host]
        self.out = torch.zeros(t, hq, d, dtype=torch.bfloat16, device="cuda")
        self.offsets = torch.tensor(np.cumsum([0, *lens]), dtype=torch.int32, device="cuda")
        self.md, self.bits = ffi.varlen_md(len(lens), t, t, hq, hk, d), S.scalar(d, "bf16")[0]
        torch.cuda.synchronize()

    def fill(self):
        for to, x in zip((self.q, self.k, self.v), self.source):
            to.copy_(x)

    def call(self):
        of = ffi.DeviceView.of
        self.ctx.attention_varlen("bf16", of(self.q), of(self.k), of(self.v), of(self.out), of(self.offsets), of(self.offsets), self.md, self.bits, True)

    def want(self):
        """the same call on operands that have long been there"""
        torch.cuda.synchronize()
        self.fill()
        torch.cuda.synchronize()
        self.call()
        torch.cuda.synchronize()
        want = self.out.clone()
        for x in (self.q, self.k, self.v, self.out):
            x.zero_()
        torch.cuda.synchronize()
        assert want.abs().sum() > 0
        return want


def calls_in_order_on_the_default_stream(ctx):
    calls_in_order(ctx, torch.cuda.default_stream())


def calls_in_order_on_another_stream(ctx):
    calls_in_order(ctx, torch.cuda.Stream())


def calls_in_order(ctx, stream):
    p = Prompt(ctx)
    with torch.cuda.stream(stream):
        ctx.set_stream(torch.cuda.current_stream())
        assert ctx.stream == stream.cuda_stream
        want = p.want()
        for _ in range(5):
            torch.cuda._sleep(20_000_000)  # some 10 ms: what follows is all queued behind it
            p.fill()
            p.call()
            got = p.out.clone()
            p.out.zero_()
            for x in (p.q, p.k, p.v):
                x.fill_(float("nan"))
            assert torch.equal(got, want)


def a_new_stream_runs_behind_the_one_before(ctx):
    p = Prompt(ctx, seed=1)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    ctx.set_stream(a)
    want = p.want()
    with torch.cuda.stream(a):
        torch.cuda._sleep(20_000_000)
        p.fill()
        p.call()
    with torch.cuda.stream(b):
        ctx.set_stream(b)
        got = p.out.clone()  # (b waits for a from the hand-over on)
    own = ffi.Context(0)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    own.close()


def captured_into_the_owners_graph(ctx):
    p = Prompt(ctx, seed=2)
    s = torch.cuda.Stream()
    ctx.set_stream(s)
    want = p.want()
    graph, got = torch.cuda.CUDAGraph(), torch.zeros_like(p.out)
    with torch.cuda.graph(graph, stream=s):
        p.fill()
        p.call()
        got.copy_(p.out)
    for _ in range(4):
        for x in (p.q, p.k, p.v, p.out, got):
            x.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        with torch.cuda.stream(s):
            p.call()  # eager work between the replays
        torch.cuda.synchronize()
        assert torch.equal(p.out, want)


def the_measured_calls_are_in_order_with_torch(ctx):
    """a pass of perf/operators.py on inputs that are still being made, its outputs taken at once, no synchronization"""
    spec = importlib.util.spec_from_file_location("measured_operators", os.path.join(ROOT, "perf", "operators.py"))
    ops = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ops)
    cases = [c for c in ops.listed() if c["name"] in ("plan_decode", "store_decode", "prompt_short", "decode_one")]
    rng = random.Random(5)
    while len(cases) < 10:
        c = ops.draw(rng)
        if ops.work(c)["flops"] < 2e10 and ops.work(c)["bytes"] < 5e7:
            cases.append(c)

    def values(out):
        return list(out.values()) if isinstance(out, dict) else [out]

    for n, case in enumerate(cases):
        plain, late = ops.prepare(case, n), ops.prepare(case, n)
        given = {k: x.clone() for k, x in late.items() if torch.is_tensor(x) and x.is_cuda}
        for x in given:
            late[x].zero_()
        torch.cuda.synchronize()
        torch.cuda._sleep(20_000_000)
        for k, x in given.items():
            late[k].copy_(x)
        ops.own = True
        try:
            got = [x.clone() for x in values(ops.run(late))]
        finally:
            ops.own = False
        for k in given:
            late[k].zero_()
        want = [x.clone() for x in values(ops.run(plain))]
        for a, b in zip(got, want):
            if a.dtype == torch.int32 or case["op"] == "store" and case["cache"] != "f8e4m3":
                assert torch.equal(a, b), case
            else:
                x, y = a.double(), b.double()
                # (roundings of P and of the output, and an 8-bit value next to a tie: far below what stale operands give)
                assert (x - y).norm() <= 2 * S.HALF_STEP[{v: k for k, v in S.TORCH.items()}[a.dtype]] * y.norm(), case


CHECKS = [calls_in_order_on_the_default_stream, calls_in_order_on_another_stream, a_new_stream_runs_behind_the_one_before, captured_into_the_owners_graph,
          the_measured_calls_are_in_order_with_torch]


def main():
    for check in CHECKS:
        ctx = ffi.Context(0)
        check(ctx)
        torch.cuda.synchronize()
        ctx.close()
        print("ok", check.__name__, flush=True)


if __name__ == "__main__":
    main()
