"""The paged cache's performance cases (perf/operators.py): their calls are in the order of the caller's stream."""
import importlib.util
import os
import random
import types

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def cases():
    spec = importlib.util.spec_from_file_location("kv_cases", os.path.join(ROOT, "perf", "operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


class Stream:
    def __init__(self, handle, seen):
        self.cuda_stream, self.seen = handle, seen

    def wait_stream(self, other):
        self.seen.append((self.cuda_stream, "waits for", other.cuda_stream))


class Rows:
    def data_ptr(self):
        return 64

    def stride(self, _):
        return 4


def state(op, seen):
    call = lambda *a, stream=None: seen.append(("call on", a[-1] if stream is None else stream))   # noqa: E731
    rows = {n: Rows() for n in ("q", "k", "v", "q_out", "out", "k_cache", "v_cache")}
    return dict(rows, M=types.SimpleNamespace(kv_append_dev=call, kv_attention_dev=call), device=0, cache=0, batch=0, prep=0, heads=4,
                scale=1.0, case={"op": op, "causal": True, "window": 0, "sinks": 0})


@pytest.mark.parametrize("op", ["append", "attention"])
@pytest.mark.parametrize("handle", [77, 0])
def test_call_is_in_the_callers_order(cases, monkeypatch, op, handle):
    """On a stream of the caller's own: on that one. On the default stream, whose handle the framework takes for another:
    behind what it holds, and it goes on behind the call."""
    seen = []
    monkeypatch.setattr(cases.torch.cuda, "current_stream", lambda *a: Stream(handle, seen))
    monkeypatch.setattr(cases, "_current", lambda *a: handle, raising=False)
    cases.own, cases._stream = True, Stream(5, seen)
    cases.run(state(op, seen))
    if handle:
        assert seen == [("call on", 77)]
    else:
        assert seen == [(5, "waits for", 0), ("call on", 5), (0, "waits for", 5)]


@pytest.mark.gpu
@pytest.mark.parametrize("default", [False, True])
def test_outputs_are_ready_on_the_callers_stream(gpu, cases, default):
    """Inputs filled in behind long work on the caller's stream, outputs read there, with no other wait."""
    import torch
    cases.own = True
    r = random.Random(3)
    drawn = [cases.draw(r) for _ in range(12)]
    for op in ("append", "attention"):
        case = next(c for c in drawn if c["op"] == op)
        print("in order", case, flush=True)
        stream = torch.cuda.default_stream() if default else torch.cuda.Stream()
        with torch.cuda.stream(torch.cuda.Stream()):
            s = cases.prepare(case, 1)
            other = cases.prepare(case, 2)
            cases.run(other)
        torch.cuda.synchronize()
        expect = (other["q_out"] if op == "append" else other["out"]).clone()
        a = torch.randn(4096, 4096, device="cuda")
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for _ in range(40):
                a = (a @ a).clamp_(-1, 1)
            for n in ("q", "k", "v", "q_out", "out", "q_norm", "k_norm", "k_cache", "v_cache", "pages", "len", "row_start"):
                if s.get(n) is not None:
                    s[n].copy_(other[n])
            got = cases.run(s)
            got = (got["q"] if op == "append" else got).clone()
        torch.cuda.synchronize()
        assert torch.equal(got, expect)
