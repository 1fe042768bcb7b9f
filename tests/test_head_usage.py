"""The usage that the documents show for heads of other sizes, run as it stands there: on the CPU
against streams that only write down who waits for whom, on the GPU for its answers."""
import contextlib
import importlib.util
import re
import types
from pathlib import Path

import numpy as np
import pytest
import torch

import head_ref

ROOT = Path(__file__).resolve().parents[1]
CALLS = ("quantize_rows_device", "linear_q8_device", "logprobs_device")


def usage():
    text = (ROOT / "INTEGRATION.md").read_text()
    block, = re.findall(r"## 8\. Heads.*?```python\n(.*?)```", text, re.S)
    return compile(block, "usage", "exec")


def inputs(device):
    g = torch.Generator().manual_seed(3)
    flows, features, classes, top = 1000, 96, 20, 4
    names = dict(flows=flows, features=features, classes=classes, top=top,
                 weight=torch.randn(classes, features, generator=g), bias=torch.randn(classes, generator=g),
                 x=torch.rand(flows, features, generator=g), logits=torch.empty(flows, classes),
                 entropy=torch.empty(flows), ids=torch.empty(flows, top, dtype=torch.int32),
                 logp=torch.empty(flows, top))
    return {n: v.to(device) if isinstance(v, torch.Tensor) else v for n, v in names.items()}


def test_usage_waits(native, monkeypatch):
    """Handle 0 is not torch's default stream but the context's own one, which waits for nothing:
    the example's calls are on a stream of a handle, behind what made the inputs, and what reads
    the answers is behind the calls."""
    log = []

    class Stream:
        def __init__(self, handle=1 << 16):
            self.cuda_stream = handle

        def wait_stream(self, other):
            log.append(("wait", self.cuda_stream, other.cuda_stream))

    class Context:
        def __init__(self, **_):
            self.at = None

        def set_stream(self, handle):
            self.at = handle or None

    for name in CALLS:
        setattr(Context, name, lambda self, *_, name=name: log.append((name, self.at)))
    current = [Stream(0)]

    @contextlib.contextmanager
    def on(stream):
        current.append(stream)
        yield
        current.pop()

    fake = types.SimpleNamespace(int8=torch.int8, uint8=torch.uint8,
                                 empty=lambda *size, device, **kw: torch.empty(*size, **kw),
                                 cuda=types.SimpleNamespace(Stream=Stream, stream=on, current_stream=lambda: current[-1]))
    monkeypatch.setattr(native, "FsxContext", Context)
    exec(usage(), dict(inputs("cpu"), torch=fake))
    calls = [i for i, e in enumerate(log) if e[0] in CALLS]
    assert [log[i][0] for i in calls] == list(CALLS)
    handle = log[calls[0]][1]
    assert handle, "the context's own stream is behind nothing that torch does"
    assert all(log[i][1] == handle for i in calls)
    assert ("wait", handle, 0) in log[:calls[0]], "inputs"
    assert ("wait", 0, handle) in log[calls[-1]:], "answers"


@pytest.mark.parametrize("op", ["quantize", "linear", "logprobs"])
def test_measured_calls_wait(native, monkeypatch, op):
    """The measured cases' program: its stream is behind whichever stream made the buffers before its
    first call on them, and the allocator knows that it uses them."""
    spec = importlib.util.spec_from_file_location("measured", ROOT / "perf" / "operators.py")
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    log = []
    mine = types.SimpleNamespace(cuda_stream=1, wait_stream=lambda other: log.append(("wait", other)))
    call = lambda name: lambda *_: log.append(("call", name))
    m._program.update(lib=native, stream=mine, ctx=types.SimpleNamespace(**{n: call(n) for n in CALLS}))
    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *size, device=None, **kw: empty(*size, **kw))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: "caller")
    monkeypatch.setattr(torch.cuda, "stream", lambda stream: contextlib.nullcontext())
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, stream: log.append(("kept", t.data_ptr(), stream)))
    f, i = torch.zeros(200, 100), torch.zeros(200, 100, dtype=torch.int8)
    v, n = torch.zeros(200), torch.zeros(200, dtype=torch.int32)
    s = dict(quantize=dict(x=f, codes=i, scale=v),
             linear=dict(x=f, x_scale=None, weight=i, weight_scale=v, bias=None, y=torch.zeros(200, 200)),
             logprobs=dict(logits=f, target=n, logprob=v, entropy=v, top_id=n, top_logprob=v))[op]
    s["case"] = dict(op=op, x="f32", y="f32", act="none", top=1)
    m._own(s)
    m._own(s)
    calls = [k for k, e in enumerate(log) if e[0] == "call"]
    assert len(calls) == 2 and ("wait", "caller") in log[:calls[0]]
    for t in s.values():
        if isinstance(t, torch.Tensor):
            assert ("kept", t.data_ptr(), mine) in log[:calls[0]]


@pytest.mark.gpu
def test_usage_answers(native):
    """Inputs made by work that is still under way when the example begins, answers read right
    behind it; no host wait anywhere."""
    names = inputs("cuda")
    x, weight = names["x"].clone(), names["weight"].clone()
    names["x"].zero_()
    names["weight"].zero_()
    busy = torch.rand(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    for _ in range(20):
        busy = busy @ busy * 1e-3
    names["x"].copy_(x)
    names["weight"].copy_(weight)
    space = dict(names, torch=torch)
    exec(usage(), space)
    got = {n: names[n].clone() for n in ("logits", "entropy", "ids", "logp")}
    torch.cuda.synchronize()
    space["ctx"].close()
    q, s = head_ref.quantize(x)
    wq, ws = head_ref.quantize(weight)
    want, tol = head_ref.linear(q, s, wq, ws, names["bias"], "none", torch.float32)
    head_ref.assert_close(got["logits"], want, tol, "logits")
    ref = head_ref.logprobs(got["logits"], None, names["top"])
    assert np.array_equal(got["ids"].cpu().numpy(), ref["top_id"])
    head_ref.assert_close(got["entropy"], ref["entropy"], ref["entropy_tol"], "entropy")
    head_ref.assert_close(got["logp"], ref["top_logprob"], ref["top_logprob_tol"], "alternatives")
