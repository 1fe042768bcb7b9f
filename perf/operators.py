"""The quantised layer and its answers, measured case by case.

Three operators that a scoring head is made of (include/fsx_hip.h):

  quantize   rows of floats to int8 codes with one scale a row (fsx_quantize_rows_device)
  linear     int8 matrix product with a scale for every row of x and every output
             channel, bias and activation (fsx_linear_q8_device); x comes as codes with
             their scales, or as floats that the call quantises
  logprobs   of every row of logits: the log probability of a given class, the entropy and
             the most probable alternatives (fsx_logprobs_device)

`run` computes them from elementary torch operations, or, where `own` is true, through
flowsentryx_amd.lib. Nothing here says how far results may be apart.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1}
SMALLEST_SCALE = 2.0 ** -126
NEG = float("-inf")


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # one row: what a serving loop quantises for each new token
        dict(name="quantize one row", op="quantize", rows=1, cols=4096, x="bf16", pad=0),
        # a whole batch of activations, or a weight matrix by output channel
        dict(name="quantize 8192 rows", op="quantize", rows=8192, cols=8192, x="bf16", pad=0),
        # one new token through a square layer: the latency of a serving step
        dict(name="linear one token", op="linear", rows=1, inf=4096, outf=4096, x="bf16", y="bf16", bias=False,
             act="none", pad=0),
        # a decode batch through a widening layer: the weights are read once for 16 rows
        dict(name="linear decode batch", op="linear", rows=16, inf=4096, outf=16384, x="f16", y="f16", bias=True,
             act="none", pad=0),
        # a prompt chunk
        dict(name="linear prompt chunk", op="linear", rows=512, inf=4096, outf=4096, x="bf16", y="bf16", bias=False,
             act="none", pad=0),
        # the largest product: activations already quantised
        dict(name="linear 8192 cubed", op="linear", rows=8192, inf=8192, outf=8192, x="i8", y="bf16", bias=False,
             act="none", pad=0),
        # sizes that fit no tile, rows at odd strides, a hidden layer's activation
        dict(name="linear odd sizes", op="linear", rows=1000, inf=1003, outf=777, x="f32", y="f32", bias=True,
             act="relu", pad=1),
        # the head over flow features: 2^22 flows of 8 features (the scoring workload), 16 classes
        dict(name="linear flow features", op="linear", rows=1 << 22, inf=8, outf=16, x="f32", y="f32", bias=True,
             act="none", pad=0),
        # the answer of one serving step: one row over a large vocabulary
        dict(name="logprobs one row", op="logprobs", rows=1, classes=131072, x="bf16", top=20, masked=0.0, pad=0),
        # a prompt's log probabilities over a large vocabulary
        dict(name="logprobs prompt", op="logprobs", rows=2048, classes=131072, x="bf16", top=8, masked=0.0, pad=0),
        # odd sizes and strides, most classes masked, one row masked altogether
        dict(name="logprobs odd masked", op="logprobs", rows=301, classes=50021, x="f16", top=20, masked=0.9, pad=3),
        # the classes of 2^22 flows
        dict(name="logprobs flow classes", op="logprobs", rows=1 << 22, classes=16, x="f32", top=3, masked=0.0, pad=0),
    ]


def _log_int(rng, lo, hi):
    """A whole number, spread over the logarithm of lo..hi."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("quantize", "linear", "linear", "logprobs", "logprobs"))
    pad = rng.choice((0, 0, 1, 8, 16))
    if op == "quantize":
        cols = _log_int(rng, 1, 16384)
        rows = _log_int(rng, 1, min(1 << 20, max(1, (1 << 26) // cols)))
        return dict(op=op, rows=rows, cols=cols, x=rng.choice(("f32", "f16", "bf16")), pad=pad)
    if op == "linear":
        inf, outf = _log_int(rng, 4, 16384), _log_int(rng, 1, 16384)
        rows = _log_int(rng, 1, max(1, min((1 << 39) // (inf * outf), (1 << 25) // max(inf, outf), 1 << 22)))
        return dict(op=op, rows=rows, inf=inf, outf=outf, x=rng.choice(("f32", "f16", "bf16", "i8")),
                    y=rng.choice(("f32", "f16", "bf16")), bias=rng.random() < 0.5,
                    act=rng.choice(("none", "none", "relu", "sigmoid")), pad=pad)
    classes = _log_int(rng, 2, 131072)
    rows = _log_int(rng, 1, max(1, min((1 << 27) // classes, 1 << 22)))
    return dict(op=op, rows=rows, classes=classes, x=rng.choice(("f32", "f16", "bf16")), top=rng.randint(1, 32),
                masked=rng.choice((0.0, 0.0, 0.5, 0.9)), pad=pad)


def work(case):
    if case["op"] == "quantize":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (SIZE[case["x"]] + 1) + 4 * case["rows"], "flops": 2 * n}
    if case["op"] == "linear":
        m, k, n = case["rows"], case["inf"], case["outf"]
        b = m * k * SIZE[case["x"]] + n * k + m * n * SIZE[case["y"]] + 4 * n * (2 if case["bias"] else 1)
        return {"bytes": b + (4 * m if case["x"] == "i8" else 0), "flops": 2 * m * k * n}
    n = case["rows"] * case["classes"]
    return {"bytes": n * SIZE[case["x"]] + case["rows"] * (12 + 8 * case["top"]), "flops": 6 * n}


# ---------------------------------------------------------------- what a program has in hand

def _rows(gen, rows, cols, pad, dtype, spread=1.0):
    """Normal values in rows that are cols + pad apart; a few columns ten times as large, as
    activations have them."""
    x = torch.randn(rows, cols + pad, generator=gen, device="cuda") * spread
    x[:, torch.randint(0, cols, (1 + cols // 200,), generator=gen, device="cuda")] *= 10
    return x.to(dtype)[:, :cols]


def _codes(gen, rows, cols, pad):
    return torch.randint(-127, 128, (rows, cols + pad), generator=gen, device="cuda", dtype=torch.int8)[:, :cols]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, pad = case["rows"], case["pad"]
    s = dict(case=case)
    if case["op"] == "quantize":
        s["x"] = _rows(gen, rows, case["cols"], pad, DTYPES[case["x"]])
        s["codes"] = torch.empty(rows, case["cols"], dtype=torch.int8, device="cuda")
        s["scale"] = torch.empty(rows, device="cuda")
    elif case["op"] == "linear":
        k, n = case["inf"], case["outf"]
        if case["x"] == "i8":
            s["x"] = _codes(gen, rows, k, pad)
            s["x_scale"] = 0.005 + 0.01 * torch.rand(rows, generator=gen, device="cuda")
        else:
            s["x"] = _rows(gen, rows, k, pad, DTYPES[case["x"]])
            s["x_scale"] = None
        s["weight"] = _codes(gen, n, k, pad)
        s["weight_scale"] = (0.5 + torch.rand(n, generator=gen, device="cuda")) / (64 * math.sqrt(k))
        s["bias"] = torch.randn(n, generator=gen, device="cuda") if case["bias"] else None
        s["y"] = torch.empty(rows, n, dtype=DTYPES[case["y"]], device="cuda")
    else:
        v, top = case["classes"], case["top"]
        x = 3 * torch.randn(rows, v + pad, generator=gen, device="cuda")
        target = torch.randint(0, v, (rows,), generator=gen, device="cuda", dtype=torch.int32)
        if case["masked"]:
            x.masked_fill_(torch.rand(rows, v + pad, generator=gen, device="cuda") < case["masked"], NEG)
            x[rows // 2] = NEG      # a row of which the mask leaves nothing
            target[::7] = -1        # rows that are asked for no class
        s["logits"] = x.to(DTYPES[case["x"]])[:, :v]
        s["target"] = target
        s["logprob"], s["entropy"] = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
        s["top_id"] = torch.empty(rows, top, dtype=torch.int32, device="cuda")
        s["top_logprob"] = torch.empty(rows, top, device="cuda")
    return s


# ---------------------------------------------------------------- the plain forms

def _plain_quantize(x):
    """(codes in float32, scales): scale = max(amax / 127, 2^-126) in 32 bits, code = x / scale
    to the nearest whole number, halves to even (the quotient in 64 bits: a half is a border).
    A row with a NaN or an infinity has codes 0 and the scale NaN."""
    x = x.float()
    amax = x.abs().amax(1)
    ok = torch.isfinite(amax)
    scale = torch.where(ok, (amax.double() / 127).float().clamp_min(SMALLEST_SCALE), float("nan"))
    codes = torch.where(ok[:, None], torch.round(x.double() / scale.double()[:, None]), 0.0)
    return codes.float(), scale


def _plain_linear(s):
    case = s["case"]
    codes, scale = (s["x"].float(), s["x_scale"]) if s["x_scale"] is not None else _plain_quantize(s["x"])
    y = (codes @ s["weight"].float().T) * scale[:, None] * s["weight_scale"]
    if s["bias"] is not None:
        y = y + s["bias"]
    if case["act"] == "relu":
        y = torch.where(y < 0, 0.0, y)
    elif case["act"] == "sigmoid":
        y = 1 / (1 + torch.exp(-y))
    return y.to(s["y"].dtype)


def _plain_logprobs(s):
    """-inf is a masked class: it has no probability and is no alternative. An empty row has
    logprob -inf and entropy 0; a row without a class asked for (-1) has logprob 0."""
    x, target, top = s["logits"].float(), s["target"].long(), s["case"]["top"]
    rows, v = x.shape
    m = x.amax(1)
    z = x - torch.where(m == NEG, 0.0, m)[:, None]
    e = torch.exp(z)
    total = e.sum(1)
    log_total = torch.log(total)
    entropy = torch.where(total > 0, log_total - torch.where(e > 0, e * z, 0.0).sum(1) / total, 0.0)
    z_target = z.gather(1, target.clamp_min(0)[:, None])[:, 0]
    logprob = torch.where(target < 0, 0.0, torch.where(z_target == NEG, NEG, z_target - log_total))
    # the values' order as whole numbers, ties by the lowest class: all keys differ
    bits = (x + 0.0).view(torch.int32).long()
    key = (torch.where(bits < 0, -1 - (bits & 0x7FFFFFFF), bits) << 20) + (v - 1 - torch.arange(v, device=x.device))
    best = key.topk(min(top, v), dim=1).values
    ids = v - 1 - (best & 0xFFFFF)
    z_top = z.gather(1, ids)
    gone = z_top == NEG
    ids = torch.where(gone, -1, ids)
    lp = torch.where(gone, NEG, z_top - log_total[:, None])
    out_id = torch.full((rows, top), -1, dtype=torch.int32, device=x.device)
    out_lp = torch.full((rows, top), NEG, device=x.device)
    out_id[:, :ids.shape[1]] = ids.int()
    out_lp[:, :ids.shape[1]] = lp
    return dict(logprob=logprob, entropy=entropy, top_id=out_id, top_logprob=out_lp)


# ---------------------------------------------------------------- the framework's operators

_program = {}


def _context():
    """The context and the stream that a program keeps for all its calls."""
    if not _program:
        from flowsentryx_amd import lib
        stream = torch.cuda.Stream()
        ctx = lib.FsxContext(max_entries=1024, max_batch=1024)
        ctx.set_stream(stream.cuda_stream)
        _program.update(lib=lib, stream=stream, ctx=ctx)
    return _program["lib"], _program["ctx"], _program["stream"]


def _ready(s, lib, stream):
    """What a program does once for its buffers: the layer, the workspace, and the stream's order behind
    what made them, whichever stream that was."""
    case = s["case"]
    if case["op"] == "linear":
        w = s["weight"]
        act = {"none": lib.ACT_NONE, "relu": lib.ACT_RELU, "sigmoid": lib.ACT_SIGMOID}[case["act"]]
        s["layer"] = lib.q8_linear(w.data_ptr(), s["weight_scale"].data_ptr(),
                                   s["bias"].data_ptr() if s["bias"] is not None else None,
                                   w.shape[1], w.shape[0], w.stride(0), act)
        size = lib.linear_q8_work(s["layer"], _dtype(lib)[case["x"]], s["x"].shape[0])
    elif case["op"] == "logprobs":
        size = lib.logprobs_work(s["logits"].shape[0], s["logits"].shape[1], case["top"])
    if case["op"] != "quantize":
        s["work"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    stream.wait_stream(torch.cuda.current_stream())
    for t in s.values():
        if isinstance(t, torch.Tensor):
            t.record_stream(stream)
    s["ready"] = True


def _dtype(lib):
    return {"f32": lib.DTYPE_F32, "f16": lib.DTYPE_F16, "bf16": lib.DTYPE_BF16, "i8": lib.DTYPE_I8}


def _own(s):
    """The call, asynchronous on the program's stream: who changes the state's buffers or reads the
    outputs on another stream waits for it first, as torch.cuda.synchronize() does."""
    lib, ctx, stream = _context()
    case = s["case"]
    dtype = _dtype(lib)
    if "ready" not in s:
        _ready(s, lib, stream)
    if case["op"] == "quantize":
        x, q = s["x"], s["codes"]
        ctx.quantize_rows_device(x.data_ptr(), dtype[case["x"]], x.shape[0], x.shape[1], x.stride(0),
                                 q.data_ptr(), q.stride(0), s["scale"].data_ptr())
        with torch.cuda.stream(stream):
            return dict(values=torch.mul(q, s["scale"][:, None]), scale=s["scale"])
    if case["op"] == "linear":
        x, y = s["x"], s["y"]
        ctx.linear_q8_device(s["layer"], x.data_ptr(), dtype[case["x"]], x.stride(0),
                             s["x_scale"].data_ptr() if s["x_scale"] is not None else None, x.shape[0],
                             y.data_ptr(), dtype[case["y"]], y.stride(0), s["work"].data_ptr(), s["work"].numel())
        return y
    x = s["logits"]
    ctx.logprobs_device(x.data_ptr(), dtype[case["x"]], x.shape[0], x.shape[1], x.stride(0), s["target"].data_ptr(),
                        s["logprob"].data_ptr(), s["entropy"].data_ptr(), case["top"], s["top_id"].data_ptr(),
                        s["top_logprob"].data_ptr(), s["work"].data_ptr(), s["work"].numel())
    return dict(logprob=s["logprob"], entropy=s["entropy"], top_id=s["top_id"], top_logprob=s["top_logprob"])


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "quantize":
        codes, scale = _plain_quantize(state["x"])
        return dict(values=codes * scale[:, None], scale=scale)
    return _plain_linear(state) if op == "linear" else _plain_logprobs(state)


# ---------------------------------------------------------------- the definition in 64 bits

def _exact_codes(x):
    """Codes and scales of a block of rows; the scale is a 32-bit number by definition."""
    top = torch.linalg.vector_norm(x.double(), ord=math.inf, dim=1)
    scale = torch.clamp((top / 127.0).float(), min=SMALLEST_SCALE).double()
    return torch.round(x.double() / scale.unsqueeze(1)), scale


def exact(case, seed):
    s = prepare(case, seed)
    rows = case["rows"]
    block = max(1, (1 << 26) // max(case.get("cols", 0), case.get("inf", 0) + case.get("outf", 0),
                                    case.get("classes", 0)))
    parts = []
    for at in range(0, rows, block):
        to = min(rows, at + block)
        if case["op"] == "quantize":
            codes, scale = _exact_codes(s["x"][at:to])
            parts.append((codes.mul_(scale.unsqueeze(1)), scale))
        elif case["op"] == "linear":
            if s["x_scale"] is None:
                codes, scale = _exact_codes(s["x"][at:to])
            else:
                codes, scale = s["x"][at:to].double(), s["x_scale"][at:to].double()
            y = torch.mm(codes, s["weight"].double().t().contiguous())
            y *= torch.outer(scale, s["weight_scale"].double())
            if case["bias"]:
                y += s["bias"].double()
            if case["act"] == "relu":
                y.clamp_(min=0)
            elif case["act"] == "sigmoid":
                y = torch.sigmoid(y)
            parts.append((y,))
        else:
            x = s["logits"][at:to].double()
            lse = torch.logsumexp(x, 1, keepdim=True)
            lp = torch.where(x == NEG, NEG, x - lse)
            entropy = torch.special.entr(torch.exp(lp)).sum(1)
            t = s["target"][at:to].long()
            given = torch.where(t < 0, 0.0, lp.gather(1, t.clamp_min(0).unsqueeze(1)).squeeze(1))
            k = min(case["top"], case["classes"])
            best = torch.full((to - at, case["top"]), NEG, dtype=torch.float64, device=x.device)
            best[:, :k] = torch.topk(lp, k, dim=1).values
            parts.append((given, entropy, best))
    got = [torch.cat(p) for p in zip(*parts)]
    if case["op"] == "quantize":
        return dict(values=got[0], scale=got[1])
    if case["op"] == "linear":
        return got[0]
    return dict(logprob=got[0], entropy=got[1], top_id=None, top_logprob=got[2])
