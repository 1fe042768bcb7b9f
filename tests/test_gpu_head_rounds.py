"""GPU: the free-size heads over more rows than their blocks take in one round. What a block
leaves in LDS and in registers from one round must not reach the next, so rows of
different kinds (plain, tied, masked, empty, with a NaN or +inf) follow one another in every block,
and every row has the bits that it has in a call of few rows. The heads behind the packet path, too,
as one run."""
import numpy as np
import pytest
import torch

import head_ref
from test_gpu_head import CANARY, FLOATS, NEG, Head, codes_of, gen_of, layer_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def head(native):
    h = Head(native)
    yield h
    h.ctx.close()


def mixed(rows, cols, pad, dtype, seed):
    """Rows of seven kinds in turn. 7 divides no grid here, so a block's next row is of another kind."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, cols + pad, generator=g, device="cuda").mul_(3)
    x[0::7] = x[0::7].round()
    some = x[1::7]
    some[torch.rand(some.shape, generator=g, device="cuda") < 0.9] = NEG
    x[2::7] = NEG
    x[3::7, cols // 2] = float("nan")
    x[4::7, cols - 1] = float("inf")
    x[5::7] *= 100
    return x.to(dtype)[:, :cols]


def slices(rows, at_once):
    return [(a, min(rows, a + at_once)) for a in range(0, rows, at_once)]


# ---------------------------------------------------------------- log probabilities

# rows, classes, dtype, top, rows of a call that takes one round
ROUNDS = [
    (600007, 7, "f16", 28, 100000),     # a lane a row, counted
    (70001, 33, "f32", 33, 8000),       # eight lanes, counted
    (70001, 100, "bf16", 20, 8000),     # sixteen lanes, one by one
    (20001, 200, "bf16", 12, 8000),     # 32 lanes, bounded
    (20001, 200, "f32", 9, 8000),       # four logits a lane, bounded
    (20001, 300, "f16", 55, 8000),      # a wave a row, one by one
    (20001, 300, "f32", 4, 8000),       # a wave a row, bounded
    (20001, 500, "bf16", 20, 8000),
    (20001, 500, "bf16", 2, 8000),      # kept in registers
    (20001, 1000, "bf16", 20, 8000),    # sixteen logits a lane, bounded
    (65600, 1100, "bf16", 0, 8000),     # a block a row
    (65600, 1100, "bf16", 4, 8000),
    (65600, 1100, "f16", 64, 8000),
    (65600, 2100, "bf16", 5, 8000),     # its waves' pieces twice as large
    (65600, 4100, "bf16", 5, 8000),     # four times
    (65600, 4100, "bf16", 0, 8000),
]


@pytest.mark.parametrize("rows,classes,dtype,top,at_once", ROUNDS)
def test_logprobs_rounds(head, rows, classes, dtype, top, at_once):
    x = mixed(rows, classes, 3, FLOATS[dtype], rows + classes + top)
    t = torch.randint(-1, classes + 1, (rows,), dtype=torch.int32, generator=gen_of("rt", rows, classes)).cuda()

    def outputs():
        return [torch.full((rows + 1,), 7.0, device="cuda"), torch.full((rows + 1,), 7.0, device="cuda"),
                torch.full((rows + 1, top), CANARY, dtype=torch.int32, device="cuda"),
                torch.full((rows + 1, top), 7.0, device="cuda")]

    def call(out, a, b):
        lp, en, ids, lps = (o[a:b] for o in out)
        head.logprobs(x[a:b], t[a:b], lp, en, ids if top else None, lps if top else None,
                      head.logprobs_work(x[a:b], top))

    whole, parts = outputs(), outputs()
    torch.cuda.synchronize()
    call(whole, 0, rows)
    for a, b in slices(rows, at_once):
        call(parts, a, b)
    torch.cuda.synchronize()
    for name, a, b in zip(("logprob", "entropy", "ids", "alternatives"), whole, parts):
        a, b = a.nan_to_num(3e38), b.nan_to_num(3e38)   # (a NaN is no row's value)
        assert torch.equal(a, b), f"{name}: rows {torch.nonzero((a != b).reshape(rows + 1, -1).any(1))[:5, 0].tolist()}"
    # the last pass against 64 bits
    last = slice(rows - 70, rows)
    ref = head_ref.logprobs(x[last], t[last], top)
    head_ref.assert_close(whole[0][last], ref["logprob"], ref["logprob_tol"], "logprob")
    head_ref.assert_close(whole[1][last], ref["entropy"], ref["entropy_tol"], "entropy")
    if top:
        assert np.array_equal(whole[2][last].cpu().numpy(), ref["top_id"])
        head_ref.assert_close(whole[3][last], ref["top_logprob"], ref["top_logprob_tol"], "alternatives")


# ---------------------------------------------------------------- row quantiser

@pytest.mark.parametrize("rows,cols,dtype,at_once", [
    (16777300, 3, "f32", 4000000), (262200, 1100, "bf16", 60000), (65540, 2049, "bf16", 16000),
    (65540, 5000, "f16", 16000), (65540, 8300, "bf16", 16000)])
def test_quantize_rounds(head, rows, cols, dtype, at_once):
    """All threads of a row, and the block's maximum where a block takes one."""
    x = mixed(rows, cols, 0, FLOATS[dtype], rows + cols)
    out = [(torch.full((rows + 1, cols), CANARY, dtype=torch.int8, device="cuda"), torch.full((rows + 1,), 7.0, device="cuda"))
           for _ in range(2)]
    torch.cuda.synchronize()
    head.quantize(x, out[0][0][:rows], out[0][1][:rows])
    for a, b in slices(rows, at_once):
        head.quantize(x[a:b], out[1][0][a:b], out[1][1][a:b])
    torch.cuda.synchronize()
    for a, b in zip(*out):
        assert torch.equal(a.nan_to_num(-1.0), b.nan_to_num(-1.0))
    q, s = head_ref.quantize(x[rows - 70:])
    assert torch.equal(out[0][0][rows - 70:rows].cpu().long(), q)
    assert torch.equal(out[0][1][rows - 70:rows].cpu().nan_to_num(-1.0), s.nan_to_num(-1.0))


# ---------------------------------------------------------------- int8 layer

@pytest.mark.parametrize("xt", [*FLOATS, "i8"])
@pytest.mark.parametrize("rows,k,n,at_once", [(1100003, 8, 16, 250000), (300007, 31, 17, 60000), (140003, 50, 70, 30000)])
def test_linear_rounds(head, xt, rows, k, n, at_once):
    """Short rows, the next ones read ahead."""
    g = gen_of("rl", rows, k, n)
    w, ws, bias = layer_of(g, n, k, 3, True)
    if xt == "i8":
        x, xs = codes_of(g, rows, k, 1), (0.005 + 0.01 * torch.rand(rows, generator=g)).cuda()
    else:
        x, xs = mixed(rows, k, 1, FLOATS[xt], rows + k), None
    layer = head.layer(w, ws, bias, "none")
    whole, parts = (torch.full((rows + 1, n), float(CANARY), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    head.linear(layer, x, xs, whole[:rows], head.linear_work(layer, x))
    for a, b in slices(rows, at_once):
        head.linear(layer, x[a:b], None if xs is None else xs[a:b], parts[a:b], head.linear_work(layer, x[a:b]))
    torch.cuda.synchronize()
    assert torch.equal(whole.nan_to_num(3e38), parts.nan_to_num(3e38))
    last = slice(rows - 70, rows)
    codes, scale = (x[last].cpu().long(), xs[last]) if xs is not None else head_ref.quantize(x[last])
    ref, tol = head_ref.linear(codes, scale, w, ws, bias, "none", torch.bfloat16)
    head_ref.assert_close(whole[last], ref, tol, "y")


def test_linear_large_copies(head):
    """Operands at odd strides whose copies take more than one round: the bits of the same operands
    at 16-byte strides."""
    g = gen_of("rc")
    for rows, n in ((400, 8300), (8300, 400)):
        k = 4103
        w, ws, bias = layer_of(g, n, k, 9, True)
        x = codes_of(g, rows, k, 9)
        assert w.stride(0) % 16 == 0 and x.stride(0) % 16 == 0
        xs = (0.005 + 0.01 * torch.rand(rows, generator=g)).cuda()
        odd_w, odd_x = codes_of(g, n, k, 2), codes_of(g, rows, k, 4)
        odd_w.copy_(w)
        odd_x.copy_(x)
        y = [torch.empty(rows, n, device="cuda") for _ in range(2)]
        layers = [head.layer(w, ws, bias, "none"), head.layer(odd_w, ws, bias, "none")]
        works = [head.linear_work(a, x) for a in layers]
        assert works[1].numel() >= n * k, "copies"
        torch.cuda.synchronize()
        head.linear(layers[0], x, xs, y[0], works[0])
        head.linear(layers[1], odd_x, xs, y[1], works[1])
        torch.cuda.synchronize()
        assert torch.equal(*y)
        ref, tol = head_ref.linear(x[-9:].cpu().long(), xs[-9:], w, ws, bias, "none", torch.float32)
        head_ref.assert_close(y[1][-9:], ref, tol, "y")


# ---------------------------------------------------------------- behind the packet path

@pytest.mark.parametrize("pipeline", [0, 1])
def test_behind_the_packets(native, oracle, pipeline):
    """Batches of packets to verdicts and flow features, the features through a layer to class answers,
    all on the context's stream with no wait of the host between, batches overlapping or not. Verdicts
    and features are the oracle's, the answers those of the features that each batch has left."""
    from flowsentryx_amd import synth
    p, s = synth.config_params(2, n=3 << 16)
    hdr, ln, ts = oracle.synth(p, s, 0, int(p.n))
    cut = [0, 50_000, 51_001, 120_000, len(ln)]
    batches = [(hdr[a:b], ln[a:b], ts[a:b]) for a, b in zip(cut, cut[1:])]
    cap, classes, top = max(len(b[1]) for b in batches), 12, 3
    g = gen_of("plane heads")
    w, ws, bias = layer_of(g, classes, 8, 0, True)
    dev = lambda a: torch.from_numpy(a.view(np.uint8).reshape(-1)).cuda()
    cfg = dict(max_entries=1 << 18, max_batch=cap)
    with native.FsxContext(**cfg) as c:
        layer = native.q8_linear(w.data_ptr(), ws.data_ptr(), bias.data_ptr(), 8, classes, 8, native.ACT_NONE)
        runs = []
        for b in batches:
            empty = lambda *size, dtype=torch.float32: torch.zeros(*size, dtype=dtype, device="cuda")
            runs.append(dict(
                d=[dev(a) for a in b], n=len(b[1]), v=empty(cap, dtype=torch.uint8), k=empty(cap, 16, dtype=torch.uint8),
                f=empty(cap, dtype=torch.uint8), x=empty(cap, 8), z=empty(cap, classes), en=empty(cap),
                ids=empty(cap, top, dtype=torch.int32), lps=empty(cap, top),
                work=torch.empty(native.linear_q8_work(layer, native.DTYPE_F32, cap), dtype=torch.uint8, device="cuda"),
                work2=torch.empty(native.logprobs_work(cap, classes, top), dtype=torch.uint8, device="cuda")))
        torch.cuda.synchronize()
        c.set_pipeline(pipeline)
        for r in runs:
            c.process_batch_device(*(t.data_ptr() for t in r["d"]), r["n"], r["v"].data_ptr(), r["k"].data_ptr(),
                                   r["f"].data_ptr(), r["x"].data_ptr(), None, None, cap)
            c.linear_q8_device(layer, r["x"].data_ptr(), native.DTYPE_F32, 8, None, cap, r["z"].data_ptr(),
                               native.DTYPE_F32, classes, r["work"].data_ptr(), r["work"].numel())
            c.logprobs_device(r["z"].data_ptr(), native.DTYPE_F32, cap, classes, classes, None, None, r["en"].data_ptr(),
                              top, r["ids"].data_ptr(), r["lps"].data_ptr(), r["work2"].data_ptr(), r["work2"].numel())
        c.sync()
        torch.cuda.synchronize()
    o = oracle.Oracle(max_entries=cfg["max_entries"])
    for r, (h, l, t) in zip(runs, batches):
        assert np.array_equal(r["v"][:r["n"]].cpu().numpy(), o.batch(h, l, t))
        ko, fo, xo = oracle.flow_features(h, l, t)
        m = len(fo)
        kg, fg, xg = r["k"][:m].cpu().numpy(), r["f"][:m].cpu().numpy(), r["x"][:m].cpu().numpy()
        og = sorted(range(m), key=lambda i: (int(fg[i]), kg[i].tobytes()))
        oo = sorted(range(m), key=lambda i: (int(fo[i]), ko[i].tobytes()))
        assert np.array_equal(kg[og], ko[oo]) and np.array_equal(xg[og].view(np.uint32), xo[oo].view(np.uint32))
        q, sc = head_ref.quantize(r["x"][:m])
        ref, tol = head_ref.linear(q, sc, w, ws, bias, "none", torch.float32)
        head_ref.assert_close(r["z"][:m], ref, tol, "logits")
        ref = head_ref.logprobs(r["z"][:m], None, top)
        head_ref.assert_close(r["en"][:m], ref["entropy"], ref["entropy_tol"], "entropy")
        assert np.array_equal(r["ids"][:m].cpu().numpy(), ref["top_id"])
        head_ref.assert_close(r["lps"][:m], ref["top_logprob"], ref["top_logprob_tol"], "alternatives")
