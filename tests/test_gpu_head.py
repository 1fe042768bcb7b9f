"""GPU: the free-size heads (row quantiser, int8 layer, log probabilities) against 64-bit
references on the CPU (tests/head_ref.py): types, odd sizes, strides, masks, what they leave
alone, streams, graphs, and a run of them together."""
import zlib

import numpy as np
import pytest
import torch

import head_ref

pytestmark = pytest.mark.gpu

FLOATS = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
NEG = float("-inf")
CANARY = 77


class Head:
    """The operators on torch tensors, on the stream of one context."""

    def __init__(self, native, stream=None):
        self.lib = native
        self.stream = stream or torch.cuda.Stream()
        self.ctx = native.FsxContext(max_entries=1024, max_batch=1024)
        self.ctx.set_stream(self.stream.cuda_stream)
        self.code = {torch.float32: native.DTYPE_F32, torch.float16: native.DTYPE_F16,
                     torch.bfloat16: native.DTYPE_BF16, torch.int8: native.DTYPE_I8}
        self.act = {"none": native.ACT_NONE, "relu": native.ACT_RELU, "sigmoid": native.ACT_SIGMOID}

    def quantize(self, x, q, scale):
        self.ctx.quantize_rows_device(x.data_ptr(), self.code[x.dtype], x.shape[0], x.shape[1], x.stride(0),
                                      q.data_ptr(), q.stride(0), scale.data_ptr())

    def layer(self, w, ws, bias, act):
        return self.lib.q8_linear(w.data_ptr(), ws.data_ptr(), None if bias is None else bias.data_ptr(), w.shape[1],
                                  w.shape[0], w.stride(0), self.act[act])

    def linear_work(self, layer, x):
        return torch.full((self.lib.linear_q8_work(layer, self.code[x.dtype], x.shape[0]),), 255, dtype=torch.uint8,
                          device="cuda")

    def linear(self, layer, x, xs, y, work):
        self.ctx.linear_q8_device(layer, x.data_ptr(), self.code[x.dtype], x.stride(0),
                                  None if xs is None else xs.data_ptr(), x.shape[0], y.data_ptr(), self.code[y.dtype],
                                  y.stride(0), work.data_ptr(), work.numel())

    def logprobs_work(self, x, top):
        return torch.full((self.lib.logprobs_work(x.shape[0], x.shape[1], top),), 255, dtype=torch.uint8,
                          device="cuda")

    def logprobs(self, x, target, logprob, entropy, ids, lps, work):
        p = [None if t is None else t.data_ptr() for t in (target, logprob, entropy, ids, lps)]
        self.ctx.logprobs_device(x.data_ptr(), self.code[x.dtype], x.shape[0], x.shape[1], x.stride(0), p[0], p[1],
                                 p[2], 0 if ids is None else ids.shape[1], p[3], p[4], work.data_ptr(), work.numel())


@pytest.fixture(scope="module")
def head(native):
    h = Head(native)
    yield h
    h.ctx.close()


def rows_of(gen, rows, cols, pad, dtype, spread=1.0):
    """Normal rows `cols + pad` apart, a few of them much smaller or larger than the others."""
    x = torch.randn(rows, cols + pad, generator=gen) * spread
    x *= 2.0 ** torch.randint(-6, 7, (rows, 1), generator=gen)
    return x.to(dtype).cuda()[:, :cols]


def codes_of(gen, rows, cols, pad, lo=-128):
    return torch.randint(lo, 128, (rows, cols + pad), generator=gen, dtype=torch.int8).cuda()[:, :cols]


def gen_of(*key):
    return torch.Generator().manual_seed(zlib.crc32(repr(key).encode()))


# ---------------------------------------------------------------- row quantiser

def run_quantize(head, x, pad=5):
    rows, cols = x.shape
    q = torch.full((rows + 1, cols + pad), CANARY, dtype=torch.int8, device="cuda")
    scale = torch.full((rows + 1,), 7.0, device="cuda")
    torch.cuda.synchronize()
    head.quantize(x, q[:rows, :cols], scale[:rows])
    torch.cuda.synchronize()
    assert (q[rows] == CANARY).all() and (q[:, cols:] == CANARY).all() and scale[rows] == 7.0
    return q[:rows, :cols].cpu(), scale[:rows].cpu()


def check_quantize(head, x, pad=5):
    q, scale = run_quantize(head, x, pad)
    wq, ws = head_ref.quantize(x)
    assert torch.equal(scale.isnan(), ws.isnan())
    assert torch.equal(scale.nan_to_num(0.0), ws.nan_to_num(0.0)), "scales are 32-bit numbers by definition"
    assert torch.equal(q.long(), wq), "codes are whole numbers by definition"


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,cols,pad", [(1, 1, 0), (1, 4096, 0), (3, 17, 0), (5, 1003, 5), (64, 16, 16), (65, 64, 0),
                                           (257, 255, 1), (4, 16385, 3), (2, 70000, 0), (4097, 8, 0), (70001, 2, 1),
                                           (33, 8192, 8), (7, 1025, 0), (130, 300, 4)])
def test_quantize(head, dtype, rows, cols, pad):
    g = gen_of("q", rows, cols)
    check_quantize(head, rows_of(g, rows, cols, pad, FLOATS[dtype]), pad=(0, 5, 16)[rows % 3])


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("cols", [15, 16, 17, 31, 33, 47, 63, 65, 95, 112, 113, 129, 200, 225, 257, 317, 511, 513, 1000, 1025,
                                  2000, 2049, 4095, 4097, 8191, 8193, 16383, 16400])
def test_quantize_row_ends(head, dtype, cols):
    """Every number of threads and chunks a row, the last chunk beginning inside the one before."""
    for rows, pad in ((1, 0), (67, 1), (300, 16)):
        check_quantize(head, rows_of(gen_of("qe", rows, cols), rows, cols, pad, FLOATS[dtype]), pad=pad)


def test_quantize_borders(head):
    """Quotients on a half and a last place beside it, for scales with all kinds of last places."""
    g = gen_of("borders")
    rows = []
    for e in range(64):
        amax = np.float32(127 * 2.0 ** (e - 32)) if e % 2 else np.float32((1 + torch.rand(1, generator=g).item()) * 2.0 ** (e - 32))
        s = np.float32(amax / np.float32(127))
        half = ((np.arange(127) + 0.5) * np.float64(s)).astype(np.float32)
        v = np.concatenate([[amax], half, np.nextafter(half, np.float32(0)), np.nextafter(half, np.float32(np.inf)),
                            -half, -np.nextafter(half, np.float32(0)), -np.nextafter(half, np.float32(np.inf))])
        rows.append(np.where(np.abs(v) > amax, amax, v))
    check_quantize(head, torch.from_numpy(np.stack(rows).astype(np.float32)).cuda())


def test_quantize_special_rows(head):
    x = torch.randn(40, 300, generator=gen_of("special"))
    x[0] = 0
    x[1, 299] = float("nan")
    x[2, 0] = float("inf")
    x[3, 7] = NEG
    x[4] = 1e-44                 # below 32-bit normal numbers
    x[5] *= 1e-38
    x[6] = torch.finfo(torch.float32).max
    x[7] = -torch.finfo(torch.float32).max
    x[8] = -0.0
    x[9, 1:] = 0
    x[10] = float("nan")
    x[11, 3], x[11, 200] = float("inf"), float("nan")
    check_quantize(head, x.cuda())
    for t in (torch.float16, torch.bfloat16):
        check_quantize(head, x.to(t).cuda())


def test_quantize_far_rows(head):
    """Rows whose elements lie beyond 2^31 elements from the first."""
    ld = (1 << 30) + 8
    big = torch.zeros(2 * ld + 64, dtype=torch.float16, device="cuda")
    x = big.as_strided((3, 50), (ld, 1))
    x.copy_(torch.randn(3, 50, generator=gen_of("far")).half())
    check_quantize(head, x)


# ---------------------------------------------------------------- int8 layer

def check_linear(head, x, xs, w, ws, bias, act, ydtype, ypad=3, want=None):
    rows, n = x.shape[0], w.shape[0]
    y = torch.full((rows + 1, n + ypad), float(CANARY), dtype=ydtype, device="cuda")
    layer = head.layer(w, ws, bias, act)
    work = head.linear_work(layer, x)
    torch.cuda.synchronize()
    head.linear(layer, x, xs, y[:rows, :n], work)
    torch.cuda.synchronize()
    assert (y[rows] == CANARY).all() and (y[:, n:] == CANARY).all(), "what is behind the rows was written"
    codes, scale = (x.cpu().long(), xs) if xs is not None else head_ref.quantize(x)
    ref, tol = head_ref.linear(codes, scale, w, ws, bias, act, ydtype)
    head_ref.assert_close(y[:rows, :n], ref, tol, "y")
    return y[:rows, :n]


def layer_of(g, n, k, pad, bias):
    w = codes_of(g, n, k, pad)
    ws = ((0.5 + torch.rand(n, generator=g)) / (64 * k ** 0.5)).cuda()
    return w, ws, torch.randn(n, generator=g).cuda() if bias else None


ROWS = [1, 2, 3, 4, 5, 15, 16, 17, 33, 64, 65, 129, 257, 600]
SHAPES = [(1, 1), (7, 5), (8, 16), (15, 3), (16, 64), (17, 65), (63, 130), (64, 1), (65, 17), (100, 33), (127, 255),
          (128, 256), (129, 48), (255, 7), (1000, 100), (1003, 777), (4096, 64), (520, 512)]


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("k,n", SHAPES)
def test_linear_codes(head, rows, k, n):
    g = gen_of("lc", rows, k, n)
    i = rows + k + n
    w, ws, bias = layer_of(g, n, k, (0, 16, 3)[i % 3], i % 2)
    x = codes_of(g, rows, k, (0, 3, 16)[rows % 3])
    xs = (0.005 + 0.01 * torch.rand(rows, generator=g)).cuda()
    check_linear(head, x, xs, w, ws, bias, ("none", "relu", "sigmoid")[i % 3], list(FLOATS.values())[rows % 3])


@pytest.mark.parametrize("xt", FLOATS)
@pytest.mark.parametrize("rows", [1, 2, 4, 5, 16, 17, 100, 513])
@pytest.mark.parametrize("k,n", [(1, 4), (8, 16), (13, 7), (40, 33), (64, 64), (70, 20), (777, 130), (4096, 256),
                                 (5001, 9)])
def test_linear_floats(head, xt, rows, k, n):
    g = gen_of("lf", rows, k, n)
    i = rows + k + n
    w, ws, bias = layer_of(g, n, k, (0, 3, 16)[i % 3], i % 2)
    x = rows_of(g, rows, k, (0, 1, 8)[rows % 3], FLOATS[xt])
    check_linear(head, x, None, w, ws, bias, ("relu", "none", "sigmoid")[i % 3], list(FLOATS.values())[i % 3])


@pytest.mark.parametrize("rows,k,n", [(1500, 1024, 2000), (4100, 264, 1030), (300, 4112, 4100), (2, 20000, 3000),
                                      (40, 8200, 520), (12, 131071, 40), (200001, 8, 16), (66000, 24, 3)])
def test_linear_large(head, rows, k, n):
    g = gen_of("ll", rows, k, n)
    w, ws, bias = layer_of(g, n, k, 0, True)
    x = rows_of(g, rows, k, 0, torch.bfloat16)
    check_linear(head, x, None, w, ws, bias, "none", torch.float32)
    q, s = head_ref.quantize(x)
    check_linear(head, q.to(torch.int8).cuda(), s.cuda(), w, ws, bias, "none", torch.bfloat16, ypad=0)


@pytest.mark.parametrize("rows", [1, 20, 300])
def test_linear_largest_sums(head, rows):
    """Every product 128 * 128 over the longest rows: the sum fills 31 bits."""
    k, n = 131071, 70
    x = torch.full((rows, k), -128, dtype=torch.int8, device="cuda")
    w = torch.full((n, k), -128, dtype=torch.int8, device="cuda")
    w[1::2] = 127
    ones = torch.ones(max(rows, n), device="cuda")
    check_linear(head, x, ones[:rows], w, ones[:n], None, "none", torch.float32)


@pytest.mark.parametrize("rows,k", [(3, 8), (3, 500), (40, 24), (40, 700), (400, 1024)])
def test_linear_special_rows(head, rows, k):
    """Rows with a NaN or an infinity give NaN, zero rows the bias, and no other row is touched."""
    g = gen_of("ls", rows, k)
    w, ws, bias = layer_of(g, 33, k, 0, True)
    x = rows_of(g, rows, k, 0, torch.float32)
    x[0, k - 1] = float("nan")
    x[1, 0] = float("inf")
    x[2] = 0
    for act in ("none", "relu", "sigmoid"):
        y = check_linear(head, x, None, w, ws, bias, act, torch.float32)
        assert y[:2].isnan().all() and not y[2:].isnan().any()


def test_linear_garbage_behind_rows(head):
    """What lies between a row's end and the next row is not read as data."""
    g = gen_of("garbage")
    for rows in (2, 40, 300):
        for k in (70, 1001, 8):
            w, ws, _ = layer_of(g, 40, k, 26, False)
            x = rows_of(g, rows, k, 10, torch.float32)
            x.as_strided((rows, 10), (k + 10, 1), k)[:] = float("nan")
            check_linear(head, x, None, w, ws, None, "none", torch.float32)


# (rows, k, n, bytes between rows of x, of the weights): strides of 16 bytes or not, one tile of
# k or several with a rest, a last tile of a few rows and channels
TILES = [(4097, 130, 4000, 14, 14), (4097, 70, 4000, 10, 10), (2300, 100, 2305, 12, 12), (2300, 300, 2305, 4, 4),
         (1700, 70, 1801, 10, 10), (1700, 200, 1801, 8, 8), (1700, 390, 1801, 10, 10), (1700, 700, 1801, 4, 4),
         (300, 65, 400, 15, 15), (300, 520, 400, 8, 8), (300, 65, 400, 0, 15), (300, 777, 403, 0, 0),
         (2100, 333, 2100, 0, 0), (2100, 333, 2100, 3, 0), (2100, 333, 2100, 0, 3), (4100, 65, 4100, 1, 2),
         (100, 5000, 200, 8, 8), (100, 5001, 200, 0, 0), (17, 2048, 100, 0, 0), (4000, 2000, 320, 0, 1), (700, 2000, 2000, 0, 15), (40, 2049, 7, 15, 15), (40, 2049, 7, 0, 15),
         (33, 131071, 65, 1, 1), (20, 4096, 16390, 0, 0), (2, 16400, 100, 0, 0), (16, 9000, 2050, 8, 8),
         (17000, 130, 50, 14, 14), (17001, 300, 64, 4, 4), (4097, 2050, 4000, 14, 14), (9, 9001, 130, 0, 0), (16, 300, 9000, 4, 4), (31, 300, 8000, 4, 5)]


@pytest.mark.parametrize("rows,k,n,xpad,wpad", TILES)
def test_linear_forms(head, rows, k, n, xpad, wpad):
    """Each way that a product of codes takes through the GPU, in a workspace of exactly its size."""
    g = gen_of("tiles", rows, k, n, xpad, wpad)
    w, ws, bias = layer_of(g, n, k, wpad, True)
    x = codes_of(g, rows, k, xpad)
    xs = (0.005 + 0.01 * torch.rand(rows, generator=g)).cuda()
    layer = head.layer(w, ws, bias, "none")
    need = head.lib.linear_q8_work(layer, head.lib.DTYPE_I8, rows)
    work = torch.full((need + 256,), 255, dtype=torch.uint8, device="cuda")
    y = torch.full((rows + 1, n + 3), float(CANARY), device="cuda")
    torch.cuda.synchronize()
    head.linear(layer, x, xs, y[:rows, :n], work[:need])
    torch.cuda.synchronize()
    assert (work[need:] == 255).all(), "behind the workspace"
    assert (y[rows] == CANARY).all() and (y[:, n:] == CANARY).all(), "what is behind the rows was written"
    ref, tol = head_ref.linear(x.cpu().long(), xs, w, ws, bias, "none", torch.float32)
    head_ref.assert_close(y[:rows, :n], ref, tol, "y")


def test_linear_forms_agree(head):
    """A row's results have the same bits in any batch, at any stride, from codes or floats."""
    g = gen_of("agree")
    for k, n, most in ((4096, 520, 700), (500, 2100, 2100), (60, 33, 300)):
        w, ws, bias = layer_of(g, n, k, 0, True)
        odd = codes_of(g, n, k, 3)
        odd.copy_(w)
        x = rows_of(g, most, k, 0, torch.bfloat16)
        q, s = torch.empty(most, k, dtype=torch.int8, device="cuda"), torch.empty(most, device="cuda")
        torch.cuda.synchronize()
        head.quantize(x, q, s)
        whole = None
        for weight in (w, odd):
            layer = head.layer(weight, ws, bias, "sigmoid")
            for rows in (most, 300, 33, 17, 5, 4, 1):
                for xx, xs in ((x[:rows], None), (q[:rows], s)):
                    y = torch.empty(rows, n, device="cuda")
                    work = head.linear_work(layer, xx)
                    torch.cuda.synchronize()
                    head.linear(layer, xx, xs, y, work)
                    torch.cuda.synchronize()
                    whole = y if whole is None else whole
                    assert torch.equal(y, whole[:rows]), (k, n, rows)


@pytest.mark.parametrize("rows,k,n,xpad,wpad", [(100, 5000, 200, 8, 8), (2100, 333, 2100, 0, 0), (1700, 390, 1801, 10, 10)])
def test_linear_forms_replayed(head, rows, k, n, xpad, wpad):
    """Products in parts and with copied operands, captured and replayed on other codes."""
    g = gen_of("replay", rows)
    w, ws, bias = layer_of(g, n, k, wpad, True)
    x = codes_of(g, rows, k, xpad)
    xs = torch.rand(rows, generator=g).cuda()
    y = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda")
    layer = head.layer(w, ws, bias, "relu")
    work = head.linear_work(layer, x)
    torch.cuda.synchronize()
    head.linear(layer, x, xs, y, work)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=head.stream):
        head.linear(layer, x, xs, y, work)
    for _ in range(4):
        x.copy_(codes_of(g, rows, k, 0))
        w.copy_(codes_of(g, n, k, 0))
        work.fill_(255)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone()
        y.zero_()
        torch.cuda.synchronize()
        head.linear(layer, x, xs, y, work)
        torch.cuda.synchronize()
        assert torch.equal(got, y)


@pytest.mark.parametrize("xt", FLOATS)
@pytest.mark.parametrize("rows,k", [(4, 8176), (4, 8177), (3, 10000), (2, 16368), (1, 32752), (1, 32753), (4, 65), (1, 16385)])
def test_linear_floats_few(head, xt, rows, k):
    """Floats quantised by every block, up to the LDS they may fill, and the sizes behind it."""
    g = gen_of("ff", rows, k)
    w, ws, bias = layer_of(g, 37, k, 3, True)
    check_linear(head, rows_of(g, rows, k, 1, FLOATS[xt]), None, w, ws, bias, "none", torch.float32)


def test_linear_floats_few_many_channels(head):
    """.. with eight waves a block instead of sixteen."""
    g = gen_of("ffn")
    w, ws, bias = layer_of(g, 8200, 300, 4, True)
    check_linear(head, rows_of(g, 3, 300, 1, torch.float16), None, w, ws, bias, "none", torch.float32)


@pytest.mark.parametrize("xt", [*FLOATS, "i8"])
@pytest.mark.parametrize("rows,k,n", [(9001, 70, 1), (9001, 130, 17), (20005, 300, 32), (140000, 65, 16), (50, 3008, 5),
                                      (50, 3009, 5), (333, 1000, 31), (17, 20000, 9), (40, 7000, 32), (33, 13000, 16),
                                      (70003, 129, 33), (8200, 520, 12), (50, 3008, 20), (8200, 3000, 20)])
def test_linear_few_channels(head, xt, rows, k, n):
    """Many rows to few channels, at strides that are multiples of 16 and odd ones."""
    g = gen_of("fc", rows, k, n)
    for pad in (-k % 16, (-k % 4) + 1):
        w, ws, bias = layer_of(g, n, k, pad, True)
        if xt == "i8":
            x, xs = codes_of(g, rows, k, pad), (0.005 + 0.01 * torch.rand(rows, generator=g)).cuda()
        else:
            x, xs = rows_of(g, rows, k, pad, FLOATS[xt]), None
        check_linear(head, x, xs, w, ws, bias, "none", torch.float32)


@pytest.mark.parametrize("xt", [*FLOATS, "i8"])
@pytest.mark.parametrize("rows,k,n", [(140001, 5, 20), (70001, 16, 100), (33000, 17, 130), (40000, 31, 65), (9000, 40, 700),
                                      (3000, 64, 3000), (2, 7, 300), (70000, 7, 12)])
def test_linear_short_rows(head, xt, rows, k, n):
    """Rows of up to 64 values to few channels and many, beside each other and apart."""
    g = gen_of("short", rows, k, n)
    for pad in (0, 3):
        w, ws, bias = layer_of(g, n, k, pad, True)
        if xt == "i8":
            x, xs = codes_of(g, rows, k, pad), (0.005 + 0.01 * torch.rand(rows, generator=g)).cuda()
        else:
            x, xs = rows_of(g, rows, k, pad, FLOATS[xt]), None
        check_linear(head, x, xs, w, ws, bias, "relu", torch.bfloat16)


def test_linear_far_rows(head):
    """x, weights and y beyond 2^31 elements from their first."""
    g = gen_of("far")
    ld = (1 << 30) + 16
    big = torch.zeros(2 * ld + 4096, dtype=torch.int8, device="cuda")
    bigy = torch.zeros(2 * ld + 4096, dtype=torch.float16, device="cuda")
    w, ws, _ = layer_of(g, 3, 200, 0, False)
    far_w = big.as_strided((3, 200), (ld, 1))
    far_w.copy_(w)
    far_x = big.as_strided((3, 200), (ld, 1), 1024)
    far_x.copy_(codes_of(g, 3, 200, 0))
    far_y = bigy.as_strided((3, 3), (ld, 1))
    xs = torch.full((3,), 0.01, device="cuda")
    layer = head.layer(far_w, ws, None, "none")
    torch.cuda.synchronize()
    head.linear(layer, far_x, xs, far_y, head.linear_work(layer, far_x))
    torch.cuda.synchronize()
    ref, tol = head_ref.linear(far_x.cpu().long(), xs, far_w, ws, None, "none", torch.float16)
    head_ref.assert_close(far_y, ref, tol, "y")


def test_linear_several_launches(head):
    """More channels than one launch takes: each part of them has the bits of its own product."""
    g = gen_of("slabs")
    n, cuts = (1 << 20) * 2 + 100, [0, 70, (1 << 20) - 5, (1 << 20) + 90, (1 << 21) + 100]
    for rows, k, xt in ((2, 8, torch.float32), (3, 70, torch.float32), (5, 70, torch.float32), (70, 66, torch.float16)):
        w = torch.randint(-128, 128, (n, k), dtype=torch.int8, device="cuda")
        ws = torch.rand(n, device="cuda")
        bias = torch.randn(n, device="cuda")
        x = rows_of(g, rows, k, 0, xt)
        y, part = torch.empty(rows, n, dtype=torch.float16, device="cuda"), torch.empty(rows, n, dtype=torch.float16, device="cuda")
        layer = head.layer(w, ws, bias, "relu")
        work = head.linear_work(layer, x)
        torch.cuda.synchronize()
        head.linear(layer, x, None, y, work)
        for a, b in zip(cuts, cuts[1:]):
            head.linear(head.layer(w[a:b], ws[a:b], bias[a:b], "relu"), x, None, part[:, a:b], work)
        torch.cuda.synchronize()
        assert torch.equal(y, part)
        check_linear(head, x, None, w[-300:], ws[-300:], bias[-300:], "relu", torch.float16)


@pytest.mark.parametrize("k,n", [(70, 12), (66, 32), (12, 20)])
def test_linear_more_rows_than_one_launch(head, k, n):
    """2^24 rows go in one launch: the few behind them have the bits of a call of their own, and all
    of one that starts in their midst."""
    rows = (1 << 24) + 9
    g = gen_of("slabrows", k, n)
    w, ws, bias = layer_of(g, n, k, 2, True)
    layer = head.layer(w, ws, bias, "relu")
    x = torch.zeros(rows, k, dtype=torch.float16, device="cuda")
    x[:40] = rows_of(g, 40, k, 0, torch.float16)
    x[-40:] = rows_of(g, 40, k, 0, torch.float16)
    x[1 << 23:(1 << 23) + 40] = x[-40:]
    q, s = torch.empty(rows, k, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    torch.cuda.synchronize()
    head.quantize(x, q, s)
    for xx, xs in ((x, None), (q, s)):
        y = torch.full((rows + 1, n), float(CANARY), dtype=torch.float16, device="cuda")
        work = head.linear_work(layer, xx)
        torch.cuda.synchronize()
        head.linear(layer, xx, xs, y[:rows], work)
        torch.cuda.synchronize()
        assert (y[rows] == CANARY).all()
        assert torch.equal(y[rows - 40:rows], y[1 << 23:(1 << 23) + 40])
        for part in (slice(0, 40), slice(rows - 40, rows)):
            z = check_linear(head, xx[part], None if xs is None else xs[part], w, ws, bias, "relu", torch.float16)
            assert torch.equal(y[part], z)
        del y, work


# ---------------------------------------------------------------- log probabilities

def check_logprobs(head, x, target=True, entropy=True, top=5):
    rows, classes = x.shape
    g = gen_of("t", rows, classes)
    t = torch.randint(0, classes, (rows,), generator=g, dtype=torch.int32)
    t[::5] = -1
    t[3::7] = classes if rows % 2 else -2
    t = t.cuda() if target is True else target
    lp, en = torch.full((rows + 1,), 7.0, device="cuda"), torch.full((rows + 1,), 7.0, device="cuda")
    ids = torch.full((rows + 1, top), CANARY, dtype=torch.int32, device="cuda")
    lps = torch.full((rows + 1, top), 7.0, device="cuda")
    work = head.logprobs_work(x, top)
    torch.cuda.synchronize()
    head.logprobs(x, t, None if t is None else lp, en if entropy else None, ids[:rows] if top else None,
                  lps[:rows] if top else None, work)
    torch.cuda.synchronize()
    assert lp[rows] == 7 and en[rows] == 7 and (ids[rows] == CANARY).all() and (lps[rows] == 7).all()
    ref = head_ref.logprobs(x, t, top)
    if t is not None:
        head_ref.assert_close(lp[:rows], ref["logprob"], ref["logprob_tol"], "logprob")
    if entropy:
        head_ref.assert_close(en[:rows], ref["entropy"], ref["entropy_tol"], "entropy")
        assert not (en[:rows] < 0).any()
    if top:
        assert np.array_equal(ids[:rows].cpu().numpy(), ref["top_id"]), "alternatives"
        head_ref.assert_close(lps[:rows], ref["top_logprob"], ref["top_logprob_tol"], "top_logprob")


def logits_of(g, rows, classes, pad, dtype, masked=0.0):
    x = 3 * torch.randn(rows, classes + pad, generator=g)
    if masked:
        x[torch.rand(rows, classes + pad, generator=g) < masked] = NEG
    return x.to(dtype).cuda()[:, :classes]


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,classes,pad,top", [
    (1, 1, 0, 1), (2, 2, 1, 5), (300, 3, 0, 3), (1000, 16, 0, 3), (77, 17, 0, 17), (65, 31, 2, 8), (40, 64, 0, 64),
    (33, 100, 4, 10), (20, 255, 1, 5), (19, 256, 0, 20), (18, 257, 8, 1), (13, 512, 0, 33), (12, 513, 0, 5),
    (9, 1000, 3, 64), (9, 1024, 0, 5), (8, 1025, 0, 5), (7, 2048, 0, 64), (5, 4097, 5, 20), (3, 8191, 0, 2),
    (2, 32003, 0, 40), (1, 131072, 0, 20), (1, 70001, 1, 64), (5, 50021, 3, 20), (600, 2100, 0, 4)])
def test_logprobs(head, dtype, rows, classes, pad, top):
    check_logprobs(head, logits_of(gen_of("l", rows, classes), rows, classes, pad, FLOATS[dtype]), top=top)


@pytest.mark.parametrize("classes", [5, 16, 130, 700, 3001, 40000])
@pytest.mark.parametrize("masked", [0.5, 0.999])
def test_logprobs_masked(head, classes, masked):
    x = logits_of(gen_of("m", classes), 40, classes, 1, torch.float16, masked)
    x[7] = NEG
    x[8] = NEG
    x[8, classes - 1] = -3.0
    check_logprobs(head, x, top=20)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("classes", [4, 16, 200, 1000, 2500, 33000])
def test_logprobs_special_rows(head, dtype, classes):
    """NaN, infinities, the type's lowest value as a mask, equal logits, rising and falling rows."""
    t = FLOATS[dtype]
    x = logits_of(gen_of("s", classes), 24, classes, 0, torch.float32)
    low = torch.finfo(t).min
    x[0, classes // 2] = float("nan")
    x[1, 0] = float("inf")
    x[2, 1], x[2, 3] = float("inf"), NEG
    x[3] = low
    x[4] = low
    x[4, 2] = 1.0
    x[5] = 0.0
    x[6] = -5.0
    x[7] = torch.linspace(-20, 20, classes)
    x[8] = torch.linspace(20, -20, classes)
    x[9, ::2] = 4.0
    x[10] = 0.0
    x[10, ::3] = -0.0
    x[11] = torch.finfo(t).max
    x[12] = 50.0
    x[12, 1] = 90.0
    x[13, :3] = NEG
    x[14] = float("nan")
    x[15] = NEG
    x[15, 0] = float("nan")
    x[16] = 1e-30
    x[17, classes - 1] = 60000.0
    check_logprobs(head, x.to(t), top=min(33, 2 * classes))


@pytest.mark.parametrize("rows,classes,top", [(1030, 1500, 64), (1030, 5003, 1), (1030, 2048, 33), (30, 9000, 64),
                                              (3, 200001, 64), (3, 60000, 1), (257, 20000, 32)])
def test_logprobs_orders(head, rows, classes, top):
    """Rows whose candidates outrun any bound: rising, equal, falling, all of a few values."""
    g = gen_of("orders", rows, classes)
    x = 3 * torch.randn(rows, classes, generator=g)
    step = torch.arange(classes) / classes
    x[0] = step * 9
    x[1] = 2.5
    if rows > 2: x[2] = -step * 9
    if rows > 3:
        x[3] = torch.randint(0, 3, (classes,), generator=g).float()
        x[4] = (torch.arange(classes) // 512 % 7).float()
        x[rows - 1] = step * 3
        x[rows - 2, 1:] = NEG
    check_logprobs(head, x.cuda(), top=top)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows", [1, 70, 300, 1100])
@pytest.mark.parametrize("classes,top", [(3, 4), (4, 64), (7, 28), (8, 4), (9, 9), (16, 5), (20, 22), (25, 4), (33, 33),
                                         (64, 4), (84, 19), (100, 20), (128, 32), (200, 20), (200, 23), (256, 9), (300, 33), (500, 55), (512, 64), (129, 6), (129, 12), (130, 64), (256, 25), (278, 30), (513, 6),
                                         (520, 40), (700, 46), (1000, 64), (1004, 20), (1023, 7)])
def test_logprobs_short_orders(head, dtype, rows, classes, top):
    """Each way that the alternatives of short rows are put in order: ties, masked and empty rows,
    more asked for than there are."""
    g = gen_of("so", rows, classes, top)
    x = 3 * torch.randn(rows, classes + 1, generator=g)
    x[::3] = torch.randint(-2, 3, (len(x[::3]), classes + 1), generator=g).float()
    x[1::4][torch.rand(len(x[1::4]), classes + 1, generator=g) < 0.9] = NEG
    x[-1] = NEG
    if rows > 40:
        x[20], x[21] = 1.0, NEG
        x[21, classes - 1] = 0.5
        x[22, classes // 2] = float("nan")
        x[23, 0] = float("inf")
        x[24] = torch.arange(classes + 1) / classes
    check_logprobs(head, x.to(FLOATS[dtype]).cuda()[:, :classes], top=top)


def test_logprobs_parts(head):
    """Each output by itself, and none of them but the alternatives."""
    for classes in (16, 300, 5000, 70000):
        x = logits_of(gen_of("p", classes), 11, classes, 0, torch.bfloat16)
        check_logprobs(head, x, top=0)
        check_logprobs(head, x, target=None, top=0)
        check_logprobs(head, x, target=None, entropy=False, top=2)
        check_logprobs(head, x, entropy=False, top=0)


def test_logprobs_many_rows(head):
    check_logprobs(head, logits_of(gen_of("many"), 300007, 16, 0, torch.float32), top=3)
    check_logprobs(head, logits_of(gen_of("many2"), 70001, 6, 2, torch.float16, 0.9), top=7)


def test_logprobs_far_rows(head):
    ld = (1 << 30) + 8
    big = torch.zeros(2 * ld + 8192, dtype=torch.float16, device="cuda")
    for classes in (40, 5000):
        x = big.as_strided((3, classes), (ld, 1))
        x.copy_(3 * torch.randn(3, classes, generator=gen_of("farl")).half())
        check_logprobs(head, x)


# ---------------------------------------------------------------- as a program uses them

def test_together(head):
    """Flow features through two layers quantised on the GPU by channel, to class answers: the
    whole run on one stream with no wait between, captured into a graph as well, replayed on new
    features several times; every replay has the bits of the eager run."""
    g = gen_of("together")
    flows, hidden, classes, top = 500, 96, 20, 4
    dims = [(8, hidden), (hidden, classes)]
    wf = [torch.randn(o, i, generator=g).cuda() / i ** 0.5 for i, o in dims]
    bias = [torch.randn(o, generator=g).cuda() for _, o in dims]
    wq = [torch.empty(o, i, dtype=torch.int8, device="cuda") for i, o in dims]
    ws = [torch.empty(o, device="cuda") for _, o in dims]
    x = torch.empty(flows, 8, device="cuda")
    h = torch.empty(flows, hidden, dtype=torch.bfloat16, device="cuda")
    z = torch.empty(flows, classes, device="cuda")
    target = torch.randint(0, classes, (flows,), generator=g, dtype=torch.int32).cuda()
    lp, en = torch.empty(flows, device="cuda"), torch.empty(flows, device="cuda")
    ids = torch.empty(flows, top, dtype=torch.int32, device="cuda")
    lps = torch.empty(flows, top, device="cuda")
    torch.cuda.synchronize()
    for w, q, s in zip(wf, wq, ws):
        head.quantize(w, q, s)
    layers = [head.layer(q, s, b, a) for q, s, b, a in zip(wq, ws, bias, ("relu", "none"))]
    works = [head.linear_work(layers[0], x), head.linear_work(layers[1], h), head.logprobs_work(z, top)]
    torch.cuda.synchronize()

    def run():
        head.linear(layers[0], x, None, h, works[0])
        head.linear(layers[1], h, None, z, works[1])
        head.logprobs(z, target, lp, en, ids, lps, works[2])

    def outputs():
        torch.cuda.synchronize()
        return [t.clone() for t in (h, z, lp, en, ids, lps)]

    graph = torch.cuda.CUDAGraph()
    x.copy_(torch.rand(flows, 8, generator=g))
    torch.cuda.synchronize()
    with torch.cuda.stream(head.stream):
        run()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=head.stream):
        run()
    for step in range(4):
        with torch.cuda.stream(head.stream):
            x.copy_(torch.rand(flows, 8, generator=g) * (step + 1))
            run()
        eager = outputs()
        for t in (h, z, lp, en, ids, lps):
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        for a, b in zip(outputs(), eager):
            assert torch.equal(a, b)
    # against 64 bits, layer by layer from the bits that each layer read
    xq, xsc = head_ref.quantize(x)
    for i, (w, q, s) in enumerate(zip(wf, wq, ws)):
        cq, cs = head_ref.quantize(w)
        assert torch.equal(q.cpu().long(), cq) and torch.equal(s.cpu(), cs)
    ref, tol = head_ref.linear(xq, xsc, wq[0], ws[0], bias[0], "relu", torch.bfloat16)
    head_ref.assert_close(h, ref, tol, "hidden")
    hq, hs = head_ref.quantize(h)
    ref, tol = head_ref.linear(hq, hs, wq[1], ws[1], bias[1], "none", torch.float32)
    head_ref.assert_close(z, ref, tol, "logits")
    ref = head_ref.logprobs(z, target, top)
    head_ref.assert_close(lp, ref["logprob"], ref["logprob_tol"], "logprob")
    assert np.array_equal(ids.cpu().numpy(), ref["top_id"])


@pytest.mark.parametrize("rows,k,n,classes", [(1, 4096, 512, 70000), (70, 1000, 300, 9000), (900, 520, 700, 300)])
def test_graph_replays(head, rows, k, n, classes):
    """Every kernel of these sizes captured once and replayed on new inputs, with eager work between."""
    g = gen_of("graph", rows)
    w, ws, bias = layer_of(g, n, k, 0, True)
    x = rows_of(g, rows, k, 0, torch.bfloat16)
    y = torch.empty(rows, n, device="cuda")
    layer = head.layer(w, ws, bias, "none")
    z = logits_of(g, rows, classes, 0, torch.bfloat16)
    q, s = torch.empty(rows, k, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    lp, en = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    ids, lps = torch.empty(rows, 9, dtype=torch.int32, device="cuda"), torch.empty(rows, 9, device="cuda")
    target = torch.randint(0, classes, (rows,), generator=g, dtype=torch.int32).cuda()
    works = [head.linear_work(layer, x), head.logprobs_work(z, 9)]

    def run():
        head.quantize(x, q, s)
        head.linear(layer, x, None, y, works[0])
        head.logprobs(z, target, lp, en, ids, lps, works[1])

    torch.cuda.synchronize()
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=head.stream):
        run()
    for step in range(4):
        x.copy_(torch.randn(rows, k, generator=g).bfloat16())
        z.copy_((2 * torch.randn(rows, classes, generator=g)).bfloat16())
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (q, s, y, lp, en, ids, lps)]
        for t in (q, s, y, lp, en, ids, lps):
            t.zero_()
        torch.cuda.synchronize()
        run()
        torch.cuda.synchronize()
        for a, b in zip(got, (q, s, y, lp, en, ids, lps)):
            assert torch.equal(a, b), step


def test_two_contexts_at_once(native):
    """Two contexts on two streams, each with its own workspace, running at the same time."""
    heads = [Head(native), Head(native)]
    g = gen_of("two")
    jobs = []
    for h, rows in zip(heads, (3, 200)):
        w, ws, bias = layer_of(g, 512, 2048, 0, True)
        x = rows_of(g, rows, 2048, 0, torch.bfloat16)
        z = logits_of(g, rows, 40000, 0, torch.bfloat16)
        y, lp, en = (torch.empty(rows, 512, device="cuda"), torch.empty(rows, device="cuda"),
                     torch.empty(rows, device="cuda"))
        layer = h.layer(w, ws, bias, "none")
        t = torch.zeros(rows, dtype=torch.int32, device="cuda")
        jobs.append((h, layer, x, y, h.linear_work(layer, x), z, t, lp, en, h.logprobs_work(z, 0), w, ws, bias))
    torch.cuda.synchronize()
    for _ in range(10):
        for h, layer, x, y, wk, z, t, lp, en, wk2, *_ in jobs:
            h.linear(layer, x, None, y, wk)
            h.logprobs(z, t, lp, en, None, None, wk2)
    torch.cuda.synchronize()
    for h, layer, x, y, wk, z, t, lp, en, wk2, w, ws, bias in jobs:
        q, s = head_ref.quantize(x)
        ref, tol = head_ref.linear(q, s, w, ws, bias, "none", torch.float32)
        head_ref.assert_close(y, ref, tol, "y")
        r = head_ref.logprobs(z, t, 0)
        head_ref.assert_close(lp, r["logprob"], r["logprob_tol"], "logprob")
        head_ref.assert_close(en, r["entropy"], r["entropy_tol"], "entropy")
        h.ctx.close()


def test_beside_the_data_plane(native):
    """A context that also runs packet batches: the head's calls go in order with them."""
    from flowsentryx_amd import synth
    from oracle import pyoracle
    pyoracle.build()
    p, s = synth.config_params(1, n=1 << 14)
    hdr, ln, ts = pyoracle.synth(p, s, 0, p.n)
    cfg = dict(pps_threshold=50, window_ns=20_000_000, block_ns=50_000_000, max_entries=4096)
    o = pyoracle.Oracle(**cfg)
    want = o.batch(hdr, ln, ts)
    with native.FsxContext(max_batch=p.n, **cfg) as c:
        x = torch.randn(64, 100, generator=gen_of("plane")).cuda()
        q, sc = torch.empty(64, 100, dtype=torch.int8, device="cuda"), torch.empty(64, device="cuda")
        torch.cuda.synchronize()
        c.quantize_rows_device(x.data_ptr(), native.DTYPE_F32, 64, 100, 100, q.data_ptr(), 100, sc.data_ptr())
        got = c.verdict_batch(hdr, ln, ts)
        c.quantize_rows_device(x.data_ptr(), native.DTYPE_F32, 64, 100, 100, q.data_ptr(), 100, sc.data_ptr())
        c.sync()
        assert np.array_equal(got, want)
        wq, ws = head_ref.quantize(x)
        assert torch.equal(q.cpu().long(), wq) and torch.equal(sc.cpu(), ws)
