"""CPU: what the free-size heads refuse (include/fsx_hip.h fsx_quantize_rows_device,
fsx_linear_q8_device, fsx_logprobs_device), their workspace sizes, and the 64-bit references'
own known answers. A refused call touches nothing but the context's message, so a zeroed block
of memory stands in for a context here."""
import ctypes as C
import random
import errno
import math

import numpy as np
import pytest
import torch

import head_ref

P = 1 << 20   # an aligned address that a refused call never reads


@pytest.fixture(scope="module")
def fake(native):
    block = C.create_string_buffer(1 << 22)
    return native.load_library(), C.addressof(block), block


def refused(fake, rc, word):
    lib, ctx, _ = fake
    assert rc == -errno.EINVAL
    assert word in lib.fsx_last_error(ctx).decode()


def quant(fake, **over):
    a = dict(x=P, dtype=0, rows=4, cols=32, ldx=32, q=P, ldq=32, scale=P)
    a.update(over)
    lib, ctx, _ = fake
    return lib.fsx_quantize_rows_device(ctx, a["x"], a["dtype"], a["rows"], a["cols"], a["ldx"], a["q"], a["ldq"],
                                        a["scale"])


@pytest.mark.parametrize("over,word", [
    (dict(dtype=3), "type"), (dict(dtype=-1), "type"), (dict(dtype=9), "type"), (dict(cols=0), "elements"),
    (dict(cols=1 << 31, ldx=1 << 31), "elements"), (dict(ldx=31), "apart"), (dict(ldq=31), "apart"),
    (dict(x=None), "null"), (dict(q=None), "null"), (dict(scale=None), "null"), (dict(x=P + 2), "misaligned"),
    (dict(scale=P + 1), "misaligned"), (dict(rows=1 << 41), "range"), (dict(ldx=1 << 58), "range"),
    (dict(dtype=2, x=P + 1), "misaligned")])
def test_quantize_refusals(fake, over, word):
    refused(fake, quant(fake, **over), word)


def lin(fake, native, work=0, work_bytes=0, **over):
    a = dict(w=P, ws=P, bias=None, k=32, n=16, ldw=32, act=0, reserved=0, x=P, xt=3, ldx=32, xs=P, rows=4, y=P,
             yt=0, ldy=16)
    a.update(over)
    layer = native.q8_linear(a["w"], a["ws"], a["bias"], a["k"], a["n"], a["ldw"], a["act"])
    layer.reserved = a["reserved"]
    lib, ctx, _ = fake
    return lib.fsx_linear_q8_device(ctx, C.byref(layer), a["x"], a["xt"], a["ldx"], a["xs"], a["rows"], a["y"],
                                    a["yt"], a["ldy"], work, work_bytes)


@pytest.mark.parametrize("over,word", [
    (dict(k=0), "features"), (dict(k=131072, ldw=131072, ldx=131072), "features"),
    (dict(n=1 << 31, ldy=1 << 31), "features"), (dict(act=3), "activation"), (dict(act=-1), "activation"),
    (dict(reserved=1), "activation"), (dict(xt=4), "type"), (dict(yt=3), "type"), (dict(yt=-1), "type"),
    (dict(ldx=31), "apart"), (dict(ldw=31), "apart"), (dict(ldy=15), "apart"), (dict(w=None), "null"),
    (dict(ws=None), "null"), (dict(x=None), "null"), (dict(xs=None), "null"), (dict(y=None), "null"),
    (dict(bias=P + 2), "misaligned"), (dict(y=P + 2), "misaligned"), (dict(yt=1, y=P + 1), "misaligned"),
    (dict(xt=0), "x scales given"), (dict(xt=2, xs=None, rows=200, n=500, ldy=500, k=500, ldx=500, ldw=500), "workspace"), (dict(rows=1 << 41), "range")])
def test_linear_refusals(fake, native, over, word):
    refused(fake, lin(fake, native, **over), word)


def test_linear_workspace(fake, native):
    layer = native.q8_linear(P, P, None, 100, 160)
    need = native.linear_q8_work(layer, native.DTYPE_F32, 1000)
    assert need >= 1000 * 104
    over = dict(xt=0, xs=None, rows=1000, k=100, n=160, ldy=160, ldw=100, ldx=100)
    refused(fake, lin(fake, native, P, need - 1, **over), "workspace")
    refused(fake, lin(fake, native, P + 8, need, **over), "workspace")
    refused(fake, lin(fake, native, None, need, **over), "workspace")
    for bad in (dict(in_features=0), dict(in_features=131072), dict(out_features=0), dict(out_features=1 << 31)):
        other = native.q8_linear(P, P, None, bad.get("in_features", 100), bad.get("out_features", 16))
        assert native.linear_q8_work(other, native.DTYPE_F32, 8) == 0
    assert native.linear_q8_work(layer, native.DTYPE_F32, 0) == 0
    assert native.linear_q8_work(layer, 7, 8) == 0
    assert native.load_library().fsx_linear_q8_work(None, 0, 8) == 0


def test_linear_workspace_before_the_weights(fake, native):
    """A program may ask before its weights are there: then the size covers any place of theirs."""
    for rows, k, n, ld in ((5000, 512, 5000, 512), (5000, 500, 5000, 500), (100, 4096, 64, 4096), (2, 9, 5, 9)):
        sizes = [native.linear_q8_work(native.q8_linear(w, P, None, k, n, ld), native.DTYPE_I8, rows) for w in (P, P + 1, None)]
        assert sizes[2] == max(sizes), (rows, k, n, ld)


def test_linear_takes_the_workspace_it_asks_for(fake, native):
    """Whatever the sizes and places, a workspace of the size asked for is enough for the call (which
    fails later here, without a GPU)."""
    if torch.cuda.device_count():
        pytest.skip("with a GPU the accepted calls would run, on addresses that are none")
    rng = random.Random(5)
    lib, ctx, _ = fake
    size = lambda top: int(round(2 ** rng.uniform(0, top)))
    cases = [(4000, 2000, 320, 3, 0, 1, 0)]
    for _ in range(4000):
        cases.append((size(20), min(131071, size(17)), size(16), rng.choice((0, 2, 3, 3)), rng.choice((0, 0, 1, 8)),
                      rng.choice((0, 0, 1, 8)), rng.choice((0, 0, 4))))
    for rows, k, n, xt, xpad, wpad, at in cases:
        ldx, ldw = k + -k % 16 + xpad, k + -k % 16 + wpad
        layer = native.q8_linear(P + at, P, None, k, n, ldw)
        need = native.linear_q8_work(layer, xt, rows)
        lin(fake, native, P, need, w=P + at, k=k, n=n, ldw=ldw, xt=xt, ldx=ldx, xs=P if xt == 3 else None, rows=rows,
            x=P + at, ldy=n)
        assert b"workspace" not in lib.fsx_last_error(ctx), (rows, k, n, xt, ldx, ldw, at, lib.fsx_last_error(ctx))


def test_linear_workspace_of_refused_layers(fake, native):
    """No size for a layer that the call refuses, whatever is wrong with it."""
    over = dict(k=1000, n=500, ldw=1000, ldx=1000, ldy=500, xt=0, xs=None, rows=100)
    assert native.linear_q8_work(native.q8_linear(P, P, None, 1000, 500), native.DTYPE_F32, 100) > 0
    for bad in (dict(act=3), dict(act=-1), dict(reserved=1), dict(ldw=999), dict(ldw=1 << 52)):
        a = {**over, **bad}
        layer = native.q8_linear(P, P, None, a["k"], a["n"], a["ldw"], a.get("act", 0))
        layer.reserved = a.get("reserved", 0)
        assert native.linear_q8_work(layer, native.DTYPE_F32, 100) == 0, bad
        assert lin(fake, native, P, 1 << 40, **a) == -errno.EINVAL, bad


@pytest.mark.parametrize("rows", [(1 << 36) - 16, 1 << 36, (1 << 36) + 16, 1 << 37, (1 << 40) - 16, 1 << 40])
def test_linear_workspace_of_many_rows(fake, native, rows):
    """Row counts whose blocks pass 32 bits: the size is worked out, and a product over so many
    rows is cut into no parts (codes need nothing, floats their codes and scales)."""
    layer = native.q8_linear(P, P, None, 16384, 16)
    assert native.linear_q8_work(layer, native.DTYPE_I8, rows) == 0
    assert native.linear_q8_work(layer, native.DTYPE_F32, rows) == rows * (16384 + 4)


def logp(fake, work=0, work_bytes=0, **over):
    a = dict(x=P, dtype=0, rows=4, classes=50, ld=50, target=P, logprob=P, entropy=P, top=3, ids=P, lps=P)
    a.update(over)
    lib, ctx, _ = fake
    return lib.fsx_logprobs_device(ctx, a["x"], a["dtype"], a["rows"], a["classes"], a["ld"], a["target"],
                                   a["logprob"], a["entropy"], a["top"], a["ids"], a["lps"], work, work_bytes)


@pytest.mark.parametrize("over,word", [
    (dict(dtype=3), "type"), (dict(classes=0), "classes"), (dict(classes=1 << 31, ld=1 << 31), "classes"),
    (dict(top=65), "top_k"), (dict(ld=49), "apart"), (dict(x=None), "null"), (dict(x=P + 1), "misaligned"),
    (dict(target=None), "together"), (dict(logprob=None), "together"), (dict(ids=None), "null"),
    (dict(lps=None), "null"), (dict(top=0), "without top_k"), (dict(entropy=P + 1), "misaligned"),
    (dict(target=P + 2), "misaligned"), (dict(rows=1 << 41), "range")])
def test_logprobs_refusals(fake, over, word):
    refused(fake, logp(fake, **over), word)


def test_parts_are_few(fake, native):
    """A call in parts has another launch that joins them, a block for a row and a thread for four
    channels: rows and products that are cut are small enough for one."""
    for classes in (8193, 70001, 131072, (1 << 31) - 1):
        for rows in list(range(1, 1100)) + [1 << 16, 1 << 36, 1 << 40]:
            assert (native.logprobs_work(rows, classes, 5) > 0) == (rows <= 170), (rows, classes)
    rng = random.Random(6)
    for _ in range(20000):
        rows, k, n = (int(2 ** rng.uniform(0, top)) for top in (41, 17, 31))
        layer = native.q8_linear(P, P, None, min(k, 131071), n, min(k, 131071) + 15 & ~15)
        copies = rows * int(layer.ld_weight) if rows * k * n >= 2.5e9 and n >= 384 else 0
        sums = native.linear_q8_work(layer, native.DTYPE_I8, min(rows, 1 << 40)) - copies
        assert sums <= 64 * 4 * (1 << 20) + 16, (rows, k, n)   # (parts, bytes, results)


def test_nothing_to_do_is_no_error(fake, native):
    assert quant(fake, rows=0) == 0
    assert lin(fake, native, rows=0) == 0
    assert lin(fake, native, n=0) == 0
    assert logp(fake, rows=0) == 0
    assert native.logprobs_work(0, 100, 3) == 0
    assert native.logprobs_work(8, 0, 3) == 0
    assert native.logprobs_work(8, 100, 65) == 0


def test_null_context(native):
    lib = native.load_library()
    layer = native.q8_linear(P, P, None, 32, 16)
    assert lib.fsx_quantize_rows_device(None, P, 0, 4, 32, 32, P, 32, P) == -errno.EINVAL
    assert lib.fsx_linear_q8_device(None, C.byref(layer), P, 3, 32, P, 4, P, 0, 16, None, 0) == -errno.EINVAL
    assert lib.fsx_linear_q8_device(C.addressof(C.create_string_buffer(1 << 22)), None, P, 3, 32, P, 4, P, 0, 16,
                                    None, 0) == -errno.EINVAL
    assert lib.fsx_logprobs_device(None, P, 0, 4, 50, 50, P, P, P, 3, P, P, None, 0) == -errno.EINVAL


def test_layer_struct_layout(native):
    assert C.sizeof(native.FsxQ8Linear) == 3 * 8 + 3 * 8 + 4 + 4


# ---- the references' own known answers

def test_reference_quantize():
    x = torch.tensor([[127.0, -0.5, 0.5, 1.5, -2.5, 0.0], [0.0] * 6, [1.0, float("nan"), 2, 3, 4, 5],
                      [float("inf"), 1, 2, 3, 4, 5]])
    q, s = head_ref.quantize(x)
    assert q.tolist() == [[127, 0, 0, 2, -2, 0], [0] * 6, [0] * 6, [0] * 6]
    assert s[0] == 1.0 and s[1] == 2.0 ** -126 and s[2:].isnan().all()


def test_reference_logprobs():
    x = torch.tensor([[0.0, 0.0, -math.inf, 0.0], [-math.inf] * 4, [1.0, math.nan, 0.0, 0.0], [0.0, math.inf, 0, 0]])
    r = head_ref.logprobs(x, torch.tensor([3, 0, 0, -1]), 5)
    assert r["top_id"].tolist() == [[0, 1, 3, -1, -1], [-1] * 5, [-1] * 5, [-1] * 5]
    assert abs(r["logprob"][0] + math.log(3)) < 1e-12 and r["logprob"][1] == -math.inf
    assert math.isnan(r["logprob"][2]) and r["logprob"][3] == 0.0
    assert abs(r["entropy"][0] - math.log(3)) < 1e-12 and r["entropy"][1] == 0.0
    assert np.isnan(r["entropy"][2:]).all()


def test_reference_linear():
    y, tol = head_ref.linear(torch.tensor([[1, -2]]), torch.tensor([0.5]), torch.tensor([[3, 4], [1, 1]]),
                             torch.tensor([2.0, 1.0]), torch.tensor([1.0, 0.0]), "relu", torch.float32)
    assert y.tolist() == [[0.0, 0.0]] and (tol > 0).all()
    y, _ = head_ref.linear(torch.tensor([[1, -2]]), torch.tensor([0.5]), torch.tensor([[3, 4]]), torch.tensor([2.0]),
                           None, "none", torch.float32)
    assert y.tolist() == [[-5.0]]
