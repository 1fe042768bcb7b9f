"""The free-size heads in 64 bits on the CPU (row quantiser, int8 layer, log probabilities),
and how far the 32-bit kernels may be from them, counted in roundings: u = 2^-24 is half a
step of a 32-bit number relative to it."""
import numpy as np
import torch

U = 2.0 ** -24
MIN_SCALE = np.float32(2.0 ** -126)
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


def quantize(x: torch.Tensor):
    """(codes int64, scales float32) of rows of floats. A 64-bit quotient decides halves as the
    exact one does: x / s of 24-bit numbers is a half exactly or at least 2^-33 away from it."""
    v = x.detach().cpu().to(torch.float64).numpy()
    amax = np.abs(v).max(axis=1)
    ok = np.isfinite(amax)
    scale = np.maximum(np.where(ok, amax, 0).astype(np.float32) / np.float32(127), MIN_SCALE)
    codes = np.rint(np.where(ok[:, None], v, 0) / scale.astype(np.float64)[:, None])
    scale = np.where(ok, scale, np.float32(np.nan)).astype(np.float32)
    return torch.from_numpy(codes.astype(np.int64)), torch.from_numpy(scale)


def linear(codes, x_scale, weight, weight_scale, bias, act, dtype):
    """(y, tolerance) in 64 bits. |sum| * scales is three roundings of 32 bits away from the
    kernel's (the sum to a float, two products), the bias' addition one more; a second-order
    term is covered by counting 4 and 2. sigmoid' = y (1 - y), its exp is within 2 u, then an
    addition and a quotient. Last the rounding to the output's type."""
    acc = codes.to(torch.float64) @ weight.cpu().to(torch.float64).T
    prod = acc * x_scale.cpu().double()[:, None] * weight_scale.cpu().double()
    y = prod + (bias.cpu().double() if bias is not None else 0.0)
    tol = 4 * U * prod.abs() + 2 * U * y.abs()
    if act == "relu":
        y = torch.where(y < 0, torch.zeros_like(y), y)
    elif act == "sigmoid":
        y = torch.sigmoid(y)
        tol = y * (1 - y) * (tol + 2 * U) * 1.01 + 4 * U * y
    # half a step above the type's largest value and beyond, a rounded result is infinite
    top = torch.finfo(dtype).max * (1 + HALF_STEP[dtype] / (2 - 2 * HALF_STEP[dtype]))
    assert not ((y.abs() - top).abs() <= 2 * tol).any(), "inputs that leave open whether a result overflows"
    y = torch.where(y.abs() >= top, torch.copysign(torch.full_like(y, float("inf")), y), y)
    tol = torch.where(y.isinf(), torch.zeros_like(tol), tol)
    return y, tol * 1.01 + HALF_STEP[dtype] * 1.01 * torch.where(y.isinf(), torch.zeros_like(y), y).abs() + TINY[dtype]


def logprobs(x: torch.Tensor, target, top: int):
    """dict of the answers in 64 bits and their tolerances ("..._tol").

    z = x - m is one rounding off, e^z as 2^(z log2 e) |z| 3 u (the product, the constant, z) and
    2 u of its own; S and T are sums of `n` parts (a thread's logits one after another, then
    joined), and each rise of the maximum (at most one for every piece of 8 logits) multiplies by
    another such e^d: d e^-d < 1/2 of what the sum holds then, so it counts 4 u."""
    v = x.detach().cpu().double().numpy()
    rows, classes = v.shape
    n = 5 * (classes // 256) // 4 + 48
    bad = np.isnan(v).any(axis=1) | np.isposinf(v).any(axis=1)
    w = np.where(bad[:, None], 0.0, v)
    m = w.max(axis=1)
    empty = np.isneginf(m)
    m = np.where(empty, 0.0, m)
    z = w - m[:, None]
    e = np.exp(z)
    zf = np.where(np.isneginf(z), 0.0, z)
    s = e.sum(axis=1)
    s1 = np.where(empty, 1.0, s)
    ls = np.log(s1)
    a1 = (np.abs(zf) * e).sum(axis=1) / s1
    a2 = (zf * zf * e).sum(axis=1) / s1
    tol_s = (n + 3 * a1 + 2) * U
    tol_t = ((n + 3) * a1 + 3 * a2) * U
    tol_ls = tol_s + 2 * U * ls
    out = {}
    entropy = np.where(bad, np.nan, np.where(empty, 0.0, ls + a1))
    out["entropy"], out["entropy_tol"] = entropy, tol_ls + tol_t + a1 * tol_s + 2 * U * (ls + a1) + U
    lp = np.where(np.isneginf(w), -np.inf, zf - ls[:, None])
    lp_tol = np.abs(zf) * U + tol_ls[:, None] + U * np.abs(np.where(np.isneginf(lp), 0, lp)) + U
    if target is not None:
        t = target.cpu().numpy().astype(np.int64)
        inside = (t >= 0) & (t < classes)
        at = np.where(inside, t, 0)
        got = lp[np.arange(rows), at]
        out["logprob"] = np.where(t == -1, 0.0, np.where(inside & ~bad, got, np.nan))
        out["logprob_tol"] = lp_tol[np.arange(rows), at]
    ids = np.full((rows, top), -1, dtype=np.int64)
    tlp = np.full((rows, top), -np.inf)
    ttol = np.zeros((rows, top))
    k = min(top, classes)
    if k:
        order = np.argsort(-w, axis=1, kind="stable")[:, :k]
        r = np.arange(rows)[:, None]
        val = lp[r, order]
        none = np.isneginf(val)
        ids[:, :k] = np.where(none, -1, order)
        tlp[:, :k] = val
        ttol[:, :k] = lp_tol[r, order]
    ids[bad] = -1
    tlp[bad] = np.nan
    out.update(top_id=ids, top_logprob=tlp, top_logprob_tol=ttol)
    return out


def assert_close(got, want, tol, what=""):
    got = np.asarray(got.detach().cpu().double() if isinstance(got, torch.Tensor) else got, dtype=np.float64)
    want, tol = np.asarray(want, dtype=np.float64), np.asarray(tol, dtype=np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN elsewhere"
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf]) and not np.isinf(got[~inf]).any(), f"{what}: infinities differ"
    fine = np.isfinite(want)
    over = np.abs(got[fine] - want[fine]) - np.broadcast_to(tol, want.shape)[fine]
    if over.size:
        i = int(over.argmax())
        assert over[i] <= 0, f"{what}: {got[fine][i]!r} for {want[fine][i]!r}, {over[i]:.3g} over its tolerance"
