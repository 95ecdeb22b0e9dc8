"""Attention over the 8-bit K/V pool in float64 with a bound, element by element, of what the kernels'
roundings may add up to.  u = 2^-24 is half a step of fp32, relative to the value.

* logits: d products summed in fp32 (each addition off by at most 2 u of the sum of magnitudes, tensor
  cores truncate); one scaling and the subtraction of the maximum, off by 4 u of the numbers involved; in
  the large-tile kernel with bfloat16 activations also the K codes times their scale, rounded to f16
  (2^-11 of each product).  An error of e in a logit is one of e relative to the weight, and reaches the
  output through the key itself and through the sum of weights.
* weights: rounded to f16 by the tensor-core kernels, 2^-11; with bfloat16 activations the large-tile
  kernel rounds the V codes times their scale to f16 too, 2^-11 again; 2^-19 for the exponential and the
  handful of fp32 operations beside it.
* weights below f16's normal range are off by up to 2^-25 of a unit.  The few-rows kernel scales the
  largest weight times V scale of a row to [2^7, 2^8); the large-tile kernel scales by the largest of a
  group of 32 keys, within 2^7 of it, and its V codes carry a factor below 2.
* fp32 sums over n keys: the tensor-core kernels add at most n / 8 + 64 terms one after another, the
  CUDA-core kernel n.
* the output: half a step of its type.
"""

import numpy as np
import torch

from tests.fp8_pool import DTYPES

U = 2.0 ** -24
ROWS, TILE, SIMT = "few rows", "large tile", "CUDA cores"


def kernel_of(c, extend):
    """The kernel that the call of a Case takes (extend: through the extend entry point)."""
    g = c.hq // c.hkv
    fast = c.dtype != "f32" and c.d in (64, 128, 256) and c.layout != "odd"
    rows = g * (max(c.ext) if extend else 1)
    if fast and (not extend or rows <= 48) and len(c.seq) * -(-rows // 32) <= 32768:
        return ROWS
    return TILE if fast and extend and g <= 16 else SIMT


def _exponent(s):
    """floor(log2 |s|), 0 for scales that are zero"""
    s = np.abs(s)
    return np.floor(np.log2(np.where(s > 0, s, 1)))


def row_terms(c, kernel, q, k, v, ks, vs, scale):
    """(out, tolerance without the output's rounding) of query rows q [M, D] over keys k, v [n, D] with
    scales ks, vs [n]: everything float64; visible keys only."""
    n, d = k.shape
    x = q @ k.T * scale
    mag_x = np.abs(q) @ np.abs(k).T * scale
    m = x.max(-1, keepdims=True)
    p = np.exp(x - m)
    p /= p.sum(-1, keepdims=True)
    out, mag = p @ v, p @ np.abs(v)
    fold = kernel == TILE and c.dtype == "bf16"
    k_err = 2 * d * U + (2.0 ** -11 * (1 + 2.0 ** -9) if fold else 0)
    if getattr(c, "alike", False):  # the same K row everywhere: the same product, whatever its error
        k_err = 0.0
    e = _exponent(vs)
    lam = mag_x * k_err + 4 * U * (np.abs(x) + np.abs(m) + np.abs(e) + np.abs(e).max(initial=0))
    w = 2.0 ** -19
    if kernel != SIMT:
        w += 2.0 ** -11 * (2 if fold else 1)
    sums = 2 * U * (n if kernel == SIMT else n / 8 + 64)
    tol = (p * lam) @ np.abs(v) + (p * lam).sum(-1, keepdims=True) * np.abs(out)
    tol = tol + mag * (w + sums) + np.abs(out) * (sums + w)
    if kernel != SIMT:
        code = np.abs(np.divide(v, vs[:, None], out=np.zeros_like(v), where=vs[:, None] != 0))
        unit = (p * np.abs(vs)).max(-1, keepdims=True)
        tol = tol + unit * code.sum(0) * (2.0 ** -32 if kernel == ROWS else 2.0 ** -17)
    return out, tol


def _act(c, t, h):
    x = c.gate[t, h].double().numpy()
    return 1 / (1 + np.exp(-x)) * (x if c.gate_mode == "silu" else 1)


def _request(c, r, slot_mode):
    s = c.r2t[c.rows[r], :c.seq[r]].numpy()
    return np.where(s < 0, s + len(c.codes) if slot_mode == "wrap" else 0, s)


def _group(c, s, h):
    """(K, V, K scale, V scale) of the slots for one kv head, float64"""
    codes = c.codes[s, h].float().double().numpy()
    sc = c.scale[s, h].double().numpy()
    return codes[:, 0] * sc[:, :1], codes[:, 1] * sc[:, 1:], sc[:, 0], sc[:, 1]


def reference(c, kernel, slot_mode="clamp"):
    """(out, tolerance) [T, Hq, D] of a Case whose scales are finite."""
    q = c.q.double().numpy()
    out, tol = np.full(q.shape, np.nan), np.full(q.shape, np.nan)
    g, t = c.hq // c.hkv, 0
    for r, (n, e) in enumerate(zip(c.seq, c.ext)):
        s = _request(c, r, slot_mode)
        for h in range(c.hkv):
            hs = slice(h * g, (h + 1) * g)
            k, v, ks, vs = _group(c, s, h)
            for i in range(e):
                m = n - e + i + 1
                if m > 0:
                    out[t + i, hs], tol[t + i, hs] = row_terms(
                        c, kernel, q[t + i, hs], k[:m], v[:m], ks[:m], vs[:m], c.d ** -0.5)
        t += e
    if c.gate_mode != "none":
        a = _act(c, slice(None), slice(None))
        out, tol = out * a, np.abs(a) * tol + 2.0 ** -19 * np.abs(out * a)
    return out, rounded(c.dtype, out, tol)


def rounded(dtype, out, tol):
    f = torch.finfo(DTYPES[dtype])
    return tol * (1 + f.eps) + f.eps / 2 * np.abs(out) + f.smallest_normal * f.eps / 2


def check(got, ref, what=""):
    out, tol = ref
    got = got.detach().double().cpu().numpy()
    assert got.shape == out.shape, (got.shape, out.shape)
    assert np.array_equal(np.isnan(got), np.isnan(out)), f"{what}: NaNs in other places"
    bad = np.abs(got - out) > tol
    assert not bad.any(), (f"{what}: {bad.sum()} of {bad.size} off, worst "
                           f"{np.nanmax(np.abs(got - out) / tol):.3g} of its tolerance")


def unseen(c, kernel, r, parts):
    """Those of the given sets of keys without which the result of request r's last query token would pass
    check in every element."""
    s = _request(c, r, "clamp")
    t = sum(c.ext[:r + 1]) - 1
    g = c.hq // c.hkv
    seen = np.zeros(len(parts), bool)
    for h in range(c.hkv):
        q = c.q[t, h * g:(h + 1) * g].double().numpy()
        k, v, ks, vs = _group(c, s, h)
        out, tol = row_terms(c, kernel, q, k, v, ks, vs, c.d ** -0.5)
        tol = rounded(c.dtype, out, tol)
        x = q @ k.T * c.d ** -0.5
        p = np.exp(x - x.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        for i, keys in enumerate(parts):
            if seen[i]:
                continue
            left = 1 - p[:, keys].sum(-1, keepdims=True)
            if len(keys) == c.seq[r] or (left < 1e-9).any():
                seen[i] = True  # nothing is left: NaN
            else:
                seen[i] = (np.abs((out - p[:, keys] @ v[keys]) / left - out) > tol).any()
    return [keys.tolist() for keys, ok in zip(parts, seen) if not ok]
