"""Inputs and tolerances shared by the tests of the 8-bit K/V pool."""

import numpy as np
import torch

from oracle import kv_fp8 as O

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# relative error of an attention weight before the fp32 sums: the tensor-core kernels hold weights
# in f16 (11 bits; half a step is 2^-12 of the value), with bfloat16 activations the large-tile kernel
# also rounds scaled codes to f16; 2^-8 and 2^-11 also admit weights in sums of e4m3 terms; the
# fp32 path's exponentials are good to a few units of 2^-24
WEIGHT_ERR = {"f32": 2.0 ** -20, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


class Case:
    """A random pool, table and batch on the host (numpy, from torch tensors of the dtype)."""

    def __init__(self, seed, dtype, hq, hkv, d, pre, ext, spare=7, gate="none", layout="adjacent",
                 device="cuda", scale_spread=0.5):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.hq, self.hkv, self.d, self.gate_mode = dtype, hq, hkv, d, gate
        self.pre, self.ext = list(pre), list(ext)
        self.seq = [p + e for p, e in zip(pre, ext)]
        n, total, t = len(self.seq), sum(self.seq), sum(self.ext)
        slots = total + spare
        dt = DTYPES[dtype]
        x = torch.randn((slots, hkv, 2, d), generator=g)
        codes, sc = O.quantize_rows(x.numpy())
        self.codes = torch.from_numpy(codes.astype(np.float32)).to(torch.float8_e4m3fn)
        self.scale = torch.from_numpy(sc) * torch.exp(
            scale_spread * torch.randn(sc.shape, generator=g))
        perm = torch.randperm(slots, generator=g)[:total]
        self.rows = torch.randperm(n + 2, generator=g)[:n]
        self.r2t = torch.full((n + 2, max(self.seq + [1]) + 3), -1, dtype=torch.int64)
        at = 0
        for r, s in zip(self.rows.tolist(), self.seq):
            self.r2t[r, :s] = perm[at:at + s]
            at += s
        self.q = torch.randn((t, hq, d), generator=g).to(dt)
        self.gate = torch.randn((t, hq, 2 * d), generator=g).to(dt)[..., d:]
        self.layout, self.device = layout, device

    def pool(self):
        """(k_buffer, v_buffer, kv_scale) on the device in the case's layout."""
        dev = self.device
        if self.layout == "adjacent":  # K and V rows of a head next to each other
            c = self.codes.to(dev)
            return c[:, :, 0], c[:, :, 1], self.scale.to(dev)
        if self.layout == "separate":  # two tensors
            c = self.codes.view(torch.uint8)
            k, v = (c[:, :, j].contiguous().view(torch.float8_e4m3fn).to(dev) for j in (0, 1))
            return k, v, self.scale.to(dev)
        # "odd": rows at odd byte offsets, scales with gaps
        s, h, _, d = self.codes.shape
        raw = torch.zeros((s, h, 2, d + 3), dtype=torch.uint8)
        raw[..., 1:d + 1] = self.codes.view(torch.uint8)
        c = raw.to(dev)[..., 1:d + 1].view(torch.float8_e4m3fn)
        sc = torch.zeros((s, h + 1, 4))
        sc[:, :h, :2] = self.scale
        return c[:, :, 0], c[:, :, 1], sc.to(dev)[:, :h, :2]

    def args(self):
        dev = self.device
        return (self.r2t.to(dev), self.rows.to(dev), torch.tensor(self.seq, device=dev))

    def run(self, force_extend=False, slot_mode="clamp", out=None, err=None):
        from tokenfactory_b200 import ops
        kw = dict(gate=None if self.gate_mode == "none" else self.gate.to(self.device),
                  gate_mode=self.gate_mode, slot_mode=slot_mode, out=out, err=err)
        q, pool, args = self.q.to(self.device), self.pool(), self.args()
        sm = self.d ** -0.5
        if all(e == 1 for e in self.ext) and not force_extend:
            return ops.paged_decode_fp8(q, *pool, *args, sm, max(self.seq), **kw)
        return ops.paged_extend_fp8(q, *pool, *args, torch.tensor(self.ext, device=self.device), sm,
                                    max(self.seq), max(self.ext), **kw)

    def reference(self, slot_mode="clamp"):
        rows = self.codes.float().double().numpy() * self.scale.double().numpy()[..., None]
        return O.attention(self.q.double().numpy(), rows[:, :, 0], rows[:, :, 1], self.r2t.numpy(),
                           self.rows.tolist(), self.seq, self.ext, self.d ** -0.5,
                           self.gate.double().numpy(), self.gate_mode, slot_mode,
                           self.scale[..., 1].double().numpy())


def check(got, ref, dtype, d, what=""):
    """got against (out, magnitude, score magnitude, step magnitude): one rounding of the output, the
    weights' error, and the fp32 sums (d products a score and as many weighted rows: each addition
    is off by at most 2^-24 of the running magnitude; the activation's exponential by 2^-20).

    The step: a sum of e4m3 terms has an absolute error too, half the subnormal step, 2^-10.  The
    weights w_j = 2^7 p_j vs_j / P are scaled by P = max_j p_j 2^ev_j <= max_j p_j max_j vs_j (2^ev_j the
    power of two below the largest vs of token j's tile), so p_j vs_j is off by at most
    2^-17 max p max vs, and a sum over the V codes by that times sum_j |code_j|."""
    out, mag, smag, step = ref
    got = got.detach().double().cpu().numpy()
    assert got.shape == out.shape, (got.shape, out.shape)
    assert np.array_equal(np.isnan(got), np.isnan(out)), f"{what}: NaNs in other places"
    tol = (torch.finfo(DTYPES[dtype]).eps / 2 * np.abs(out)
           + mag * (WEIGHT_ERR[dtype] + 2 * d * 2.0 ** -24 * (1 + smag) + 2.0 ** -20) + 1e-30)
    if dtype != "f32":
        tol = tol + 2.0 ** -17 * step
    if dtype == "f16":
        tol = tol + 2.0 ** -25  # half a step of a subnormal output
    bad = np.abs(got - out) > tol
    assert not bad.any(), (f"{what}: {bad.sum()} of {bad.size} off, worst "
                           f"{np.nanmax(np.abs(got - out) / tol):.3g} of its tolerance")
