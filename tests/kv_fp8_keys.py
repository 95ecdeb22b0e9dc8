"""Cases in which every key counts: a result that lacks any block of 32 keys, or any key at the end of one,
is outside the bound of kv_fp8_bounds.py.  Lengths end at, before and behind the kernels' tiles (32 and 128
keys), the shares of their CTAs and their splits."""

import numpy as np
import torch

from tests import kv_fp8_bounds as B
from tests.fp8_pool import Case

# name: (dtype, hq, hkv, d, prefixes, new tokens)
DECODE = {
    "one_long": ("bf16", 8, 1, 256, [9000], [1]),
    "one_long_f16": ("f16", 8, 2, 128, [7000], [1]),
    "ragged": ("bf16", 16, 2, 128, [0, 31, 32, 95, 1000, 2047, 1663, 300, 14, 63, 2500, 640, 127], [1] * 13),
    "ragged_f16": ("f16", 16, 2, 64, [0, 31, 32, 95, 1000, 2047, 1663, 300, 14, 63, 2500, 640, 127], [1] * 13),
    "batch": ("bf16", 8, 4, 64, [(97 * i) % 701 for i in range(60)], [1] * 60),
    "wide_batch": ("bf16", 32, 4, 256, [(389 * i) % 1601 for i in range(24)], [1] * 24),
    "gqa24": ("bf16", 48, 2, 128, [700, 31, 1500], [1, 1, 1]),
    "cuda_cores": ("bf16", 4, 2, 80, [31, 32, 700], [1, 1, 1]),
    "cuda_cores_f32": ("f32", 8, 2, 64, [31, 32, 900], [1, 1, 1]),
}
EXTEND = {
    "drafts": ("bf16", 32, 4, 256, [900, 30, 513, 3000], [4, 1, 3, 2]),
    "drafts_f16": ("f16", 8, 2, 128, [1900, 0, 62], [2, 5, 2]),
    "two_passes": ("bf16", 32, 4, 128, [900, 30, 513, 2000], [6, 1, 3, 5]),
    "edges": ("bf16", 8, 2, 128, [127, 128, 129, 0, 63], [13, 1, 128, 127, 65]),
    "edges_f16": ("f16", 8, 2, 256, [127, 128, 129, 0, 63], [13, 1, 30, 127, 65]),
    "edges_d64": ("bf16", 16, 2, 64, [127, 128, 129, 0, 63], [13, 1, 30, 127, 65]),
    "split": ("bf16", 8, 1, 256, [5000, 0, 1], [40, 1, 90]),
    "split_f16": ("f16", 8, 1, 128, [4100, 0], [70, 1]),
    "cuda_cores": ("bf16", 4, 2, 80, [20, 64], [33, 1]),
    "cuda_cores_f32": ("f32", 8, 2, 64, [20, 96], [10, 33]),
}


def case(name, extend, alike):
    """alike: all K rows of a head are the same, so that every key has the same weight; the V rows at the
    ends of every 32 keys are 16 times larger."""
    dtype, hq, hkv, d, pre, ext = (EXTEND if extend else DECODE)[name]
    c = Case(60, dtype, hq, hkv, d, pre, ext, scale_spread=0.0 if alike else 0.3)
    c.alike = alike
    if alike:
        c.codes.view(torch.uint8)[:, :, 0] = c.codes.view(torch.uint8)[:1, :, 0].clone()
        c.scale[..., 0] = c.scale[:1, :, 0].clone()
        for r, n in enumerate(c.seq):
            s = c.r2t[c.rows[r], :n]
            c.scale[s[0::32], :, 1] *= 16
            c.scale[s[31::32], :, 1] *= 16
    return c, B.kernel_of(c, extend)


def parts(c, r, alike):
    """What a result of request r must not lack: every block of 32 keys, and (alike) every key at the end of
    one."""
    n = c.seq[r]
    out = [np.arange(j, min(j + 32, n)) for j in range(0, n, 32)]
    if alike:
        out += [np.array([j]) for j in range(n) if j % 32 in (0, 31)]
    return out
