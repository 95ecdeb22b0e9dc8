"""The 8-bit K/V pool at the ends of its range: rows of zeros, rows near the activations' largest value,
tokens whose size or scale must not reach the queries that do not see them."""

import numpy as np
import pytest

from oracle import kv_fp8 as O
from tests.fp8_pool import DTYPES, Case, check

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _put(c, req, pos, which, x):
    """Stores row x [D] (which: 0 K, 1 V) of every kv head for the request's token at pos."""
    s = int(c.r2t[c.rows[req], pos])
    x = torch.as_tensor(x, dtype=torch.float32).expand(c.hkv, c.d).to(DTYPES[c.dtype]).float()
    codes, scale = O.quantize_rows(x.numpy())
    c.codes[s, :, which] = torch.from_numpy(codes.astype(np.float32)).to(torch.float8_e4m3fn)
    c.scale[s, :, which] = torch.from_numpy(scale)


# name: (hq, hkv, d, prefixes, new tokens); the first takes the split large-tile kernel, the last two the
# few-rows and the CUDA-core kernel
SHAPES = {
    "split": (8, 1, 256, [3000, 0, 1], [70, 1, 200]),
    "d256": (8, 2, 256, [0, 40], [150, 77]),
    "d128": (8, 2, 128, [0, 40], [150, 77]),
    "d64": (8, 2, 64, [0, 40], [150, 77]),
    "gqa6": (24, 4, 128, [10, 0], [70, 96]),
    "few": (8, 2, 128, [0, 40], [5, 9]),
    "simt": (8, 2, 80, [0, 40], [5, 49]),
}


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("name", list(SHAPES))
def test_extend_of_zero_rows(name, dtype):
    """Queries and K rows of zeros: every key has the same weight, the output is the mean of V."""
    hq, hkv, d, pre, ext = SHAPES[name]
    c = Case(41, dtype, hq, hkv, d, pre, ext)
    c.q.zero_()
    for r, n in enumerate(c.seq):
        for j in range(n):
            _put(c, r, j, 0, 0.0)
    check(c.run(), c.reference(), dtype, d, name)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("name", list(SHAPES))
def test_extend_of_a_zero_token_among_others(name, dtype):
    """One token of zeros (q, k and v) at the start of each request, and one in the middle."""
    hq, hkv, d, pre, ext = SHAPES[name]
    c = Case(42, dtype, hq, hkv, d, pre, ext)
    t = 0
    for r, (p, e) in enumerate(zip(pre, ext)):
        for i in (0, e // 2):
            c.q[t + i] = 0
            _put(c, r, p + i, 0, 0.0)
            _put(c, r, p + i, 1, 0.0)
        t += e
    check(c.run(), c.reference(), dtype, d, name)


@pytest.mark.parametrize("name", list(SHAPES))
def test_extend_over_a_pool_of_zero_scales(name):
    """Rows that were never stored (codes and scales 0) have logits of zero and values of zero."""
    hq, hkv, d, pre, ext = SHAPES[name]
    c = Case(43, "bf16", hq, hkv, d, pre, ext)
    c.q[::3] = 0
    c.scale.zero_()
    check(c.run(), c.reference(), "bf16", d, name)
