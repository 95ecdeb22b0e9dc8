"""The 8-bit K/V pool at the ends of its range: rows of zeros, rows near the activations' largest value,
tokens whose size or scale must not reach the queries that do not see them."""

import numpy as np
import pytest

from oracle import kv_fp8 as O
from tests import kv_fp8_bounds as B
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


# rows of very different size beside each other: what is hidden from a query, or seen with next to no
# weight, must not cost the others their bits.  dtype, (hq, hkv, d, prefixes, new tokens), and whether
# single tokens go through decode
MIXED = {
    "decode": ("bf16", 8, 2, 128, [399, 0, 70], [1, 1, 1]),
    "decode_f16": ("f16", 8, 1, 256, [399, 0, 70], [1, 1, 1]),
    "drafts": ("bf16", 8, 2, 256, [300, 0, 61], [5, 1, 8]),
    "drafts_f16": ("f16", 8, 2, 64, [300, 0, 61], [5, 1, 8]),
    "tile": ("bf16", 8, 2, 256, [0, 40], [150, 77]),
    "tile_f16": ("f16", 8, 2, 128, [0, 40], [150, 77]),
    "tile_d64": ("bf16", 8, 2, 64, [0, 40], [150, 77]),
    "tile_split": ("bf16", 8, 1, 256, [3000, 0, 1], [70, 1, 200]),
    "tile_split_f16": ("f16", 8, 1, 256, [3000, 0, 1], [70, 1, 200]),
    "simt": ("bf16", 8, 2, 80, [0, 40], [5, 49]),
}


def _check_bound(c, what):
    ext = any(e != 1 for e in c.ext)
    B.check(c.run(force_extend=ext), B.reference(c, B.kernel_of(c, ext)), what)


@pytest.mark.parametrize("name", [n for n in MIXED if "decode" not in n])
@pytest.mark.parametrize("which", [0, 1])
def test_large_rows_hidden_from_earlier_queries(name, which):
    """K or V rows of the type's largest size (bf16: 3e38, a scale of 2^119) at the last new token of each
    request, which only the last query sees; its queries are zeros, so that no logit overflows."""
    dtype, hq, hkv, d, pre, ext = MIXED[name]
    c = Case(44, dtype, hq, hkv, d, pre, ext)
    big = 0.9 * torch.finfo(DTYPES[dtype]).max
    g = torch.Generator().manual_seed(1)
    at = np.cumsum(ext) - 1
    for r, n in enumerate(c.seq):
        x = torch.rand(d, generator=g) * 2 - 1
        x[0] = 1
        _put(c, r, n - 1, which, big * x)
        c.q[at[r]] = 0
    _check_bound(c, name)


@pytest.mark.parametrize("name", list(MIXED))
def test_large_values_beside_small_ones(name):
    """Every seventh V row is 2^20 (fp16: 2^12) larger and meets logits far below the others' (its K row
    points away from the queries): weights of about 2^-45 beside ordinary ones."""
    dtype, hq, hkv, d, pre, ext = MIXED[name]
    c = Case(45, dtype, hq, hkv, d, pre, ext, scale_spread=0.0)
    u = torch.zeros(d)
    u[::2] = 1
    c.q = (c.q.float() * 0.5 + u).to(DTYPES[dtype])
    v = torch.randn(d, generator=torch.Generator().manual_seed(2))
    for r, n in enumerate(c.seq):
        for j in range(3, n, 7):
            _put(c, r, j, 0, -(64.0 / d ** 0.5) * u)
            _put(c, r, j, 1, (2.0 ** 20 if dtype == "bf16" else 2.0 ** 12) * v)
    _check_bound(c, name)


@pytest.mark.parametrize("name", list(MIXED))
def test_rows_of_every_size(name):
    """K and V scales spread over 2^+-40 (fp16 outputs: V over 2^-30 to 2^6), query sizes to match, so that
    logits stay ordinary."""
    dtype, hq, hkv, d, pre, ext = MIXED[name]
    c = Case(46, dtype, hq, hkv, d, pre, ext, scale_spread=0.0)
    g = torch.Generator().manual_seed(3)
    n = len(c.scale)
    lo, hi = (-40, 40) if dtype == "bf16" else (-30, 6)
    c.scale[..., 1] *= torch.exp2(torch.randint(lo, hi, (n, hkv), generator=g).float())
    c.scale[..., 0] *= torch.exp2(torch.randint(-40, 1, (n, hkv), generator=g).float())
    _check_bound(c, name)


@pytest.mark.parametrize("name", [n for n in MIXED if MIXED[n][0] == "bf16"])
def test_groups_of_large_values_far_above_the_others(name):
    """V rows 2^110 larger in whole groups of keys, with logits 14 below the others': they make the output, the
    others its sum of weights."""
    dtype, hq, hkv, d, pre, ext = MIXED[name]
    c = Case(47, dtype, hq, hkv, d, pre, ext, scale_spread=0.0)
    u = torch.zeros(d)
    u[::2] = 1
    c.q = (c.q.float() * 0.5 + u).to(DTYPES[dtype])
    g = torch.Generator().manual_seed(4)
    for r, n in enumerate(c.seq):
        for j in range(128, 256) if n > 256 else range(32, min(n, 64)):
            _put(c, r, j, 0, -(28.0 / d ** 0.5) * u)
            _put(c, r, j, 1, 2.0 ** 110 * torch.randn(d, generator=g))
    _check_bound(c, name)


@pytest.mark.parametrize("extend", [False, True])
def test_empty_requests_before_a_dependent_launch(extend):
    """A call in which no request has tokens or queries, a read of its output right behind it, and another
    call whose scratch may be the first one's."""
    from tokenfactory_b200 import ops
    c = Case(48, "bf16", 8, 2, 128, [0, 0], [1, 1])
    busy = Case(49, "bf16", 8, 2, 128, [700, 90], [1, 1])
    zero = torch.zeros(2, dtype=torch.int64, device="cuda")
    q, pool, (r2t, rows, _) = c.q.cuda(), c.pool(), c.args()
    qb, poolb, argsb = busy.q.cuda(), busy.pool(), busy.args()
    out = torch.empty_like(q)
    seen, kept = [], []
    for _ in range(50):
        out.fill_(3)
        if extend:
            ops.paged_extend_fp8(q, *pool, r2t, rows, zero, zero, 128 ** -0.5, 1, 1, out=out)
        else:
            ops.paged_decode_fp8(q, *pool, r2t, rows, zero, 128 ** -0.5, 1, out=out)
        seen.append(out.clone())
        kept.append(ops.paged_decode_fp8(qb, *poolb, *argsb, 128 ** -0.5, max(busy.seq)))
    seen, want = torch.stack(seen), B.reference(busy, B.ROWS)
    assert (seen == 3).all() if extend else torch.isnan(seen).all()
    for k in kept:
        B.check(k, want)


@pytest.mark.parametrize("dtype,d", [("f32", 64), ("bf16", 48), ("f16", 80), ("bf16", 128)])
@pytest.mark.parametrize("extend", [False, True])
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
def test_scales_that_are_not_finite_make_the_rows_that_see_them_nan(dtype, d, extend, which, value):
    """A K or V scale that is not finite, its codes all 1 and the queries negative (logits of -inf): NaN in
    every element of the rows of its head that see the token, and nothing in the others."""
    ext = [9, 4] if extend else [1, 1]
    c = Case(50, dtype, 8, 2, d, [40, 20], ext)
    c.q = -c.q.abs()
    slot = int(c.r2t[c.rows[0], 42 if extend else 10])
    c.codes.view(torch.uint8)[slot, 1] = 0x38  # 1.0
    c.scale[slot, 1, which] = value
    got = c.run(force_extend=extend).double().cpu().numpy()
    nan = np.zeros(got.shape, bool)
    nan[2 if extend else 0:ext[0], 4:] = True
    assert np.array_equal(np.isnan(got), nan)
    c.scale[slot, 1, which] = 1e-3
    ref, tol = B.reference(c, B.kernel_of(c, extend))
    assert (np.abs(got - ref)[~nan] <= tol[~nan]).all()


@pytest.mark.parametrize("name", list(MIXED))
@pytest.mark.parametrize("what", ["q", "gate"])
def test_queries_and_gates_that_are_not_finite(name, what):
    """Infinities and NaNs in one query row (or one element of its gate) make that row (element) NaN and leave
    every other one alone."""
    dtype, hq, hkv, d, pre, ext = MIXED[name]
    c = Case(51, dtype, hq, hkv, d, pre, ext, gate="sigmoid")
    extend = any(e != 1 for e in ext)
    t = len(c.q)
    ref, tol = B.reference(c, B.kernel_of(c, extend))
    nan = np.zeros(ref.shape, bool)
    for i, x in enumerate((float("inf"), -float("inf"), float("nan"))):
        row, head = min(i * 2, t - 1), (3 * i) % hq
        if what == "q":
            c.q[row, head, 5 * i + 1] = x
            nan[row, head] = True
        elif i == 2:
            c.gate = c.gate.clone()
            c.gate[row, head, 7] = x
            nan[row, head, 7] = True
    got = c.run(force_extend=extend).double().cpu().numpy()
    assert np.array_equal(np.isnan(got), nan)
    assert (np.abs(got - ref)[~nan] <= tol[~nan]).all()


@pytest.mark.parametrize("name", list(MIXED))
def test_results_repeat_whatever_the_scales(name):
    dtype, hq, hkv, d, pre, ext = MIXED[name]
    c = Case(52, dtype, hq, hkv, d, pre, ext)
    c.scale *= torch.exp2(torch.randint(-12, 13, c.scale.shape).float())
    extend = any(e != 1 for e in ext)
    a = c.run(force_extend=extend)
    for _ in range(3):
        assert torch.equal(a, c.run(force_extend=extend))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_a_model_on_a_prompt_of_zeros(dtype):
    """Hidden states of zero through the full-attention layers and their 8-bit pool: zeros, as from a 16-bit
    pool, and later tokens are finite."""
    from tests.test_gpu_kv_fp8_model import _model, _step
    from tokenfactory_b200.hybrid_model import HybridCachePool
    dt = DTYPES[dtype]
    cfg, model = _model(128, 8, 1, dt)
    with torch.no_grad():
        model.model.language_model.embed_tokens.weight[0] = 0
    r2t = torch.arange(300, device="cuda").view(1, 300)
    outs = []
    for kv in (torch.float8_e4m3fn, None):
        pool = HybridCachePool(cfg, 300, 2, dtype=dt, kv_dtype=kv)
        first = _step(model, pool, r2t, [0], [0], [150], torch.zeros(150, dtype=torch.int64))
        later = _step(model, pool, r2t, [0], [150], [1], torch.tensor([7]))
        outs.append(first)
        assert torch.isfinite(first).all() and torch.isfinite(later).all()
    assert (outs[0] == 0).all() and (outs[1] == 0).all()


@pytest.mark.parametrize("name,size", [(n, 2.0 ** s) for n in MIXED
                                       for s in (8, 15, 24, 29, 33, 60, 100)
                                       if s < 16 or MIXED[n][0] == "bf16"])
def test_logits_of_every_size(name, size):
    """One K row of a given size in the middle of each request, and one twice that size a little behind it:
    where a query's logit is positive it takes all the weight, where it is negative it takes none."""
    dtype, hq, hkv, d, pre, ext = MIXED[name]
    extend = any(e != 1 for e in ext)
    c = Case(53, dtype, hq, hkv, d, pre, ext)
    g = torch.Generator().manual_seed(5)
    for r, n in enumerate(c.seq):
        for at, f in ((n // 2, 0.5), (min(n // 2 + 5, n - 1), 1.0)):
            x = torch.rand(d, generator=g) * 2 - 1
            x[0] = 1
            _put(c, r, at, 0, f * size * x)
    got = c.run(force_extend=extend).double().cpu().numpy()
    kernel, t = B.kernel_of(c, extend), 0
    q, sure, rows = c.q.double().numpy(), 0, 0
    for r, (n, e) in enumerate(zip(c.seq, c.ext)):
        s = c.r2t[c.rows[r], :n].numpy()
        for h in range(hkv):
            k, v, ks, vs = B._group(c, s, h)
            for i in range(e):
                m = n - e + i + 1
                for hh in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                    rows += 1
                    x = k[:m] @ q[t + i, hh] * d ** -0.5
                    # fp32 logits are off by 2^-18 of their terms' sum (bfloat16's large extends 2^-10); a lead of more than
                    # that and 40 (2^-57 of weight) leaves the leader alone
                    err = (np.abs(k[:m]) @ np.abs(q[t + i, hh]) * d ** -0.5).max() * 2.0 ** -10
                    top = np.argsort(x)[::-1]
                    if m > 1 and x[top[0]] - x[top[1]] > 2 * err + 40:
                        want, tol = v[top[0]], 2.0 ** -9 * np.abs(v[top[0]])
                    elif np.abs(x).max() < 40:
                        want, tol = B.row_terms(c, kernel, q[t + i, hh][None], k[:m], v[:m], ks[:m],
                                                vs[:m], d ** -0.5)
                        want, tol = want[0], tol[0]
                    elif x.max() < 40 and x[x > -60].size:  # the large rows take nothing: the others' average
                        keep = np.flatnonzero(x > -60 - 2 * err * (np.abs(x) > 60))
                        keep = keep[np.abs(x[keep]) < 60]
                        if (np.abs(np.delete(x, keep)) < 60 + 4 * err).any():
                            continue
                        want, tol = B.row_terms(c, kernel, q[t + i, hh][None], k[keep], v[keep],
                                                ks[keep], vs[keep], d ** -0.5)
                        want, tol = want[0], tol[0]
                    else:
                        continue
                    sure += 1
                    assert (np.abs(got[t + i, hh] - want) <= B.rounded(dtype, want, tol)).all(), (
                        r, i, hh, np.abs(got[t + i, hh] - want).max(), x[top[:2]])
        t += e
    assert sure > rows // 4
