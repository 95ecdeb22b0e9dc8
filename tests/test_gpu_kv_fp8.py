"""The 8-bit K/V pool on the GPU: store, prologue, decode and extend against float64."""

import numpy as np
import pytest

from oracle import fp8 as OF
from oracle import kv_fp8 as O
from tests.fp8_pool import DTYPES, Case, check

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _codes(x):
    return OF.e4m3_decode(x.contiguous().view(torch.uint8).cpu().numpy())


# ------------------------------------------------------------------------------------------------
# store
# ------------------------------------------------------------------------------------------------
def _empty_pool(slots, hkv, d, layout="adjacent", g=None):
    raw = torch.randint(0, 120, (slots, hkv, 2, d + (3 if layout == "odd" else 0)),
                        dtype=torch.uint8, device="cuda")
    if layout == "odd":
        raw = raw[..., 1:d + 1]
    c = raw.view(torch.float8_e4m3fn)
    sc = torch.rand((slots, hkv, 2), device="cuda")
    return c[:, :, 0], c[:, :, 1], sc


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hkv,d,layout", [(1, 64, "adjacent"), (4, 128, "adjacent"),
                                          (3, 256, "adjacent"), (2, 80, "adjacent"),
                                          (1, 1, "adjacent"), (2, 256, "odd")])
@pytest.mark.parametrize("tokens", [1, 37])
def test_store_is_bit_exact(dtype, hkv, d, layout, tokens):
    from tokenfactory_b200 import ops
    torch.manual_seed(tokens * d)
    slots = tokens + 9
    kb, vb, sc = _empty_pool(slots, hkv, d, layout)
    before = kb.contiguous().view(torch.uint8).clone(), sc.clone()
    dt = DTYPES[dtype]
    # k strided (a view of a wider projection), v with rows of very different size
    k = torch.randn((tokens, hkv, 2 * d), device="cuda").to(dt)[..., :d]
    v = (torch.randn((tokens, hkv, d), device="cuda")
         * torch.exp(4 * torch.randn((tokens, hkv, 1), device="cuda"))).to(dt)
    v[0, 0] = 0
    loc = torch.randperm(slots, device="cuda")[:tokens]
    neg = loc.clone()
    neg[0] -= slots  # torch's wrap
    ops.kv_store_fp8(kb, vb, sc, neg, k, v)
    for j, (buf, x) in enumerate(((kb, k), (vb, v))):
        codes, scale = O.quantize_rows(x.float().cpu().numpy())
        np.testing.assert_array_equal(_codes(buf.view(torch.uint8)[loc]),
                                      codes)
        np.testing.assert_array_equal(sc[loc, :, j].cpu().numpy(), scale)
    rest = torch.ones(slots, dtype=torch.bool, device="cuda")
    rest[loc] = False
    assert torch.equal(kb.contiguous().view(torch.uint8)[rest], before[0][rest])
    assert torch.equal(sc[rest], before[1][rest])


@pytest.mark.parametrize("d", [64, 256, 48])
def test_store_of_rows_that_are_not_finite(d):
    from tokenfactory_b200 import ops
    kb, vb, sc = _empty_pool(6, 2, d)
    k = torch.randn((4, 2, d), device="cuda", dtype=torch.bfloat16)
    v = torch.randn((4, 2, d), device="cuda", dtype=torch.bfloat16)
    k[0, 1, d - 1], k[2, 0, 5], v[3, 1, 0] = float("inf"), float("nan"), -float("inf")
    loc = torch.tensor([5, 0, 2, 3], device="cuda")
    ops.kv_store_fp8(kb, vb, sc, loc, k, v)
    for j, (buf, x) in enumerate(((kb, k), (vb, v))):
        codes, scale = O.quantize_rows(x.float().cpu().numpy())
        np.testing.assert_array_equal(_codes(buf.view(torch.uint8)[loc]), codes)
        np.testing.assert_array_equal(sc[loc, :, j].cpu().numpy(), scale)


def test_store_skips_and_records_bad_locations():
    from tokenfactory_b200 import _capi, ops
    kb, vb, sc = _empty_pool(6, 2, 64)
    before = kb.contiguous().view(torch.uint8).clone()
    k = torch.randn((3, 2, 64), device="cuda", dtype=torch.bfloat16)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.kv_store_fp8(kb, vb, sc, torch.tensor([6, 1, -7], device="cuda"), k, k, err=err)
    assert err.item() == _capi.TF_KERR_SLOT_RANGE
    after = kb.contiguous().view(torch.uint8)
    keep = [0, 2, 3, 4, 5]
    assert torch.equal(after[keep], before[keep]) and not torch.equal(after[1], before[1])


# ------------------------------------------------------------------------------------------------
# prologue
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hq,hkv,d,rot", [(32, 4, 256, 64), (8, 2, 64, 16), (4, 1, 128, 32),
                                          (6, 2, 128, 128), (2, 2, 256, 96), (3, 1, 64, 2)])
@pytest.mark.parametrize("mrope", [None, True, False])
def test_prologue(dtype, hq, hkv, d, rot, mrope):
    from tokenfactory_b200 import ops
    if mrope is not None and rot < 6:
        pytest.skip("three sections need three angles")
    g = torch.Generator().manual_seed(d + rot)
    t, slots = 7, 19
    dt = DTYPES[dtype]
    q = torch.randn((t, hq, 2 * d), generator=g).to(dt)[..., :d]
    k, v = (torch.randn((t, hkv, d), generator=g).to(dt) for _ in range(2))
    wq, wk = ((1 + 0.2 * torch.randn(d, generator=g)) for _ in range(2))
    if dtype != "f32" and hkv != 2:
        wq, wk = wq.to(dt), wk.to(dt)  # otherwise fp32 weights beside 16-bit activations
    pos = torch.randint(0, 1 << 20, (t,) if mrope is None else (3, t), generator=g)
    inv = 1.0 / 1e7 ** (torch.arange(0, rot, 2, dtype=torch.float32) / rot)
    h = rot // 2
    sec = (h - 2 * (h // 3), h // 3, h // 3)
    loc = torch.randperm(slots, generator=g)[:t]
    kb, vb, sc = _empty_pool(slots, hkv, d)
    got = ops.attn_prologue_fp8(q.cuda(), k.cuda(), v.cuda(), wq.cuda(), wk.cuda(), pos.cuda(),
                                inv.cuda(), kb, vb, sc, loc.cuda(), eps=1e-6, mrope_section=sec,
                                mrope_interleaved=bool(mrope))
    args = (pos.numpy(), inv.numpy(), 1e-6, sec, bool(mrope))
    wantq = O.norm_rotate(q.double().numpy(), wq.double().numpy(), *args)
    wantk = O.norm_rotate(k.double().numpy(), wk.double().numpy(), *args)
    # fp32 norm and rotation: a dozen operations of at most 2^-23 each of the row's largest value
    slack = 2.0 ** -19 * max(np.abs(wantq).max(), np.abs(wantk).max())
    tol = torch.finfo(dt).eps / 2 * np.abs(wantq) + slack
    assert (np.abs(got.double().cpu().numpy() - wantq) <= tol).all()
    scale = sc[loc.cuda()].double().cpu().numpy()
    rows = [_codes(b.view(torch.uint8)[loc.cuda()]).astype(np.float64) * scale[..., j, None]
            for j, b in enumerate((kb, vb))]
    for r, want, s, sl in ((rows[0], wantk, scale[..., 0], slack),
                           (rows[1], v.double().numpy(), scale[..., 1], 0)):
        amax = np.abs(want).max(-1)
        assert (np.abs(s - amax / 448) <= 2.0 ** -22 * amax / 448 + sl / 448).all()
        # half a step of e4m3: 2^-4 of the value, 2^-10 of the scale below 2^-6
        half = np.maximum(2.0 ** -4 * np.abs(want), 2.0 ** -10 * s[..., None])
        assert (np.abs(r - want) <= half * (1 + 2.0 ** -18) + 2 * sl).all()


def test_prologue_unaligned_and_bad_location():
    from tokenfactory_b200 import _capi, ops
    t, hq, hkv, d = 5, 4, 2, 128
    kb, vb, sc = _empty_pool(8, hkv, d, "odd")
    k8, v8, sc8 = _empty_pool(8, hkv, d)
    x = torch.randn((t, hq + 2 * hkv, d + 1), device="cuda", dtype=torch.bfloat16)[..., 1:]
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    w = torch.ones(d, device="cuda", dtype=torch.bfloat16)
    pos = torch.arange(t, device="cuda")
    inv = torch.rand(16, device="cuda")
    loc = torch.tensor([3, 8, 0, 5, -1], device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    a = ops.attn_prologue_fp8(q, k, v, w, w, pos, inv, kb, vb, sc, loc, err=err)
    assert err.item() == _capi.TF_KERR_SLOT_RANGE
    b = ops.attn_prologue_fp8(q.contiguous(), k.contiguous(), v.contiguous(), w, w, pos, inv, k8,
                              v8, sc8, loc)
    ok = torch.tensor([3, 0, 5, 7], device="cuda")
    # the two forms of the kernel may contract their products differently: an ulp of the output
    torch.testing.assert_close(a.float(), b.float(), rtol=2.0 ** -7, atol=1e-5)
    torch.testing.assert_close(sc[ok], sc8[ok], rtol=1e-5, atol=0)
    torch.testing.assert_close(kb.view(torch.uint8)[ok].view(torch.float8_e4m3fn).float(),
                               k8.view(torch.uint8)[ok].view(torch.float8_e4m3fn).float(),
                               rtol=2.0 ** -3, atol=2.0 ** -8)
    assert torch.equal(vb.view(torch.uint8)[ok], v8.view(torch.uint8)[ok])


# ------------------------------------------------------------------------------------------------
# decode
# ------------------------------------------------------------------------------------------------
DECODE = {
    # name: (dtype, hq, hkv, d, lengths, more)
    "one_token": ("bf16", 8, 1, 256, [1], {}),
    "lengths": ("bf16", 32, 4, 256, [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129], {}),
    "empty": ("bf16", 8, 2, 128, [0, 5, 0, 33, 0], {}),
    "all_empty": ("f16", 8, 2, 64, [0, 0], {}),
    "gqa1": ("bf16", 4, 4, 64, [7, 70, 300], {}),
    "gqa3": ("f16", 12, 4, 128, [100, 9, 257], {}),
    "gqa6": ("bf16", 24, 4, 256, [40, 555], {}),
    "gqa7_h3": ("bf16", 21, 3, 128, [40, 222, 1], {}),
    "gqa16": ("bf16", 32, 2, 64, [40, 100], {}),
    "mqa_f16": ("f16", 8, 1, 256, [700, 3], {}),
    "heads8": ("bf16", 16, 8, 64, [90, 17, 1, 260], {}),
    "heads16": ("bf16", 16, 16, 64, [90, 17], {}),
    "f32": ("f32", 8, 2, 64, [17, 96, 40, 1], {}),
    "d80": ("bf16", 4, 2, 80, [33, 64], {}),
    "d32_f16": ("f16", 8, 2, 32, [33, 64], {}),
    "long": ("bf16", 8, 1, 256, [9001, 100, 2500], {}),
    "long_f16": ("f16", 8, 2, 128, [7001, 13], {}),
    "separate": ("bf16", 8, 2, 256, [50, 300], dict(layout="separate")),
    "odd": ("bf16", 8, 2, 128, [50, 130], dict(layout="odd")),
    "spread": ("bf16", 8, 2, 128, [400, 130], dict(scale_spread=4.0)),
    "spread_f16": ("f16", 8, 2, 256, [400, 130], dict(scale_spread=4.0)),
    "silu": ("bf16", 8, 2, 128, [50, 130], dict(gate="silu")),
    "sigmoid": ("bf16", 32, 4, 256, [50, 1300, 5], dict(gate="sigmoid")),
    "sigmoid_f32": ("f32", 8, 2, 64, [50, 5], dict(gate="sigmoid")),
    "batch": ("bf16", 8, 2, 64, [(37 * i) % 301 + 1 for i in range(200)], dict(gate="silu")),
}


@pytest.mark.parametrize("name", list(DECODE))
def test_decode(name):
    dtype, hq, hkv, d, seq, more = DECODE[name]
    c = Case(11, dtype, hq, hkv, d, [s - 1 for s in seq], [1] * len(seq), **more)
    check(c.run(), c.reference(), dtype, d, name)


def test_decode_reads_negative_entries_as_the_sibling_does():
    c = Case(5, "bf16", 8, 2, 128, [40, 20], [1, 1])
    c.r2t[c.rows[0], 3] = -1
    for mode in ("clamp", "wrap"):
        check(c.run(slot_mode=mode), c.reference(mode), "bf16", 128, mode)


def test_decode_records_bad_entries():
    from tokenfactory_b200 import _capi
    c = Case(5, "bf16", 8, 2, 128, [40, 20], [1, 1])
    slots = c.codes.shape[0]
    c.r2t[c.rows[1], 3] = slots
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = c.run(err=err)
    assert err.item() == _capi.TF_KERR_SLOT_RANGE
    c.r2t[c.rows[1], 3] = 0  # what it is read as
    check(got, c.reference(), "bf16", 128)
    c.rows = c.rows.clone()
    c.rows[0] = c.r2t.shape[0]
    err.zero_()
    c.run(err=err)
    assert err.item() == _capi.TF_KERR_REQ_RANGE


@pytest.mark.parametrize("d,hkv", [(256, 4), (128, 1), (64, 2), (48, 2)])
def test_decode_of_scales_that_are_not_finite(d, hkv):
    """NaN, infinite and zero scales reach the requests that see their tokens and no other; the last
    tile of a shorter request ends inside its rows."""
    c = Case(6, "bf16", 4 * hkv, hkv, d, [40, 20, 60, 33], [1, 1, 1, 1])
    s0, s1, s2 = (int(c.r2t[c.rows[i], 10]) for i in (0, 1, 2))
    c.scale[s0, 0, 0] = float("nan")
    c.scale[s1, 0, 1] = float("inf")
    c.codes.view(torch.uint8)[s1, 0, 1] = 0
    c.scale[s2, :, :] = 0
    check(c.run(), c.reference(), "bf16", d)


def test_decode_at_the_end_of_a_pool_past_32_bit_offsets():
    from tokenfactory_b200 import ops
    hkv, d, slots = 4, 256, 2_300_000  # 4.7 GB of codes
    small = Case(8, "bf16", 32, hkv, d, [300, 1000], [1, 1])
    n = small.codes.shape[0]
    codes = torch.empty((slots, hkv, 2, d), dtype=torch.float8_e4m3fn, device="cuda")
    sc = torch.empty((slots, hkv, 2), device="cuda")
    codes.view(torch.uint8)[slots - n:] = small.codes.view(torch.uint8).cuda()
    sc[slots - n:] = small.scale.cuda()
    r2t, rows, seq = small.args()
    r2t = torch.where(r2t >= 0, r2t + (slots - n), r2t)
    got = ops.paged_decode_fp8(small.q.cuda(), codes[:, :, 0], codes[:, :, 1], sc, r2t, rows, seq,
                               d ** -0.5, max(small.seq))
    check(got, small.reference(), "bf16", d)
    got = ops.paged_extend_fp8(small.q.cuda(), codes[:, :, 0], codes[:, :, 1], sc, r2t, rows, seq,
                               torch.ones_like(seq), d ** -0.5, max(small.seq), 1)
    check(got, small.reference(), "bf16", d)


# ------------------------------------------------------------------------------------------------
# extend
# ------------------------------------------------------------------------------------------------
EXTEND = {
    # name: (dtype, hq, hkv, d, prefixes, new tokens, more)
    "one": ("bf16", 8, 1, 256, [0], [1], {}),
    "prompt": ("bf16", 8, 2, 128, [0, 0], [129, 5], {}),
    "prefix": ("bf16", 32, 4, 256, [100, 0, 257], [33, 64, 17], {}),
    "edges": ("bf16", 8, 2, 128, [127, 128, 129, 0, 63], [1, 1, 128, 127, 65], {}),
    "drafts": ("bf16", 32, 4, 256, [900, 30, 513, 2000], [4, 1, 3, 8], dict(gate="sigmoid")),
    "drafts_f16": ("f16", 8, 2, 128, [1900, 0], [2, 5], {}),
    "drafts_d64": ("bf16", 16, 8, 64, [300, 7, 640], [3, 2, 6], dict(gate="silu")),
    "long_prefix": ("bf16", 8, 1, 256, [6000], [40], {}),
    "f16": ("f16", 8, 2, 256, [77, 0, 5], [40, 200, 1], {}),
    "f16_d64": ("f16", 8, 2, 64, [77, 0], [40, 100], {}),
    "f32": ("f32", 8, 2, 64, [20, 0], [10, 33], dict(gate="sigmoid")),
    "gqa1": ("bf16", 4, 4, 64, [10, 200], [150, 3], {}),
    "gqa3": ("bf16", 12, 4, 128, [50], [70], {}),
    "gqa6": ("bf16", 24, 4, 256, [50, 9], [70, 11], {}),
    "gqa16": ("bf16", 32, 2, 128, [50], [30], {}),
    "d80": ("bf16", 4, 2, 80, [20], [33], {}),
    "separate": ("bf16", 8, 2, 256, [50, 300], [40, 3], dict(layout="separate")),
    "odd": ("bf16", 8, 2, 128, [50, 130], [40, 3], dict(layout="odd")),
    "spread": ("bf16", 8, 2, 128, [200, 130], [40, 300], dict(scale_spread=4.0)),
    "spread_f16": ("f16", 8, 2, 256, [200, 130], [40, 300], dict(scale_spread=4.0)),
    "silu": ("bf16", 8, 2, 128, [50, 0], [140, 60], dict(gate="silu")),
    "some_empty": ("bf16", 8, 2, 128, [0, 30, 0, 8], [0, 20, 0, 3], {}),
}


@pytest.mark.parametrize("name", list(EXTEND))
def test_extend(name):
    dtype, hq, hkv, d, pre, ext, more = EXTEND[name]
    c = Case(12, dtype, hq, hkv, d, pre, ext, **more)
    check(c.run(force_extend=True), c.reference(), dtype, d, name)


def test_decode_batch_through_extend():
    c = Case(13, "bf16", 32, 4, 256, [499, 0, 1200, 16], [1, 1, 1, 1], gate="sigmoid")
    check(c.run(force_extend=True), c.reference(), "bf16", 256)


def test_extend_leaves_rows_behind_the_last_request():
    c = Case(14, "bf16", 8, 2, 128, [30, 9], [20, 7])
    t = c.q.shape[0]
    extra = torch.randn((5, 8, 128)).to(c.q)
    q, c.q = c.q, torch.cat((c.q, extra))
    out = torch.full(c.q.shape, 3.0, dtype=c.q.dtype, device="cuda")
    c.run(out=out)
    assert (out[t:] == 3).all()
    c.q = q
    check(out[:t], c.reference(), "bf16", 128)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_extend_hidden_tokens_do_not_reach_earlier_rows(d):
    """Scales of NaN and infinity on new tokens: rows before them are untouched, rows that see them
    are NaN."""
    c = Case(15, "bf16", 8, 2, d, [70, 3], [60, 200])
    s = int(c.r2t[c.rows[0], 70 + 30])
    c.scale[s, 0, 1] = float("nan")
    s = int(c.r2t[c.rows[1], 3 + 150])
    c.scale[s, 1, 0] = float("inf")
    got, ref = c.run(), c.reference()
    g = got.double().cpu().numpy()
    assert np.isfinite(g[:30]).all() and np.isnan(g[30:60, :4]).all()
    assert np.isfinite(g[30:60, 4:]).all()
    assert np.isfinite(g[60:210]).all() and np.isnan(g[210:, 4:]).all()
    ref[0][30:60, :4] = np.nan
    ref[0][210:, 4:] = np.nan
    check(got, ref, "bf16", d)


def test_extend_records_lengths_the_table_cannot_hold():
    from tokenfactory_b200 import _capi, ops
    c = Case(16, "bf16", 8, 2, 128, [30, 9], [20, 7])
    r2t, rows, seq = c.args()
    seq[0] = r2t.shape[1] + 1
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.full(c.q.shape, 3.0, dtype=c.q.dtype, device="cuda")
    ops.paged_extend_fp8(c.q.cuda(), *c.pool(), r2t, rows, seq,
                         torch.tensor(c.ext, device="cuda"), 128 ** -0.5, max(c.seq), max(c.ext),
                         out=out, err=err)
    assert err.item() == _capi.TF_KERR_SLOT_RANGE
    assert (out[:20] == 3).all() and torch.isfinite(out[20:].float()).all()


# ------------------------------------------------------------------------------------------------
# streams, graphs, strides
# ------------------------------------------------------------------------------------------------
def test_strided_query_and_output():
    from tokenfactory_b200 import ops
    c = Case(17, "bf16", 8, 2, 128, [300, 40], [1, 1])
    wide = torch.zeros((2, 8, 300), dtype=torch.bfloat16, device="cuda")
    q = wide[..., 3:131]
    q.copy_(c.q)
    out = torch.zeros((2, 9, 133), dtype=torch.bfloat16, device="cuda")
    o = ops.paged_decode_fp8(q, *c.pool(), *c.args(), 128 ** -0.5, 301, out=out[:, 1:, 2:130])
    check(o, c.reference(), "bf16", 128)
    assert (out[:, 0] == 0).all() and (out[:, :, :2] == 0).all() and (out[:, :, 130:] == 0).all()
    ext = torch.ones(2, dtype=torch.int64, device="cuda")
    out.zero_()
    o = ops.paged_extend_fp8(q, *c.pool(), *c.args(), ext, 128 ** -0.5, 301, 1,
                             out=out[:, 1:, 2:130])
    check(o, c.reference(), "bf16", 128)
    assert (out[:, 0] == 0).all() and (out[:, :, :2] == 0).all() and (out[:, :, 130:] == 0).all()


@pytest.mark.parametrize("extend", [False, True])
def test_two_graphs_and_eager_calls_interleaved(extend):
    """Two captured calls of different batches and an eager one, on their own streams at once: none
    uses another's scratch; replays follow changed lengths."""
    from tokenfactory_b200 import ops
    cases = [Case(20 + i, "bf16", 8, 1, 256, pre, [3 if extend else 1] * len(pre))
             for i, pre in enumerate(([3000, 50], [700, 1500, 9], [2500]))]
    dev = []
    for c in cases:
        dev.append(dict(q=c.q.cuda(), pool=c.pool(), args=c.args(),
                        ext=torch.tensor(c.ext, device="cuda")))

    def call(c, x):
        if extend:
            return ops.paged_extend_fp8(x["q"], *x["pool"], *x["args"], x["ext"], 1 / 16,
                                        max(c.seq), 3)
        return ops.paged_decode_fp8(x["q"], *x["pool"], *x["args"], 1 / 16, max(c.seq))

    want = [c.reference() for c in cases]
    for c, x in zip(cases, dev):
        call(c, x)
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in cases]
    for c, x in zip(cases[:2], dev[:2]):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(c, x))
        graphs.append(g)
    for _ in range(5):
        for o in outs:
            o.fill_(7)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            eager = call(cases[2], dev[2])
        torch.cuda.synchronize()
        for o, w in zip(outs + [eager], want):
            check(o, w, "bf16", 256)
    # the captured call reads its lengths on the device
    c = cases[0]
    seq = [s - 17 for s in c.seq]
    dev[0]["args"][2].copy_(torch.tensor(seq))
    c.seq = seq
    graphs[0].replay()
    torch.cuda.synchronize()
    check(outs[0], c.reference(), "bf16", 256)
    del graphs


def test_results_repeat():
    c = Case(30, "bf16", 32, 4, 256, [4000, 77, 1500], [1, 1, 1], gate="sigmoid")
    a, b = c.run(), c.run()
    assert torch.equal(a, b)
    a, b = c.run(force_extend=True), c.run(force_extend=True)
    assert torch.equal(a, b)


# many requests in one CTA's share, head groups above a tile's, batches above the plan's, and large
# extends whose key blocks end at every place
EDGES = {
    # name: (dtype, hq, hkv, d, prefixes, new tokens, more)
    "decode_many_tiny": ("bf16", 4, 2, 64, [i % 3 - 1 for i in range(20000)], [1] * 20000, {}),
    "decode_beyond_the_plan": ("bf16", 2, 1, 64, [0] * 33000, [1] * 33000, {}),
    "decode_gqa40": ("bf16", 40, 1, 128, [70, 3, 300], [1, 1, 1], dict(gate="sigmoid")),
    "decode_gqa64": ("f16", 64, 1, 64, [70, 3, 300], [1, 1, 1], {}),
    "decode_gqa1_h20": ("bf16", 20, 20, 128, [70, 3, 0], [1, 1, 1], {}),
    "extend_many_tiny": ("bf16", 8, 2, 128, [i % 5 for i in range(6000)],
                         [i % 4 for i in range(6000)], {}),
    "extend_many_and_one_large": ("bf16", 8, 2, 64, [i % 5 for i in range(2000)],
                                  [200 if i == 777 else i % 3 for i in range(2000)], {}),
    "extend_gqa24": ("bf16", 24, 1, 128, [33], [40], {}),
    "extend_gqa24_drafts": ("bf16", 24, 1, 128, [33, 250], [2, 1], dict(gate="silu")),
    "extend_two_passes": ("bf16", 32, 4, 256, [900, 30, 513, 2000], [6, 1, 3, 5], dict(gate="sigmoid")),
    "extend_two_passes_f16": ("f16", 12, 2, 64, [300, 7, 0], [8, 2, 1], {}),
    "extend_d64": ("bf16", 8, 2, 64, [500, 0], [301, 129], dict(gate="silu")),
    "extend_d64_f16": ("f16", 16, 2, 64, [333, 1], [150, 257], {}),
    "extend_split": ("bf16", 8, 1, 256, [3000, 0, 1], [70, 1, 200], dict(gate="sigmoid")),
    "extend_split_f16": ("f16", 8, 1, 128, [2900, 0], [70, 1], {}),
    "extend_gqa5": ("bf16", 10, 2, 256, [200, 14], [37, 90], {}),
}


@pytest.mark.parametrize("name", list(EDGES))
def test_edges(name):
    dtype, hq, hkv, d, pre, ext, more = EDGES[name]
    c = Case(13, dtype, hq, hkv, d, pre, ext, **more)
    check(c.run(), c.reference(), dtype, d, name)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("ext", [[1] * 9, [80, 1, 90]])
def test_a_row_of_one_key_is_that_key(d, ext):
    """float16: the only key's value, off by the output's rounding (half a step, 2^-11 of the value) and
    a few fp32 operations (2^-20), whatever the weight's rounding was."""
    c = Case(17, "f16", 8, 2, d, [0] * len(ext), ext, scale_spread=2.0)
    got = c.run().double().cpu().numpy()
    ref = c.reference()[0]
    first = np.cumsum([0] + ext[:-1])
    tol = (2.0 ** -11 + 2.0 ** -20) * np.abs(ref[first]) + 2.0 ** -25
    assert (np.abs(got[first] - ref[first]) <= tol).all()


def test_more_than_64_query_heads_per_kv_head_are_refused():
    from tokenfactory_b200 import _capi
    for ext in (1, 2):
        with pytest.raises(_capi.TFAttnError, match="64 query heads"):
            Case(13, "bf16", 65, 1, 64, [70, 3], [ext, ext]).run()


def test_refusals():
    from tokenfactory_b200 import _capi, ops
    c = Case(31, "bf16", 8, 2, 128, [30, 9], [1, 1])
    q, (kb, vb, sc), args = c.q.cuda(), c.pool(), c.args()

    def dec(q=q, kb=kb, vb=vb, sc=sc, args=args, **kw):
        return ops.paged_decode_fp8(q, kb, vb, sc, *args, 128 ** -0.5, 31, **kw)

    with pytest.raises(TypeError):
        dec(kb=kb.float(), vb=vb.float())
    with pytest.raises(TypeError):
        dec(sc=sc.half())
    with pytest.raises(ValueError):
        dec(sc=sc[:-1])
    with pytest.raises(ValueError):
        dec(sc=sc.transpose(1, 2))
    with pytest.raises(ValueError):
        dec(q=q[:, :7])
    with pytest.raises(ValueError):
        dec(q=q[..., :64])
    with pytest.raises(ValueError):
        dec(args=(args[0], args[1], args[2][:1]))
    with pytest.raises(ValueError):
        dec(out=torch.empty((2, 8, 64), dtype=q.dtype, device="cuda"))
    with pytest.raises(TypeError):
        dec(out=torch.empty((2, 8, 128), dtype=torch.float16, device="cuda"))
    with pytest.raises(TypeError):
        dec(q=q.double())
    with pytest.raises(KeyError):
        dec(gate_mode="tanh")
    with pytest.raises(_capi.TFAttnError):
        dec(gate_mode="silu")  # no gate given
    with pytest.raises(_capi.TFAttnError):
        ops.paged_decode_fp8(q, kb, vb, sc, *args, 0.1, args[0].shape[1] + 1)
    with pytest.raises(ValueError):
        ops.paged_extend_fp8(q, kb, vb, sc, *args, args[2][:1], 0.1, 31, 1)
    k = torch.zeros((2, 2, 128), dtype=torch.bfloat16, device="cuda")
    loc = torch.tensor([0, 1], device="cuda")
    with pytest.raises(ValueError):
        ops.kv_store_fp8(kb, vb, sc, loc[:1], k, k)
    with pytest.raises(ValueError):
        ops.kv_store_fp8(kb, vb, sc, loc, k[..., :64], k[..., :64])
    with pytest.raises(ValueError):  # a pool of the activation dtype
        ops.kv_store_fp8(k, k, sc[:2], loc, k, k)
    with pytest.raises(ValueError):
        ops.kv_store_fp8(kb, vb, sc, loc, k, k.half())
    with pytest.raises(TypeError):
        ops.kv_store_fp8(kb, vb, sc, loc.int(), k, k)
    w = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    inv = torch.ones(16, device="cuda")
    with pytest.raises(TypeError):
        ops.attn_prologue_fp8(q, k, k, w, w, loc, inv, k, k, sc[:2], loc)
    with pytest.raises(ValueError):
        ops.attn_prologue_fp8(q, k, k, w, w, loc, inv, kb, vb, sc, loc, q_out=q[:1].clone())
    with pytest.raises(_capi.TFAttnError):
        ops.attn_prologue_fp8(q, k, k, w, w, loc, torch.ones(65, device="cuda"), kb, vb, sc, loc)
    # empty calls do nothing
    e = torch.zeros(0, dtype=torch.int64, device="cuda")
    assert ops.paged_decode_fp8(q[:0], kb, vb, sc, args[0], e, e, 0.1, 1).shape == (0, 8, 128)
    assert ops.paged_extend_fp8(q[:0], kb, vb, sc, args[0], e, e, e, 0.1, 1, 1).shape == (0, 8, 128)
    ops.kv_store_fp8(kb, vb, sc, e, k[:0], k[:0])
