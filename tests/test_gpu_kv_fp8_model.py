"""The 8-bit K/V pool under the model: the operators run together as a serving step calls them
(prompts, a chunk on a cached prefix, drafts, single tokens), a layer's pool rows against those of a
16-bit pool, and a captured step."""

import numpy as np
import pytest

from oracle import kv_fp8 as O
from tests.fp8_pool import check

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _model(d, hq, hkv, dtype):
    from tokenfactory_b200.hybrid_model import HybridConfig, HybridForCausalLM
    torch.manual_seed(3)
    cfg = HybridConfig(hidden_size=256, num_attention_heads=hq, num_key_value_heads=hkv, head_dim=d,
                       linear_num_key_heads=2, linear_num_value_heads=4, linear_key_head_dim=128,
                       linear_value_head_dim=128, vocab_size=512, intermediate_size=320,
                       num_hidden_layers=3,
                       layer_types=["full_attention", "linear_attention", "full_attention"])
    prev = torch.get_default_dtype()
    torch.set_default_dtype(dtype)  # (.to(dtype) would round the rotary frequencies)
    try:
        model = HybridForCausalLM(cfg)
    finally:
        torch.set_default_dtype(prev)
    with torch.no_grad():
        for n, p in model.named_parameters():
            if n.endswith("A_log"):
                p.uniform_(0.0, 1.5)
            elif p.dim() == 1:
                p.uniform_(0.5, 1.5)
            else:
                p.normal_(0.0, 0.1)
    return cfg, model.eval().cuda()


def _step(model, pool, r2t, rows, pre, ext, ids):
    from tokenfactory_b200 import ForwardBatch
    dev = "cuda"
    seq = [p + e for p, e in zip(pre, ext)]
    pos = torch.cat([torch.arange(p, n) for p, n in zip(pre, seq)]).to(dev)
    loc = torch.cat([r2t[r, p:n] for r, p, n in zip(rows, pre, seq)])
    fb = ForwardBatch(batch_size=len(rows), req_pool_indices=torch.tensor(rows, device=dev),
                      seq_lens=torch.tensor(seq, device=dev),
                      prefix_lens=torch.tensor(pre, device=dev), extend_lens=list(ext),
                      out_cache_loc=loc, req_to_token=r2t, is_prefill=max(ext) > 1,
                      max_seq_len=max(seq), max_extend_len=max(ext),
                      extend_lens_tensor=torch.tensor(ext, device=dev))
    return model(ids.to(dev), pos, pool, fb)


class _Spy:
    """Records the calls of the pool's operators that the layers make."""

    NAMES = ("kv_store_fp8", "attn_prologue_fp8", "paged_decode_fp8", "paged_extend_fp8")

    def __init__(self, monkeypatch):
        from tokenfactory_b200 import hybrid_attention, ops
        self.calls = []
        for name in self.NAMES:
            real = getattr(ops, name)

            def fn(*a, _real=real, _name=name, **kw):
                out = _real(*a, **kw)
                # the operands that later calls change, as they were read
                keep = [x.clone() if torch.is_tensor(x) else x for x in a]
                self.calls.append((_name, keep, kw, None if out is None else out.clone()))
                return out

            monkeypatch.setattr(hybrid_attention.ops, name, fn)


def _check_attention(name, a, kw, out, dtype, d):
    q, kb, vb, sc = (x.float().double().cpu().numpy() for x in a[:4])
    r2t, rows, seq = (x.cpu().numpy() for x in a[4:7])
    ext = [1] * len(seq) if name == "paged_decode_fp8" else a[7].tolist()
    scale = a[7] if name == "paged_decode_fp8" else a[8]
    gate = kw["gate"].double().cpu().numpy()
    ref = O.attention(q, kb * sc[..., :1], vb * sc[..., 1:], r2t, rows.tolist(), seq.tolist(), ext,
                      scale, gate, kw["gate_mode"], kw["slot_mode"], sc[..., 1])
    check(out, ref, dtype, d, name)


@pytest.mark.parametrize("dtype,d,hq,hkv", [("bf16", 256, 8, 2), ("bf16", 128, 8, 1),
                                            ("f16", 64, 8, 4), ("bf16", 32, 4, 2),
                                            ("f32", 64, 4, 2)])
def test_steps_of_a_model(monkeypatch, dtype, d, hq, hkv):
    """Prompts, a chunk next to drafts, and single tokens of up to three requests: every call's
    result from the pool as that call found it, and the rows that the first layer stores against a
    16-bit pool's."""
    from tests.fp8_pool import DTYPES
    from tokenfactory_b200.hybrid_model import HybridCachePool
    dt = DTYPES[dtype]
    cfg, model = _model(d, hq, hkv, dt)
    g = torch.Generator().manual_seed(4)
    slots, width = 650, 200
    r2t = torch.full((4, width), -1, dtype=torch.int64)
    r2t[:3] = torch.randperm(slots, generator=g)[:3 * width].view(3, width)
    r2t = r2t.cuda()
    p8 = HybridCachePool(cfg, slots, 4, dtype=dt, kv_dtype=torch.float8_e4m3fn)
    p16 = HybridCachePool(cfg, slots, 4, dtype=dt)
    assert p8.k_buffer.dtype == torch.float8_e4m3fn and p8.get_full_kv_scales(0) is not None
    assert p16.get_full_kv_scales(0) is None
    spy = _Spy(monkeypatch)
    steps = [([0, 1], [0, 0], [70, 9]),           # prompts
             ([0, 2, 1], [70, 0, 9], [33, 1, 3]),  # a chunk, a first token, drafts
             ([0, 1, 2], [103, 12, 1], [1, 1, 1]),
             ([2], [2], [1]),                      # a batch of one
             ([1, 2], [13, 3], [1, 1])]
    for rows, pre, ext in steps:
        ids = torch.randint(0, cfg.vocab_size, (sum(ext),), generator=g)
        logits = _step(model, p8, r2t, rows, pre, ext, ids)
        _step(model, p16, r2t, rows, pre, ext, ids)
        assert logits.shape == (len(rows), cfg.vocab_size) and torch.isfinite(logits).all()
        names = [c[0] for c in spy.calls]
        attend = "paged_decode_fp8" if max(ext) == 1 else "paged_extend_fp8"
        assert len(names) == 4 and names[1] == names[3] == attend, names
        assert names[0] in ("attn_prologue_fp8", "kv_store_fp8") and names[0] == names[2]
        assert (d in (64, 128, 256)) == (names[0] == "attn_prologue_fp8"), names
        for name, a, kw, out in spy.calls:
            if name == attend:
                _check_attention(name, a, kw, out, dtype, d)
        spy.calls.clear()
    # layer 0 sees the same input from both pools: its K/V differ by the codes' rounding only
    written = torch.cat([r2t[0, :104], r2t[1, :14], r2t[2, :4]])
    rest = torch.ones(slots, dtype=torch.bool, device="cuda")
    rest[written] = False
    k8, v8 = p8.get_full_kv_buffers(0)
    sc = p8.get_full_kv_scales(0)
    assert (k8.view(torch.uint8)[rest] == 0).all() and (sc[rest] == 0).all()
    k16, v16 = (x[written].double().cpu().numpy() for x in p16.get_full_kv_buffers(0))
    s = sc[written].double().cpu().numpy()
    k, v = (x[written].float().double().cpu().numpy() * s[..., j:j + 1]
            for j, x in enumerate((k8, v8)))
    # V is stored as it is: half a step of e4m3 (2^-4 of the value; 2^-10 of the scale below 2^-6)
    half = np.maximum(2.0 ** -4 * np.abs(v16), 2.0 ** -10 * s[..., 1:])
    assert (np.abs(v - v16) <= half * (1 + 2.0 ** -20)).all()
    # K of the 16-bit pool is rounded too, at most at the norm's two products, the rotation's sine,
    # cosine, two products and sum (seven roundings of at most half a step of a value no larger than
    # the row's largest rotated pair, sqrt(2) amax)
    amax = np.abs(k16).max(-1, keepdims=True)
    slack = 7 * torch.finfo(dt).eps / 2 * 1.5 * amax + 1e-5 * amax
    half = np.maximum(2.0 ** -4 * (np.abs(k16) + slack), 2.0 ** -10 * s[..., :1])
    assert (np.abs(k - k16) <= half * (1 + 2.0 ** -20) + slack).all()


def test_captured_decode_step_of_a_model():
    """A decode step captured once and replayed over changing lengths and places equals the eager
    one; the bound on lengths is the table's."""
    from tokenfactory_b200 import ForwardBatch
    from tokenfactory_b200.hybrid_model import HybridCachePool
    from tokenfactory_b200.runner import CapturedStep
    cfg, model = _model(128, 8, 2, torch.bfloat16)
    g = torch.Generator().manual_seed(5)
    n, width = 3, 96
    r2t = torch.randperm(n * width, generator=g).view(n, width).cuda()
    rows = torch.arange(n, device="cuda")
    ones = torch.ones(n, dtype=torch.long, device="cuda")

    def step(pool):
        def fn(ids, lens, loc):
            fb = ForwardBatch(batch_size=n, req_pool_indices=rows, seq_lens=lens,
                              prefix_lens=lens - 1, extend_lens=[1] * n, out_cache_loc=loc,
                              req_to_token=r2t, is_prefill=False, max_seq_len=width,
                              max_extend_len=1, extend_lens_tensor=ones,
                              req_pool_indices_list=list(range(n)))
            return model(ids, lens - 1, pool, fb)
        return fn

    pools = [HybridCachePool(cfg, n * width, n, kv_dtype=torch.float8_e4m3fn) for _ in range(2)]
    start = [40, 1, 17]
    ids = torch.randint(0, cfg.vocab_size, (sum(start),), generator=g)
    for p in pools:
        _step(model, p, r2t, [0, 1, 2], [0, 0, 0], start, ids)

    def inputs(i):
        lens = torch.tensor([s + 1 + i for s in start], device="cuda")
        gi = torch.Generator().manual_seed(i)
        return dict(ids=torch.randint(0, cfg.vocab_size, (n,), generator=gi).cuda(), lens=lens,
                    loc=r2t[rows, lens - 1])

    cap = CapturedStep(step(pools[0]), inputs(0),
                       state=[v for v in vars(pools[0]).values() if torch.is_tensor(v)])
    eager = step(pools[1])
    for i in range(6):
        a, b = cap(**inputs(i)).clone(), eager(**inputs(i))
        assert torch.equal(a, b), i
    assert torch.equal(pools[0].k_buffer.view(torch.uint8), pools[1].k_buffer.view(torch.uint8))
    assert torch.equal(pools[0].kv_scale, pools[1].kv_scale)


def test_slot_based_attention_of_an_8_bit_pool():
    from tests.fp8_pool import Case
    from tokenfactory_b200 import ForwardBatch
    from tokenfactory_b200.hybrid_attention import slot_based_attention
    for pre, ext in (([30, 4], [20, 1]), ([50, 0], [1, 1]), ([8], [1])):
        c = Case(21, "bf16", 8, 2, 128, pre, ext)
        r2t, rows, seq = c.args()
        fb = ForwardBatch(batch_size=len(ext), req_pool_indices=rows, seq_lens=seq,
                          prefix_lens=torch.tensor(pre, device="cuda"), extend_lens=list(ext),
                          out_cache_loc=seq[:0], req_to_token=r2t, is_prefill=max(ext) > 1)
        kb, vb, sc = c.pool()
        got = slot_based_attention(c.q.cuda(), kb, vb, fb, 128 ** -0.5, sc)
        check(got, c.reference("wrap" if len(ext) == 1 else "clamp"), "bf16", 128)
