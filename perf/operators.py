"""Timed cases of the operators on a K/V pool held in 8 bits.

The pool keeps every K and V row (one slot, one kv head, head_dim values) as e4m3 codes with one
float32 scale, so a row stands for ``codes * scale``.  Four operators work on it:

* ``kv_store``:  x -> codes = e4m3(x * (448 / amax)), scale = amax / 448 with
  amax = max(max |x|, 1e-12) of the row, written at each token's slot;
* ``prologue``:  q and k RMSNorm, rotation of the first rotary_dim values, then kv_store of the
  rotated k and of v; returns the rotated q;
* ``decode``:    softmax(q K^T scale) V of one query token per request over its seq_len tokens,
  read through req_to_token, times the output gate's activation;
* ``extend``:    the same for extend_len new tokens per request, causal over prefix + extend.

``own`` selects the framework's kernels; otherwise ``run`` computes the plain form in 32 bits.
"""

import math

import torch

own = False

FP8 = torch.float8_e4m3fn
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-6
THETA = 1e7

# heads (query, kv) and head sizes of the repository's full-attention layers: the 27B shape, the
# module default, their shards on 2 and 4 ranks, the small test model, and plain multi-head
HEADS = [(32, 4), (24, 4), (16, 2), (8, 1), (8, 2), (4, 4)]


def _case(name, op, dtype="bf16", hq=32, hkv=4, d=256, **kw):
    return dict(name=name, op=op, dtype=dtype, hq=hq, hkv=hkv, d=d, **kw)


def listed():
    return [
        # one decode step of 48 running requests writes one token each
        _case("store_step_48", "store", tokens=48, slots=8192),
        # a prefill batch of about 20K new tokens
        _case("store_prefill_20011", "store", tokens=20011, slots=65536),
        # the attention prologue of a decode step, 128 requests at far positions
        _case("prologue_step_128", "prologue", tokens=128, slots=8192, pos=8192),
        # the prologue of a prefill batch, ragged
        _case("prologue_prefill_7001", "prologue", dtype="f16", hq=24, tokens=7001, slots=16384,
              pos=32768),
        # the small fp32 model: four requests, prompts of 16 to 64 tokens, 32 decode steps
        _case("decode_small_f32", "decode", dtype="f32", hq=8, hkv=2, d=64, batch=4, lo=17, hi=96,
              gate="sigmoid"),
        # a single user's decode step over one long context: latency
        _case("decode_one_8191", "decode", batch=1, lo=8191, hi=8191, gate="sigmoid"),
        # a few ragged requests, down to a context of one token, on one of two ranks
        _case("decode_ragged_13", "decode", dtype="f16", hq=16, hkv=2, d=128, batch=13, lo=1,
              hi=3001, gate="none"),
        # a full serving batch: 128 requests of 512 to 8192 tokens
        _case("decode_batch_128", "decode", batch=128, lo=512, hi=8192, gate="sigmoid"),
        # scoring a few drafted tokens per request over long contexts
        _case("extend_drafts_24", "extend", batch=24, lo=300, hi=6000, elo=2, ehi=5,
              gate="sigmoid"),
        # a small ragged prefill of the two-kv-head model
        _case("extend_small_f16", "extend", dtype="f16", hq=8, hkv=2, d=128, batch=3, lo=0, hi=77,
              elo=1, ehi=333, gate="none"),
        # one chunk of a long prompt
        _case("extend_chunk_512", "extend", batch=1, lo=28000, hi=28000, elo=512, ehi=512,
              gate="sigmoid"),
        # prefill over cached prefixes of up to 4096 tokens, 512 to 2048 new ones
        _case("extend_prefix_4", "extend", batch=4, lo=0, hi=4096, elo=512, ehi=2048,
              gate="sigmoid"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["store", "prologue", "decode", "decode", "extend", "extend"])
    hq, hkv = rng.choice(HEADS)
    c = dict(op=op, dtype=rng.choice(["bf16", "bf16", "f16"]), hq=hq, hkv=hkv,
             d=rng.choice([64, 128, 256, 256]))
    if op in ("store", "prologue"):
        c["tokens"] = _log(rng, 1, 20011 if op == "store" else 7001)
        c["slots"] = c["tokens"] + _log(rng, 64, 16384)
        if op == "prologue":
            c["pos"] = c["tokens"] + _log(rng, 64, 65536)
        return c
    c["gate"] = rng.choice(["none", "silu", "sigmoid"])
    if op == "decode":
        c["batch"] = _log(rng, 1, 160)
        c["lo"] = _log(rng, 1, 2000)
        c["hi"] = c["lo"] + _log(rng, 1, min(30000, 900000 // c["batch"] + 1))
        while c["batch"] * (c["lo"] + c["hi"]) > 1100000:
            c["batch"] = (c["batch"] + 1) // 2
        return c
    c["batch"] = _log(rng, 1, 16)
    c["elo"] = _log(rng, 1, 700)
    c["ehi"] = c["elo"] + _log(rng, 1, 1300)
    if rng.random() < 0.4:  # a few tokens per request
        c["elo"], c["ehi"] = 1, rng.randint(1, 12)
    c["lo"] = rng.choice([0, 0, _log(rng, 1, 2000)])
    c["hi"] = c["lo"] + _log(rng, 1, 12000)
    while _pairs(c) * hq * c["d"] > 8e10:  # at most about the largest listed case
        c["batch"] = (c["batch"] + 1) // 2
        c["hi"] = (c["lo"] + c["hi"]) // 2
        c["ehi"] = (c["elo"] + c["ehi"]) // 2
    return c


def _spread(lo, hi, n, phase):
    """n lengths spread evenly over [lo, hi] in a fixed shuffled order."""
    if n == 1:
        return [hi]
    order = sorted(range(n), key=lambda i: math.modf(i * 0.6180339887 + phase)[0])
    return [lo + (hi - lo) * r // (n - 1) for r in sorted(range(n), key=lambda i: order[i])]


def _lengths(case):
    """(prefix lengths, new-token lengths) of the case's requests."""
    n = case["batch"]
    if case["op"] == "decode":
        return [x - 1 for x in _spread(case["lo"], case["hi"], n, 0.3)], [1] * n
    return _spread(case["lo"], case["hi"], n, 0.3), _spread(case["elo"], case["ehi"], n, 0.7)


def _pairs(case):
    """visible (query, key) pairs of one query head"""
    return sum(e * p + e * (e + 1) // 2 for p, e in zip(*_lengths(case)))


def work(case):
    hq, hkv, d, eb = case["hq"], case["hkv"], case["d"], BYTES[case["dtype"]]
    if case["op"] in ("store", "prologue"):
        t = case["tokens"]
        b = t * (hkv * 2 * (d * eb + d + 4) + 8)
        f = t * hkv * d * 4
        if case["op"] == "prologue":
            b += t * (2 * hq * d * eb + 8)
            f += t * (hq + hkv) * d * 6
        return {"bytes": b, "flops": f}
    pre, ext = _lengths(case)
    t, total = sum(ext), sum(pre) + sum(ext)
    rows = 3 if case["gate"] != "none" else 2
    return {"bytes": total * (hkv * (2 * d + 8) + 8) + rows * t * hq * d * eb,
            "flops": 4 * hq * d * _pairs(case)}


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _pool(case, slots, g):
    """The pool as a serving process allocates it: codes [slots, Hkv, 2, D] with the K and the V
    row of a head next to each other, scales [slots, Hkv, 2].  Rows are those of normal values whose
    size differs from token to token and head to head."""
    hkv, d = case["hkv"], case["d"]
    codes = torch.empty((slots, hkv, 2, d), dtype=FP8, device="cuda")
    scale = torch.empty((slots, hkv, 2), dtype=torch.float32, device="cuda")
    for s in range(0, slots, 1 << 16):
        n = min(1 << 16, slots - s)
        x = torch.randn((n, hkv, 2, d), generator=g, device="cuda")
        x *= torch.exp(0.3 * torch.randn((n, hkv, 2, 1), generator=g, device="cuda"))
        amax = x.abs().amax(-1, keepdim=True)
        scale[s:s + n] = amax.squeeze(-1) / 448
        codes[s:s + n] = (x * (448 / amax)).clamp(-448, 448).to(FP8)
    return codes, scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(dt)

    st = dict(op=case["op"], scaling=d ** -0.5)
    if case["op"] in ("store", "prologue"):
        t, slots = case["tokens"], case["slots"]
        codes, st["kv_scale"] = _pool(case, slots, g)
        st["k_buffer"], st["v_buffer"] = codes[:, :, 0], codes[:, :, 1]
        st["loc"] = torch.randperm(slots, generator=g, device="cuda")[:t]
        st["k"], st["v"] = normal(t, hkv, d), normal(t, hkv, d)
        if case["op"] == "prologue":
            rot = d // 4
            st["q"] = normal(t, hq, 2 * d)[..., :d]  # the q half of the fused q/gate projection
            st["wq"] = (1 + 0.1 * normal(d).float()).to(dt)
            st["wk"] = (1 + 0.1 * normal(d).float()).to(dt)
            first = int(torch.randint(0, case["pos"] - t + 1, (1,), generator=g, device="cuda"))
            st["positions"] = torch.arange(first, first + t, device="cuda")
            st["inv_freq"] = (1.0 / THETA ** (torch.arange(0, rot, 2, dtype=torch.float32)
                                              / rot)).cuda()
        return st
    pre, ext = _lengths(case)
    n, seq = len(pre), [p + e for p, e in zip(pre, ext)]
    total, t = sum(seq), sum(ext)
    slots = total + total // 4 + 16
    codes, st["kv_scale"] = _pool(case, slots, g)
    st["k_buffer"], st["v_buffer"] = codes[:, :, 0], codes[:, :, 1]
    perm = torch.randperm(slots, generator=g, device="cuda")[:total]
    r2t = torch.full((n + 3, max(seq) + 8), -1, dtype=torch.int64, device="cuda")
    rows = torch.randperm(n + 3, generator=g, device="cuda")[:n]
    at = 0
    for r, s in zip(rows.tolist(), seq):
        r2t[r, :s] = perm[at:at + s]
        at += s
    st["req_to_token"], st["rows"] = r2t, rows
    st["seq_lens"] = torch.tensor(seq, device="cuda")
    st["extend_lens"] = torch.tensor(ext, device="cuda")
    st["max_seq"], st["max_ext"], st["tokens"] = max(seq), max(ext), t
    st["q"] = normal(t, hq, d)
    st["gate_mode"] = case["gate"]
    # the gate is the second half of the fused q/gate projection: a strided view
    st["gate"] = normal(t, hq, 2 * d)[..., d:] if case["gate"] != "none" else None
    return st


# ------------------------------------------------------------------------------------------------
# the plain forms, in 32 bits
# ------------------------------------------------------------------------------------------------
def _quantize_rows(x):
    amax = x.abs().amax(-1, keepdim=True).clamp(min=1e-12)
    return (x * (448 / amax)).clamp(-448, 448).to(FP8), (amax / 448).squeeze(-1)


def _store(st, k, v):
    kc, ks = _quantize_rows(k)
    vc, vs = _quantize_rows(v)
    st["k_buffer"].view(torch.uint8)[st["loc"]] = kc.view(torch.uint8)
    st["v_buffer"].view(torch.uint8)[st["loc"]] = vc.view(torch.uint8)
    st["kv_scale"][st["loc"]] = torch.stack((ks, vs), dim=-1)


def _norm_rotate(x, w, positions, inv_freq):
    x = x.float()
    y = w.float() * (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS))
    ang = positions.double()[:, None] * inv_freq.double()
    c, s = ang.cos().float()[:, None], ang.sin().float()[:, None]
    h = inv_freq.numel()
    a, b = y[..., :h], y[..., h:2 * h]
    return torch.cat((a * c - b * s, b * c + a * s, y[..., 2 * h:]), dim=-1)


def _rows(buf, scale, slots):
    """float32 rows [..., Hkv, D] of the slots"""
    return buf.view(torch.uint8)[slots].view(FP8).float() * scale[slots].unsqueeze(-1)


def _attend(st):
    q, ext, seq = st["q"], st["extend_lens"], st["seq_lens"]
    n, e, l = ext.numel(), st["max_ext"], st["max_seq"]
    t, hq, d = q.shape
    hkv = st["k_buffer"].shape[1]
    g = hq // hkv
    dev = q.device
    slots = st["req_to_token"][st["rows"]][:, :l].clamp(min=0)
    start = ext.cumsum(0) - ext
    i = torch.arange(e, device=dev)
    tok = (start[:, None] + i).clamp(max=t - 1)                      # [n, e]
    rows = q[tok].float().reshape(n, e, hkv, g, d).permute(0, 2, 1, 3, 4).reshape(n, hkv, e * g, d)
    s = torch.matmul(rows, _rows(st["k_buffer"], st["kv_scale"][..., 0], slots).permute(0, 2, 3, 1))
    s.mul_(st["scaling"])
    seen = torch.arange(l, device=dev) <= (seq - ext)[:, None, None] + i[:, None]  # [n, e, l]
    s = s.view(n, hkv, e, g, l).masked_fill_(~seen[:, None, :, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    s.div_(s.sum(-1, keepdim=True))
    o = torch.matmul(s.view(n, hkv, e * g, l),
                     _rows(st["v_buffer"], st["kv_scale"][..., 1], slots).permute(0, 2, 1, 3))
    o = o.view(n, hkv, e, g, d).permute(0, 2, 1, 3, 4).reshape(n, e, hq, d)
    of = torch.repeat_interleave(torch.arange(n, device=dev), ext, output_size=t)
    o = o[of, torch.arange(t, device=dev) - start[of]]
    if st["gate"] is not None:
        x = st["gate"].float()
        sg = 1 / (1 + torch.exp(-x))
        o = o * (x * sg if st["gate_mode"] == "silu" else sg)
    return o.to(q.dtype)


def run(st):
    if own:
        return _run_own(st)
    if st["op"] == "store":
        _store(st, st["k"].float(), st["v"].float())
        return st["k_buffer"], st["v_buffer"], st["kv_scale"]
    if st["op"] == "prologue":
        q = _norm_rotate(st["q"], st["wq"], st["positions"], st["inv_freq"]).to(st["q"].dtype)
        k = _norm_rotate(st["k"], st["wk"], st["positions"], st["inv_freq"])
        _store(st, k, st["v"].float())
        return q, st["k_buffer"], st["v_buffer"], st["kv_scale"]
    return _attend(st)


# ------------------------------------------------------------------------------------------------
# the framework's kernels
# ------------------------------------------------------------------------------------------------
def _run_own(st):
    from tokenfactory_b200 import ops
    pool = st["k_buffer"], st["v_buffer"], st["kv_scale"]
    if st["op"] == "store":
        ops.kv_store_fp8(*pool, st["loc"], st["k"], st["v"])
        return pool
    if st["op"] == "prologue":
        q = ops.attn_prologue_fp8(st["q"], st["k"], st["v"], st["wq"], st["wk"], st["positions"],
                                  st["inv_freq"], *pool, st["loc"], eps=EPS)
        return (q, *pool)
    if st["op"] == "decode":
        return ops.paged_decode_fp8(st["q"], *pool, st["req_to_token"], st["rows"],
                                    st["seq_lens"], st["scaling"], st["max_seq"],
                                    gate=st["gate"], gate_mode=st["gate_mode"])
    return ops.paged_extend_fp8(st["q"], *pool, st["req_to_token"], st["rows"], st["seq_lens"],
                                st["extend_lens"], st["scaling"], st["max_seq"], st["max_ext"],
                                gate=st["gate"], gate_mode=st["gate_mode"])


# ------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def _e4m3_64(x):
    """float64 values rounded to the nearest e4m3 value (ties to even), saturated at 448"""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _store_64(st, k, v):
    out = []
    scales = st["kv_scale"].double()
    for j, (buf, x) in enumerate(((st["k_buffer"], k), (st["v_buffer"], v))):
        amax = x.abs().amax(-1).clamp(min=1e-12)
        codes = buf.double()
        codes[st["loc"]] = _e4m3_64(x * (448 / amax)[..., None])
        scales[st["loc"], :, j] = amax / 448
        out.append(codes)
    return out[0], out[1], scales


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "store":
        return _store_64(st, st["k"].double(), st["v"].double())
    if case["op"] == "prologue":
        ang = st["positions"].double().outer(st["inv_freq"].double())
        turn = torch.polar(torch.ones_like(ang), ang)[:, None]
        done = []
        for x, w in ((st["q"], st["wq"]), (st["k"], st["wk"])):
            y = x.double()
            y = w.double() * y / (y.square().mean(-1, keepdim=True) + EPS).sqrt()
            h = ang.shape[1]
            z = torch.complex(y[..., :h], y[..., h:2 * h]) * turn
            done.append(torch.cat((z.real, z.imag, y[..., 2 * h:]), dim=-1))
        return (done[0], *_store_64(st, done[1], st["v"].double()))
    hq, hkv = case["hq"], case["hkv"]
    out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for r, p, e in zip(st["rows"].tolist(), *_lengths(case)):
        slots = st["req_to_token"][r, :p + e]
        for h in range(hkv):
            sc = st["kv_scale"][slots, h].double()
            k = st["k_buffer"][:, h].view(torch.uint8)[slots].view(FP8).double() * sc[:, :1]
            v = st["v_buffer"][:, h].view(torch.uint8)[slots].view(FP8).double() * sc[:, 1:]
            for a in range(0, e, 256):
                m = min(256, e - a)
                heads = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
                s = torch.einsum("igd,jd->igj", st["q"][at + a:at + a + m, heads].double(), k)
                late = (torch.arange(p + e, device="cuda")[None]
                        > p + a + torch.arange(m, device="cuda")[:, None])
                w = torch.softmax((s * st["scaling"]).masked_fill(late[:, None], -math.inf), -1)
                out[at + a:at + a + m, heads] = torch.einsum("igj,jd->igd", w, v)
        at += e
    if st["gate"] is not None:
        x = st["gate"].double()
        out *= torch.sigmoid(x) * (x if case["gate"] == "silu" else 1)
    return out
