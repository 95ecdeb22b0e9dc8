"""The K/V pool held in 8 bits, in float64 numpy: quantization of rows to e4m3 codes and a scale, the
prologue over it and attention over it (formulas in include/tfattn.h; the reference has no such
pool).  The oracle of the tf_*_fp8 entry points; the product path never touches it."""

import numpy as np

E4M3_MAX = 448.0
MIN_AMAX = 1e-12


def round_e4m3(x: np.ndarray) -> np.ndarray:
    """Nearest e4m3 value, ties to even, saturated at 448."""
    x = np.asarray(x, np.float64)
    step = np.exp2(np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -6))) - 3)
    return np.clip(np.round(x / step) * step, -E4M3_MAX, E4M3_MAX)


def quantize_rows(x: np.ndarray):
    """(code values float64, scale float32) of the rows of x (last axis), with the fp32 operations
    of the definition: amax = max(max |x|, 1e-12), code = e4m3(x * (448 / amax)), scale =
    amax / 448; a row that is not finite gets codes 0 and scale NaN."""
    x = np.asarray(x, np.float32)
    finite = np.isfinite(x).all(-1)
    amax = np.maximum(np.abs(np.where(finite[..., None], x, 0)).max(-1), np.float32(MIN_AMAX))
    amax = amax.astype(np.float32)
    mul = (np.float32(E4M3_MAX) / amax).astype(np.float32)
    codes = round_e4m3(np.where(finite[..., None], x, 0) * mul[..., None])
    scale = np.where(finite, amax / np.float32(E4M3_MAX), np.float32(np.nan)).astype(np.float32)
    return codes, scale


def norm_rotate(x, w, positions, inv_freq, eps, mrope_section=(11, 11, 10), interleaved=True):
    """RMSNorm then rotation of the first 2 * len(inv_freq) values (rotate_half convention), in
    float64; positions [T] or [3, T]."""
    x = np.asarray(x, np.float64)
    y = np.asarray(w, np.float64) * x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    h = len(inv_freq)
    j = np.arange(h)
    pos = np.asarray(positions)
    if pos.ndim == 1:
        p = np.repeat(pos[:, None], h, 1)
    else:
        if interleaved:
            row = np.where((j % 3 == 1) & (j < 3 * mrope_section[1]), 1,
                           np.where((j % 3 == 2) & (j < 3 * mrope_section[2]), 2, 0))
        else:
            row = np.repeat([0, 1, 2], mrope_section)
        p = pos[row].T
    ang = p.astype(np.float64) * np.asarray(inv_freq, np.float64)
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    a, b = y[..., :h], y[..., h:2 * h]
    return np.concatenate([a * c - b * s, b * c + a * s, y[..., 2 * h:]], -1)


def attention(q, k_rows, v_rows, req_to_token, req_pool_indices, seq_lens, extend_lens, scale,
              gate=None, gate_mode="none", slot_mode="clamp", v_scale=None):
    """(out, magnitude, score magnitude, step magnitude) [T, Hq, D] float64 of paged attention over
    dequantized pool rows k_rows / v_rows [slots, Hkv, D].  magnitude is the same sum with |v| and
    |act(gate)|: what a relative error of the weights is multiplied by; score magnitude is the row's
    largest scale * sum_d |q_d k_d|: what a relative error of the products adds to a score; step
    magnitude, with v_scale [slots, Hkv] given, is max_j p_j * max_j v_scale_j * sum_j |v code_j|
    |act(gate)|: what an error of each weight * scale relative to the largest possible one is
    multiplied by.  Requests without keys give NaN."""
    q = np.asarray(q, np.float64)
    smag, step = np.zeros(q.shape), np.zeros(q.shape)
    hkv = k_rows.shape[1]
    g = q.shape[1] // hkv
    out, mag = np.full(q.shape, np.nan), np.full(q.shape, np.nan)
    t = 0
    for r, n, e in zip(req_pool_indices, seq_lens, extend_lens):
        s = req_to_token[r, :n]
        s = np.where(s < 0, s + len(k_rows) if slot_mode == "wrap" else 0, s)
        for i in range(e):
            m = n - e + i + 1
            if m > 0:
                k, v = k_rows[s[:m]], v_rows[s[:m]]
                for h in range(hkv):
                    hs = slice(h * g, (h + 1) * g)
                    smag[t, hs] = (np.abs(q[t, hs]) @ np.abs(k[:, h]).T).max(-1)[:, None] * scale
                    x = q[t, hs] @ k[:, h].T * scale
                    x = np.exp(x - x.max(-1, keepdims=True))
                    x /= x.sum(-1, keepdims=True)
                    out[t, hs], mag[t, hs] = x @ v[:, h], x @ np.abs(v[:, h])
                    if v_scale is not None:
                        vs = np.abs(v_scale[s[:m], h])
                        ok = np.isfinite(vs) & (vs > 0)
                        codes = (np.abs(v[ok, h]) / vs[ok, None]).sum(0)
                        step[t, hs] = x.max(-1)[:, None] * vs[ok].max(initial=0) * codes
            t += 1
    if gate_mode != "none":
        x = np.asarray(gate, np.float64)
        act = 1 / (1 + np.exp(-x)) * (x if gate_mode == "silu" else 1)
        out, mag, step = out * act, mag * np.abs(act), step * np.abs(act)
    return out, mag, smag, step
