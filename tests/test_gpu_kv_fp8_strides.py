"""8-bit attention with query, gate and output rows at odd places, through every kernel."""

import pytest

from tests import kv_fp8_bounds as B
from tests.fp8_pool import Case

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

# name: (dtype, hq, hkv, d, prefixes, new tokens)
SHAPES = {
    "decode": ("bf16", 8, 2, 128, [300, 40], [1, 1]),
    "decode_f16": ("f16", 8, 1, 256, [2000], [1]),
    "drafts": ("bf16", 8, 2, 256, [300, 40], [3, 5]),
    "tile": ("bf16", 8, 2, 256, [30, 0], [70, 129]),
    "tile_f16": ("f16", 8, 2, 128, [30, 0], [70, 129]),
    "tile_d64": ("bf16", 6, 2, 64, [30, 0], [70, 129]),
    "tile_split": ("bf16", 8, 1, 256, [3000, 1], [70, 20]),
    "cuda_cores": ("bf16", 8, 2, 80, [30, 0], [7, 50]),
}


@pytest.mark.parametrize("odd", ["q", "gate", "out", "all", "none"])
@pytest.mark.parametrize("gate", ["none", "sigmoid", "silu"])
@pytest.mark.parametrize("name", list(SHAPES))
def test_rows_at_odd_places(name, gate, odd):
    """q, gate or out with rows that start two bytes off and strides that are no multiple of 16 bytes; the
    output's surroundings stay as they were."""
    from tokenfactory_b200 import ops
    dtype, hq, hkv, d, pre, ext = SHAPES[name]
    c = Case(70, dtype, hq, hkv, d, pre, ext, gate=gate)
    t = len(c.q)

    def place(x, off):
        wide = torch.full((t, hq + 1, d + 13), 9.0, dtype=c.q.dtype, device="cuda")
        view = wide[:, 1:, off:off + d] if off else torch.full_like(x, 9.0, device="cuda")
        view.copy_(x)
        return wide, view

    _, q = place(c.q, 3 if odd in ("q", "all") else 0)
    _, g = place(c.gate.contiguous(), 5 if odd in ("gate", "all") else 0)
    out = torch.zeros_like(c.q)
    around, out = place(out, 1 if odd in ("out", "all") else 0)
    kw = dict(out=out, gate=None if gate == "none" else g, gate_mode=gate)
    sm, extend = d ** -0.5, any(e > 1 for e in ext)
    if extend:
        got = ops.paged_extend_fp8(q, *c.pool(), *c.args(), torch.tensor(ext, device="cuda"), sm,
                                   max(c.seq), max(ext), **kw)
    else:
        got = ops.paged_decode_fp8(q, *c.pool(), *c.args(), sm, max(c.seq), **kw)
    assert got.data_ptr() == out.data_ptr()
    B.check(got, B.reference(c, B.kernel_of(c, extend)), name)
    if odd in ("out", "all"):
        assert (around[:, 0] == 9).all() and (around[:, :, 0] == 9).all()
        assert (around[:, :, d + 1:] == 9).all()
