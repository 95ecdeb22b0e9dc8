"""8-bit attention: entries of the tables that are negative, outside the pool or shared between requests, through
every kernel."""

import pytest

from tests import kv_fp8_bounds as B
from tests.fp8_pool import Case

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

# name: (dtype, hq, hkv, d, prefixes, new tokens)
SHAPES = {
    "decode": ("bf16", 8, 2, 128, [300, 40], [1, 1]),
    "drafts": ("f16", 8, 2, 256, [300, 40], [3, 5]),
    "tile": ("bf16", 8, 2, 256, [30, 0], [70, 129]),
    "tile_f16": ("f16", 8, 2, 64, [30, 0], [70, 129]),
    "tile_split": ("bf16", 8, 1, 256, [3000, 1], [70, 20]),
    "cuda_cores": ("bf16", 8, 2, 80, [30, 0], [7, 50]),
}


def _case(name):
    dtype, hq, hkv, d, pre, ext = SHAPES[name]
    c = Case(80, dtype, hq, hkv, d, pre, ext)
    extend = any(e > 1 for e in ext)
    return c, extend, B.kernel_of(c, extend)


@pytest.mark.parametrize("mode", ["clamp", "wrap"])
@pytest.mark.parametrize("name", list(SHAPES))
def test_negative_entries(name, mode):
    c, extend, kernel = _case(name)
    for r, n in enumerate(c.seq):
        c.r2t[c.rows[r], [0, n // 2, n - 1]] = torch.tensor([-1, -3, -len(c.codes)])
    B.check(c.run(force_extend=extend, slot_mode=mode), B.reference(c, kernel, mode), name)


@pytest.mark.parametrize("name", list(SHAPES))
def test_entries_outside_the_pool_are_recorded_and_read_as_slot_0(name):
    from tokenfactory_b200 import _capi
    c, extend, kernel = _case(name)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    row = c.r2t[c.rows[1]]
    row[3], row[c.seq[1] - 1] = len(c.codes), 1 << 40
    got = c.run(force_extend=extend, err=err)
    assert err.item() == _capi.TF_KERR_SLOT_RANGE
    row[3], row[c.seq[1] - 1] = 0, 0
    B.check(got, B.reference(c, kernel), name)


@pytest.mark.parametrize("bad", [-1, 1 << 33])
@pytest.mark.parametrize("name", list(SHAPES))
def test_requests_outside_the_table_are_recorded(name, bad):
    from tokenfactory_b200 import _capi
    c, extend, kernel = _case(name)
    c.r2t[0] = torch.where(c.r2t[0] < 0, 0, c.r2t[0])  # what such a request reads
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    rows = c.rows.clone()
    c.rows = rows.clone()
    c.rows[0] = bad
    got = c.run(force_extend=extend, err=err)
    assert err.item() == _capi.TF_KERR_REQ_RANGE
    c.rows[0] = 0
    B.check(got, B.reference(c, kernel), name)


@pytest.mark.parametrize("name", list(SHAPES))
def test_shared_slots_and_rows(name):
    """Two requests on one table row, whose tokens lie partly in the same slots."""
    c, extend, kernel = _case(name)
    long = int(max(range(2), key=lambda r: c.seq[r]))
    c.rows = c.rows[[long, long]]
    row = c.r2t[c.rows[0]]
    n = max(c.seq)
    row[n // 2:n // 2 + 9] = row[:9].clone()
    B.check(c.run(force_extend=extend), B.reference(c, kernel), name)
