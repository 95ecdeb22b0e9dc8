"""8-bit attention against the derived bound where every key counts: none is lost at the end of a tile, of a
CTA's share or of a split."""

import pytest

from tests import kv_fp8_bounds as B
from tests import kv_fp8_keys as K

pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("alike", [True, False])
@pytest.mark.parametrize("extend,name", [(False, n) for n in K.DECODE] + [(True, n) for n in K.EXTEND])
def test_every_key(extend, name, alike):
    c, kernel = K.case(name, extend, alike)
    B.check(c.run(force_extend=extend), B.reference(c, kernel), name)
