"""The bound of the 8-bit attention tests, without a GPU: no result that lacks keys is inside it, and its
values are the oracle's."""

import numpy as np
import pytest

from tests import kv_fp8_bounds as B
from tests import kv_fp8_keys as K


@pytest.mark.parametrize("extend,name", [(False, n) for n in K.DECODE] + [(True, n) for n in K.EXTEND])
def test_missing_keys_are_seen(extend, name):
    c, kernel = K.case(name, extend, alike=True)
    for r in range(len(c.seq)):
        if c.ext[r] == 0:
            continue
        missing = B.unseen(c, kernel, r, K.parts(c, r, True))
        assert not missing, f"request {r} of {c.seq[r]} keys: {missing[:5]} would not be missed"


@pytest.mark.parametrize("extend,name", [(False, "ragged"), (False, "cuda_cores"), (True, "drafts"),
                                         (True, "edges_f16"), (True, "edges"), (False, "ragged_f16")])
def test_reference_is_the_oracle(extend, name):
    from oracle import kv_fp8 as O
    c, kernel = K.case(name, extend, alike=False)
    out, _ = B.reference(c, kernel)
    rows = c.codes.float().double().numpy() * c.scale.double().numpy()[..., None]
    want = O.attention(c.q.double().numpy(), rows[:, :, 0], rows[:, :, 1], c.r2t.numpy(),
                       c.rows.tolist(), c.seq, c.ext, c.d ** -0.5)[0]
    np.testing.assert_allclose(out, want, rtol=1e-9, atol=1e-12)
