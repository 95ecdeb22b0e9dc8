"""The 8-bit pool's prologue: cosines and sines of far positions, element by element."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,rot", [(256, 64), (128, 32), (64, 64), (256, 96)])
@pytest.mark.parametrize("t", [64, 1200])
def test_rotation_by_angles_of_far_positions(d, rot, t):
    """Rows with one value whose norm is exactly 1 come out as the angle's cosine and sine.  sincosf is off by
    at most 2 units (2^-23 of the value each); the angle, positions times frequencies below 2^17 in fp64, by
    2^-36, and one product and one sum more round in fp32 (2^-24 each, of at most the value)."""
    from tokenfactory_b200 import ops
    h = rot // 2
    g = torch.Generator().manual_seed(d + t)
    pos = torch.randint(0, 1 << 17, (t,), generator=g)
    inv = 1.0 / 1e7 ** (torch.arange(0, rot, 2, dtype=torch.float32) / rot)
    q = torch.zeros((t, h, d))
    q[:, torch.arange(h), torch.arange(h)] = 1  # head j: 1 at dim j
    w = torch.full((d,), 1.0)
    pool = torch.zeros((t, 1, 2, d), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    sc = torch.zeros((t, 1, 2), device="cuda")
    kv = torch.zeros((t, 1, d), device="cuda")
    # eps 1 - 1/d: the mean square 1/d of a row plus eps is 1 to 2^-24
    got = ops.attn_prologue_fp8(q.cuda(), kv, kv, w.cuda(), w.cuda(), pos.cuda(), inv.cuda(),
                                pool[:, :, 0], pool[:, :, 1], sc, torch.arange(t, device="cuda"),
                                eps=1 - 1 / d).double().cpu().numpy()
    ang = pos.numpy()[:, None].astype(np.float64) * inv.numpy().astype(np.float64)
    j = np.arange(h)
    for value, want in ((got[:, j, j], np.cos(ang)), (got[:, j, j + h], np.sin(ang))):
        tol = (2 * 2.0 ** -23 + 4 * 2.0 ** -24) * np.abs(want) + 2.0 ** -35
        bad = np.abs(value - want) > tol
        assert not bad.any(), (bad.sum(), (np.abs(value - want) / tol).max())
