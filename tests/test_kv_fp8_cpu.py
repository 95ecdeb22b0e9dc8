"""The 8-bit K/V pool without a GPU: the oracle's rounding against torch's conversion, the argument
checks of the C entry points and of their torch front end."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import fp8 as OF
from oracle import kv_fp8 as O


def test_oracle_rounds_like_torch():
    rng = np.random.default_rng(3)
    x = np.concatenate([rng.normal(0, s, 5000) for s in (1e-3, 0.05, 1, 30, 200)]
                       + [np.arange(-480, 481) / 64.0, [0.0, 448.0, 460.0, -448.0, 2.0 ** -10]])
    x = x.astype(np.float32)
    want = torch.from_numpy(np.clip(x, -448, 448)).to(torch.float8_e4m3fn).float().numpy()
    np.testing.assert_array_equal(O.round_e4m3(x), want)
    codes = np.array([b for b in range(256) if b & 0x7f != 0x7f], np.uint8)
    v = OF.e4m3_decode(codes)
    np.testing.assert_array_equal(O.round_e4m3(v), v)


def test_oracle_rows():
    x = np.zeros((5, 8), np.float32)
    x[1] = np.linspace(-3, 2, 8)
    x[2, 3] = 1e-20
    x[3, 0], x[4, 1] = np.inf, np.nan
    codes, scale = O.quantize_rows(x)
    assert (codes[0] == 0).all() and scale[0] == np.float32(1e-12) / np.float32(448)
    assert np.abs(codes[1]).max() == 448
    assert (np.abs(codes[1] * scale[1] - x[1]) <= 2.0 ** -4 * np.abs(x[1]) + 1e-6).all()
    assert (codes[2:] == 0).all() and np.isnan(scale[3:]).all()


def test_oracle_attention_of_one_key_is_its_value():
    q = np.ones((1, 2, 4))
    k = v = np.arange(8.0).reshape(2, 1, 4)
    out, mag, _, _ = O.attention(q, k, v, np.array([[1]]), [0], [1], [1], 0.5)
    assert (out == v[1, 0]).all() and (mag == np.abs(v[1, 0])).all()


FAKE = 0x1000


def _paged(**kw):
    from tokenfactory_b200 import _capi
    base = dict(q=FAKE, k_buffer=FAKE, v_buffer=FAKE, req_to_token=FAKE, req_pool_indices=FAKE,
                seq_lens=FAKE, extend_lens=FAKE, out=FAKE, batch_size=2, num_tokens=2,
                num_q_heads=8, num_kv_heads=2, head_dim=64, num_slots=9, r2t_rows=2, r2t_cols=16,
                r2t_stride=16, max_seq_len=8, max_extend_len=1, dtype=1, scale=0.125)
    return _capi.PagedAttnArgs(**{**base, **kw})


def test_c_entry_points_check_before_any_cuda_call():
    from tokenfactory_b200 import _capi as C
    lib = C.load()
    good = C.KVScale(data=FAKE, stride_slot=4, stride_head=2)
    calls = [
        (lib.tf_paged_decode_fp8, _paged(), (None, 0, None)),
        (lib.tf_paged_extend_fp8, _paged(), (None, 0, None)),
        (lib.tf_kv_store_fp8,
         C.KVStoreArgs(k_buffer=FAKE, v_buffer=FAKE, num_slots=4, k=FAKE, v=FAKE,
                       out_cache_loc=FAKE, num_tokens=3, num_kv_heads=2, head_dim=64, dtype=1),
         (None,)),
        (lib.tf_attn_prologue_fp8,
         C.AttnPrologueArgs(q=FAKE, k=FAKE, v=FAKE, q_norm_weight=FAKE, k_norm_weight=FAKE,
                            positions=FAKE, inv_freq=FAKE, q_out=FAKE, k_buffer=FAKE,
                            v_buffer=FAKE, out_cache_loc=FAKE, num_slots=8, num_tokens=4,
                            num_q_heads=8, num_kv_heads=2, head_dim=256, rotary_dim=64, pos_rows=1,
                            dtype=1, norm_weight_dtype=1),
         (None,)),
    ]
    for fn, a, rest in calls:
        p = ctypes.byref(a)
        assert fn(None, ctypes.byref(good), *rest) == C.TF_ERR_INVALID_ARG
        assert fn(p, None, *rest) == C.TF_ERR_INVALID_ARG
        assert b"scales" in lib.tf_last_error()
        assert fn(p, ctypes.byref(C.KVScale(stride_slot=4)), *rest) == C.TF_ERR_INVALID_ARG
        for bad in (C.KVScale(data=FAKE + 4, stride_slot=4, stride_head=2),
                    C.KVScale(data=FAKE, stride_slot=3, stride_head=2),
                    C.KVScale(data=FAKE, stride_slot=4, stride_head=1)):
            assert fn(p, ctypes.byref(bad), *rest) == C.TF_ERR_ALIGNMENT
    s = ctypes.byref(good)
    for fn in (lib.tf_paged_decode_fp8, lib.tf_paged_extend_fp8):
        for kw, want in ((dict(q=None), C.TF_ERR_INVALID_ARG),
                         (dict(num_q_heads=7), C.TF_ERR_INVALID_ARG),
                         (dict(head_dim=257), C.TF_ERR_UNSUPPORTED),
                         (dict(dtype=5), C.TF_ERR_INVALID_ARG),
                         (dict(gate_mode=2), C.TF_ERR_INVALID_ARG),
                         (dict(slot_mode=7), C.TF_ERR_INVALID_ARG),
                         (dict(num_slots=0), C.TF_ERR_INVALID_ARG),
                         (dict(max_seq_len=17), C.TF_ERR_INVALID_ARG)):
            assert fn(ctypes.byref(_paged(**kw)), s, None, 0, None) == want, kw
        assert fn(ctypes.byref(_paged(batch_size=0, num_tokens=0)), s, None, 0, None) == C.TF_OK
    bad = calls[3][1]
    bad.rotary_dim = 63
    assert lib.tf_attn_prologue_fp8(ctypes.byref(bad), s, None) == C.TF_ERR_UNSUPPORTED
    bad.rotary_dim, bad.head_dim = 64, 96
    assert lib.tf_attn_prologue_fp8(ctypes.byref(bad), s, None) == C.TF_ERR_UNSUPPORTED


def test_ctypes_layout_of_the_scale_structure(tmp_path):
    import os
    import shutil
    import subprocess

    from tokenfactory_b200 import _capi
    from tests.test_capi_abi import HEADER
    if shutil.which("gcc") is None:
        pytest.skip("needs a host C compiler")
    c = tmp_path / "l.c"
    c.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "tfattn.h"\nint main(void){'
                 'printf("%zu %zu %zu %zu", sizeof(tf_kv_scale), offsetof(tf_kv_scale, data), '
                 'offsetof(tf_kv_scale, stride_slot), offsetof(tf_kv_scale, stride_head));return 0;}')
    subprocess.run(["gcc", "-I", os.path.dirname(HEADER), str(c), "-o", str(tmp_path / "l")],
                   check=True)
    out = subprocess.run([str(tmp_path / "l")], capture_output=True, text=True, check=True).stdout
    s = _capi.KVScale
    assert out.split() == [str(x) for x in (ctypes.sizeof(s), s.data.offset, s.stride_slot.offset,
                                            s.stride_head.offset)]


def test_cpu_tensors_are_refused():
    from tokenfactory_b200 import ops
    q = torch.zeros((2, 8, 64), dtype=torch.bfloat16)
    pool = torch.zeros((4, 2, 64), dtype=torch.uint8).view(torch.float8_e4m3fn)
    sc, i = torch.zeros(4, 2, 2), torch.zeros(2, dtype=torch.int64)
    k = torch.zeros((2, 2, 64), dtype=torch.bfloat16)
    w = torch.ones(64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv_store_fp8(pool, pool, sc, i, k, k)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_decode_fp8(q, pool, pool, sc, i.view(1, 2), i, i, 0.125, 1)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_extend_fp8(q, pool, pool, sc, i.view(1, 2), i, i, i, 0.125, 1, 1)
    with pytest.raises(ValueError, match="CUDA"):
        ops.attn_prologue_fp8(q, k, k, w, w, i, torch.ones(8), pool, pool, sc, i)


def test_cache_pool_in_8_bits():
    from tokenfactory_b200.hybrid_model import HybridCachePool, HybridConfig
    cfg = HybridConfig(num_hidden_layers=8, num_key_value_heads=2, head_dim=64)
    p = HybridCachePool(cfg, 10, 2, device="cpu", kv_dtype=torch.float8_e4m3fn)
    k, v = p.get_full_kv_buffers(7)
    sc = p.get_full_kv_scales(7)
    assert k.shape == v.shape == (10, 2, 64) and k.dtype == v.dtype == torch.float8_e4m3fn
    assert sc.shape == (10, 2, 2) and sc.dtype == torch.float32 and sc.is_contiguous()
    assert v.data_ptr() - k.data_ptr() == 64 and k.stride() == v.stride() == (256, 128, 1)
    assert sc.data_ptr() - p.get_full_kv_scales(3).data_ptr() == 10 * 2 * 2 * 4
    plain = HybridCachePool(cfg, 10, 2, device="cpu")
    assert plain.kv_scale is None and plain.get_full_kv_scales(3) is None
    assert plain.k_buffer.dtype == plain.v_buffer.dtype == torch.bfloat16
    assert plain.k_buffer.is_contiguous() and plain.v_buffer.is_contiguous()
    with pytest.raises(TypeError):
        HybridCachePool(cfg, 10, 2, device="cpu", kv_dtype=torch.float16)


@pytest.mark.parametrize("hq,max_ext", [(64, 0), (64, 9), (8, 4000), (2, 1 << 20)])
def test_decode_workspace_does_not_follow_the_extend_fields(hq, max_ext):
    """A caller that shares one argument structure between extend and decode calls: the decode's size
    is that of one query row per head, whatever the extend fields say."""
    from tokenfactory_b200 import _capi
    lib = _capi.load()
    kw = dict(num_q_heads=hq, num_kv_heads=2, head_dim=128)
    want = lib.tf_paged_decode_fp8_workspace_size(
        ctypes.byref(_paged(extend_lens=None, max_extend_len=1, **kw)))
    got = lib.tf_paged_decode_fp8_workspace_size(
        ctypes.byref(_paged(extend_lens=FAKE, max_extend_len=max_ext, **kw)))
    assert want > 0 and got == want
