"""Refusals of the transformer-block operators' C entry points, on a machine without a GPU: a bad call returns its error code before anything
is launched, an empty one returns at once."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def R():
    import revisiting_at_amd as R
    R._lib.load()
    return R


NULL, ARG, SIZE, DTYPE = -1, -4, -2, -3
S12, S24 = (ctypes.c_int64 * 12)(), (ctypes.c_int64 * 24)()
P = 4096                                                        # a pointer that no refused call follows


def mha_fwd(lib, q=P, k=P, v=P, out=P, ws=P, strides=S12, dtype=1, B=1, Nq=4, Nk=4, H=2, Hkv=1, d=64, scale=0.125):
    return lib.cnx_mha_fwd(q, k, v, out, None, None, None, ws, strides, dtype, B, Nq, Nk, H, Hkv, d, 0, scale, None)


def mha_bwd(lib, q=P, dq=P, lse=P, dvec=P, dk=P, ws=P, strides=S24, dtype=1, B=1, Nq=4, Nk=4, H=2, Hkv=1, d=64, scale=0.125):
    return lib.cnx_mha_bwd(q, P, P, P, P, lse, dq, dk, P, dvec, None, None, ws, strides, dtype, B, Nq, Nk, H, Hkv, d, 0, scale, None)


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), NULL), (dict(strides=None), NULL), (dict(dtype=0), DTYPE), (dict(dtype=7), DTYPE), (dict(d=32), ARG), (dict(d=96), ARG),
    (dict(H=3, Hkv=2), ARG), (dict(H=0), SIZE), (dict(Hkv=0), SIZE), (dict(B=-1), SIZE), (dict(Nq=-1), SIZE), (dict(Nk=-1), SIZE),
    (dict(scale=0.0), ARG), (dict(scale=-1.0), ARG), (dict(scale=float("nan")), ARG), (dict(scale=float("inf")), ARG),
    (dict(Nq=2 ** 31 - 1), SIZE), (dict(Nk=2 ** 31 - 1), SIZE), (dict(B=2 ** 40), SIZE), (dict(B=0), 0), (dict(B=0, q=None), 0)])
def test_mha_refuses(R, kw, code):
    lib = R._lib.load()
    assert mha_fwd(lib, **kw) == code
    assert mha_bwd(lib, **kw) == code


def test_mha_refuses_missing_outputs_and_workspace(R):
    lib = R._lib.load()
    assert mha_fwd(lib, out=None) == NULL and mha_fwd(lib, k=None) == NULL and mha_fwd(lib, v=None) == NULL
    assert mha_bwd(lib, dq=None) == NULL and mha_bwd(lib, lse=None) == NULL and mha_bwd(lib, dvec=None) == NULL and mha_bwd(lib, dk=None) == NULL
    assert lib.cnx_mha_ws_floats(1, 1, 5000, 2, 1, 64) > 0                     # few rows: the keys are split
    assert mha_fwd(lib, ws=None, Nq=1, Nk=5000) == NULL
    assert lib.cnx_mha_bwd_ws_floats(1, 5000, 100, 2, 1, 64, 0) > 0 == lib.cnx_mha_ws_floats(1, 5000, 100, 2, 1, 64)     # few key tiles: the rows
    assert mha_bwd(lib, ws=None, Nq=5000, Nk=100, H=2, Hkv=1) == NULL
    assert lib.cnx_mha_bwd_ws_floats(1, 5000, 100, 2, 1, 80, 0) == 0 and lib.cnx_mha_bwd_ws_floats(64, 1025, 1025, 6, 6, 64, 0) == 0
    assert lib.cnx_mha_ws_floats(1, 1, 5000, 2, 1, 80) == 0 and lib.cnx_mha_ws_floats(0, 1, 1, 1, 1, 64) == 0
    assert mha_fwd(lib, Nq=0) == 0 and mha_bwd(lib, Nq=0, Nk=0) == 0
    assert [lib.cnx_mha_supported(d) for d in (0, 32, 64, 96, 128, 256)] == [0, 0, 1, 0, 1, 0]


def attn_bwd(lib, qkv=P, out=P, dqkv=P, ws=P, strides=S24, dtype=1, pos=P, pos_dtype=2, axes=2, sections=(16, 16), inv=P, B=1, N=4, H=2, d=64, dw=None,
             norm=1, scale=0.125):
    sec = None if sections is None else (ctypes.c_int32 * len(sections))(*sections)
    return lib.cnx_attention_rope_bwd(qkv, P, P, out, P, P, dqkv, dw, dw, ws, strides, dtype, None, None, pos, pos_dtype, 0, axes, sec, inv, B, N, H, d,
                                      1e-6, norm, 0, scale, None)


@pytest.mark.parametrize("kw,code", [
    (dict(qkv=None), NULL), (dict(out=None), NULL), (dict(dqkv=None), NULL), (dict(ws=None), NULL), (dict(strides=None), NULL), (dict(dtype=0), DTYPE),
    (dict(d=32), ARG), (dict(H=0), SIZE), (dict(B=0), 0), (dict(N=0), 0), (dict(N=-1), SIZE), (dict(scale=0.0), ARG), (dict(norm=0, pos=None), ARG),
    (dict(dw=P, norm=0), ARG), (dict(inv=None), NULL), (dict(sections=None), NULL), (dict(pos_dtype=3), DTYPE), (dict(axes=5), ARG),
    (dict(sections=(16, 17)), ARG), (dict(B=2 ** 40), SIZE)])
def test_attention_rope_backward_refuses(R, kw, code):
    assert attn_bwd(R._lib.load(), **kw) == code


def test_attention_rope_workspaces_and_forward_refusals(R):
    lib = R._lib.load()
    size = lib.cnx_attention_rope_bwd_ws_floats
    assert size(2, 17, 2, 64, 1) - size(2, 17, 2, 64, 0) == 17 * 64 and size(2, 17, 2, 64, 0) >= 68 + 17 * 64 + 2 * 4 * 64
    assert size(1, 1000, 1, 64, 0) > size(1, 1000, 1, 64, 0) - lib.cnx_mha_bwd_ws_floats(1, 1000, 1000, 1, 1, 64, 0) > 0        # rows split
    assert size(1, 17, 2, 96, 0) == 0 and size(0, 17, 2, 64, 0) == 0

    def fwd(qkv=P, y=P, out=P, ws=P, dtype=1, w=None, w_dtype=0, pos=P, axes=2, sections=(16, 16), B=1, N=4, H=2, d=64, norm=1, scale=0.125):
        sec = (ctypes.c_int32 * len(sections))(*sections)
        return lib.cnx_attention_rope_fwd(qkv, y, y, out, None, ws, dtype, w, w, w_dtype, pos, 2, 0, axes, sec, P, B, N, H, d, 1e-6, norm, 0, scale, None)
    for kw, code in ((dict(qkv=None), NULL), (dict(y=None), NULL), (dict(out=None), NULL), (dict(ws=None, N=1000), NULL), (dict(dtype=0), DTYPE),
                     (dict(w=P, w_dtype=2), DTYPE), (dict(d=32), ARG), (dict(axes=0), ARG), (dict(sections=(1, 2)), ARG), (dict(H=0), SIZE),
                     (dict(N=-1), SIZE), (dict(scale=-1.0), ARG), (dict(B=0, qkv=None), 0), (dict(N=0), 0)):
        assert fwd(**kw) == code, kw


def rope(lib, fwd=True, q=P, out=P, strides=S24, dtype=1, w=None, w_dtype=0, pos=P, pos_dtype=2, axes=2, sections=(16, 16), inv=P, B=1, N=4, Hq=2,
         Hk=2, d=64, dw=None, ws=None, norm=1):
    sec = None if sections is None else (ctypes.c_int32 * len(sections))(*sections)
    tail = (dtype, strides, w, w, w_dtype, pos, pos_dtype, 0, axes, sec, inv, B, N, Hq, Hk, d, 1e-6, norm, 0, None)
    if fwd:
        return lib.cnx_qk_norm_rope_fwd(q, P, out, P, *tail)
    return lib.cnx_qk_norm_rope_bwd(P, P, q, P, out, P, dw, dw, ws, *tail)


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), NULL), (dict(out=None), NULL), (dict(strides=None), NULL), (dict(dtype=3), DTYPE), (dict(d=24), ARG), (dict(d=8), ARG),
    (dict(d=272), ARG), (dict(inv=None), NULL), (dict(sections=None), NULL), (dict(pos_dtype=3), DTYPE), (dict(axes=0), ARG), (dict(axes=5), ARG),
    (dict(sections=(16, 15)), ARG), (dict(sections=(33, -1)), ARG), (dict(B=-1), SIZE), (dict(N=-1), SIZE), (dict(Hq=-1), SIZE),
    (dict(Hk=1 << 21), SIZE), (dict(B=2 ** 40, N=2 ** 40), SIZE), (dict(w=P, w_dtype=2), DTYPE), (dict(B=0), 0), (dict(N=0), 0),
    (dict(Hq=0, Hk=0), 0)])
def test_qk_norm_rope_refuses(R, kw, code):
    lib = R._lib.load()
    assert rope(lib, True, **kw) == code
    assert rope(lib, False, **kw) == code


def test_qk_norm_rope_refuses_weight_gradients_without_a_workspace(R):
    lib = R._lib.load()
    assert rope(lib, False, w=P, dw=P, ws=None) == NULL
    assert lib.cnx_qk_norm_rope_ws_floats(64) > 0 and lib.cnx_qk_norm_rope_ws_floats(24) == 0


def test_operators_have_no_cpu_path(R):
    x = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16)
    for f in (lambda: R.ops.mha(x, x, x), lambda: R.ops.qk_norm_rope(x, x), lambda: R.ops.attention_rope(torch.zeros(1, 4, 384, dtype=torch.bfloat16), 2)):
        with pytest.raises(R._lib.ApgdHipError):
            f()
