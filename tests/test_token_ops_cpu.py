"""Refusals of the token operators, without a GPU."""
import ctypes as C

import numpy as np
import pytest
import torch

from ccnet_amd import _lib, ops


def test_token_ops_refuse_bad_arguments_before_any_launch():
    """The C entry points of the token operators turn bad sizes, types and pointers into CCNET_EINVAL with a message, and have nothing to
    do for empty problems; the Python wrappers refuse CPU tensors.  No GPU is touched."""
    L = _lib.lib()
    H = _lib.Heads
    null, ok, odd = H(None, 0, 0, 0), H(1 << 20, 1024, 256, 128), H((1 << 20) + 2, 1024, 256, 128)
    skew = H(1 << 20, 1024, 256, 130)
    p = C.c_void_p(1 << 20)

    def rope(q=ok, k=null, dt=1, B=2, T=4, Hq=2, Hk=0, D=128, pos=p, freqs=p, rot=128, eps=1e-6, qo=ok):
        return L.ccnet_qk_norm_rope(q, k, dt, B, T, Hq, Hk, D, None, None, eps, pos, 4, freqs, rot, 0, qo, null, None)

    for bad in (dict(dt=2), dict(D=12), dict(D=264), dict(D=0), dict(rot=130), dict(rot=127), dict(rot=-2), dict(pos=None), dict(freqs=None), dict(eps=-1.0), dict(q=null), dict(q=odd),
                dict(q=skew), dict(qo=null), dict(Hk=1), dict(Hq=0), dict(B=-1), dict(T=-1)):
        assert rope(**bad) == -1, bad
    assert b"qk_norm_rope" in L.ccnet_last_error()
    assert rope(B=0) == 0 and rope(T=0, q=null, qo=null) == 0

    def write(k=ok, v=ok, dt=1, B=2, T=4, Hh=2, D=128, fmt=0, kc=p, ks=p, pages=8, page=16, tab=p, width=4, start=p):
        return L.ccnet_kv_cache_write(k, v, dt, B, T, Hh, D, fmt, kc, p, ks, p, pages, page, tab, width, start, None, None)

    for bad in (dict(dt=5), dict(fmt=2), dict(D=24), dict(D=272), dict(page=8), dict(page=48), dict(page=256), dict(kc=None), dict(ks=None), dict(tab=None), dict(start=None), dict(k=null),
                dict(v=odd), dict(v=skew), dict(B=70000), dict(Hh=0), dict(width=-1), dict(pages=-1), dict(width=1 << 28), dict(kc=C.c_void_p((1 << 20) + 8))):
        assert write(**bad) == -1, bad
    assert write(B=0) == 0 and write(T=0) == 0 and write(width=0) == 0 and write(pages=0) == 0
    assert L.ccnet_kv_cache_read(p, p, p, p, 0, 8, 16, p, 4, None, 1, 2, 4, 2, 128, ok, ok, None) == -1   # no lengths
    assert L.ccnet_kv_cache_read(p, p, p, p, 0, 8, 16, p, 4, p, 1, 2, 4, 2, 128, ok, null, None) == -1

    def cache(q=ok, dt=1, B=2, Sq=1, Hq=4, kc=p, fmt=1, pages=8, Hh=2, page=16, D=128, tab=p, width=4, lens=p, out=ok):
        return L.ccnet_cache_attention(q, dt, B, Sq, Hq, kc, p, p, p, fmt, pages, Hh, page, D, tab, width, lens, 0.1, 0, out, None, None)

    for bad in (dict(dt=3), dict(fmt=7), dict(Hq=3), dict(Hq=0), dict(D=40), dict(page=20), dict(kc=None), dict(tab=None), dict(lens=None), dict(q=null), dict(q=odd), dict(out=skew),
                dict(B=-2), dict(width=1 << 29)):
        assert cache(**bad) == -1, bad
    assert b"cache_attention" in L.ccnet_last_error()
    assert cache(B=0) == 0 and cache(Sq=0) == 0

    def cross(q=ok, k=ok, v=ok, dt=1, B=2, Sq=1, Sk=9, Hq=4, Hk=2, D=128, out=ok):
        return L.ccnet_cross_attention(q, k, v, dt, B, Sq, Sk, Hq, Hk, D, None, None, 0, 0.1, out, None, None)

    for bad in (dict(dt=-1), dict(Hq=5), dict(Hk=0), dict(D=20), dict(D=512), dict(q=odd), dict(k=null), dict(v=skew), dict(out=null), dict(Sk=-1), dict(B=1 << 20)):
        assert cross(**bad) == -1, bad
    assert cross(B=0) == 0 and cross(Sq=0) == 0
    # the Python layer
    t = torch.zeros(1, 2, 2, 64)
    with pytest.raises(ValueError, match="GPU"):
        ops.cross_attention(t, t, t, t)
    with pytest.raises(ValueError, match="GPU"):
        ops.qk_norm_rope(t, None, None, None, torch.zeros(1, 2, dtype=torch.int32), ops.rope_freqs(64), t, None)
    with pytest.raises(ValueError, match="16, 32, 64 or 128"):
        ops.Cache8.empty(2, 8, 1, 64, torch.int8, "cpu")
    with pytest.raises(ValueError, match="GPU"):
        ops.Cache8.empty(2, 16, 1, 64, torch.int8, "cpu")
    assert np.allclose(ops.rope_freqs(4, base=100.0).numpy(), [1.0, 0.1])
    assert not ops.Recorder.active()


def test_cache_attention_from_refuses_what_cache_attention_does_and_a_missing_start():
    """No GPU is touched: bad arguments are CCNET_EINVAL, empty problems have nothing to do."""
    L, H, p = _lib.lib(), _lib.Heads, C.c_void_p(1 << 20)
    ok, odd = H(1 << 20, 1024, 256, 128), H((1 << 20) + 2, 1024, 256, 128)

    def call(q=ok, dt=1, B=2, Sq=1, Hq=4, kc=p, D=128, page=16, lens=p, start=p, out=ok):
        return L.ccnet_cache_attention_from(q, dt, B, Sq, Hq, kc, p, p, p, 1, 8, 2, page, D, p, 4, lens, start, 0.1, out, None, None)

    for bad in (dict(start=None), dict(dt=3), dict(Hq=3), dict(D=40), dict(page=20), dict(kc=None), dict(lens=None), dict(q=odd)):
        assert call(**bad) == -1, bad
    assert call(B=0, start=None) == 0 and call(Sq=0) == 0


def test_cache_attention_splits_keys_by_the_grid_it_launches():
    """A call splits its keys to make 512 workgroups, so one whose row tiles alone make them needs no workspace.  64 query rows are one workgroup's in
    bfloat16 to 128 dims, two workgroups' in bfloat16 beyond and in float32 to 128 dims, four in float32 beyond.  Recorded, so nothing is launched."""
    L, H, p = _lib.lib(), _lib.Heads, C.c_void_p(1 << 20)
    for dt, D, per in ((1, 64, 1), (1, 128, 1), (1, 256, 2), (0, 64, 2), (0, 128, 2), (0, 256, 4)):
        x = H(1 << 20, 64 * 256, 256, 256)
        plan = C.c_void_p()
        assert L.ccnet_plan_begin(C.byref(plan)) == 0
        try:
            for B in (512, 256, 128, 64):
                rc = L.ccnet_cache_attention(x, dt, B, 64, 1, p, p, p, p, 0, 8, 1, 64, D, p, 64, p, 0.1, 0, x, None, None)
                assert (rc == 0) == (B * per > 256), (dt, D, B)   # (two ranges from half of 512 down)
                assert L.ccnet_cache_attention_workspace_bytes(B, 64, 1, 1, D, 64, 64) > 0 or rc == 0
        finally:
            L.ccnet_plan_end()
            L.ccnet_plan_destroy(plan)


def test_rope_freqs_refuses_an_odd_count_of_dims():
    """Seven dims are three pairs and a half: they gave four frequencies, a rotation of eight."""
    for bad in (7, 1, -2):
        with pytest.raises(ValueError, match="even"):
            ops.rope_freqs(bad)
    assert ops.rope_freqs(0).shape == (0,) and ops.rope_freqs(0).dtype == torch.float64 and ops.rope_freqs(6).shape == (3,)
