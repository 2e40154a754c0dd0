"""Refusals of the RMS norms, before anything reaches a GPU."""
import pytest

from nlearn_amd import _lib


def test_rms_norm_refusals_of_the_library():
    lib = _lib.load()
    fwd = lambda rows=4, D=16, dt=1, x=256, ldx=16, r=None, s=None, g=512, eps=1e-5, y=768: lib.nl_rms_norm_fwd(  # noqa: E731
        None, rows, D, dt, x, ldx, r, 16, s, 16, g, eps, y, 16, None)
    assert fwd(rows=0) == _lib.NL_OK
    for bad in (dict(rows=-1), dict(D=0), dict(D=16385), dict(dt=2), dict(x=None), dict(ldx=15), dict(g=None),
                dict(y=None), dict(eps=0.0), dict(eps=float("nan")), dict(eps=2.0), dict(r=1024)):
        assert fwd(**bad) == _lib.NL_EINVAL, bad
        assert lib.nl_last_error()
    for bad in (dict(x=257), dict(dt=0, x=258), dict(g=514), dict(y=769)):
        assert fwd(**bad) == _lib.NL_EALIGN, bad
    f8 = lambda ldq=128, lds=1, q=4096, sc=8192: lib.nl_rms_norm_fp8(  # noqa: E731
        None, 4, 16, 1, 256, 16, None, 0, None, 0, 512, 1e-5, q, ldq, sc, lds)
    assert f8(ldq=112) == f8(lds=0) == f8(q=None) == f8(sc=None) == _lib.NL_EINVAL
    assert f8(ldq=136) == f8(q=4104) == _lib.NL_EALIGN
    bwd = lambda dy=256, dg=1024, ws=4096, wsb=1 << 20, dx=2048, ld=16: lib.nl_rms_norm_bwd(  # noqa: E731
        None, 4, 16, 1, dy, ld, 512, 16, 768, 1280, None, 0, dx, 16, dg, 0, ws, wsb)
    assert bwd(dy=None) == bwd(dx=None) == bwd(ws=None) == bwd(wsb=16) == bwd(ld=8) == _lib.NL_EINVAL
    assert bwd(dy=257) == bwd(ws=4104) == bwd(dg=1026) == _lib.NL_EALIGN
    assert lib.nl_rms_norm_bwd_ws_bytes(4, 16) >= 64 and lib.nl_rms_norm_bwd_ws_bytes(0, 16) == 0
    assert lib.nl_rms_norm_bwd_ws_bytes(1 << 30, 16384) <= 1 << 26


def test_rms_norm_refusals_in_python():
    import torch
    from nlearn_amd.kernels.fp8 import add_rms_norm_fp8, rms_norm_fp8
    from nlearn_amd.kernels.fused import add_rms_norm, rms_norm

    x, gamma = torch.zeros((3, 64)), torch.ones(64)
    for norm, add in ((rms_norm, add_rms_norm), (rms_norm_fp8, add_rms_norm_fp8)):
        with pytest.raises(RuntimeError, match="HIP device"):
            norm(x, gamma)
        with pytest.raises(ValueError, match="bfloat16 or float32"):
            norm(x.half(), gamma)
        with pytest.raises(ValueError, match="gamma"):
            norm(x, gamma[:63])
        with pytest.raises(ValueError, match="gamma"):
            norm(x, gamma.double())
        with pytest.raises(ValueError, match="elements"):
            norm(torch.zeros((3, 0)), gamma[:0])
        with pytest.raises(ValueError, match="elements"):
            norm(torch.zeros((1, 16385)), torch.ones(16385))
        for eps in (0.0, -1.0, 2.0, float("nan"), float("inf")):
            with pytest.raises(ValueError, match="eps"):
                norm(x, gamma, eps)
        with pytest.raises(ValueError, match="residual"):
            add(x, x[:2], gamma)
        with pytest.raises(ValueError, match="residual"):
            add(x, x.bfloat16(), gamma)
        with pytest.raises(ValueError, match="one device"):
            norm(x, torch.ones(64, device="meta"))
        with pytest.raises(ValueError, match="2\\^31"):
            norm(torch.zeros(1).expand(1 << 31, 1), torch.ones(1))
