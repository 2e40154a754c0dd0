"""Refusals of the RMS norms, the global norm and the products, before anything reaches a GPU."""
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
    assert lib.nl_rms_norm_bwd_ws_bytes((1 << 31) - 1, 1) == lib.nl_rms_norm_bwd_ws_bytes(1 << 20, 1) > 0


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


def test_global_norm_refusals_of_the_library():
    import ctypes

    lib = _lib.load()

    def leaf(g=256, out=256, rows=1, cols=8, ld=8, ldo=8, dtype=0):
        return (ctypes.c_int64 * 7)(g or 0, out or 0, rows, cols, ld, ldo, dtype)

    clip = lambda t=None, n=1, most=1.0, norm=512, ws=1024, wsb=8192: lib.nl_clip_by_global_norm(  # noqa: E731
        None, n, t if t is not None else leaf(), most, norm, ws, wsb)
    bad = [dict(n=-1), dict(most=0.0), dict(most=float("nan")), dict(norm=None), dict(ws=None), dict(wsb=8191),
           dict(t=leaf(g=None)), dict(t=leaf(out=None)), dict(t=leaf(rows=-1)), dict(t=leaf(cols=-1)),
           dict(t=leaf(dtype=2)), dict(t=leaf(rows=2, ld=7)), dict(t=leaf(rows=2, ldo=7)),
           dict(t=leaf(rows=2, ld=8, ldo=9))]
    for kw in bad:
        assert clip(**kw) == _lib.NL_EINVAL, kw
    for kw in (dict(t=leaf(g=258)), dict(t=leaf(out=257, dtype=1)), dict(ws=1028), dict(norm=514)):
        assert clip(**kw) == _lib.NL_EALIGN, kw
    for t in (leaf(rows=1 << 31), leaf(rows=2, cols=1 << 31, ld=1 << 31, ldo=1 << 31), leaf(cols=1 << 41)):
        assert clip(t) == _lib.NL_EUNSUPPORTED
    assert lib.nl_global_norm_multi(None, 1, leaf(g=None), 512, 1024, 8192) == _lib.NL_EINVAL
    assert lib.nl_global_norm_multi(None, 1, None, 512, 1024, 8192) == _lib.NL_EINVAL
    assert lib.nl_global_norm_multi(None, 1, leaf(out=None), None, 1024, 8192) == _lib.NL_EINVAL


def test_global_norm_refusals_in_python():
    import torch
    from nlearn_amd.kernels.clip import clip_by_global_norm, global_norm, rows_of

    x = torch.ones(8)
    for most in (0.0, -1.0, float("nan"), float("inf"), 1e300):
        with pytest.raises(ValueError, match="max_norm"):
            clip_by_global_norm([x], most)
    for call in (global_norm, lambda t: clip_by_global_norm(t, 1.0)):
        with pytest.raises(ValueError, match="no "):
            call([])
        with pytest.raises(ValueError, match="float32 or bfloat16"):
            call([x.double()])
        with pytest.raises(RuntimeError, match="HIP device"):
            call([x])
    with pytest.raises(ValueError, match="twice"):
        clip_by_global_norm([x, x], 1.0, inplace=True)
    # how a tensor is walked: (rows, columns, row stride)
    m = torch.zeros((6, 10))
    assert rows_of(m) == (1, 60, 60) and rows_of(m.t()) == (1, 60, 60)
    assert rows_of(m[:, :7]) == (6, 7, 10) and rows_of(m[:, :7].t()) == (6, 7, 10)
    assert rows_of(m[:, 3]) == (6, 1, 10) and rows_of(m[2]) == (1, 10, 10)
    assert rows_of(m[::2]) == (3, 10, 20) and rows_of(torch.zeros(())) == (1, 1, 1)
    assert rows_of(m[1:2, 2:9:2]) == (4, 1, 2)
    c = torch.zeros((4, 5, 8))
    assert rows_of(c[..., :6]) == (20, 6, 8) and rows_of(c[:, :3, :6]) is None and rows_of(c[:, :3]) == (4, 24, 40)
    assert rows_of(c.permute(1, 0, 2)) == (1, 160, 160)
    assert rows_of(x.expand(3, 8)) is None and rows_of(x[:1].expand(4)) is None
    assert rows_of(torch.as_strided(m, (4, 5), (3, 1))) is None


def test_fused_product_refusals_of_the_library():
    lib = _lib.load()

    def product(M=4, N=16, K=128, bias=None, bdt=0, act=0, res=None, ldr=16, rnd=0, aux=None, ldaux=16, C=1024, dt=1, ldc=16,
                sc=None, ldsc=0):
        return lib.nl_gemm_fp8_fused(None, M, N, K, 256, 128, 512, 4, 1, 4096, 128, 768, 4, 128, bias, bdt, act, res, ldr, rnd,
                                     aux, ldaux, C, dt, ldc, sc, ldsc, None, 0)

    assert product(M=0) == product(N=0) == _lib.NL_OK
    for bad in (dict(M=-1), dict(act=4), dict(act=-1), dict(C=None), dict(ldc=8), dict(dt=3), dict(res=2048, ldr=8),
                dict(aux=2048, ldaux=8), dict(dt=2, ldc=128, sc=None), dict(dt=2, ldc=64, sc=64, ldsc=1),
                dict(dt=2, ldc=128, sc=64, ldsc=0), dict(dt=2, ldc=128, sc=64, ldsc=1, aux=2048),
                dict(dt=2, ldc=128, sc=64, ldsc=1, rnd=1), dict(bias=256, bdt=2)):
        assert product(**bad) == _lib.NL_EINVAL, bad
        assert lib.nl_last_error()
    for bad in (dict(bias=258), dict(bias=257, bdt=1), dict(res=2056), dict(res=2048, ldr=20), dict(aux=2056), dict(C=1032), dict(ldc=20),
                dict(dt=2, ldc=136, sc=64, ldsc=1)):
        assert product(**bad) == _lib.NL_EALIGN, bad
    for bad in (dict(res=2048, ldr=1 << 22), dict(aux=2048, ldaux=1 << 22), dict(ldc=1 << 22)):
        assert product(**bad) == _lib.NL_EUNSUPPORTED, bad
    # the plain product has no 8-bit result
    assert lib.nl_gemm_fp8(None, 4, 16, 128, 256, 128, 512, 4, 1, 4096, 128, 768, 4, 128, 1024, 2, 128, None,
                           0) == _lib.NL_EINVAL


def test_output_gradient_refusals_of_the_library():
    lib = _lib.load()

    def dact(rows=4, cols=16, dy=256, dt=1, ld=16, u=512, ldu=16, act=2, q=1024, ldq=128, s=64, lds=1, db=None, bdt=0,
             ws=None, wsb=0):
        return lib.nl_quantize_fp8_dact(None, rows, cols, dy, dt, ld, u, ldu, act, q, ldq, s, lds, None, 0, None, 0, db, bdt,
                                        ws, wsb)

    assert dact(rows=0) == dact(cols=0) == _lib.NL_OK
    need = lib.nl_quantize_fp8_dact_ws_bytes(4, 16)
    assert need == 64 and lib.nl_quantize_fp8_dact_ws_bytes(0, 16) == 0
    for bad in (dict(act=4), dict(u=None), dict(ldu=8), dict(dy=None), dict(q=None), dict(dt=2), dict(ld=8), dict(s=None),
                dict(db=2048), dict(db=2048, ws=4096, wsb=need - 1), dict(db=2048, bdt=2, ws=4096, wsb=need)):
        assert dact(**bad) == _lib.NL_EINVAL, bad
    for bad in (dict(u=513), dict(dy=257), dict(db=2050, ws=4096, wsb=need),
                dict(db=2049, bdt=1, ws=4096, wsb=need), dict(ws=4098), dict(q=1032)):
        assert dact(**bad) == _lib.NL_EALIGN, bad
    assert dact(cols=(1 << 25) + 1, ld=1 << 26, ldu=1 << 26, ldq=1 << 26, lds=1 << 19, db=2048, ws=4096,
                wsb=1 << 60) == _lib.NL_EUNSUPPORTED
    # a layer: the same checks, and its buffers
    assert lib.nl_linear_fp8_fused_ws_bytes(64, 32, 16, 1, 1, 1, 1) == (
        lib.nl_linear_fp8_ws_bytes(64, 32, 16, 1, 1, 1) + lib.nl_quantize_fp8_dact_ws_bytes(64, 16))
    fwd = lambda act=2, ws=4096, bias=None: lib.nl_linear_fp8_fused_fwd(  # noqa: E731
        None, 64, 32, 16, 256, 1, 32, 512, 0, 16, bias, 0, act, None, 0, 8192, 16, 1024, 1, 16, 0, 0, None, 0, ws, 1 << 20)
    assert fwd(ws=None) == _lib.NL_EINVAL and fwd(ws=4104) == _lib.NL_EALIGN
    bwd = lambda act=2, u=512, wsb=1 << 20, db=2048: lib.nl_linear_fp8_fused_bwd(  # noqa: E731
        None, 64, 32, 16, 256, 1, 16, u, 16, act, db, 0, 4096, 1 << 20, 1, 0, 1024, 1, 32, None, 0, 0, 8192, wsb)
    assert bwd(act=7) == bwd(u=None) == bwd(wsb=64) == _lib.NL_EINVAL
    assert bwd(db=2050) == _lib.NL_EALIGN


def test_fused_product_refusals_in_python():
    import torch
    from nlearn_amd.kernels.fp8 import Fp8Blocks, Fp8Weight, _gemm_fp8_fused, _readable, gemm_fp8, linear_fp8

    x, W = torch.zeros((3, 64), dtype=torch.bfloat16), torch.zeros((64, 20))
    bias, res = torch.zeros(20), torch.zeros((3, 20), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="HIP device"):
        linear_fp8(x, W, bias=bias, activation="gelu", residual=res)
    for kw, what in ((dict(activation="tanh"), "activation"), (dict(activation=True), "activation"),
                     (dict(bias=bias[:19]), "bias"), (dict(bias=bias.double()), "bias"), (dict(bias=bias[None]), "bias"),
                     (dict(residual=res.float()), "residual"), (dict(residual=res[:2]), "residual"),
                     (dict(residual=res[:1].expand(3, 20)[:, :19]), "residual")):
        for w in (W, Fp8Weight(Fp8Blocks.empty(20, 64, 128, "cpu"), Fp8Blocks.empty(64, 20, 128, "cpu"))):
            with pytest.raises(ValueError, match=what):
                linear_fp8(x, w, **kw)
    many = torch.zeros((1, 1), dtype=torch.bfloat16).expand((1 << 30) + 1, 1)
    with pytest.raises(ValueError, match="bias gradient"):
        linear_fp8(many, torch.zeros((1, 1)), bias=torch.zeros(1, requires_grad=True))
    a, b = Fp8Blocks.empty(3, 64, 1, "cpu"), Fp8Blocks.empty(20, 64, 1, "cpu")
    with pytest.raises(RuntimeError, match="HIP device"):
        gemm_fp8(a, b, bias=bias)
    bf, e4 = torch.bfloat16, torch.float8_e4m3fn
    for args, what in (((bf, None, None, None, "swish", None), "activation"), ((bf, None, None, bias[:3], None, None), "bias"),
                       ((torch.float16, None, None, None, None, None), "result"),
                       ((bf, None, None, None, None, res.float()), "residual"), ((e4, None, None, None, None, res.float()), "residual"),
                       ((torch.float32, None, None, None, None, res), "residual"),
                       ((bf, None, None, None, None, res[:2]), "residual"),
                       ((bf, torch.zeros((3, 20), dtype=e4), None, bias, None, None), "result"),
                       ((bf, res[:1].expand(3, 20), None, bias, None, None), "overlap"),
                       ((bf, None, torch.zeros((4, 4))[:, :2], bias, None, None), "workspace")):
        with pytest.raises(ValueError, match=what):
            _gemm_fp8_fused(a, b, *args)
    # what the epilogue may read of a matrix over C: whole rows of 8, the last one's too
    t = torch.zeros((5, 24))
    assert _readable(t) is t and _readable(t[:, :16]).data_ptr() == t.data_ptr()
    assert _readable(t[:, :20]).data_ptr() == t.data_ptr()
    tight = torch.zeros(4 * 24 + 20).as_strided((5, 20), (24, 1))
    copy = _readable(tight)
    assert copy.data_ptr() != tight.data_ptr() and copy.stride(0) % 8 == 0 and torch.equal(copy, tight)
    assert copy.untyped_storage().nbytes() >= 4 * (4 * copy.stride(0) + 24)
    for odd in (t[:, 1:17], t[:, ::2], t.t(), t[:1].expand(5, 24)):
        copy = _readable(odd)
        assert copy.data_ptr() % 16 == 0 and copy.stride(1) == 1 and torch.equal(copy, odd)
