"""CPU checks of the 8-bit and distillation calls: what they refuse, on the host and before any launch,
workspace sizes, and the float64 definitions against each other."""
import numpy as np
import pytest

from oracle import distill_fp8 as orc


def test_e4m3_table_and_rounding():
    import torch

    t = orc.e4m3_table()
    want = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(t, want)
    # every byte is its own nearest, and a midpoint goes to the even neighbour
    fin = np.isfinite(t)
    np.testing.assert_array_equal(orc.e4m3_bytes(t)[fin], np.arange(256)[fin])
    pos = np.arange(0, 0x7e)
    mid = (t[pos] + t[pos + 1]) / 2
    np.testing.assert_array_equal(orc.e4m3_bytes(mid), np.where(pos % 2 == 0, pos, pos + 1))
    x = np.random.default_rng(0).uniform(-448, 448, 20000) * 2.0 ** np.random.default_rng(1).integers(-12, 1, 20000)
    np.testing.assert_array_equal(orc.e4m3_bytes(x), torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy())


def test_quantize_definition():
    rng = np.random.default_rng(2)
    x = rng.standard_normal((130, 300)) * 2.0 ** rng.integers(-30, 30, (130, 1))
    for group in (1, 128):
        q, s = orc.quantize(x, group)
        v = orc.values(q, s, group)[:, :300]
        # half a step: 2^-4 of the value, or 2^-10 of the scale below the normal range
        f = np.repeat(np.repeat(2.0 ** (s.astype(float) - 127), group, 0)[:130], 128, 1)[:, :300]
        assert (np.abs(v - x) <= np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10 * f)).all()
        assert (np.abs(x) <= 448 * f).all()


def test_distill_definition_is_the_gradient():
    """The formula's dlogits against central differences of the formula's loss."""
    rng = np.random.default_rng(3)
    z, v = rng.standard_normal((3, 12)), rng.standard_normal((3, 4))
    ids = np.array([[0, 3, 3, -1], [5, 6, 7, 11], [-1, -1, -1, -1]])
    for lse in (None, rng.standard_normal(3) + 2):
        loss, d, _, _ = orc.distill(z, ids, v, lse, 1.7, 1.0)
        assert loss[2] == 0 and (d[2] == 0).all()
        for m in range(3):
            for c in range(12):
                hi, lo = z.copy(), z.copy()
                hi[m, c] += 1e-5
                lo[m, c] -= 1e-5
                num = (orc.distill(hi, ids, v, lse, 1.7, 1.0)[0][m] - orc.distill(lo, ids, v, lse, 1.7, 1.0)[0][m]) / 2e-5
                assert abs(num - d[m, c]) < 1e-8


def test_python_refusals():
    import torch
    from nlearn_amd.kernels import distill, fp8

    bf, f8, e8 = torch.bfloat16, torch.float8_e4m3fn, torch.float8_e8m0fnu
    x = torch.zeros((4, 130), dtype=bf)
    with pytest.raises(RuntimeError, match="HIP device"):
        fp8.quantize_fp8(x)
    for bad, what in ((torch.zeros(4, dtype=bf), "2-D"), (torch.zeros((4, 4), dtype=torch.float16), "bfloat16 or float32"),
                      (torch.zeros((4, 4), dtype=torch.int32), "bfloat16 or float32")):
        with pytest.raises(ValueError, match=what):
            fp8.quantize_fp8(bad)
    with pytest.raises(ValueError, match="1 or 128"):
        fp8.quantize_fp8_both(x, group=64)
    q, s = torch.zeros((4, 256), dtype=torch.uint8).view(f8), torch.zeros((4, 2), dtype=torch.uint8).view(e8)
    fp8.Fp8Blocks(q, s, (4, 130), 1)
    fp8.Fp8Blocks(q, s[:1], (4, 256), 128)
    wide = torch.zeros((4, 264), dtype=torch.uint8).view(f8)
    for args, what in (((q, s, (4, 300), 1), "q must be"), ((q, s, (5, 130), 1), "q must be"),
                       ((q.view(torch.uint8), s, (4, 130), 1), "q must be"), ((q, s, (4, 130), 128), "scale must be"),
                       ((q, s.view(torch.uint8), (4, 130), 1), "scale must be"), ((q, s, (4, 130), 2), "1 or 128"),
                       ((wide[:, :256], s, (4, 130), 1), "16-byte"), ((q[:1].expand(4, 256), s, (4, 130), 1), "of their own"),
                       ((q, s[:1].expand(4, 2), (4, 130), 1), "of their own"),
                       ((wide[:, 8:], s, (4, 130), 1), "16-byte")):
        with pytest.raises(ValueError, match=what):
            fp8.Fp8Blocks(*args)
    a = fp8.Fp8Blocks(q, s, (4, 130), 1)
    with pytest.raises(ValueError, match="inner dimensions"):
        fp8.gemm_fp8(a, fp8.Fp8Blocks(q, s, (4, 256), 1))
    with pytest.raises(RuntimeError, match="HIP device"):
        fp8.gemm_fp8(a, a)
    with pytest.raises(ValueError, match="features"):
        fp8.linear_fp8(x, torch.zeros((8, 8)))
    with pytest.raises(ValueError, match="2 dims"):
        fp8.linear_fp8(x, torch.zeros(130))
    with pytest.raises(ValueError, match=">= 2 dims"):
        fp8.linear_fp8(x[0], torch.zeros((130, 8)))
    with pytest.raises(ValueError, match="bfloat16 or float32"):
        fp8.linear_fp8(x.half(), torch.zeros((130, 8)))
    with pytest.raises(ValueError, match="bfloat16 or float32"):
        fp8.linear_fp8(x, torch.zeros((130, 8), dtype=torch.float16))
    with pytest.raises(RuntimeError, match="HIP device"):
        fp8.linear_fp8(x, torch.zeros((130, 8)))

    for k in (0, 131, 257):
        with pytest.raises(ValueError, match="1 <= k"):
            distill.top_logits(x, k)
    for t in (0.0, -1.0, float("nan"), float("inf"), 1e-9):
        with pytest.raises(ValueError, match="temperature"):
            distill.top_logits(x, 3, t)
    with pytest.raises(ValueError, match="bfloat16"):
        distill.top_logits(x.float(), 3)
    with pytest.raises(ValueError, match="unit stride"):
        distill.top_logits(torch.zeros((130, 4), dtype=bf).t(), 3)
    with pytest.raises(ValueError, match="empty vocabulary"):
        distill.top_logits(torch.zeros((4, 0), dtype=bf), 3)
    with pytest.raises(RuntimeError, match="HIP device"):
        distill.top_logits(x, 3)
    ids, v = torch.zeros((4, 3), dtype=torch.int32), torch.zeros((4, 3))
    d = distill.distill_cross_entropy
    for args, what in (((x, ids[:3], v[:3]), "must both be"), ((x, ids, v[:, :2]), "must both be"),
                       ((x, ids[:, :0], v[:, :0]), "1 <= k"), ((x, ids.short(), v), "int32 or int64"),
                       ((x, ids, v.double()), "bfloat16 or float32"), ((x, ids, v, torch.zeros(3)), "lse must be"),
                       ((x, ids, v, torch.zeros(4, dtype=bf)), "lse must be"), ((x, ids, v, None, 0.0), "temperature"),
                       ((x.float(), ids, v), "bfloat16"), ((x, ids, v.clone().requires_grad_(True)), "no gradient"),
                       ((x[:1].expand(4, 130), ids, v, None, 1.0, True), "inplace")):
        with pytest.raises(ValueError, match=what):
            d(*args)
    with pytest.raises(RuntimeError, match="HIP device"):
        d(x, ids, v)


def test_c_abi_refusals_and_sizes():
    """Argument errors of the C entry points, found before any HIP call."""
    from nlearn_amd import _lib

    L = _lib.load()
    E, A, U, ok = _lib.NL_EINVAL, _lib.NL_EALIGN, _lib.NL_EUNSUPPORTED, _lib.NL_OK
    # quantize: rows, cols, x, dtype, ldx, group, q, ldq, scale, lds, qt, ldqt, scale_t, ldst
    base = dict(rows=4, cols=130, x=256, dt=1, ldx=136, group=1, q=512, ldq=256, s=1024, lds=2, qt=2048, ldqt=128, st=4096,
                ldst=1)

    def quantize(**kw):
        a = {**base, **kw}
        return L.nl_quantize_fp8(None, a["rows"], a["cols"], a["x"], a["dt"], a["ldx"], a["group"], a["q"], a["ldq"],
                                 a["s"], a["lds"], a["qt"], a["ldqt"], a["st"], a["ldst"])

    assert quantize(rows=0, qt=None) == ok and quantize(cols=0, q=None) == ok
    for kw, rc in ((dict(rows=-1), E), (dict(dt=2), E), (dict(group=64), E), (dict(q=None, qt=None), E), (dict(x=None), E),
                   (dict(ldx=129), E), (dict(ldq=130), E), (dict(ldq=264), A), (dict(q=520), A), (dict(lds=1), E),
                   (dict(s=None), E), (dict(ldqt=100), E), (dict(st=None), E), (dict(x=257), A), (dict(x=258, dt=0), A),
                   (dict(rows=1 << 31), E), (dict(rows=1 << 30, cols=8, qt=None, ldq=128, lds=1, ldx=8), U)):
        assert quantize(**kw) == rc, kw
    # gemm: M, N, K, A, lda, sa, ldsa, ga, B, ldb, sb, ldsb, gb, C, dtype, ldc, ws, bytes
    g0 = dict(M=4, N=5, K=130, A=256, lda=256, sa=512, ldsa=2, ga=1, B=1024, ldb=256, sb=2048, ldsb=2, gb=128, C=4096, dt=1,
              ldc=8)

    def gemm(**kw):
        a = {**g0, **kw}
        return L.nl_gemm_fp8(None, a["M"], a["N"], a["K"], a["A"], a["lda"], a["sa"], a["ldsa"], a["ga"], a["B"], a["ldb"],
                             a["sb"], a["ldsb"], a["gb"], a["C"], a["dt"], a["ldc"], None, 0)

    assert gemm(M=0) == ok and gemm(N=0) == ok
    for kw, rc in ((dict(M=-1), E), (dict(dt=3), E), (dict(ga=2), E), (dict(lda=192), E), (dict(lda=264), A),
                   (dict(A=264), A), (dict(A=None), E), (dict(sb=None), E), (dict(ldsb=1), E), (dict(C=None), E),
                   (dict(ldc=4), E), (dict(ldc=12), A), (dict(C=4100), A), (dict(lda=1 << 23), U),
                   (dict(ldc=1 << 21), U)):
        assert gemm(**kw) == rc, kw
    assert L.nl_gemm_fp8_ws_bytes(8192, 8192, 8192) == 0 and L.nl_gemm_fp8_ws_bytes(0, 4, 4) == 0
    # a small output with a long sum is split: whole fp32 partials, at least 2 of them
    n = L.nl_gemm_fp8_ws_bytes(512, 512, 16384)
    assert n % (512 * 512 * 4) == 0 and n >= 2 * 512 * 512 * 4
    # linear: sizes, workspaces
    assert L.nl_linear_fp8_saved_bytes(4, 130, 200, 0, 0) == 0
    # W (130 rows of 256 bytes, 2 rows of 4 scale bytes), X^T (130 rows of 128 bytes and 4 scale bytes)
    w, xt = (130 * 256 + 2 * 4 + 15) // 16 * 16, (130 * 128 + 130 * 4 + 15) // 16 * 16
    assert L.nl_linear_fp8_saved_bytes(4, 130, 200, 1, 0) == w and L.nl_linear_fp8_saved_bytes(4, 130, 200, 1, 1) == w + xt
    fwd = L.nl_linear_fp8_ws_bytes(4, 130, 200, 0, 1, 1)
    f = (None, 4, 130, 200, 256, 1, 136, 512, 0, 200, 1024, 1, 200, 1, 1)
    assert L.nl_linear_fp8_fwd(*f, 2048, w + xt - 1, 4096, fwd) == E and b"saved" in L.nl_last_error()
    assert L.nl_linear_fp8_fwd(*f, 2048, w + xt, 4096, fwd - 1) == E and b"workspace" in L.nl_last_error()
    assert L.nl_linear_fp8_fwd(*f, 2056, w + xt, 4096, fwd) == A
    assert L.nl_linear_fp8_fwd(*f, 2048, w + xt, None, fwd) == E
    assert L.nl_linear_fp8_fwd(*(f[:1] + (0,) + f[2:]), 2048, w + xt, 4096, fwd) == E
    b = (None, 4, 130, 200, 256, 1, 200, 2048, w + xt)
    assert L.nl_linear_fp8_bwd(*b, 0, 0, None, 0, 0, None, 0, 0, None, 0) == ok       # nothing wanted
    assert L.nl_linear_fp8_bwd(*b, 1, 1, 512, 1, 136, 1024, 0, 200, 4096, 16) == E
    # top, distill
    assert L.nl_top_logits(None, 0, 100, None, 100, 3, 1.0, None, None, None) == ok
    for args, rc in (((4, 0, 256, 100, 3, 1.0), E), ((4, 100, 256, 99, 3, 1.0), E), ((4, 100, 256, 100, 0, 1.0), E),
                     ((4, 100, 256, 100, 101, 1.0), E), ((4, 1000, 256, 1000, 257, 1.0), E), ((4, 100, 257, 100, 3, 1.0), A),
                     ((4, 100, None, 100, 3, 1.0), E), ((4, 100, 256, 100, 3, 0.0), E), ((4, 100, 256, 100, 3, -1.0), E),
                     ((4, 100, 256, 100, 3, float("nan")), E), ((4, 100, 256, 100, 3, float("inf")), E),
                     ((4, 1 << 24, 256, 1 << 24, 3, 1.0), E), ((1 << 27, 8, 256, 8, 3, 1.0), U)):
        assert L.nl_top_logits(None, *args, 512, 1024, 2048) == rc, args
    assert L.nl_top_logits(None, 4, 100, 256, 100, 3, 1.0, None, 1024, 2048) == E
    d0 = dict(M=4, V=100, z=256, ld=100, k=3, ids=512, v=1024, dt=0, T=1.0, loss=2048, d=4096, ldd=100)

    def dist(**kw):
        a = {**d0, **kw}
        return L.nl_distill_fwd_bwd(None, a["M"], a["V"], a["z"], a["ld"], a["k"], a["ids"], 0, a["v"], a["dt"], None, a["T"],
                                    a["loss"], None, 0.25, a["d"], a["ldd"])

    assert dist(M=0) == ok
    for kw, rc in ((dict(k=0), E), (dict(k=257), E), (dict(dt=5), E), (dict(ids=None), E), (dict(v=None), E),
                   (dict(loss=None), E), (dict(ldd=99), E), (dict(d=4097), A), (dict(d=256, ldd=104), E), (dict(T=0.0), E),
                   (dict(ld=50), E), (dict(z=None), E), (dict(V=0), E)):
        assert dist(**kw) == rc, kw


def test_sizes_past_32_bits_are_refused():
    """The kernels count rows in 32 bits: more of them raise, and are not cut to their low bits."""
    import torch
    from nlearn_amd.kernels import distill, fp8

    n = (1 << 32) + 8
    blocks = fp8.Fp8Blocks.empty(n, 0, 1, "cpu")
    with pytest.raises(ValueError, match=r"2\^31"):
        fp8.gemm_fp8(blocks, fp8.Fp8Blocks.empty(4, 0, 1, "cpu"))
    x = torch.zeros((1, 8), dtype=torch.bfloat16).expand(n, 8)
    with pytest.raises(ValueError, match=r"2\^31"):
        fp8.linear_fp8(x, torch.zeros((8, 8)))
    with pytest.raises(ValueError, match=r"2\^31"):
        distill.top_logits(x, 3)
    with pytest.raises(ValueError, match=r"2\^31"):
        distill.distill_cross_entropy(x, torch.zeros((1, 3), dtype=torch.int32).expand(n, 3), torch.zeros((1, 3)).expand(n, 3))


def test_main_grad_of_another_shape_is_refused():
    """The weight gradient is written with the buffer's row stride: a buffer that is not W's shape would be overrun."""
    import torch
    from nlearn_amd.kernels import fp8

    W = torch.zeros((128, 40), requires_grad=True)
    assert fp8._main_grad(W) is None
    W.main_grad = torch.zeros((128, 40))
    assert fp8._main_grad(W) is W.main_grad
    for shape in ((40, 128), (128, 41), (127, 40), (5120,), (128, 40, 1)):
        W.main_grad = torch.zeros(shape)
        with pytest.raises(ValueError, match="main_grad"):
            fp8._main_grad(W)
    W.main_grad = torch.zeros((128, 40), device="meta")
    with pytest.raises(ValueError, match="main_grad"):
        fp8._main_grad(W)


def test_launches_of_2_to_the_32_threads_are_refused():
    """16 blocks of 128 a workgroup of 256: the last count below 2^28 that fits is 2^28 - 16."""
    from nlearn_amd import _lib

    L = _lib.load()
    for rows in ((1 << 28) - 15, (1 << 28) - 1, 1 << 28):
        assert L.nl_quantize_fp8(None, rows, 8, 256, 1, 8, 1, 512, 128, 1024, 1, None, 0, None, 0) == _lib.NL_EUNSUPPORTED
        assert b"blocks" in L.nl_last_error()
    # tiles of 128 x 128 and 512 threads: 2^23 of them
    assert L.nl_quantize_fp8(None, 1 << 29, 256, 256, 1, 256, 128, 512, 256, 1024, 2, None, 0, None, 0) == _lib.NL_EUNSUPPORTED
    assert b"tiles" in L.nl_last_error()


def test_forward_refuses_what_its_backward_would():
    import torch
    from nlearn_amd import _lib
    from nlearn_amd.kernels import fp8

    L = _lib.load()

    def forward(M, K, N, dx, dw):
        saved, ws = L.nl_linear_fp8_saved_bytes(M, K, N, dx, dw), L.nl_linear_fp8_ws_bytes(M, K, N, 0, dx, dw)
        return L.nl_linear_fp8_fwd(None, M, K, N, 256, 1, K, 512, 0, N, 1024, 1, (N + 7) // 8 * 8, dx, dw, 2048, saved, 4096,
                                   ws)

    for M, K, N, dx, dw, what in ((8388481, 16, 8, 0, 1, b"8388480 rows"), (8388608, 16, 8, 1, 1, b"8388480 rows"),
                                  (4, 2097024, 8, 1, 0, b"columns"), (1 << 27, 16, 256, 1, 0, b"blocks")):
        assert forward(M, K, N, dx, dw) == _lib.NL_EUNSUPPORTED and what in L.nl_last_error(), (M, K, N)

    def frozen(M, K, N):
        W = fp8.Fp8Weight.__new__(fp8.Fp8Weight)
        W.shape = (K, N)
        return fp8.linear_fp8(torch.zeros((1, 1), dtype=torch.bfloat16).expand(M, K).requires_grad_(True), W)

    for shape in ((4, 2097024, 8), (1 << 27, 16, 256)):
        with pytest.raises(ValueError, match="no input gradient"):
            frozen(*shape)
