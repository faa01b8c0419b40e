"""Models in 4 bits: quantisation, its inverse, and prediction from the codes,
against the definitions in float64.

Tolerances.  Codes and scales are exact: the values they stand for have to be
equal to the definition's, rounded once to the type.  A prediction is a sum of
nf products in float; whatever the order, each of the at most nf + 16
additions and scalings is off by at most 2^-23 (tensor cores cut where they
add) of the sum of magnitudes so far, so
|Yhat - Yhat64| <= (nf + 16) 2^-23 sum|x q s| + eps/2 |Yhat64|.
"""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - collected on CPU boxes too
    pytest.skip("needs a CUDA device", allow_module_level=True)

from gpu_algos_b200 import capi, glm  # noqa: E402

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _values(M, group):
    """q*s of the definition, in float64."""
    out = torch.zeros(M.shape, dtype=torch.float64, device=M.device)
    for lo in range(0, M.shape[2], group):
        w = M[:, :, lo:lo + group].double()
        top = w.abs().amax(2, keepdim=True)
        s = (top / 7).to(M.dtype).double()
        s = torch.where(torch.isfinite(w).all(2, keepdim=True), s, math.nan)
        q = torch.where(s > 0, torch.round(w / torch.where(s > 0, s, 1.0)).clamp(-7, 7), torch.zeros_like(w))
        out[:, :, lo:lo + group] = q * s
    return out


def _model(shape, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g)
            * torch.exp(torch.randn(shape[0], shape[1], 1, device="cuda", generator=g))).to(dtype)


def _equal(a, b):
    return bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", [64, 128])
@pytest.mark.parametrize("shape", [(1, 1, 1), (1, 1, 63), (2, 16, 64), (1, 17, 65), (3, 15, 128), (1, 33, 129),
                                   (64, 16, 256), (1, 100, 777), (2, 5, 1000), (1, 300, 192)])
def test_quantize_round_trip(shape, group, dtype):
    M = _model(shape, dtype)
    before = M.clone()
    q = glm.quantize_q4(M, group)
    out = glm.dequantize_q4(q)
    assert torch.equal(M, before)
    assert _equal(out, _values(M, group).to(dtype))
    # again into the same model, on what it stands for
    assert glm.quantize_q4(out, group, out=q) is q
    assert _equal(glm.dequantize_q4(q), _values(out, group).to(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_borders_and_special_values(dtype):
    M = torch.zeros(1, 20, 128, dtype=dtype, device="cuda")
    tiny, top = torch.finfo(dtype).smallest_normal, torch.finfo(dtype).max
    half = torch.arange(128, device="cuda") % 29 / 2.0 - 7.0  # every multiple of 1/2 in -7..7: ties
    M[0, 0] = half.to(dtype)
    M[0, 1] = (half * tiny).to(dtype)
    M[0, 2] = (half / 7.0 * top).to(dtype)
    M[0, 3] = (half * 3.0).to(dtype)
    M[0, 4, 5] = 1.0
    M[0, 5, 5] = math.nan
    M[0, 6, 5] = math.inf
    M[0, 7, 5] = -math.inf
    M[0, 8] = -torch.finfo(dtype).max
    M[0, 9] = (half * tiny * torch.finfo(dtype).eps).to(dtype)  # subnormal: scales that round a lot
    M[0, 10] = (half * tiny * torch.finfo(dtype).eps * 8).to(dtype)
    M[0, 11] = torch.nextafter(half, torch.full_like(half, 100.0)).to(dtype)
    M[0, 12] = torch.nextafter(half, torch.full_like(half, -100.0)).to(dtype)
    M[0, 11, 0] = M[0, 12, 0] = 7.0
    g = torch.Generator(device="cuda").manual_seed(1)
    M[0, 13:] = torch.randn(7, 128, device="cuda", generator=g).to(dtype)
    for group in (64, 128):
        out = glm.dequantize_q4(glm.quantize_q4(M, group))
        assert _equal(out, _values(M, group).to(dtype)), group


def _check_predict(Y, X, M, group):
    W = _values(M, group)
    ref = torch.einsum("otf,tgf->otg", X.double(), W)
    size = torch.einsum("otf,tgf->otg", X.double().abs(), W.abs())
    tol = (X.shape[2] + 16) * 2.0**-23 * size + torch.finfo(Y.dtype).eps / 2 * ref.abs()
    if Y.dtype == torch.float16:
        tol = tol + 2.0**-25  # half a step among the subnormals
    err = (Y.double() - ref).abs()
    assert bool((err <= tol).all()), (tuple(X.shape), tuple(M.shape), group, float((err / (tol + 1e-300)).max()))


def _predict(shape, nobs, dtype, group, seed=0, **kw):
    M = _model(shape, dtype, seed) / 4
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    X = torch.randn(nobs, shape[0], shape[2], device="cuda", generator=g).to(dtype)
    q = glm.quantize_q4(M, group)
    return glm.predict_q4(X, q, **kw), X, M, q


NOBS = [1, 2, 3, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 200, 256, 257, 700]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nobs", NOBS)
def test_predict_over_observations(nobs, dtype):
    for shape, group in (((1, 150, 520), 128), ((2, 40, 333), 64)):
        Y, X, M, _ = _predict(shape, nobs, dtype, group)
        _check_predict(Y, X, M, group)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", [64, 128])
@pytest.mark.parametrize("shape", [(1, 1, 1), (1, 1, 5000), (3, 5, 63), (1, 16, 64), (64, 16, 256), (1, 129, 65),
                                   (2, 1000, 7), (1, 257, 1025), (1, 2048, 512), (5, 130, 192)])
def test_predict_over_models(shape, group, dtype):
    for nobs in (1, 5, 24, 90, 300):
        Y, X, M, _ = _predict(shape, nobs, dtype, group, 2)
        _check_predict(Y, X, M, group)


# longer than shared memory holds at once, more row blocks to a CTA than it takes together, features over clusters
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,nobs", [((1, 2500, 9000), 8), ((1, 2400, 20000), 13), ((1, 16, 70000), 3),
                                        ((1, 40000, 130), 2), ((1, 40000, 130), 16), ((300, 7, 100), 5),
                                        ((3, 700, 12000), 40), ((1, 20, 30000), 200)])
def test_predict_long_and_many(shape, nobs, dtype):
    for group in (64, 128):
        Y, X, M, _ = _predict(shape, nobs, dtype, group, 6)
        _check_predict(Y, X, M, group)


def test_a_copied_model_stands_alone():
    import copy
    import io

    M = _model((1, 40, 200), torch.bfloat16)
    q = glm.quantize_q4(M, 64)
    X = torch.ones(3, 1, 200, device="cuda", dtype=torch.bfloat16)
    Y = glm.predict_q4(X, q)
    twin = copy.deepcopy(q)
    buf = io.BytesIO()
    torch.save(q, buf)
    buf.seek(0)
    loaded = torch.load(buf, weights_only=False)
    glm.quantize_q4(torch.zeros_like(M), 64, out=q)  # the first one is overwritten
    assert torch.equal(glm.predict_q4(X, twin), Y) and torch.equal(glm.predict_q4(X, loaded), Y)
    assert torch.count_nonzero(glm.predict_q4(X, q)) == 0


def test_wrappers_refuse_what_does_not_fit():
    q = glm.quantize_q4(torch.ones(2, 3, 8, device="cuda"), 64)
    before = capi.launch_count()
    X = torch.ones(4, 2, 8, device="cuda")
    for bad in (X.half(), X[:, :1], X[:, :, :4], X.transpose(0, 1).contiguous().transpose(0, 1), X.cpu()):
        with pytest.raises(ValueError):
            glm.predict_q4(bad, q)
    with pytest.raises(ValueError):
        glm.predict_q4(X, q, out=torch.empty(4, 2, 4, device="cuda"))
    with pytest.raises(ValueError):
        glm.predict_q4(X, q, workspace=torch.empty(16, dtype=torch.uint8))
    with pytest.raises(ValueError):
        glm.quantize_q4(torch.ones(2, 3, 8, device="cuda"), 128, out=q)
    with pytest.raises(ValueError):
        glm.dequantize_q4(q, out=torch.empty(2, 3, 8, device="cuda", dtype=torch.float16))
    assert capi.launch_count() == before


def test_predict_without_features_or_observations():
    q = glm.quantize_q4(torch.zeros(2, 3, 0, device="cuda"))
    Y = glm.predict_q4(torch.zeros(4, 2, 0, device="cuda"), q)
    assert tuple(Y.shape) == (4, 2, 3) and torch.count_nonzero(Y) == 0
    q = glm.quantize_q4(torch.ones(2, 3, 8, device="cuda"))
    assert glm.predict_q4(torch.zeros(0, 2, 8, device="cuda"), q).numel() == 0


@pytest.mark.parametrize("nobs", [1, 6, 40, 150])
def test_nan_and_infinity_stay_where_they_belong(nobs):
    for dtype in DTYPES:
        M = _model((1, 50, 200), dtype, 3)
        M[0, 7, 150] = math.nan
        M[0, 20, 3] = math.inf
        X = torch.ones(nobs, 1, 200, device="cuda", dtype=dtype)
        X[0, 0, 10] = math.nan
        Y = glm.predict_q4(X, glm.quantize_q4(M, 64))
        bad = torch.zeros(nobs, 1, 50, dtype=torch.bool, device="cuda")
        bad[0] = True
        bad[:, :, 7] = True
        bad[:, :, 20] = True
        assert torch.equal(torch.isnan(Y), bad)


@pytest.mark.parametrize("nobs", [1, 20, 130])
def test_unaligned_pointers_and_guard_bands(nobs):
    for dtype in DTYPES:
        shape, group = (2, 37, 200), 64
        Y, X, M, q = _predict(shape, nobs, dtype, group, 4)
        buf = torch.zeros(X.numel() + 1, dtype=dtype, device="cuda")
        buf[1:].copy_(X.reshape(-1))
        out = torch.full((Y.numel() + 17,), 77.0, dtype=dtype, device="cuda")
        view = out[1:1 + Y.numel()].view(Y.shape)
        got = glm.predict_q4(buf[1:].view(X.shape), q, out=view)
        _check_predict(got, X, M, group)
        assert bool((out[:1] == 77).all()) and bool((out[1 + Y.numel():] == 77).all())
        mbuf = torch.zeros(M.numel() + 1, dtype=dtype, device="cuda")
        mbuf[1:].copy_(M.reshape(-1))
        q2 = glm.quantize_q4(mbuf[1:].view(M.shape), group)
        assert torch.equal(q2.codes, q.codes) and torch.equal(q2.scales, q.scales)
        dbuf = torch.full((M.numel() + 9,), 77.0, dtype=dtype, device="cuda")
        d = glm.dequantize_q4(q, out=dbuf[1:1 + M.numel()].view(M.shape))
        assert _equal(d, _values(M, group).to(dtype))
        assert float(dbuf[0]) == 77 and bool((dbuf[1 + M.numel():] == 77).all())


@pytest.mark.parametrize("nobs", [1, 12, 50, 260])
def test_workspace_repeats_stream_and_graph(nobs):
    for dtype in DTYPES:
        shape, group = (1, 300, 1000), 128
        Y, X, M, q = _predict(shape, nobs, dtype, group, 5)
        need = glm.predict_q4_workspace_bytes(dtype, 1000, 300, 1, nobs, group)
        ws = torch.full((need + 64,), 0xA5, dtype=torch.uint8, device="cuda")
        assert torch.equal(Y, glm.predict_q4(X, q, workspace=ws[:need]))
        assert bool((ws[need:] == 0xA5).all())
        if need:
            with pytest.raises(capi.GlmbError, match="workspace"):
                glm.predict_q4(X, q, workspace=ws[:need - 1])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        out = glm.predict_q4(X, q, stream=side)
        side.synchronize()
        assert torch.equal(out, Y)
        static_in, static_out = X.clone(), torch.empty_like(Y)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            glm.predict_q4(static_in, q, out=static_out, workspace=ws)
        for _ in range(2):
            static_in.mul_(-0.5)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(static_out, glm.predict_q4(static_in, q))


def test_model_through_the_library():
    """gradient -> orthogonal_step -> quantize_q4 -> predict_q4, as a program
    uses them, each against its definition."""
    from tests.test_gpu_ortho import DEFAULT, _step_reference, _tolerance

    g = torch.Generator(device="cuda").manual_seed(8)
    nobs, ntasks, nt, nf = 500, 2, 24, 160
    X = torch.randn(nobs, ntasks, nf, device="cuda", generator=g)
    truth = torch.randn(ntasks, nt, nf, device="cuda", generator=g) / math.sqrt(nf)
    Y = torch.einsum("otf,tgf->otg", X, truth).contiguous()
    M, V = torch.zeros_like(truth), torch.zeros_like(truth)
    for _ in range(3):
        grad = glm.gradient(X, M, Y, regularize=False)
        exact = 2 * torch.einsum("otg,otf->tgf", torch.einsum("otf,tgf->otg", X.double(), M.double()) - Y.double(),
                                 X.double())
        assert float((grad.double() - exact).norm() / exact.norm()) <= 1e-5  # the library's float gradient
        refM, refV, U, O = _step_reference(M, grad, V, 0.05, 0.9, True, 0.0, 1.0)
        glm.orthogonal_step(M, grad, V, 0.05, mu=0.9)
        for t in range(ntasks):
            tol = 0.05 * _tolerance(U[t], O[t], (DEFAULT,) * 5, torch.float32)
            # 0.05 and 0.9 are rounded to float: 2^-24 of the momentum and of the update
            tol += 2.0**-22 * float(M[t].norm()) + 2.0**-24 * 4 * 0.05 * 485 * float(O[t].norm())
            assert float((M[t].double() - refM[t]).norm()) <= tol
    q = glm.quantize_q4(M, 64)
    assert _equal(glm.dequantize_q4(q), _values(M, 64).float())
    _check_predict(glm.predict_q4(X, q), X, M, 64)
    _check_predict(glm.predict_q4(X[:1].contiguous(), q), X[:1], M, 64)
