"""Newton-Schulz orthogonalisation and the model update built on it, against
the same steps in float64.

Tolerance.  A step's products are exact to about 2^-20 of their operands'
size (two operands of at least 22 bits, sums of at least float precision), and a
perturbation of X before the remaining steps is multiplied by at most the
largest slope of the polynomials that follow, |P'|, over the singular values
between 0 and |X|_2.  So  |O - O64|_F <= steps * 2^-19 * amp * s1 * sqrt(m)
with s1 the largest singular value of X0, amp the largest slope of the whole
chain over [0, s1] (2^-19: a factor 2 for the products' terms b and c), m the
shorter side; plus half a step of the output's rounding, eps/2 * |O64|_F.
"""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - collected on CPU boxes too
    pytest.skip("needs a CUDA device", allow_module_level=True)

from gpu_algos_b200 import capi, glm  # noqa: E402

DEFAULT = (3.4445, -4.7750, 2.0315)
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _reference(G, coefs):
    out = []
    for T in G.double():
        n = T.norm()
        X = T / n if float(n) != 0 else T
        tall = X.shape[0] > X.shape[1]
        X = X.T if tall else X
        for a, b, c in coefs:
            A = X @ X.T
            X = a * X + (b * A + c * (A @ A)) @ X
        out.append(X.T if tall else X)
    return torch.stack(out)


def _tolerance(T, ref, coefs, dtype):
    """Frobenius bound of one task's error."""
    n = float(T.double().norm())
    if n == 0:
        return 0.0
    s1 = float(torch.linalg.matrix_norm(T.double() / n, 2))
    x = torch.linspace(0, s1, 20001, dtype=torch.float64)
    slope = torch.ones_like(x)
    for a, b, c in coefs:
        slope = slope * (a + 3 * b * x**2 + 5 * c * x**4).abs()
        x = a * x + b * x**3 + c * x**5
    amp = max(1.0, float(slope.max()))
    m = min(T.shape)
    return (len(coefs) * 2.0**-19 * amp * s1 * math.sqrt(m)
            + torch.finfo(dtype).eps / 2 * float(ref.norm()))


def _check(out, G, coefs=(DEFAULT,) * 5):
    ref = _reference(G, coefs)
    for o, r, g in zip(out, ref, G):
        err = float((o.double() - r).norm())
        assert err <= _tolerance(g, r, coefs, out.dtype), (tuple(G.shape), err, float(r.norm()))


def _gradient(shape, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ntasks, nt, nf = shape
    r = max(1, min(nt, nf, 8))
    strong = torch.randn(ntasks, nt, r, device="cuda", generator=g) @ torch.randn(ntasks, r, nf, device="cuda",
                                                                                  generator=g)
    return (0.1 * strong + 0.1 * torch.randn(ntasks, nt, nf, device="cuda", generator=g)).to(dtype)


SHAPES = [(1, 1, 1), (1, 1, 8), (3, 1, 300), (2, 5, 1), (64, 16, 256), (2, 16, 16), (1, 17, 33), (2, 33, 40),
          (1, 31, 5000), (70, 3, 7), (1, 48, 48), (1, 64, 100), (1, 65, 64), (1, 129, 257), (1, 200, 200),
          (2, 300, 77), (1, 256, 1024), (1, 511, 640), (3, 1021, 333), (1, 1024, 520), (1, 2500, 40), (5, 96, 4100)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_shapes(shape, dtype):
    G = _gradient(shape, dtype)
    before = G.clone()
    out = glm.orthogonalize(G)
    _check(out, G)
    assert torch.equal(G, before)


# tiles of pairs, K over clusters of sixteen and over two halves, and their tall counterparts
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1300, 2600), (1, 2600, 1300), (1, 100, 9000), (1, 9000, 100), (2, 600, 640),
                                   (40, 130, 140)])
def test_cuts(shape, dtype):
    G = _gradient(shape, dtype, 12)
    _check(glm.orthogonalize(G), G)


def test_wrappers_refuse_what_does_not_fit():
    G = torch.ones(2, 40, 50, device="cuda")
    before = capi.launch_count()
    for bad in (G.transpose(1, 2), G[:, ::2], G.cpu(), G[0], G.double()):
        with pytest.raises(ValueError):
            glm.orthogonalize(bad)
    with pytest.raises(ValueError):
        glm.orthogonalize(G, out=torch.empty(2, 50, 40, device="cuda"))
    with pytest.raises(ValueError):
        glm.orthogonal_step(G, G.half(), torch.zeros_like(G), 0.1)
    with pytest.raises(ValueError):
        glm.orthogonal_step(G, torch.ones_like(G), torch.zeros_like(G).half(), 0.1)
    with pytest.raises(capi.GlmbError):
        glm.orthogonal_step(G, G, torch.zeros_like(G), 0.1)  # the gradient is the model
    with pytest.raises(capi.GlmbError):
        glm.orthogonalize(G, steps=0)
    assert capi.launch_count() == before


@pytest.mark.parametrize("shape", [(2, 16, 100), (2, 150, 130), (1, 700, 300)])
@pytest.mark.parametrize("coefs", [[(1.5, -0.5, 0.0)] * 3, [(2.0, -1.5, 0.5)] * 12, [DEFAULT],
                                   [(3.0, -4.0, 1.75), (2.0, -1.5, 0.5), (1.875, -1.25, 0.375)],
                                   [(1.0, 0.0, 0.0)] * 16])
def test_coefficients(shape, coefs):
    G = _gradient(shape, torch.float32, 1)
    out = glm.orthogonalize(G, steps=len(coefs), coefficients=coefs)
    _check(out, G, coefs)


@pytest.mark.parametrize("shape", [(4, 8, 50), (4, 140, 200)])
def test_zero_nan_and_infinite_tasks(shape):
    for dtype in DTYPES:
        G = _gradient(shape, dtype, 2)
        G[1] = 0
        G[2, 3, 5] = math.nan
        G[3, 0, 0] = math.inf
        out = glm.orthogonalize(G)
        _check(out[:1], G[:1])
        assert torch.count_nonzero(out[1]) == 0
        assert torch.isnan(out[2]).all() and torch.isnan(out[3]).all()


@pytest.mark.parametrize("shape", [(1, 8, 50), (1, 140, 200), (1, 200, 140)])
@pytest.mark.parametrize("rank", [1, 3])
def test_low_rank(shape, rank):
    g = torch.Generator(device="cuda").manual_seed(3)
    _, nt, nf = shape
    G = (torch.randn(1, nt, rank, device="cuda", generator=g) @ torch.randn(1, rank, nf, device="cuda", generator=g))
    _check(glm.orthogonalize(G), G)


@pytest.mark.parametrize("shape", [(1, 8, 50), (1, 140, 200)])
@pytest.mark.parametrize("magnitude", [1e-36, 1e-20, 1e18, 1e36])
def test_magnitude_does_not_matter(shape, magnitude):
    G = _gradient(shape, torch.float32, 4)
    big = G * magnitude
    _check(glm.orthogonalize(big), big)
    half = (_gradient(shape, torch.float16, 4) * 60000.0).clamp(-65504, 65504)
    _check(glm.orthogonalize(half), half)


@pytest.mark.parametrize("shape", [(2, 16, 100), (1, 300, 130), (1, 130, 300)])
def test_in_place_repeats_and_workspace(shape):
    for dtype in DTYPES:
        G = _gradient(shape, dtype, 5)
        out = glm.orthogonalize(G)
        ntasks, nt, nf = shape
        need = glm.orthogonal_workspace_bytes(dtype, nf, nt, ntasks)
        ws = torch.full((need + 64,), 0xA5, dtype=torch.uint8, device="cuda")
        again = glm.orthogonalize(G, workspace=ws[:need])
        assert torch.equal(out, again)  # no order of sums depends on timing
        assert bool((ws[need:] == 0xA5).all())
        if need:
            with pytest.raises(capi.GlmbError, match="workspace"):
                glm.orthogonalize(G, workspace=ws[:need - 1])
        inplace = G.clone()
        assert glm.orthogonalize(inplace, out=inplace) is inplace
        assert torch.equal(out, inplace)


def _step_reference(M, g, V, lr, mu, nesterov, wd, scale, coefs=(DEFAULT,) * 5):
    V = (V.double() * mu + g.double()).float()
    U = g.float().double() + mu * V.double() if nesterov else V.double()
    O = _reference(U, coefs)
    return M.double() * (1 - lr * wd) - lr * scale * O, V, U, O


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("shape", [(1, 1, 5), (64, 16, 256), (2, 33, 17), (1, 100, 777), (2, 777, 100), (1, 300, 512)])
def test_step(shape, nesterov, dtype):
    g = torch.Generator(device="cuda").manual_seed(6)
    grad = _gradient(shape, dtype, 6)
    M = torch.randn(shape, device="cuda", generator=g).to(dtype)
    V = torch.randn(shape, device="cuda", generator=g)
    lr, mu, wd = 0.25, 0.9375, 0.125  # exact in float
    scale = math.sqrt(max(1.0, shape[1] / shape[2]))
    refM, refV, U, O = _step_reference(M, grad, V, lr, mu, nesterov, wd, scale)
    oldM = M.clone()
    assert glm.orthogonal_step(M, grad, V, lr, mu=mu, nesterov=nesterov, weight_decay=wd) is M
    # one product and one sum, each rounded once at most
    assert torch.all((V.double() - refV.double()).abs() <= 2.0**-22 * (refV.double().abs() + grad.double().abs()))
    for t in range(shape[0]):
        tol = lr * scale * _tolerance(U[t], O[t], (DEFAULT,) * 5, torch.float32)
        tol += (torch.finfo(dtype).eps / 2 + 2.0**-22) * float(refM[t].norm() + oldM[t].double().norm())
        assert float((M[t].double() - refM[t]).norm()) <= tol


def test_step_of_a_zero_gradient_only_decays():
    M = torch.ones(2, 40, 50, device="cuda")
    Z = torch.zeros_like(M)
    V = torch.zeros_like(M)
    glm.orthogonal_step(M, Z, V, 0.5, weight_decay=0.5)
    assert torch.equal(M, torch.full_like(M, 0.75)) and torch.count_nonzero(V) == 0


@pytest.mark.parametrize("shape", [(2, 16, 100), (1, 300, 130)])
def test_stream_and_graph(shape):
    G = _gradient(shape, torch.float32, 7)
    ref = glm.orthogonalize(G)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out = glm.orthogonalize(G, stream=side)
    side.synchronize()
    assert torch.equal(out, ref)
    # captured and replayed on new data, with the caller's workspace and without
    ntasks, nt, nf = shape
    for ws in (torch.empty(max(1, glm.orthogonal_workspace_bytes(G.dtype, nf, nt, ntasks)), dtype=torch.uint8,
                           device="cuda"), None):
        static_in, static_out = G.clone(), torch.empty_like(G)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            glm.orthogonalize(static_in, out=static_out, workspace=ws)
        for seed in (8, 9):
            static_in.copy_(_gradient(shape, torch.float32, seed))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(static_out, glm.orthogonalize(static_in))


def test_two_calls_side_by_side():
    a, b = _gradient((1, 600, 500), torch.float32, 10), _gradient((1, 500, 600), torch.bfloat16, 11)
    ra, rb = glm.orthogonalize(a), glm.orthogonalize(b)
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = [(glm.orthogonalize(a, stream=sa), glm.orthogonalize(b, stream=sb)) for _ in range(4)]
    torch.cuda.synchronize()
    for oa, ob in outs:
        assert torch.equal(oa, ra) and torch.equal(ob, rb)
