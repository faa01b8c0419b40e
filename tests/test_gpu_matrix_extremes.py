"""The whole-matrix operators past 2^32 elements and past 65535 tasks, and
captured graphs that run side by side."""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - collected on CPU boxes too
    pytest.skip("needs a CUDA device", allow_module_level=True)

from gpu_algos_b200 import glm  # noqa: E402
from tests import ortho_bits as ob  # noqa: E402
from tests.test_gpu_q4 import _check_predict, _equal, _values  # noqa: E402

BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def _room():
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 80 GB free")
    yield
    torch.cuda.empty_cache()


def _randn(shape, seed, dtype=torch.float32):
    return torch.randn(shape, device="cuda", dtype=dtype, generator=torch.Generator(device="cuda").manual_seed(seed))


def test_models_past_2_to_the_32_weights():
    nt, nf, group = 110000, 40000, 128
    M = _randn((1, nt, nf), 51, BF16)
    q = glm.quantize_q4(M, group)
    W = glm.dequantize_q4(q)
    rows = torch.cat([torch.arange(0, 8), torch.arange(53680, 53700), torch.arange(107366, 107382),
                      torch.arange(nt - 24, nt)]).cuda()  # about 2^31 and 2^32 elements in, and the ends
    part = M[:, rows].contiguous()
    assert _equal(W[:, rows], _values(part, group).to(BF16))
    del W
    for nobs in (1, 12, 40):
        X = _randn((nobs, 1, nf), 52, BF16)
        _check_predict(glm.predict_q4(X, q)[:, :, rows], X, part, group)


@pytest.mark.parametrize("dtype,nf", [(BF16, 64), (torch.float32, 72)])
def test_predictions_past_2_to_the_32(dtype, nf):
    nobs, nt, group = 66000, 66000, 64
    M, X = _randn((1, nt, nf), 53, dtype), _randn((nobs, 1, nf), 54, dtype)
    Y = glm.predict_q4(X, glm.quantize_q4(M, group))
    obs = torch.cat([torch.arange(0, 3), torch.arange(32530, 32545), torch.arange(65070, 65080),
                     torch.arange(nobs - 5, nobs)]).cuda()
    _check_predict(Y[obs], X[obs], M, group)


def test_matrices_past_2_to_the_32_entries():
    shape = (2, 40, 56_000_000)
    G = torch.empty(shape, device="cuda", dtype=BF16)
    for t in range(2):
        G[t] = _randn(shape[1:], 55 + t, BF16)
    out = glm.orthogonalize(G)
    for t in range(2):
        # O = P X with P a polynomial of X X^T, which is summed in pieces
        gram = torch.zeros(40, 40, device="cuda", dtype=torch.float64)
        for c in G[t].split(4_000_000, 1):
            gram += c.double() @ c.double().T
        norm = math.sqrt(float(gram.diagonal().sum()))
        A, P = gram / norm**2, torch.eye(40, device="cuda", dtype=torch.float64)
        eye = P.clone()
        for a, b, c in ob.DEFAULT:
            Q = a * eye + b * A + c * A @ A
            A, P = Q @ A @ Q, Q @ P
        # An entry of X X^T is a sum of 875 thousand blocks over sixteen CTAs, in float registers: 55 thousand
        # additions each off by 2^-24 of the sum at most.  X has sigma = 1/sqrt(40) throughout, so the steps turn a
        # relative error of X X^T into |sigma F'(sigma) / F(sigma)| / 2 of it in O, F the whole chain.
        x = torch.tensor(40 ** -0.5, dtype=torch.float64, requires_grad=True)
        F = x
        for a, b, c in ob.DEFAULT:
            F = a * F + b * F**3 + c * F**5
        F.backward()
        grown = abs(float((x * x.grad / F).detach())) / 2 * 875e3 / 16 * 2.0**-24
        for lo in (0, 27_999_000, 53_687_000, 55_999_000):
            ref = P @ G[t][:, lo:lo + 1000].double() / norm
            err = (out[t][:, lo:lo + 1000].double() - ref).norm(dim=0)
            assert bool((err <= (torch.finfo(BF16).eps / 2 + grown) * ref.norm(dim=0)).all())


@pytest.mark.parametrize("dtype", [torch.float32, BF16])
def test_many_tasks(dtype):
    ntasks = 140001
    M, X = _randn((ntasks, 3, 9), 56, dtype), _randn((2, ntasks, 9), 57, dtype)
    q = glm.quantize_q4(M, 64)
    assert _equal(glm.dequantize_q4(q), _values(M, 64).to(dtype))
    _check_predict(glm.predict_q4(X, q), X, M, 64)
    X = _randn((20, ntasks, 9), 58, dtype)
    _check_predict(glm.predict_q4(X, q), X, M, 64)
    out = glm.orthogonalize(M)
    for t in (0, 1, 65534, 65535, 65536, 131070, 131071, ntasks - 1):
        ref = ob.definition(M[t], ob.DEFAULT)
        limit = ob.bound(ref, ob.plain(M[t], ob.DEFAULT)) + torch.finfo(dtype).eps / 2 * float(ref.norm())
        assert float((out[t].double() - ref).norm()) <= limit


def test_captured_training_and_serving_side_by_side():
    """One graph updates a model and quantises it, another predicts from a
    second model meanwhile; each has its own workspace and stream."""
    nt, nf, nobs = 300, 520, 50
    M, V, grad = _randn((1, nt, nf), 59) / 8, torch.zeros(1, nt, nf, device="cuda"), _randn((1, nt, nf), 60)
    served, X = glm.quantize_q4(_randn((1, nt, nf), 61), 64), _randn((nobs, 1, nf), 62)
    trained = glm.quantize_q4(M, 64)
    Y = torch.empty(nobs, 1, nt, device="cuda")
    ws = [torch.empty(n, dtype=torch.uint8, device="cuda")
          for n in (glm.orthogonal_workspace_bytes(torch.float32, nf, nt, 1),
                    glm.predict_q4_workspace_bytes(torch.float32, nf, nt, 1, nobs, 64))]
    M2, V2 = M.clone(), V.clone()
    streams, graphs = [torch.cuda.Stream(), torch.cuda.Stream()], [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    torch.cuda.synchronize()
    with torch.cuda.graph(graphs[0], stream=streams[0]):
        glm.orthogonal_step(M, grad, V, 0.1, workspace=ws[0])
        glm.quantize_q4(M, 64, out=trained)
    with torch.cuda.graph(graphs[1], stream=streams[1]):
        glm.predict_q4(X, served, out=Y, workspace=ws[1])
    expected = glm.predict_q4(X, served)
    for _ in range(5):
        glm.orthogonal_step(M2, grad, V2, 0.1)
        Y.zero_()
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                for _ in range(1 if graph is graphs[0] else 20):
                    graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(Y, expected) and torch.equal(M, M2) and torch.equal(V, V2)
        assert _equal(glm.dequantize_q4(trained), _values(M2, 64).float())
