"""Prediction from 4-bit models near both ends of float's range: sums whose
result is a finite number come out finite and to the usual error, however
large the observations; small ones lose what bfloat16's subnormals cannot hold.

Tolerance, beside the (nf + 16) 2^-23 sum|x q s| + eps/2 |Yhat64| of ordinary
sizes (each of nf products and 16 scalings and joins rounded, or cut, once):
* a float observation is the sum of three bfloat16 terms; bits of it below
  bfloat16's smallest step, 2^-133, are lost: half a step, 2^-134, of each x;
* group sums carry 2^-10 of their value (so that 128 products of up to 7 times
  the largest float stay in range): where a result is below 2^-116 each group
  is rounded to 2^-149 of that, half a step of 2^-139.
"""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - collected on CPU boxes too
    pytest.skip("needs a CUDA device", allow_module_level=True)

from gpu_algos_b200 import glm  # noqa: E402

SHAPES = [((1, 150, 520), 128), ((2, 40, 333), 64), ((1, 40, 9000), 128)]
NOBS = [1, 6, 12, 40, 150]


def _check(X, M, group):
    q = glm.quantize_q4(M, group)
    Y = glm.predict_q4(X, q)
    # q*s in float64; a type's own rounding of q*s would overflow near its end, which prediction does not do
    top = torch.nn.functional.pad(M, (0, -M.shape[2] % group)).double().unflatten(2, (-1, group))
    s = (top.abs().amax(3) / 7).to(M.dtype).double()
    W = (torch.round(top / s[..., None].clamp(min=1e-300)).clamp(-7, 7) * s[..., None]).flatten(2)[..., :M.shape[2]]
    ref = torch.einsum("otf,tgf->otg", X.double(), W)
    size = torch.einsum("otf,tgf->otg", X.double().abs(), W.abs())
    assert float(ref.abs().max()) < torch.finfo(M.dtype).max  # the case asks for finite results
    tol = (X.shape[2] + 16) * 2.0**-23 * size + torch.finfo(Y.dtype).eps / 2 * ref.abs()
    tol = tol + W.abs().sum(2) * 2.0**-134 + s.shape[2] * 2.0**-139
    if Y.dtype != torch.float32:
        tol = tol + torch.finfo(Y.dtype).smallest_normal * torch.finfo(Y.dtype).eps / 2
    assert bool(torch.isfinite(Y).all())
    err = (Y.double() - ref).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


def _randn(shape, seed):
    return torch.randn(shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nobs", NOBS)
def test_large_observations_and_small_scales(nobs, dtype):
    for shape, group in SHAPES:
        # all of one sign with weights of one sign in the first rows: group sums as large as they get
        M = _randn(shape, 31) * 2.0**-20
        M[:, :8] = M[:, :8].abs()
        X = (1.0 + _randn((nobs, shape[0], shape[2]), 32).abs().clamp(max=1.0)) * 2.0**126
        X[0, :, ::3] = torch.finfo(dtype).max
        _check(X.to(dtype), M.to(dtype), group)
        X[:, :, 1::2] *= -1.0
        X[0, :, 1::3] = -torch.finfo(dtype).max
        _check(X.to(dtype), M.to(dtype), group)


@pytest.mark.parametrize("nobs", NOBS)
def test_float_observations_past_bfloat16s_largest(nobs):
    most = torch.finfo(torch.float32).max
    for shape, group in SHAPES:
        X = torch.zeros(nobs, shape[0], shape[2], device="cuda")
        X[:, :, 5] = most
        X[:, :, 70] = -3.3961e38  # bfloat16 would round it to infinity
        _check(X, _randn(shape, 33) * 2.0**-6, group)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("exponent", [-139, -130, -118])
@pytest.mark.parametrize("nobs", NOBS)
def test_small_observations_and_large_scales(nobs, exponent, dtype):
    for shape, group in SHAPES:
        X = (_randn((nobs, shape[0], shape[2]), 34).double() * 2.0**exponent).to(dtype)
        _check(X, (_randn(shape, 35) * 2.0**100).to(dtype), group)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nobs", NOBS)
def test_small_results(nobs, dtype):
    for shape, group in SHAPES:
        X = (_randn((nobs, shape[0], shape[2]), 36) * 2.0**-62).to(dtype)
        _check(X, (_randn(shape, 37) * 2.0**-63).to(dtype), group)
