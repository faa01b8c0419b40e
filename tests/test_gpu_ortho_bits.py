"""The orthogonalisation to the bits its planes carry (tests/ortho_bits.py has
the bound and its reasons, tests/test_ortho_bits.py that it sees a single
missing plane), over every way the products are cut; the 16-bit types are the
float result of the same matrix, rounded once."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - collected on CPU boxes too
    pytest.skip("needs a CUDA device", allow_module_level=True)

from gpu_algos_b200 import glm  # noqa: E402
from tests import ortho_bits as ob  # noqa: E402

SHAPES = [(2, 16, 256), (1, 31, 5000), (2, 33, 40), (1, 40, 33), (1, 48, 48), (1, 64, 100), (1, 65, 64), (1, 100, 64),
          (1, 129, 257), (1, 200, 200), (2, 300, 77), (1, 256, 1024), (1, 511, 640), (3, 1021, 333), (1, 1024, 520),
          (1, 2500, 40), (5, 96, 4100), (1, 1300, 2600), (1, 2600, 1300), (1, 100, 9000), (1, 9000, 100),
          (2, 600, 640), (40, 130, 140), (1, 256, 4096), (1, 1000, 777), (1, 2048, 8192), (1, 4096, 2304)]


@pytest.fixture(autouse=True)
def _plain_float32():
    was = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    yield
    torch.backends.cuda.matmul.allow_tf32 = was


def _matrices(shape, kind, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ntasks, nt, nf = shape
    noise = torch.randn(shape, device="cuda", generator=g)
    if kind == "noise":
        return noise
    r = min(8, nt, nf)
    return (0.1 * torch.randn(ntasks, nt, r, device="cuda", generator=g)
            @ torch.randn(ntasks, r, nf, device="cuda", generator=g) + 0.1 * noise)


@pytest.mark.parametrize("schedule", ob.SCHEDULES)
@pytest.mark.parametrize("kind", ["noise", "gradient"])
@pytest.mark.parametrize("shape", SHAPES)
def test_float_result_and_its_rounding(shape, kind, schedule):
    coefs = ob.SCHEDULES[schedule]
    G = _matrices(shape, kind, 41)
    out = glm.orthogonalize(G, steps=len(coefs), coefficients=coefs)
    for o, g in zip(out, G):
        ref = ob.definition(g, coefs)
        assert float((o.double() - ref).norm()) <= ob.bound(ref, ob.plain(g, coefs))
    for dtype in (torch.float16, torch.bfloat16):
        g16 = G.to(dtype)
        wide = glm.orthogonalize(g16.float(), steps=len(coefs), coefficients=coefs)
        assert torch.equal(glm.orthogonalize(g16, steps=len(coefs), coefficients=coefs), wide.to(dtype))


@pytest.mark.parametrize("shape", [(48, 300), (140, 200), (77, 640), (600, 2000)])
def test_features_of_small_scale(shape):
    U = _matrices((1, *shape), "noise", 42)
    U[:, :, ::3] *= 1e-8
    U[:, :, 1::3] *= 1e-5
    out = glm.orthogonalize(U)[0].double()
    ref, pl = ob.definition(U[0], ob.DEFAULT), ob.plain(U[0], ob.DEFAULT).double()
    limit = (4.0 * (pl - ref).norm(dim=0) + 2.0**-20 * ref.norm(dim=0)
             + ob.small_entries_bound(shape[0], ob.DEFAULT))
    assert bool(((out - ref).norm(dim=0) <= limit).all())
