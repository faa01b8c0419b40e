"""CPU checks of the bound that the GPU tests hold the orthogonalisation to:
the tensor-core path's arithmetic keeps it with room to spare, and with the low
plane left out of any one term of any product -- a mistake in one descriptor,
say -- it is broken on every shape."""
import pytest

torch = pytest.importorskip("torch")

from tests import ortho_bits as ob  # noqa: E402

SHAPES = [(33, 40), (40, 33), (48, 48), (64, 100), (129, 257), (200, 200), (300, 77), (256, 1024), (96, 4100)]


def _matrix(shape, kind, seed):
    g = torch.Generator().manual_seed(seed)
    noise = torch.randn(*shape, generator=g)
    if kind == "noise":
        return noise
    r = min(8, *shape)
    return 0.1 * torch.randn(shape[0], r, generator=g) @ torch.randn(r, shape[1], generator=g) + 0.1 * noise


@pytest.mark.parametrize("schedule", ob.SCHEDULES)
@pytest.mark.parametrize("kind", ["noise", "gradient"])
@pytest.mark.parametrize("shape", SHAPES)
def test_the_bound_tells_whole_pairs_from_missing_planes(shape, kind, schedule):
    coefs = ob.SCHEDULES[schedule]
    U = _matrix(shape, kind, 3)
    ref = ob.definition(U, coefs)
    limit = ob.bound(ref, ob.plain(U, coefs))

    def err(drop):
        return float((ob.model(U, coefs, drop).double() - ref).norm())

    assert err(None) <= 0.5 * limit
    for product in ob.PRODUCTS:
        for side in ("left", "right"):
            assert err((product, side)) > limit, (product, side)


@pytest.mark.parametrize("shape", [(48, 300), (140, 200), (77, 640)])
def test_features_of_small_scale(shape):
    U = _matrix(shape, "noise", 5)
    U[:, ::3] *= 1e-8
    U[:, 1::3] *= 1e-5
    ref, pl, out = ob.definition(U, ob.DEFAULT), ob.plain(U, ob.DEFAULT), ob.model(U, ob.DEFAULT).double()
    limit = (4.0 * (pl.double() - ref).norm(dim=0) + 2.0**-20 * ref.norm(dim=0)
             + ob.small_entries_bound(shape[0], ob.DEFAULT))
    assert bool(((out - ref).norm(dim=0) <= limit).all())
