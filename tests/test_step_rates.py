"""CPU check: a model update whose rates leave float's range is refused before
any device is touched.  The kernels take mu, 1 - lr*weight_decay and lr*scale
as floats; an infinite one would turn the model into infinities and NaN."""
import pytest

from gpu_algos_b200 import capi

INVALID = capi.GLMB_ERR_INVALID_VALUE
P, Q, R = 0x10000, 0x20000, 0x30000  # never dereferenced: every call here is refused or empty


@pytest.mark.parametrize("sfx", capi.MATRIX)
def test_rates_past_float_are_refused(sfx):
    step = getattr(capi.lib(), f"glmm_orthogonal_step_{sfx}")
    before = capi.launch_count()

    def run(lr=0.1, mu=0.9, wd=0.0, scale=1.0, sizes=(4, 4, 1)):
        return step(P, Q, R, *sizes, lr, mu, wd, scale, 0, None, 5, None, 0, None)

    for kw in ({"mu": 1e39}, {"mu": -1e300}, {"lr": 1e39}, {"lr": 1e30, "scale": 1e30}, {"lr": 1e200, "scale": 1e200},
               {"lr": 1e30, "wd": -1e30, "scale": 0.0}, {"lr": 1e308, "wd": 1e308, "scale": 0.0}):
        assert run(**kw) == INVALID, kw
        assert run(**kw, sizes=(0, 4, 1)) == INVALID, kw  # whatever the sizes
    # the largest that fit are taken (no work: an empty model)
    for kw in ({"mu": 3e38}, {"lr": 1e19, "scale": 1e19}, {"lr": 1e300, "scale": 1e-280, "wd": 1e-280}):
        assert run(**kw, sizes=(0, 4, 1)) == 0, kw
    assert capi.launch_count() == before
