"""CPU checks of the whole-matrix entry points (include/glm_matrix_b200.h):
declared and exported alike, and invalid arguments refused before any device
is touched, by the C ABI and by the torch wrappers."""
import ctypes
import math
import os
import re
import subprocess

import pytest

from gpu_algos_b200 import capi

torch = pytest.importorskip("torch")

from gpu_algos_b200 import glm  # noqa: E402

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(REPO, "include", "glm_matrix_b200.h")
INVALID, TOO_LARGE = capi.GLMB_ERR_INVALID_VALUE, capi.GLMB_ERR_TOO_LARGE
P, Q, R = 0x10000, 0x20000, 0x30000  # never dereferenced: every call here is refused or empty


def _doubles(*v):
    return (ctypes.c_double * len(v))(*v)


def test_declared_symbols_are_exported():
    src = subprocess.run(["gcc", "-E", "-P", "-x", "c", "-I", os.path.dirname(HEADER), HEADER], check=True,
                         capture_output=True, text=True).stdout
    declared = sorted(set(re.findall(r"\b(glmm_\w+)\s*\(", src)))
    out = subprocess.run(["nm", "-D", "--defined-only", capi.LIB_PATH], check=True, capture_output=True,
                         text=True).stdout
    exported = sorted({line.split()[-1] for line in out.splitlines() if " T glmm_" in line})
    assert declared == exported == sorted(capi.matrix_symbols())
    assert len(declared) == 2 + 7 * 3


@pytest.mark.parametrize("sfx", capi.MATRIX)
def test_orthogonal_refusals(sfx):
    L = capi.lib()
    orth, step = getattr(L, f"glmm_orthogonalize_{sfx}"), getattr(L, f"glmm_orthogonal_step_{sfx}")
    before = capi.launch_count()
    for bad in ((-1, 4, 1), (4, -1, 1), (4, 4, -1)):
        assert orth(P, Q, *bad, None, 5, None, 0, None) == INVALID
    assert orth(None, Q, 4, 4, 1, None, 5, None, 0, None) == INVALID
    assert orth(P, None, 4, 4, 1, None, 5, None, 0, None) == INVALID
    assert orth(P, P + 16, 8, 8, 1, None, 5, None, 0, None) == INVALID        # partial overlap
    assert orth(P, Q, 4, 4, 1, None, 5, R + 8, 1 << 20, None) == INVALID     # workspace alignment
    for steps in (0, -1, 17):
        assert orth(P, Q, 4, 4, 1, None, steps, None, 0, None) == INVALID
    for coef in ((math.nan, 0, 0), (math.inf, 0, 0), (2000.0, 0, 0), (17.0, 0, 0), (1.0, 0, 2000.0)):
        assert orth(P, Q, 4, 4, 1, _doubles(*coef), 1, None, 0, None) == INVALID
    # a schedule whose first step is fine and whose second outgrows the limit
    assert orth(P, Q, 4, 4, 1, _doubles(8.0, 0, 0, 3.0, 0, 0), 2, None, 0, None) == INVALID
    # 7x - 20x^3 + 14x^5 reaches 1.67 at x = 0.37, which the next steps take past 16
    assert orth(P, Q, 4, 4, 1, _doubles(7.0, -20.0, 14.0, 4.0, -6.0, 2.5, 1.875, -1.25, 0.375), 3, None, 0,
                None) == INVALID
    assert orth(P, Q, 1 << 39, 1 << 39, 1, None, 5, None, 0, None) == TOO_LARGE
    # empty problems succeed
    for empty in ((0, 4, 1), (4, 0, 1), (4, 4, 0)):
        assert orth(None, None, *empty, None, 5, None, 0, None) == 0

    def run(lr=0.1, mu=0.9, wd=0.0, scale=1.0, flags=0, M=P, g=Q, V=R, steps=5):
        return step(M, g, V, 4, 4, 1, lr, mu, wd, scale, flags, None, steps, None, 0, None)

    for kw in ({"lr": math.nan}, {"mu": math.inf}, {"wd": math.nan}, {"scale": -math.inf}, {"flags": 2}, {"M": None},
               {"g": None}, {"V": None}, {"g": P}, {"V": P}, {"V": Q + 4}, {"steps": 0}):
        assert run(**kw) == INVALID, kw
    assert step(None, None, None, 4, 0, 1, 0.1, 0.9, 0.0, 1.0, 0, None, 5, None, 0, None) == 0
    assert capi.launch_count() == before


@pytest.mark.parametrize("sfx", capi.MATRIX)
def test_q4_refusals(sfx):
    L = capi.lib()
    quant, deq, pred = (getattr(L, f"glmm_{n}_{sfx}") for n in ("quantize_q4", "dequantize_q4", "predict_q4"))
    before = capi.launch_count()
    for f in (quant, deq):
        assert f(P, Q, R, -1, 4, 1, 64, None) == INVALID
        for group in (0, 32, 65, 256, -64):
            assert f(P, Q, R, 4, 4, 1, group, None) == INVALID
        for args in ((None, Q, R), (P, None, R), (P, Q, None)):
            assert f(*args, 4, 4, 1, 64, None) == INVALID
        assert f(None, None, None, 0, 4, 1, 64, None) == 0
        assert f(P, Q, R, 1 << 39, 1 << 39, 1, 64, None) == TOO_LARGE
        for args in ((P, P, R), (P, P + 16, R), (P, Q, P), (P, Q, P + 28), (P, Q, Q + 16)):
            assert f(*args, 4, 4, 1, 64, None) == INVALID          # overlaps
    assert quant(Q + 960, Q, R, 4, 4, 1, 64, None) == INVALID  # the weights end inside the codes
    assert deq(P, Q, P + 992, 4, 4, 1, 64, None) == INVALID
    assert quant(P, Q + 8, R, 4, 4, 1, 64, None) == INVALID   # codes alignment
    assert deq(P + 8, Q, R, 4, 4, 1, 64, None) == INVALID
    Y = 0x90000
    assert pred(P, Q, R, Y, 4, 4, 1, -1, 64, None, 0, None) == INVALID
    assert pred(P, Q, R, Y, 4, 4, 1, 2, 96, None, 0, None) == INVALID
    for args in ((None, Q, R, Y), (P, None, R, Y), (P, Q, None, Y), (P, Q, R, None), (P, Q, R, P), (P, Q + 4, R, Y),
                 (P, Q, R, Q + 16), (P, Q, R, R), (P, Q, Q + 512, Y)):
        assert pred(*args, 4, 4, 1, 2, 64, None, 0, None) == INVALID
    assert pred(P, Q, R, Y, 4, 4, 1, 2, 64, R + 16, 1 << 20, None) == INVALID
    for nf, nt, ntasks, nobs in ((4, 0, 1, 2), (4, 4, 0, 2), (4, 4, 1, 0)):
        assert pred(None, None, None, None, nf, nt, ntasks, nobs, 64, None, 0, None) == 0
    assert capi.launch_count() == before


def test_q4_sizes():
    L = capi.lib()
    # 16 x 64 blocks of 512 bytes; scales padded to 16 targets; features to a multiple of 128
    assert L.glmm_q4_codes_bytes(256, 16, 64) == 64 * 4 * 512
    assert L.glmm_q4_codes_bytes(65, 17, 1) == 2 * 2 * 512
    assert L.glmm_q4_scales_count(65, 17, 3, 64) == 3 * 32 * 2
    assert L.glmm_q4_scales_count(129, 1, 1, 128) == 16 * 2
    assert L.glmm_q4_codes_bytes(8, 4, 1) == 2 * 512 and L.glmm_q4_scales_count(8, 4, 1, 64) == 16 * 2
    assert L.glmm_q4_codes_bytes(0, 4, 1) == 0 and L.glmm_q4_codes_bytes(-1, 4, 1) == 0
    assert L.glmm_q4_scales_count(64, 4, 1, 32) == 0


def test_wrappers_refuse_before_any_launch():
    cpu = torch.zeros(1, 4, 8)
    before = capi.launch_count()
    with pytest.raises(ValueError, match="CUDA"):
        glm.orthogonalize(cpu)
    with pytest.raises(ValueError, match="CUDA"):
        glm.orthogonal_step(cpu, cpu, cpu, 0.1)
    with pytest.raises(ValueError, match="CUDA"):
        glm.quantize_q4(cpu)
    with pytest.raises(ValueError, match="float64"):
        glm.orthogonalize(cpu.double())
    with pytest.raises(ValueError, match="int8"):
        glm.quantize_q4(cpu.to(torch.int8))
    with pytest.raises(ValueError, match="ntargets"):
        glm.orthogonalize(cpu[0])
    with pytest.raises(ValueError, match="group"):
        glm.Q4Model((1, 4, 8), torch.float32, 32, "cpu")
    model = glm.Q4Model((1, 4, 8), torch.float32, 64, "cpu")
    assert model.codes.numel() == 1024 and model.scales.numel() == 32 and model.device.type == "cpu"
    with pytest.raises(ValueError, match="CUDA"):
        glm.predict_q4(torch.zeros(2, 1, 8), model)
    assert capi.launch_count() == before


def test_coefficients_argument():
    one = glm._coefficients((1.5, -0.5, 0.0), 3)
    assert list(one) == [1.5, -0.5, 0.0] * 3
    many = glm._coefficients([(2, -1.5, 0.5), (1.5, -0.5, 0)], 2)
    assert list(many) == [2.0, -1.5, 0.5, 1.5, -0.5, 0.0]
    assert glm._coefficients(None, 5) is None
    for bad in ([(1, 2, 3)], [(1, 2)] * 2, (1, 2)):
        with pytest.raises((ValueError, TypeError)):
            glm._coefficients(bad, 2)
