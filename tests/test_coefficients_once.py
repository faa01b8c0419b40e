"""CPU check: coefficients are read once, also where a call enters another
stream's context first, so that an iterator (a schedule's generator) does for
one call with and without ``stream``.  The launch itself is replaced."""
import contextlib

import pytest

torch = pytest.importorskip("torch")

from gpu_algos_b200 import glm  # noqa: E402

ROWS = [(3.0, -4.0, 1.75), (2.0, -1.5, 0.5), (1.875, -1.25, 0.375)]


@pytest.fixture
def launched(monkeypatch):
    calls = []
    monkeypatch.setattr(glm, "_need_on", lambda *a: None)
    monkeypatch.setattr(glm, "_on", lambda device, stream: None if stream is None else contextlib.nullcontext())
    monkeypatch.setattr(glm, "_run", lambda name, sfx, device, args: calls.append((name, args)))
    return calls


@pytest.mark.parametrize("stream", [None, object()])
def test_an_iterator_does(launched, stream):
    G = torch.ones(1, 4, 8)
    flat = [v for row in ROWS for v in row]
    assert glm.orthogonalize(G, 3, iter(ROWS), stream=stream).shape == G.shape
    V = torch.zeros_like(G)
    assert glm.orthogonal_step(G, G, V, 0.1, steps=3, coefficients=(r for r in ROWS), stream=stream) is G
    assert [name for name, _ in launched] == ["glmm_orthogonalize", "glmm_orthogonal_step"]
    assert list(launched[0][1][5]) == flat and list(launched[1][1][11]) == flat
    out = torch.empty_like(G)
    assert glm.orthogonalize(G, 1, (1.5, -0.5, 0.0), out=out, stream=stream) is out
    assert launched[2][1][1] == out.data_ptr() and list(launched[2][1][5]) == [1.5, -0.5, 0.0]
