"""The model update reads the momentum that the same call has just written.

With M = 0, no decay, lr * scale = 1 and no Nesterov term the updated model is
-O(V') exactly, V' the new momentum: the same bits as orthogonalising V' by a
call of its own, which reads it after it has long been written.  A stale
momentum anywhere would show.  Odd row lengths, and tasks that start inside a
32-byte sector, put neighbouring blocks' elements into one sector."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - collected on CPU boxes too
    pytest.skip("needs a CUDA device", allow_module_level=True)

from gpu_algos_b200 import glm  # noqa: E402


@pytest.mark.parametrize("shape", [(1, 40, 51), (7, 35, 37), (3, 131, 77), (1, 1000, 777), (1, 300, 5001), (2, 5001, 67)])
def test_update_sees_the_new_momentum(shape):
    g = torch.Generator(device="cuda").manual_seed(21)
    ntasks, nt, nf = shape
    ws = torch.empty(glm.orthogonal_workspace_bytes(torch.float32, nf, nt, ntasks), dtype=torch.uint8, device="cuda")
    V = torch.randn(shape, device="cuda", generator=g)
    M = torch.empty_like(V)
    for _ in range(40):
        grad = torch.randn(shape, device="cuda", generator=g) * 3.0
        M.zero_()
        before = V.clone()
        glm.orthogonal_step(M, grad, V, 1.0, mu=0.5, nesterov=False, scale=1.0, workspace=ws)
        # mu = 1/2 is exact, so V' = V/2 + g is rounded once on either side
        assert torch.equal(V, (before.double() * 0.5 + grad.double()).float())
        assert torch.equal(M, -glm.orthogonalize(V))
