"""More edges of the matrix operators on the GPU: chains in which most SM pairs have no tile, and
what else the size lists of test_gpu_matrix.py do not reach. Bounds as derived there."""
import pytest
import torch

from test_gpu_matrix import ORTHO_TOL, ortho64, rel

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _status_clean():
    from turboadam_b200 import matrix

    yield
    assert matrix.read_status() == 0


# ---------------------------------------------------------------------------
def test_ortho_pairs_without_tiles():
    """Phases of one size of tile list beside phases of another: in a 300 x 9000 matrix the Gram
    matrix's split sum occupies many pairs and its square two, so the other pairs pass a phase with
    nothing to do and take part in the next. Other work on the GPU shifts their warps against each
    other; every repetition gives the same bits and no wait runs out."""
    from turboadam_b200 import orthogonalize

    side = torch.cuda.Stream()
    noise = torch.randn(1 << 24, device="cuda")
    for shape in ((300, 9000), (9000, 300), (64, 20000), (2, 260, 3000)):
        x = torch.randn(*shape, device="cuda")
        first = orthogonalize(x, dtype=torch.float32)
        assert rel(first, ortho64(x)) <= ORTHO_TOL
        torch.cuda.synchronize()
        for i in range(30):
            with torch.cuda.stream(side):
                noise.mul_(1.0)
            assert torch.equal(orthogonalize(x, dtype=torch.float32), first)
