"""Orthogonalisation and the Muon transition in the kernels that large and many matrices take: pairs of blocks,
mirrored tiles, split sums, several launches.  Reference, measure and tolerances are those of
test_gpu_orthogonalize.py.
"""

import pytest
import torch

from test_gpu_orthogonalize import BAR, BF16, DEV, F16, F32, FP32_BAR, _matrix, _off, _reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n", [(4096, 4096), (1536, 2048), (2500, 1100)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_pairs_of_blocks_give_the_same_bits(m, n, dtype):
    """Every operand that one block of a pair fetches is in place before the other block's products read it."""
    from pbg_b200.optim import orthogonalize, orthogonalize_error

    gen = torch.Generator(device=DEV).manual_seed(m + n)
    x = _matrix("low", m, n, gen).to(dtype)
    got = orthogonalize(x)
    for _ in range(10):
        other = orthogonalize(torch.randn(700, 900, generator=gen, device=DEV))  # other operands in the same shared memory
        assert bool(other.isfinite().all())
        assert torch.equal(got, orthogonalize(x))
    assert orthogonalize_error(DEV) == 0
