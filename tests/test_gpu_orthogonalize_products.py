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


@pytest.mark.parametrize("m,n,kind", [(4096, 512, "noise"), (1024, 640, "noise"), (1536, 2048, "noise"), (513, 700, "steep"),
                                      (520, 8000, "noise"), (4096, 4096, "low")])
def test_bf16_outputs_are_fp32_results_rounded_once(m, n, kind):
    """The error is the rounding's own, and what fp32 accuracy may add: FP32_BAR of the result; the rounding of
    so slightly other values is another sample of the same million roundings and more, taken as 1 % apart."""
    from pbg_b200.optim import orthogonalize, orthogonalize_error

    x = _matrix(kind, m, n, torch.Generator(device=DEV).manual_seed(m + 3 * n)).bfloat16()
    ref = _reference(x)
    assert _off(orthogonalize(x), ref) <= 1.01 * _off(ref.bfloat16(), ref) + FP32_BAR
    assert _off(orthogonalize(x, out_dtype=F16), ref) <= BAR[F16]
    assert orthogonalize_error(DEV) == 0
