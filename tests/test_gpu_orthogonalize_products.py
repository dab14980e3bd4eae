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


def _fp32_products(x):
    x = x.float()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / (torch.linalg.matrix_norm(x.double()).float() + 1e-7)
    for _ in range(5):
        g = x @ x.mT
        x = 3.4445 * x + (-4.7750 * g + 2.0315 * (g @ g)) @ x
    return x.mT if tall else x


@pytest.mark.parametrize("m,n", [(1, 1), (1, 7), (1, 300), (3, 2), (3, 500), (9, 64), (64, 64), (65, 130), (128, 384), (1, 4096),
                                 (5000, 3), (20, 3000), (129, 257), (256, 1024), (200, 5000), (1024, 640)])
def test_errors_are_those_of_fp32_products(m, n):
    """Pairs of fp16 numbers hold 22 bits, operands 2^-23 off where fp32's are 2^-24: twice the error of fp32 products
    at most, on average over matrices (a single small one may by chance come out exact in fp32)."""
    from pbg_b200.optim import orthogonalize

    allowed = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        ours = theirs = 0.0
        for seed in range(24 if m * n < 5000 else 6):
            x = _matrix("low" if seed % 3 == 2 else "noise", m, n, torch.Generator(device=DEV).manual_seed(1000 + seed))
            ref = _reference(x)
            ours, theirs = ours + _off(orthogonalize(x), ref), theirs + _off(_fp32_products(x), ref)
    finally:
        torch.backends.cuda.matmul.allow_tf32 = allowed
    assert ours <= 2.0 * theirs


@pytest.mark.parametrize("m,n", [(1, 5), (64, 200), (128, 1600), (200, 300), (1536, 2048)])
def test_zeros_without_an_epsilon(m, n):
    """A matrix of zeros gives zeros, and moves its master by the decay alone, where epsilon is 0 too."""
    from pbg_b200.optim import FlatMuon, orthogonalize

    x = torch.zeros(2, m, n, device=DEV)
    x[1].normal_(generator=torch.Generator(device=DEV).manual_seed(m))
    got = orthogonalize(x, epsilon=0.0)
    assert bool((got[0] == 0).all())
    assert _off(got[1], _reference(x[1], eps=0.0)) <= FP32_BAR
    x[0, 0, 1] = float("nan")
    assert bool(orthogonalize(x[0], epsilon=0.0).isnan().all())
    master = torch.randn(2 * m * n, generator=torch.Generator(device=DEV).manual_seed(n), device=DEV)
    step = FlatMuon(master, [(0, m, n), (m * n, m, n)], epsilon=0.0, lr=0.5, decay=0.5)
    before = master.clone()
    step.grad[m * n:].copy_(x[1].flatten())
    step.step()
    assert int(step.skipped) == 0 and bool(master.isfinite().all())
    assert torch.equal(master[:m * n], 0.75 * before[:m * n]) and not torch.equal(master[m * n:], 0.75 * before[m * n:])


@pytest.mark.parametrize("m,n", [(200, 300), (192, 192), (256, 8192), (1536, 2048), (300, 170)])
@pytest.mark.parametrize("steps,k", [(1, (3.4445, -4.7750, 2.0315)), (4, (3.4445, -4.7750, 2.0315)), (12, (1.5, -0.5, 0.0)),
                                     (10, (1.875, -1.25, 0.375)), (6, (2.0, -1.5, 0.5)), (3, (1.0, 0.0, 0.0)),
                                     (2, (0.5, 0.25, 0.125))])
def test_polynomials_and_step_counts(m, n, steps, k):
    """Single blocks, an odd number of 64-wide blocks, split sums and pairs, with and without a square."""
    from pbg_b200.optim import orthogonalize, orthogonalize_error

    x = _matrix("low", m, n, torch.Generator(device=DEV).manual_seed(m + n))
    ref = _reference(x, steps, 0.5, k)
    for dtype in (F32, BF16):
        got = orthogonalize(x, steps=steps, coefficients=k, epsilon=0.5, out_dtype=dtype)
        assert _off(got, ref) <= BAR[dtype]
    assert orthogonalize_error(DEV) == 0


def test_a_batch_of_more_tiles_than_one_launch_works_in():
    """18 matrices of 2,048 x 2,048: 69 MB of tiles each, 15 a launch within 1 GB."""
    from pbg_b200.optim import orthogonalize, orthogonalize_error

    gen = torch.Generator(device=DEV).manual_seed(11)
    x = torch.randn(18, 2048, 2048, generator=gen, device=DEV)
    got = orthogonalize(x)
    for i in (0, 14, 15, 17):
        assert _off(got[i], _reference(x[i])) <= FP32_BAR
    for i in (3, 16):
        assert _off(got[i], orthogonalize(x[i]).double()) <= 2 * FP32_BAR  # another tile shape may serve one matrix
    assert torch.equal(got, orthogonalize(x)) and orthogonalize_error(DEV) == 0


def test_a_transition_of_more_tiles_than_one_launch_works_in():
    """Launches of their own for what passes 1 GB, one matrix with split sums, and teams, in one list."""
    from pbg_b200.optim import FlatMuon, orthogonalize_error

    gen = torch.Generator(device=DEV).manual_seed(12)
    sizes = [(2048, 2048)] * 17 + [(256, 8192), (100, 300), (300, 64), (130, 131)]
    mats, at = [], 0
    for r, c in sizes:
        mats.append((at, r, c))
        at += (r * c + 3) // 4 * 4
    step = FlatMuon(torch.randn(at, generator=gen, device=DEV), mats, lr=0.05, momentum=0.9, decay=0.1)
    assert int(step._plan[2]) >= 2
    twin = FlatMuon(step.master.clone(), mats, lr=0.05, momentum=0.9, decay=0.1)
    for _ in range(2):
        step.grad.normal_(generator=gen)
        twin.grad.copy_(step.grad)
        before, old = step.master.clone(), step.momentum.clone()
        step.step(), twin.step()
        assert int(step.skipped) == 0 and torch.equal(step.master, twin.master)
        for i in (0, 13, 14, 15, 16, 17, 18, 19, 20):
            o, r, c = mats[i]
            s = slice(o, o + r * c)
            w, m, g = before[s].double(), old[s].double(), step.grad[s].double()
            m = 0.9 * m + 0.1 * g
            f = 0.05 * max(1.0, r / c) ** 0.5
            want = w * (1 - 0.05 * 0.1) - f * _reference((0.9 * m + 0.1 * g).view(r, c)).reshape(-1)
            bar = f * FP32_BAR * 1.3 * min(r, c) ** 0.5 + 2.0 ** -23 * float(want.norm())
            assert float((step.master[s].double() - want).norm()) <= bar, i
            assert float((step.momentum[s].double() - m).norm()) <= 2.0 ** -22 * float(m.norm() + g.norm())
    assert orthogonalize_error(DEV) == 0
