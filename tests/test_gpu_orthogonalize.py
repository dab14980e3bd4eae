"""Matrices orthogonalised by Newton-Schulz products, and the transition that uses it, against float64.

Tolerances, in the 2-norm of the difference over the 2-norm of the result.  An error in an iterate grows by
at most max |p'| = 3.9 a step in its direction (p(s) = a s + b s^3 + c s^5 on [0, 1.2]) while the iterate's
own norm grows too.  Operands kept to 2^-22 and fp32 sums give local errors of a few 2^-22; float32 operands
(2^-24, but sums of up to some thousand terms) reach 1.5e-5 at the steepest spectra below, so 2e-5 is what
"fp32 accuracy" means here.  bf16 outputs add half a step, 2^-8 relative at most, fp16 outputs 2^-11; the
single-pass form for large bf16 outputs has operands of 2^-12 in A and B, 3.9e-3 with the rounding.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
A, B, C = 3.4445, -4.7750, 2.0315
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
FP32_BAR = 2e-5
BAR = {F32: FP32_BAR, F16: 2.0 ** -11 + FP32_BAR, BF16: 2.0 ** -8}


def _reference(x, steps=5, eps=1e-7, coefficients=(A, B, C)):
    a, b, c = coefficients
    x = x.double()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + eps)
    for _ in range(steps):
        g = x @ x.mT
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.mT if tall else x


def _off(got, ref):
    return float((got.double() - ref).norm() / ref.norm())


def _matrix(kind, m, n, gen):
    if kind == "noise":
        return torch.randn(m, n, generator=gen, device=DEV)
    if kind == "low":  # a low-rank part and noise, as gradients have
        r = max(1, min(m, n) // 8)
        low = torch.randn(m, r, generator=gen, device=DEV) @ torch.randn(r, n, generator=gen, device=DEV)
        return low / math.sqrt(r) + 0.2 * torch.randn(m, n, generator=gen, device=DEV)
    k = min(m, n)
    u = torch.linalg.qr(torch.randn(m, k, generator=gen, device=DEV, dtype=torch.float64))[0]
    v = torch.linalg.qr(torch.randn(n, k, generator=gen, device=DEV, dtype=torch.float64))[0]
    s = torch.arange(1, k + 1, device=DEV, dtype=torch.float64) ** -(1.0 if kind == "steep" else 0.5)
    return ((u * s) @ v.T).float()


SHAPES = [(1, 1), (1, 300), (300, 1), (2, 3), (9, 64), (64, 64), (65, 130), (128, 128), (128, 384), (384, 128), (127, 129),
          (129, 257), (192, 192), (256, 1024), (1024, 88), (407, 512), (513, 700), (200, 5000), (1024, 640)]


@pytest.mark.parametrize("m,n", SHAPES)
@pytest.mark.parametrize("kind", ["noise", "low", "steep"])
def test_matches_float64(m, n, kind):
    from pbg_b200.optim import orthogonalize, orthogonalize_error

    gen = torch.Generator(device=DEV).manual_seed(m * 31 + n)
    x = _matrix(kind, m, n, gen)
    ref = _reference(x)
    got = orthogonalize(x)
    assert orthogonalize_error(DEV) == 0
    assert _off(got, ref) <= FP32_BAR
    assert torch.equal(got, orthogonalize(x))  # the same bits again
    for dtype in (BF16, F16):
        assert _off(orthogonalize(x, out_dtype=dtype), ref) <= BAR[dtype]


@pytest.mark.parametrize("m,n", [(1536, 2048), (2500, 1100), (4096, 512)])
def test_large_matrices(m, n):
    from pbg_b200.optim import orthogonalize, orthogonalize_error

    gen = torch.Generator(device=DEV).manual_seed(m)
    x = _matrix("low", m, n, gen)
    ref = _reference(x)
    assert _off(orthogonalize(x), ref) <= FP32_BAR
    assert _off(orthogonalize(x.bfloat16(), out_dtype=BF16), _reference(x.bfloat16())) <= BAR[BF16]
    assert orthogonalize_error(DEV) == 0


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_batches_types_strides_and_in_place(dtype):
    from pbg_b200.optim import orthogonalize

    gen = torch.Generator(device=DEV).manual_seed(3)
    x = (torch.randn(3, 5, 70, 200, generator=gen, device=DEV) * torch.rand(3, 5, 1, 1, generator=gen, device=DEV)).to(dtype)
    ref = _reference(x)
    got = orthogonalize(x)
    assert got.dtype == dtype and got.shape == x.shape
    for i in range(3):
        for j in range(5):
            assert _off(got[i, j], ref[i, j]) <= BAR[dtype]
            assert torch.equal(got[i, j], orthogonalize(x[i, j]))  # a batch is its matrices, one by one
    assert torch.equal(orthogonalize(x[:, ::2, :, 3:90]), orthogonalize(x[:, ::2, :, 3:90].contiguous()))
    y = x.clone()
    assert orthogonalize(y, out=y) is y and torch.equal(y, got)
    assert orthogonalize(x[:0]).shape == (0, 5, 70, 200)
    assert orthogonalize(x[..., :0]).shape == (3, 5, 70, 0)


def test_scales_zeros_and_non_finite_matrices():
    from pbg_b200.optim import orthogonalize

    gen = torch.Generator(device=DEV).manual_seed(4)
    x = torch.randn(6, 90, 140, generator=gen, device=DEV)
    x[1] *= 1e25   # squares past fp32
    x[2] *= 1e-12  # epsilon outweighs the norm
    x[3] = 0
    x[4, 7, 9] = float("nan")
    x[5, 80, 3] = float("inf")
    got = orthogonalize(x)
    ref = _reference(x)
    for i in (0, 1, 2):
        assert _off(got[i], ref[i]) <= FP32_BAR
    assert bool((got[3] == 0).all()) and bool(got[4:].isnan().all())


def test_steps_coefficients_and_epsilon():
    from pbg_b200._native import NativeError
    from pbg_b200.optim import orthogonalize

    gen = torch.Generator(device=DEV).manual_seed(5)
    x = torch.randn(100, 180, generator=gen, device=DEV)
    for steps, k in ((1, (A, B, C)), (2, (A, B, C)), (7, (A, B, C)), (12, (1.5, -0.5, 0.0)), (10, (1.875, -1.25, 0.375))):
        ref = _reference(x, steps, 0.5, k)
        assert _off(orthogonalize(x, steps=steps, coefficients=k, epsilon=0.5), ref) <= FP32_BAR
    # the cubic converges: its result has orthonormal rows
    q = orthogonalize(x, steps=25, coefficients=(1.5, -0.5, 0.0))
    assert float((q.double() @ q.double().T - torch.eye(100, device=DEV)).abs().max()) <= 1e-4
    for bad in (dict(steps=0), dict(steps=101), dict(coefficients=(6.0, 0.0, 0.0)), dict(coefficients=(float("nan"), 0, 0)),
                dict(epsilon=-1.0), dict(out_dtype=torch.float64), dict(out=x[:, :3])):
        with pytest.raises(NativeError):
            orthogonalize(x, **bad)
    with pytest.raises(NativeError):
        orthogonalize(x[0])
    with pytest.raises(NativeError):
        orthogonalize(x.double())


def _muon_reference(w, m, g, mats, lr, mu, decay, nesterov, rule, scale=1.0):
    w, m, g = w.double().clone(), m.double().clone(), g.double() / scale
    for at, r, c in mats:
        s = slice(at, at + r * c)
        m[s] = mu * m[s] + (1 - mu) * g[s]
        u = mu * m[s] + (1 - mu) * g[s] if nesterov else m[s]
        f = math.sqrt(max(1.0, r / c)) if rule == "shape" else 0.2 * math.sqrt(max(r, c))
        w[s] = w[s] * (1 - lr * decay) - lr * f * _reference(u.view(r, c)).reshape(-1)
    return w, m


MATRICES = [(3, 128, 128), (16400, 512, 96), (65600, 3, 128), (66000, 130, 61), (74000, 1, 7), (74007, 256, 700), (253300, 9, 1)]


@pytest.mark.parametrize("nesterov,rule", [(True, "shape"), (False, "rms")])
def test_transition_matches_float64(nesterov, rule):
    from pbg_b200.optim import FlatMuon, orthogonalize_error

    gen = torch.Generator(device=DEV).manual_seed(6)
    n = 253400
    master = torch.randn(n, generator=gen, device=DEV)
    step = FlatMuon(master, MATRICES, lr=0.05, momentum=0.9, decay=0.1, nesterov=nesterov, adjust=rule, scale=128.0)
    before = master.clone()
    inside = torch.zeros(n, dtype=torch.bool, device=DEV)
    for at, r, c in MATRICES:
        inside[at:at + r * c] = True
    w, m = master.double(), step.momentum.double()
    for _ in range(3):
        g = torch.randn(n, generator=gen, device=DEV)
        step.grad.copy_(g)
        w, m = _muon_reference(step.master, step.momentum, g, MATRICES, 0.05, 0.9, 0.1, nesterov, rule, 128.0)
        assert step.step() is step.skipped
        assert int(step.skipped) == 0 and torch.equal(step.grad, g)
        # the update's error, and the roundings of the momentum (3 of 2^-24) and the master (2 of 2^-24)
        for at, r, c in MATRICES:
            s = slice(at, at + r * c)
            f = 0.05 * (math.sqrt(max(1.0, r / c)) if rule == "shape" else 0.2 * math.sqrt(max(r, c)))
            bar = f * FP32_BAR * 1.3 * math.sqrt(min(r, c)) + 2.0 ** -23 * float(w[s].norm())
            assert float((step.master[s].double() - w[s]).norm()) <= bar
            assert float((step.momentum[s].double() - m[s]).norm()) <= 2.0 ** -22 * float(m[s].norm() + g[s].norm() / 128)
    assert torch.equal(step.master[~inside], before[~inside]) and bool((step.momentum[~inside] == 0).all())
    assert orthogonalize_error(DEV) == 0


def test_transition_skips_when_a_direction_is_not_finite():
    from pbg_b200.optim import FlatMuon

    gen = torch.Generator(device=DEV).manual_seed(7)
    master = torch.randn(40000, generator=gen, device=DEV)
    step = FlatMuon(master, [(0, 100, 100), (10000, 50, 300)])
    step.grad.normal_(generator=gen)
    step.step()
    w, m = step.master.clone(), step.momentum.clone()
    step.grad.normal_(generator=gen)
    step.grad[17000] = float("inf")
    tail = step.grad[25000:].clone()
    assert int(step.step()) == 1
    assert torch.equal(step.master, w) and torch.equal(step.momentum, m)
    assert bool((step.grad[:25000] == 0).all()) and torch.equal(step.grad[25000:], tail)
    step.grad.normal_(generator=gen)
    assert int(step.step()) == 0 and not torch.equal(step.master[:25000], w[:25000])


def test_graph_replay_controls_and_two_optimizers():
    from pbg_b200.optim import FlatMuon, orthogonalize

    gen = torch.Generator(device=DEV).manual_seed(8)
    mats = [(0, 256, 300), (76800, 300, 64)]
    masters = [torch.randn(96000, generator=gen, device=DEV) for _ in range(2)]
    eager = [FlatMuon(m.clone(), mats) for m in masters]
    caught = [FlatMuon(m.clone(), mats) for m in masters]
    x = torch.randn(4, 33, 77, generator=gen, device=DEV)
    graphs, outs = [], []
    for c in caught:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.step()
            outs.append(orthogonalize(x))
        graphs.append(g)
    for i in range(3):
        for e, c in zip(eager, caught):
            e.grad.normal_(generator=gen)
            c.grad.copy_(e.grad)
            e.controls[0] = c.controls[0] = 0.01 * (i + 1)
            e.step()
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
    for e, c in zip(eager, caught):
        assert torch.equal(e.master, c.master) and torch.equal(e.momentum, c.momentum)
    assert all(torch.equal(o, orthogonalize(x)) for o in outs)


@pytest.mark.parametrize("batch,m,n", [(1, 256, 2048), (1, 129, 16391), (1, 65536, 256), (3, 200, 4097), (1, 640, 8192)])
def test_long_sides_are_summed_in_parts(batch, m, n):
    """Few matrices with a long side: several blocks sum each Gram tile, in an order of their own, the same every call."""
    from pbg_b200.optim import orthogonalize, orthogonalize_error

    gen = torch.Generator(device=DEV).manual_seed(m + n)
    x = torch.stack([_matrix("low", m, n, gen) for _ in range(batch)])
    ref = _reference(x)
    got = orthogonalize(x)
    half = orthogonalize(x, out_dtype=BF16)
    for i in range(batch):
        assert _off(got[i], ref[i]) <= FP32_BAR
        assert _off(half[i], ref[i]) <= BAR[BF16]
    for _ in range(3):
        orthogonalize(x[:, :150, :150])  # other work in the same workspace
        assert torch.equal(got, orthogonalize(x))
    assert orthogonalize_error(DEV) == 0


def test_transition_with_long_matrices():
    from pbg_b200.optim import FlatMuon, orthogonalize_error

    gen = torch.Generator(device=DEV).manual_seed(9)
    mats = [(0, 256, 8192), (2097152, 160, 160), (2122752, 7000, 192), (3466752, 64, 90)]
    n = 3472512
    step = FlatMuon(torch.randn(n, generator=gen, device=DEV), mats, lr=0.05, momentum=0.9)
    twin = FlatMuon(step.master.clone(), mats, lr=0.05, momentum=0.9)
    for _ in range(2):
        g = torch.randn(n, generator=gen, device=DEV)
        step.grad.copy_(g), twin.grad.copy_(g)
        w, m = _muon_reference(step.master, step.momentum, g, mats, 0.05, 0.9, 0.0, True, "shape")
        step.step(), twin.step()
        for at, r, c in mats:
            s = slice(at, at + r * c)
            bar = 0.05 * math.sqrt(max(1.0, r / c)) * FP32_BAR * 1.3 * math.sqrt(min(r, c)) + 2.0 ** -23 * float(w[s].norm())
            assert float((step.master[s].double() - w[s]).norm()) <= bar
        assert torch.equal(step.master, twin.master)
    assert orthogonalize_error(DEV) == 0


def test_transition_refusals():
    from pbg_b200.optim import FlatMuon

    master = torch.zeros(100, device=DEV)
    for matrices, more in (([], {}), ([(0, 10, 11)], {}), ([(-1, 2, 2)], {}), ([(0, 0, 5)], {}), ([(0, 5, 5), (24, 2, 2)], {}),
                           ([(0, 5, 5)], dict(momentum=1.0)), ([(0, 5, 5)], dict(adjust="none")),
                           ([(0, 5, 5)], dict(grad=torch.zeros(99, device=DEV)))):
        with pytest.raises(ValueError):
            FlatMuon(master, matrices, **more)
    with pytest.raises(ValueError):
        FlatMuon(master.double(), [(0, 5, 5)])
