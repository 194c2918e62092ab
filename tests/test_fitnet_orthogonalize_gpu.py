"""Newton-Schulz orthogonalisation (fitnet.orthogonalize) against the iteration in 64 bits.

Tolerances: the same iteration in float32 (torch) has an error against 64 bits; the kernels may have 16 times that, and at least 2^-20 of
the result's norm (their sums are ordered otherwise). Results of 16 bits are rounded once; rounding the operands of their products to 11
bits may cost as much again as that (u of the type times two, of the norm)."""
import pytest
import torch

import fitnet_ref as ref

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from ai2pot_b200 import fitnet


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    fitnet.check()

MUON = (3.4445, -4.7750, 2.0315)
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def gradient_like(batch, m, n, dtype, seed=0, spread=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed + m + 3 * n)
    rows = 2 * max(m, n)
    gz, x = torch.randn(batch, rows, m, generator=g, device="cuda"), torch.randn(batch, rows, n, generator=g, device="cuda")
    x *= 10.0 ** (-spread * torch.rand(n, generator=g, device="cuda"))
    return (gz.mT @ x / rows).to(dtype)


def check(g, got, steps=5, coefficients=MUON, eps=1e-7):
    assert got.shape == g.shape and got.dtype == g.dtype
    want = ref.orthogonalize(g, steps, coefficients, eps)
    torch.backends.cuda.matmul.allow_tf32 = False
    plain = ref.orthogonalize(g, steps, coefficients, eps, torch.float32)
    norm = lambda t: torch.linalg.vector_norm(t.double(), dim=(-2, -1))
    err, own, size = norm(got - want), norm(plain - want), norm(want)
    u = ref.U[g.dtype]
    tol = 16 * own + 2.0 ** -20 * size + (0 if g.dtype == torch.float32 else 2 * u * size + (ref.TINY[g.dtype] * (g.shape[-1] * g.shape[-2]) ** 0.5))
    assert bool((err <= tol).all()), (err / size, tol / size)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,m,n", [(1, 1, 1), (1, 1, 7), (2, 9, 1), (3, 30, 20), (2, 17, 64), (1, 64, 64), (4, 65, 33), (2, 100, 300), (3, 128, 128), (1, 240, 240), (2, 257, 131),
                                       (1, 500, 20), (8, 96, 160), (1, 3, 30000), (2, 20000, 4)])
def test_shapes(batch, m, n, dtype):
    g = gradient_like(batch, m, n, dtype)
    check(g, fitnet.orthogonalize(g))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,m,n", [(1, 1024, 1024), (2, 513, 700), (1, 1537, 300), (1, 40, 2048), (3, 384, 512)])
def test_larger_matrices(batch, m, n, dtype):
    g = gradient_like(batch, m, n, dtype)
    check(g, fitnet.orthogonalize(g))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("steps,coefficients", [(0, MUON), (1, MUON), (3, (1.5, -0.5, 0.0)), (8, (1.875, -1.25, 0.375))])
def test_steps_and_coefficients(steps, coefficients, dtype):
    for shape in ((2, 48, 80), (1, 200, 150)):
        g = gradient_like(*shape, dtype)
        check(g, fitnet.orthogonalize(g, steps, coefficients), steps, coefficients)


@pytest.mark.parametrize("dtype", TYPES)
def test_low_rank_and_zero(dtype):
    """A dominant direction of rank one over a weak rest; a matrix of zeros stays zero; both next to an ordinary one."""
    g = gradient_like(3, 160, 224, torch.float32)
    u, v = torch.randn(160, 1, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)), torch.randn(1, 224, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    g[0] = u @ v + 1e-3 * g[0]
    g[1] = 0
    g = g.to(dtype)
    got = fitnet.orthogonalize(g)
    check(g, got)
    assert not bool(got[1].any())


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e6, 1e30])
def test_scales(scale):
    g = gradient_like(2, 50, 70, torch.float32) * scale
    check(g, fitnet.orthogonalize(g, eps=0.0), eps=0.0)
    g = gradient_like(1, 300, 200, torch.float32) * scale
    check(g, fitnet.orthogonalize(g, eps=0.0), eps=0.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_batch_is_independent_and_repeatable(dtype):
    for shape in ((5, 60, 40), (3, 256, 320)):
        g = gradient_like(*shape, dtype)
        got = fitnet.orthogonalize(g)
        assert torch.equal(got, fitnet.orthogonalize(g))
        assert torch.equal(got[1], fitnet.orthogonalize(g[1]))
        bad = g.clone()
        bad[0] = float("nan")
        again = fitnet.orthogonalize(bad)
        assert torch.equal(again[1:], got[1:]) and bool(again[0].isnan().all())


def test_layouts_and_more_dimensions():
    g = gradient_like(6, 40, 56, torch.float32)
    want = fitnet.orthogonalize(g)
    assert torch.equal(fitnet.orthogonalize(g.view(2, 3, 40, 56)).view(6, 40, 56), want)
    assert torch.equal(fitnet.orthogonalize(g.mT.contiguous().mT), want)
    assert torch.equal(fitnet.orthogonalize(g[0]), want[0])
    assert fitnet.orthogonalize(g[:0]).shape == (0, 40, 56)


def test_on_another_stream():
    g = gradient_like(2, 200, 260, torch.bfloat16)
    want = fitnet.orthogonalize(g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fitnet.orthogonalize(g)
    side.synchronize()
    assert torch.equal(want, got)


def test_refusals():
    g = gradient_like(1, 8, 9, torch.float32)
    for call, text in [(lambda: fitnet.orthogonalize(g.double()), "float32, bfloat16 or float16"), (lambda: fitnet.orthogonalize(g.cpu()), "CUDA"),
                       (lambda: fitnet.orthogonalize(g[0, 0]), r"\[..., m, n\]"), (lambda: fitnet.orthogonalize(g, steps=-1), "steps"),
                       (lambda: fitnet.orthogonalize(g[:, :, :0]), r"\[..., m, n\]"), (lambda: fitnet.orthogonalize(g, eps=-1.0), "eps"),
                       (lambda: fitnet.orthogonalize(g.clone().requires_grad_()), "no gradient")]:
        with pytest.raises(RuntimeError, match=text):
            call()
