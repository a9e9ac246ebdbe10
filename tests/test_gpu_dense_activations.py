"""GPU: the activations of the dense operators and their derivatives by relative error, in the tails as well, where a formula that
cancels loses all of a small result and an absolute tolerance does not see it. The product before them is one with an identity,
so z reaches them as it is.

Tolerances: a dozen roundings of 2^-24 in fp32 (the hardware's 2^x and reciprocal count two each, the fit of the normal tail
four), 2^-20 in all; sums of two terms may lose a factor of 2 to 4 where they do not cross zero. bf16 adds half a step of the
result, 2^-8, and its shorter fit of the normal tail, 5.7e-7."""
import pytest
import torch

from test_gpu_dense import D, HALF, TYPES, act64, matrix, run_backward, run_forward, slope64

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    torch.cuda.set_device(0)


def values(kind, lo, hi):
    """64 columns of z over [lo, hi]."""
    return torch.linspace(lo, hi, 64 * 500, device="cuda", dtype=torch.float64).to(TYPES[kind][1]).view(-1, 64)


def off_by(got, want):
    return float(((got.double() - want).abs() / want.abs()).max())


def check(kind, act, lo, hi, slack, derivative):
    dtype = TYPES[kind][1]
    z, eye = values(kind, lo, hi), torch.eye(64, dtype=dtype, device="cuda")
    allowed = slack * 2.0 ** -20 + (HALF[dtype] + slack * 5.7e-7 if dtype == torch.bfloat16 else 0.0)
    if derivative:
        got, want = run_backward(kind, torch.ones_like(z), z, act, matrix(z.shape[0], 64, dtype, 1), eye, ("dx",))["dx"], slope64(act, z.double())
    else:
        got, want = run_forward(kind, z, eye, None, act, None, False)[0], act64(act, z.double())
    assert off_by(got, want) <= allowed


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("lo,hi", [(-12, -8), (-8, -6), (-6, -5), (-5, -4), (-4, -2), (-2, -1e-3), (1e-3, 4), (4, 12), (12, 100)])
def test_gelu(kind, lo, hi):
    check(kind, D.ACT_GELU, lo, hi, 1, False)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("lo,hi", [(-12, -8), (-8, -6), (-6, -5), (-5, -4), (-4, -2), (-0.5, 4), (4, 12), (12, 100)])
def test_gelu_derivative(kind, lo, hi):
    check(kind, D.ACT_GELU, lo, hi, 4, True)      # (it is 0 at -0.75)
