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


SIGMOID_RANGES = [(-85, -17), (-17, -8), (-8, -2), (-2, -1e-3), (1e-3, 4), (4, 10), (10, 17), (17, 85)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("lo,hi", SIGMOID_RANGES)
@pytest.mark.parametrize("act", [D.ACT_SILU, D.ACT_SIGMOID])
def test_silu_and_sigmoid(kind, act, lo, hi):
    check(kind, act, lo, hi, 1, False)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("lo,hi", SIGMOID_RANGES)
def test_sigmoid_derivative(kind, lo, hi):
    check(kind, D.ACT_SIGMOID, lo, hi, 1, True)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("lo,hi", [(-85, -17), (-17, -8), (-8, -2), (-1, -1e-3), (1e-3, 4), (4, 10), (10, 17), (17, 85)])
def test_silu_derivative(kind, lo, hi):
    check(kind, D.ACT_SILU, lo, hi, 4, True)      # (it is 0 at -1.28)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("act", [D.ACT_GELU, D.ACT_SILU, D.ACT_SIGMOID])
def test_far_values(kind, act):
    """Where the exponential is 0 or would overflow: the limits, no NaN; of infinities and NaN what the formula has."""
    dtype = TYPES[kind][1]
    z = torch.tensor([-3e38, -1e20, -1e4, -200.0, 200.0, 1e4, 1e20, 3e38, float("inf"), float("nan")] + [0.0] * 54, device="cuda").to(dtype).view(-1, 1)
    one = torch.ones(1, 1, dtype=dtype, device="cuda")
    y, _ = run_forward(kind, z, one, None, act, None, False)
    low, high = y[:4].float(), y[4:9].float()
    assert bool((low.abs() < 1e-30).all()) and bool(torch.isnan(y[9, 0]))
    assert torch.equal(high, torch.ones_like(high) if act == D.ACT_SIGMOID else z[4:9].float())
    assert float(y[10]) == (0.5 if act == D.ACT_SIGMOID else 0.0)
    d = run_backward(kind, torch.ones_like(z[:8]).contiguous(), z[:8].contiguous(), act, z[:8].contiguous(), one, ("db", "dx"))["dx"].float()
    assert bool((d[:4].abs() < 1e-30).all())
    assert torch.equal(d[4:], torch.zeros_like(d[4:]) if act == D.ACT_SIGMOID else torch.ones_like(d[4:]))
