"""GPU tests of the half-precision affine layer's activations and of their slopes where they are small (kaldi_amd.cumatrix.AffinePerRow / DiffAffinePerRow), against float64, with bounds
relative to the value: one weight of 1 makes the layer the activation alone.

Bounds.  An exponential's argument is rounded twice, so e^-a is off by 2 a half steps U of float32, and one of -z^2 / 2 by 1.5 z^2; a dozen roundings, reciprocals and a series of relative
error 2 U follow: (4 |z| + 16) U, for gelu (1.5 z^2 + 16) U, of the magnitudes of the terms that are added up (those of swish's and gelu's slopes cancel near their zero).  An exponential
below 2^-126 is 0, and is multiplied by |z| < 128 at most: 2^-119.  Then a result is rounded to its type: half a step."""
import math, pytest, torch
from tests.rowop_cases import U32, half_step, assert_within
from tests.test_affine_gpu import act64, slope64
pytestmark = pytest.mark.gpu

HALVES = [torch.float16, torch.bfloat16]
SMALLEST = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -119}      # half the smallest step, or the float32 exponential's

def points(dtype):
    a = torch.cat([torch.arange(0, 12, 0.0625), torch.arange(12, 88, 0.5)]); return torch.cat([-a.flip(0), a]).cuda().to(dtype)      # (multiples of 1/16 below 12 have 8 bits or are rounded here)

def relative(act, z): return ((1.5 * z * z if act == "gelu" else 4 * z.abs()) + 16) * U32

def slope_terms(act, z):
    s, c = torch.sigmoid(z), torch.sigmoid(-z)
    return {"sigmoid": s * c, "tanh": 4 * torch.sigmoid(2 * z) * torch.sigmoid(-2 * z), "swish": s * (1 + z.abs() * c), "gelu": 0.5 * torch.erfc(-z / math.sqrt(2)) + z.abs() * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)}[act]

def slopes(act, dtype):
    from kaldi_amd.cumatrix import DiffAffinePerRow
    z = points(dtype); n = z.numel(); one = torch.ones(1, 1, device="cuda").to(dtype)
    db = torch.empty(n, device="cuda"); DiffAffinePerRow(one, one.expand(n, 1).contiguous(), z[None], act, one.expand(1, n).contiguous(), bias_params_deriv=db)
    dx = torch.empty(n, 1, dtype=dtype, device="cuda"); DiffAffinePerRow(z[:, None], one, z[:, None], act, one.expand(n, 1).contiguous(), dx)
    z = z.double(); s, c = torch.sigmoid(z), torch.sigmoid(-z); want = {"sigmoid": s * c, "tanh": slope_terms("tanh", z), "swish": s * (1 + z * c), "gelu": slope64("gelu", z)}[act]
    off = relative(act, z) * slope_terms(act, z) + 2.0 ** -119; assert_within(db, want, off, "slope")
    assert_within(dx[:, 0], want, half_step(dtype) * (want.abs() + off) * 2.01 + off + 2 * SMALLEST[dtype], "dx")      # (rounded for the product, and the product once more)

@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("act", ["sigmoid", "tanh", "swish"])
def test_slopes_in_the_tails(act, dtype): slopes(act, dtype)

@pytest.mark.parametrize("dtype", HALVES)
def test_gelus_slope_in_the_tails(dtype): slopes("gelu", dtype)

@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("act", ["sigmoid", "tanh", "swish", "gelu"])
def test_values_in_the_tails(act, dtype):
    """tanh between -0.1 and 0.1 is a series, beside it a difference from 1 that is off by 2 half steps of 1"""
    from kaldi_amd.cumatrix import AffinePerRow
    z = points(dtype); y = torch.empty(z.numel(), 1, dtype=dtype, device="cuda"); AffinePerRow(z[:, None], torch.ones(1, 1, device="cuda").to(dtype), None, act, None, y)
    want = act64(act, z.double()); off = relative(act, z.double()) * want.abs() + (4 * U32 if act == "tanh" else 0.0) + 2.0 ** -119
    assert_within(y[:, 0], want, half_step(dtype) * (want.abs() + off) + off + SMALLEST[dtype], "value")
