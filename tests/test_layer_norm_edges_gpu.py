"""GPU tests of layer norm (kaldi_amd.cumatrix) on rows that are not finite."""
import pytest, torch
from tests.rowop_cases import TYPES, generator
pytestmark = pytest.mark.gpu

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [3, 100, 770, 5000, 13000, 20011])      # one wavefront, several, the loop
def test_a_row_with_an_infinity_or_a_nan_has_no_statistics(cols, dtype):
    """mean = what the values add up to, inv_std NaN, and every value of the row NaN, in the derivative too; the rows beside it as without it"""
    from kaldi_amd.cumatrix import LayerNormPerRow, DiffLayerNormPerRow
    inf, nan = float("inf"), float("nan"); clean = torch.randn(9, cols, generator=generator(cols), device="cuda").to(dtype); x = clean.clone(); bad = [1, 3, 5, 7]
    x[1, cols // 2] = inf; x[3, 0] = -inf; x[5, 1] = inf; x[5, 2] = -inf; x[7, cols - 1] = nan
    def run(x):
        y, m, r, dx = torch.empty_like(x), torch.empty(9, device="cuda"), torch.empty(9, device="cuda"), torch.empty_like(x); LayerNormPerRow(x, None, None, 1e-5, y, m, r); DiffLayerNormPerRow(x, clean, None, m, r, dx); return y, m, r, dx
    y, m, r, dx = run(x); want = run(clean); good = [0, 2, 4, 6, 8]
    assert torch.isnan(r[bad]).all() and m[1] == inf and m[3] == -inf and torch.isnan(m[[5, 7]]).all() and torch.isnan(y[bad].float()).all() and torch.isnan(dx[bad].float()).all()
    assert all(torch.equal(a[good], b[good]) for a, b in zip((y, m, r, dx), want))
