"""What ops.orthogonalize loses, beyond the rounding of its result: against the iteration in 64 bits.

Tolerances.  ``UNIT``: sides of 1 : 4 keep the singular values of X0 within a factor of 3 of each other, so relative errors are
not amplified; every one of 5 steps rounds X, A and the polynomial (operands and stored results: 6 roundings to 22 bits) and
sums in fp32 (3 products, 2^-24 sqrt(K) each).  A result r = round(x) of x = want + d is off by |round(want) - want| + 2 |d|
at most, as the nearest value to x is no further from x than round(want) is."""
import pytest
import torch

from tests.test_tokens_gpu import BF16, DEV, F16, F32, gen, half_step, newton_schulz64

pytestmark = pytest.mark.gpu


def unit(k):
  return 5 * 6 * 2.0 ** -22 + 15 * 2.0 ** -24 * k ** 0.5


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m,n", [(16, 70), (64, 256), (40, 301), (261, 65), (129, 517), (517, 129), (300, 1203), (1203, 300), (701, 2810),
                                 (2811, 702)])
def test_only_the_result_is_rounded(m, n, dtype):
  """In Frobenius norm and for every element, those at the remainders of tiles, vectors and quads among them."""
  from derl_amd import ops
  g = torch.randn(2, m, n, generator=gen(m + n), device=DEV).to(dtype)
  got = ops.orthogonalize(g)
  for k in range(2):
    want, norms = newton_schulz64(g[k], 5)
    rounded = want.to(dtype).double()
    d = unit(max(m, n)) * norms[-1]
    off = (got[k].double() - want).abs()
    assert float(off.norm()) <= float((rounded - want).norm()) + 2 * d, (float(off.norm()), float((rounded - want).norm()), d)
    assert bool((off <= half_step(want, dtype) + 2 * d).all()), float((off - half_step(want, dtype)).max() / d)
    for edge in (off[-1], off[:, -1], off[-4:, -4:]):  # rows and columns that end inside a tile or a vector
      assert float(edge.norm()) <= float(half_step(want, dtype).max()) * edge.numel() ** 0.5 + 2 * d
