"""What ops.orthogonalize loses, beyond the rounding of its result: against the iteration in 64 bits.

Tolerances.  ``UNIT``: sides of 1 : 4 keep the singular values of X0 within a factor of 3 of each other, so relative errors are
not amplified; every one of 5 steps rounds X, A and the polynomial (operands and stored results: 6 roundings to 22 bits) and
sums in fp32 (3 products, 2^-24 sqrt(K) each).  A result r = round(x) of x = want + d is off by |round(want) - want| + 2 |d|
at most, as the nearest value to x is no further from x than round(want) is."""
import pytest
import torch

from tests.test_tokens_gpu import A, B, BF16, C, DEV, F16, F32, gen, half_step, newton_schulz64

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


SCALED = [(17, 70), (32, 300), (60, 200), (200, 60), (93, 96), (64, 576), (256, 512), (512, 256), (300, 1203), (1203, 300), (701, 1410)]


@pytest.mark.parametrize("scale", [1e-4, 1e-6, 1e-9])
@pytest.mark.parametrize("m,n", SCALED)
def test_rows_and_columns_of_any_size(m, n, scale):
  """Every eighth row, every seventh column, or both, are far smaller than the rest (rare tokens, units that are nearly dead; the
  iteration amplifies just those): each row and column is as accurate as its own size allows.  Relative errors of a row are those
  of ``unit``: it starts, as all rows do, with growth of `a` a step for all of its parts."""
  from derl_amd import ops
  for which in ("rows", "columns", "both"):
    g = torch.randn(m, n, generator=gen(m + n), device=DEV)
    if which != "columns":
      g[3::8] *= scale
    if which != "rows":
      g[:, 2::7] *= scale
    got = ops.orthogonalize(g).double()
    want, _ = newton_schulz64(g, 5)
    off = got - want
    bound = 2 * unit(max(m, n))
    for dim in (0, 1):
      worst = float((off.norm(dim=dim) / want.norm(dim=dim)).max())
      assert worst <= bound, (which, dim, worst, bound)
    if which == "both":
      corner = float(off[3::8, 2::7].norm() / want[3::8, 2::7].norm())
      assert corner <= bound, (corner, bound)


@pytest.mark.parametrize("m,n", [(20, 90), (60, 60), (96, 90), (130, 600), (600, 130)])
def test_a_norm_far_below_eps(m, n):
  """X0 is close to 0: every step multiplies it by `a` (five steps of a product and a sum, X0's two roundings and the norm's:
  14 half steps of an entry) and adds (b A + c A^2) X, whose entry (i, j) is off by ``unit`` / 5 of |M_i| |x_j| at most (the norms of
  a row and a column), |M_i| <= (|b| + |c| s^2) s |x_i| with s the largest singular value; step k has |x|, |x_i|, s of a^k those of
  X0 at most and its error is multiplied by `a` in the 4 - k steps behind it.  Twice that, as the errors of X move M as well."""
  from derl_amd import ops
  for norm in (1e-12, 1e-20, 1e-30):
    g = torch.randn(m, n, generator=gen(m), device=DEV) * norm
    got = ops.orthogonalize(g).double()
    want, _ = newton_schulz64(g, 5)
    x = g.double() / (g.double().norm() + 1e-7)
    s = float(torch.linalg.matrix_norm(x, 2))
    outer = x.norm(dim=1)[:, None] * x.norm(dim=0)[None]
    moved = 2 * unit(max(m, n)) / 5 * (-B + C * s * s * A ** 8) * s * outer * sum(A ** (4 + 2 * k) for k in range(5))
    assert bool(((got - want).abs() <= 14 * 2.0 ** -24 * want.abs() + moved).all()), norm


@pytest.mark.parametrize("m,n", [(24, 90), (60, 64), (90, 96), (200, 800), (800, 200)])
@pytest.mark.parametrize("coefficients,steps", [((3.0, 0.0, 0.0), 6), ((1.5, -0.5, 0.0), 12), ((2.0, -1.5, 0.5), 7), ((0.25, 0.0, 0.0), 5),
                                                ((15 / 8, -10 / 8, 3 / 8), 9), ((-1.0, 0.5, 0.0), 4), ((1.0, 2.0, 0.0), 4)])
def test_other_coefficients(m, n, coefficients, steps):
  """Singular values that pass 8, shrink, change sign or converge.  A step's rounding is ``unit`` / 5 of the magnitudes of its
  terms, |a| s + |b| s^3 + |c| s^5 for the largest singular value s, and what it moves is multiplied by the slope |a| + 3 |b| s^2
  + 5 |c| s^4 at most in the steps behind it."""
  from derl_amd import ops
  g = torch.randn(m, n, generator=gen(5), device=DEV)
  got = ops.orthogonalize(g, steps=steps, coefficients=coefficients).double()
  a, b, c = coefficients
  x = g.double() / g.double().norm()
  s = torch.linalg.svdvals(x)
  bound = 0.0
  for _ in range(steps):
    slope = abs(a) + 3 * abs(b) * s.max() ** 2 + 5 * abs(c) * s.max() ** 4
    terms = (abs(a) * s + abs(b) * s ** 3 + abs(c) * s ** 5).norm()
    bound = float(slope) * bound + unit(max(m, n)) / 5 * float(terms)
    s = (a * s + b * s ** 3 + c * s ** 5).abs()
  want, _ = newton_schulz64(g, steps, coefficients, eps=1e-7)
  assert float((got - want).norm()) <= bound, (float((got - want).norm()), bound)


@pytest.mark.parametrize("shape", [(3, 20, 60), (2, 60, 60), (3, 96, 90), (2, 130, 200)])
def test_any_number_of_steps(shape):
  """Coefficients whose iteration converges (slope 0 at 1): the last steps leave their own rounding alone; more steps than the
  one-launch kernel holds the scales of."""
  from derl_amd import ops
  g = torch.randn(shape, generator=gen(3), device=DEV)
  coefficients = (15 / 8, -10 / 8, 3 / 8)
  got = ops.orthogonalize(g, steps=45, coefficients=coefficients)
  for k in range(shape[0]):
    want, norms = newton_schulz64(g[k], 45, coefficients)
    assert float((got[k].double() - want).norm()) <= unit(max(shape)) * norms[-1]
  again = g.clone()
  assert torch.equal(ops.orthogonalize(again, steps=45, coefficients=coefficients, out=again), got)


def test_memory_of_many_small_matrices():
  from derl_amd import ops
  g = torch.randn(20000, 64, 64, generator=gen(1), device=DEV)
  out = torch.empty_like(g)
  torch.cuda.synchronize()
  torch.cuda.reset_peak_memory_stats()
  before = torch.cuda.memory_allocated()
  ops.orthogonalize(g, out=out)
  torch.cuda.synchronize()
  assert torch.cuda.max_memory_allocated() - before < 16e6
  for k in (0, 19999):
    assert torch.equal(out[k], ops.orthogonalize(g[k]))


@pytest.mark.parametrize("m,n", [(20, 60), (60, 64), (130, 500), (500, 130)])
def test_denormal_values(m, n):
  """Entries below 2^-126, with what digits they have: a power of two times them, exactly, gives the same result."""
  from derl_amd import ops
  g = torch.randn(m, n, generator=gen(9), device=DEV) * 2.0 ** -100 * 2.0 ** -38
  assert float(g.abs().max()) < 2.0 ** -126
  want = ops.orthogonalize(g * 2.0 ** 100, eps=0.0)
  assert float((ops.orthogonalize(g, eps=0.0) - want).abs().max()) <= 2.0 ** -18


def matrix_of(kind, m, n):
  g = torch.randn(m, n, generator=gen(m + 3 * n), device=DEV)
  k = min(m, n)
  if kind == "low rank":
    return g[:, :3].mm(g[:3]) + 1e-3 * g
  if kind == "rank one":
    return torch.ones(m, n, device=DEV)
  if kind == "one large row":
    g[1] *= 1e4
    return g
  if kind == "orthogonal":
    q = torch.linalg.qr(g if m >= n else g.t())[0]
    return (q if m >= n else q.t()).contiguous()
  if kind == "sparse":
    return torch.where(torch.rand(m, n, generator=gen(2), device=DEV) < 0.02, g, 0.0)
  g = torch.zeros(m, n, device=DEV)
  if kind == "diagonal":
    g[torch.arange(k), torch.arange(k)] = torch.logspace(0, -6, k, device=DEV)
  elif kind == "blocks":
    g[:m // 2, :n // 3] = 1e-5 * torch.randn(m // 2, n // 3, generator=gen(4), device=DEV)
    g[m // 2:, n // 3:] = torch.randn(m - m // 2, n - n // 3, generator=gen(5), device=DEV)
  return g


@pytest.mark.parametrize("kind", ["low rank", "rank one", "one large row", "orthogonal", "sparse", "diagonal", "blocks"])
@pytest.mark.parametrize("m,n", [(20, 33), (64, 64), (60, 200), (96, 90), (130, 300), (513, 200), (700, 1500)])
def test_matrices_that_are_not_gaussian(m, n, kind):
  """Each step's rounding, ``unit`` / 5 of X's norm, passed on by the polynomial's slope, 4 at most (its derivative
  a + 3 b s^2 + 5 c s^4 has its extremes 3.44, -1.61 and 3.97 on [0, 1.2024], where a step leaves every singular value); all three types against the same iteration, and zeros stay zeros."""
  from derl_amd import ops
  for dtype in (F32, BF16, F16):
    g = matrix_of(kind, m, n).to(dtype)
    want, norms = newton_schulz64(g, 5)
    got = ops.orthogonalize(g)
    d = unit(max(m, n)) / 5 * sum(4.0 ** (4 - k) * norm for k, norm in enumerate(norms[:5]))
    off = (got.double() - want).abs()
    assert float(off.norm()) <= float((want.to(dtype).double() - want).norm()) + 2 * d, (dtype, float(off.norm()), d)
    if kind in ("diagonal", "blocks"):
      assert not got[g.any(1).logical_not()].any()
