"""Host-side checks of the orthogonalised update that need no GPU."""
from derl_amd import _lib


def test_workspace_of_matrices_that_take_one_launch():
  """They use none of it: what one matrix's launches would take, and 256 bytes each."""
  size = _lib.load().dx_orthogonalize_workspace
  assert size(0, 1, 64, 64) < 1 << 18
  assert size(0, 65535, 64, 64) < 20 << 20
  assert size(2, 65535, 64, 200) == size(2, 1, 64, 200) + 65534 * 256
  # others: the batch's matrices side by side, 16 bytes an element of X and 12 of A at least
  assert size(0, 4, 512, 512) - size(0, 3, 512, 512) >= 28 * 512 * 512
