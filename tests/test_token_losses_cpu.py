"""Host-side checks of the token losses' scaled gradients: refusals that need no GPU."""
import pytest

from derl_amd import _lib
from tests.test_tokens_cpu import FAKE, status


@pytest.mark.parametrize("changes,code,message", [
    (dict(factor=None), -1, "null"), (dict(dz=None), -1, "null"), (dict(dz=FAKE), -1, "read again"), (dict(ws=None), -1, "null"),
    (dict(old=None), -1, "null"), (dict(dz_pitch=3), -1, "overlap"), (dict(ref_lp=FAKE, ref_z=FAKE), -1, "not both"),
    (dict(dz=FAKE + 1025), -1, "aligned"), (dict(ws_count=16), -4, "workspace"), (dict(vocab=0), -1, "vocab"), (dict(dtype=7), -1, "dtype")])
def test_policy_gradient_refuses(changes, code, message):
  args = dict(logits=FAKE, dtype=2, rows=4, vocab=10, pitch=10, actions=FAKE, old=FAKE, adv=FAKE, ref_lp=None, ref_z=None, ref_pitch=10,
              mask=None, clip=0.2, kl=0.0, ent=0.0, batch=0, dz=FAKE + 1024, dz_pitch=10, ws=FAKE, ws_count=_lib.DX_TOKEN_WORKSPACE,
              factor=FAKE, stream=None)
  assert status("dx_token_policy_grad_scaled", *{**args, **changes}.values()) == code
  assert message in _lib.last_error()


@pytest.mark.parametrize("changes,code,message", [
    (dict(factor=None), -1, "null"), (dict(dz=None), -1, "null"), (dict(dz=FAKE), -1, "read again"), (dict(stats=None), -1, "null"),
    (dict(stats=FAKE + 4), -1, "misaligned"), (dict(dz_pitch=3), -1, "overlap"), (dict(actions=None), -1, "null")])
def test_preference_gradient_refuses(changes, code, message):
  args = dict(logits=FAKE, dtype=2, rows=4, vocab=10, pitch=10, actions=FAKE, stats=FAKE, dz=FAKE + 1024, dz_pitch=10, factor=FAKE, stream=None)
  assert status("dx_preference_grad_scaled", *{**args, **changes}.values()) == code
  assert message in _lib.last_error()


def test_no_rows_is_nothing_to_do():
  assert status("dx_preference_grad_scaled", None, 0, 0, 10, 10, None, None, None, 10, FAKE, None) == 0
