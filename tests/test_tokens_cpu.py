"""Host-side checks of the token losses and the orthogonalised update: refusals that need no GPU."""
import pytest
import torch

from derl_amd import _lib, ops

FAKE = 1 << 20  # an address no check dereferences


def status(name, *args):
  return getattr(_lib.load(), name)(*args)


def policy_args(**changes):
  args = dict(logits=FAKE, dtype=0, rows=4, vocab=10, pitch=10, actions=FAKE, old=FAKE, adv=FAKE, ref_lp=None, ref_z=None, ref_pitch=10,
              mask=None, clip=0.2, kl=0.0, ent=0.0, batch=0, dz=FAKE, dz_pitch=10, lp=FAKE, ws=FAKE, ws_count=_lib.DX_TOKEN_WORKSPACE,
              loss=FAKE, stream=None)
  args.update(changes)
  return list(args.values())


@pytest.mark.parametrize("changes,code,message", [
    (dict(dtype=3), -1, "dtype"), (dict(rows=-1), -1, "rows"), (dict(rows=1 << 31), -1, "rows"), (dict(vocab=0), -1, "vocab"),
    (dict(vocab=(1 << 30) + 1, pitch=1 << 31), -1, "vocab"), (dict(pitch=9), -1, "overlap"), (dict(logits=None), -1, "null"),
    (dict(actions=None), -1, "null"), (dict(old=None), -1, "null"), (dict(dz=None), -1, "null"), (dict(loss=None), -1, "null"),
    (dict(ws=None), -1, "null"), (dict(ref_lp=FAKE, ref_z=FAKE), -1, "not both"), (dict(dz_pitch=3), -1, "overlap"),
    (dict(ref_z=FAKE, ref_pitch=3), -1, "overlap"), (dict(logits=FAKE + 2), -1, "aligned"), (dict(dz=FAKE + 1), -1, "aligned"),
    (dict(dtype=1, logits=FAKE + 1), -1, "aligned"), (dict(ws_count=16), -4, "workspace")])
def test_policy_loss_refuses(changes, code, message):
  assert status("dx_token_policy_loss", *policy_args(**changes)) == code
  assert message in _lib.last_error()


@pytest.mark.parametrize("changes,code,message", [
    (dict(pairs=0), -1, "pairs"), (dict(smooth=1.1), -1, "label_smoothing"), (dict(smooth=float("nan")), -1, "label_smoothing"),
    (dict(offsets=None), -1, "null"), (dict(stats=None), -1, "null"), (dict(stats=FAKE + 4), -1, "misaligned"),
    (dict(ws_count=0), -4, "workspace"), (dict(vocab=-3), -1, "vocab")])
def test_preference_loss_refuses(changes, code, message):
  args = dict(logits=FAKE, dtype=2, rows=4, vocab=10, pitch=10, actions=FAKE, offsets=FAKE, pairs=1, ref=None, mask=None, beta=0.1,
              smooth=0.0, batch=0, dz=FAKE, dz_pitch=10, seq=FAKE, stats=FAKE, ws=FAKE, ws_count=_lib.DX_TOKEN_WORKSPACE, loss=FAKE,
              stream=None)
  args.update(changes)
  assert status("dx_preference_loss", *args.values()) == code
  assert message in _lib.last_error()


def test_other_entry_points_refuse():
  assert status("dx_token_log_prob", None, 0, 4, 10, 10, None, None, None, None, FAKE, 1 << 20, None) == -1
  assert status("dx_token_log_prob", FAKE, 0, 4, 10, 10, FAKE, None, FAKE, None, FAKE, 4, None) == -4
  assert status("dx_token_log_prob", None, 0, 0, 10, 10, None, None, None, None, None, 0, None) == 0  # no rows: nothing to do
  assert status("dx_sequence_log_prob", None, None, 3, 2, None, None) == -1
  assert status("dx_sequence_log_prob", None, None, 3, 0, None, None) == 0
  assert status("dx_scale_rows", FAKE, 0, 2, 10, 9, FAKE, None) == -1
  assert status("dx_scale_rows", FAKE + 2, 0, 2, 10, 10, FAKE, None) == -1
  assert status("dx_muon_momentum_f32", FAKE, FAKE, FAKE, 4, None, 0, 0.5, 0.95, 1, None, None) == -1
  assert "partial sums" in _lib.last_error()
  assert status("dx_muon_apply_f32", None, FAKE, 4, 1.0, 0.1, None) == -1


def test_orthogonalize_shapes():
  size = _lib.load().dx_orthogonalize_workspace
  assert size(0, 1, 512, 3136) > 2 * 4 * 512 * 3136 and size(1, 1, 512, 3136) < size(0, 1, 512, 3136)
  assert size(0, 1, 512, 3136) == size(0, 1, 3136, 512) and size(0, 3, 64, 64) - size(0, 2, 64, 64) == size(0, 2, 64, 64) - size(0, 1, 64, 64) > 0
  assert size(1, 65535, 1, 1) > 0 and size(0, 1, 65536, 65536) > 1 << 32
  for bad in ((3, 1, 4, 4), (0, -1, 4, 4), (0, 65536, 4, 4), (0, 1, 0, 4), (0, 1, 4, 65537)):
    assert size(*bad) == -1
  args = lambda **kw: list({**dict(g=FAKE, dtype=0, batch=1, m=4, n=4, steps=5, a=1.0, b=1.0, c=1.0, eps=0.0, out=FAKE, ws=FAKE,  # noqa: E731
                                   bytes=1 << 30, stream=None), **kw}.values())
  for changes, code in ((dict(steps=0), -1), (dict(g=None), -1), (dict(out=FAKE + 2), -1), (dict(ws=FAKE + 16), -1), (dict(bytes=8), -4),
                        (dict(m=-4), -1)):
    assert status("dx_orthogonalize", *args(**changes)) == code
  assert status("dx_orthogonalize", *args(batch=0)) == 0


def test_cpu_tensors_are_refused():
  z, act = torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64)
  for call in (lambda: ops.token_log_prob(z, act), lambda: ops.token_policy_loss(z, act, z[:, 0], z[:, 0], 0.2),
               lambda: ops.preference_loss(z, act, act.int(), None, 0.1), lambda: ops.orthogonalize(z),
               lambda: ops.sequence_log_prob(z, act, act.int()), lambda: ops.scale_rows(z, z[0, :1]), lambda: ops.muon_apply(z, z, 1, 1),
               lambda: ops.muon_momentum(z, z, z, None, None, 0.9)):
    with pytest.raises(ValueError, match="no CPU path"):
      call()
