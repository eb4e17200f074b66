"""Losses over wide logits (ops.token_log_prob / token_policy_loss / preference_loss) and the orthogonalised update
(ops.orthogonalize, optim.Muon) on the GPU against their definitions in 64 bits.

Tolerances.  A row's sums are fp32: per thread up to V / threads sequential additions, then 12 across the workgroup,
each off by 2^-24 at most; an exponential is off by 2^-23 and its argument's rounding (|z - m| 2^-24).  ``slack(V)``
bounds the relative error of a row's sums; log-probabilities and entropies have it as their absolute error (the
logarithm turns one into the other), next to the rounding of values of their size.  A gradient element is a product of
such factors: 8 slack of its terms' magnitudes, and half a step of its own type."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
INF = float("inf")


def gen(seed):
  return torch.Generator(device=DEV).manual_seed(seed)


def slack(vocab):
  return (vocab / 64 + 48) * 2.0 ** -24 if vocab <= 4096 else (vocab / 256 + 48) * 2.0 ** -24


def logits_of(rows, vocab, dtype, seed=0, banned=True):
  z = (torch.randn(rows, vocab, generator=gen(seed), device=DEV) * 2).to(dtype)
  if banned and vocab >= 16:
    z[:, 3::8] = -INF
  actions = (torch.randint(0, max(1, vocab // 8), (rows,), generator=gen(seed + 1), device=DEV) * 8).clamp_(max=vocab - 1)
  if vocab >= 16:
    actions = torch.where(actions % 8 == 3, actions - 1, actions)
  return z, actions


def mask_of(rows, kind, seed=0):
  if kind == "none":
    return None
  if kind == "all":
    return torch.zeros(rows, dtype=torch.bool, device=DEV)
  keep = torch.rand(rows, generator=gen(seed + 9), device=DEV) < 0.7
  keep[0] = True
  return keep


def rows64(z, actions):
  """(p, log p, entropy, log-probability) in 64 bits."""
  logp = torch.log_softmax(z.double(), 1)
  p = logp.exp()
  entropy = -torch.where(p > 0, p * logp, 0.0).sum(1)
  return p, logp, entropy, logp.gather(1, actions[:, None])[:, 0]


def half_step(x, dtype):
  tiny = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -24}[dtype]
  return x.abs() * (torch.finfo(dtype).eps / 2) * 1.01 + tiny


def within(got, want, tolerance, what=""):
  got, want = got.double(), want.double()
  bad = ~((got - want).abs() <= tolerance)
  assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() / tolerance).max()):.3g} tolerances"


SIZES = [(5, 1), (5, 2), (7, 18), (300, 18), (9, 63), (4, 64), (1, 65), (6, 513), (33, 1000), (3, 2048), (3, 2049), (5, 4099),
         (2, 16384), (3, 16391), (2, 40003), (2, 65536), (1, 65541), (2, 131072), (1, 131075), (1, 262147)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,vocab", SIZES)
def test_token_log_prob(rows, vocab, dtype):
  from derl_amd import ops
  z, actions = logits_of(rows, vocab, dtype, rows + vocab)
  mask = mask_of(rows, "some", vocab)
  lp, entropy = ops.token_log_prob(z, actions, mask=mask)
  _, _, h64, lp64 = rows64(z, actions)
  keep = mask.double()
  within(lp, lp64 * keep, slack(vocab) + 2.0 ** -23 * (lp64.abs() + 16), "log_prob")
  # the entropy is log S - sum e d / S: twice the sums' error, of terms up to log V
  within(entropy, h64 * keep, 2 * slack(vocab) * (1 + math.log(vocab + 1)) + 2.0 ** -22 * (h64 + 1), "entropy")
  lp2, _ = ops.token_log_prob(z, actions)
  assert torch.equal(lp2[mask], lp[mask])


def policy_oracle(z, actions, old, adv, clip, ck, ch, ref_lp, ref_z, mask, batch=0):
  """Terms, gradient and the magnitude of the gradient's terms, in 64 bits."""
  p, logp, entropy, lp = rows64(z, actions)
  keep = torch.ones(z.shape[0], dtype=torch.bool, device=z.device) if mask is None else mask.bool()
  count = int(keep.sum())
  adv = adv.double()
  ratio = (lp - old.double()).exp()
  unclipped = -ratio * adv
  clipped = unclipped if clip is None else -ratio.clamp(1 - clip, 1 + clip) * adv
  active = unclipped >= clipped
  policy = torch.where(active, unclipped, clipped)
  g = torch.where(active, unclipped, 0.0)
  gsize = g.abs()
  kl = torch.zeros_like(lp)
  gap = torch.zeros_like(p)
  if ref_lp is not None:
    d = ref_lp.double() - lp
    kl = torch.expm1(d) - d
    g = g - ck * torch.expm1(d)
    # g = -r A - c (e^d - 1) may cancel: an error x of lp moves the first term by |r A| x and the second by c e^d x,
    # whatever their difference is, so those are the magnitudes that the relative errors apply to
    gsize = gsize + ck * torch.exp(d)
  if ref_z is not None:
    logq = torch.log_softmax(ref_z.double(), 1)
    gap = torch.where(p > 0, logp - logq, 0.0)
    kl = (p * gap).sum(1)
  onehot = torch.zeros_like(p).scatter_(1, actions[:, None].clamp(0, z.shape[1] - 1), 1.0)
  finite = torch.where(p > 0, logp, 0.0)
  w = 1.0 / (batch or max(count, 1))
  dz = g[:, None] * (onehot - p) + ch * p * (finite + entropy[:, None])
  size = gsize[:, None] * (onehot + p) + ch * p * (finite.abs() + entropy[:, None])
  if ref_z is not None:
    dz = dz + ck * p * (gap - kl[:, None])
    size = size + ck * p * (finite.abs() + gap.abs() + kl.abs()[:, None] + 8)
  dz, size = (torch.where(keep[:, None], x * w, 0.0) for x in (dz, size))
  mean = lambda x: float(x[keep].sum()) / count if count else 0.0
  outside = torch.zeros_like(lp) if clip is None else ((ratio < 1 - clip) | (ratio > 1 + clip)).double()
  terms = [mean(policy) - ch * mean(entropy) + ck * mean(kl)] + [mean(v) for v in (policy, entropy, kl, outside, ratio, lp)] + [count]
  return terms, dz, size, torch.where(keep, lp, 0.0)


def policy_inputs(rows, vocab, dtype, seed, clip=0.2):
  z, actions = logits_of(rows, vocab, dtype, seed)
  _, _, _, lp = rows64(z, actions)
  drift = 0.3 * torch.randn(rows, generator=gen(seed + 2), device=DEV, dtype=torch.float64)
  if clip:  # no ratio on a border, where the loss has no derivative
    for border in (math.log1p(-clip), math.log1p(clip)):
      drift = torch.where((drift - border).abs() < 1e-3, drift + 3e-3, drift)
  adv = torch.randn(rows, generator=gen(seed + 3), device=DEV)
  ref_lp = (lp - 0.3 * torch.randn(rows, generator=gen(seed + 4), device=DEV)).float()
  ref_z = (z.float() + 0.3 * torch.randn(z.shape, generator=gen(seed + 5), device=DEV)).to(dtype)
  return z, actions, (lp - drift).float(), adv, ref_lp, ref_z


def check_policy(got, want, vocab, dtype):
  terms, dz, size, lp = want
  loss, dlogits, log_prob = got
  s = slack(vocab)
  within(log_prob, lp, s + 2.0 ** -23 * (lp.abs() + 16), "log_prob")
  within(dlogits, dz, 8 * s * size + half_step(dz, dtype), "dlogits")
  t = torch.tensor(terms, dtype=torch.float64, device=loss.device)
  # means of per-row values whose errors are those above, times the values' magnitudes (ratios and advantages of a few)
  within(loss[:7], t[:7], 16 * s * (1 + math.log(vocab + 1)) + 2.0 ** -22 * (t[:7].abs() + 16), "terms")
  assert loss[7].item() == terms[7]


@pytest.mark.parametrize("ref", ["none", "log_prob", "logits"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,vocab", SIZES)
def test_token_policy_loss(rows, vocab, dtype, ref):
  from derl_amd import ops
  z, actions, old, adv, ref_lp, ref_z = policy_inputs(rows, vocab, dtype, 7 * rows + vocab)
  ref_lp = ref_lp if ref == "log_prob" else None
  ref_z = ref_z if ref == "logits" else None
  mask = mask_of(rows, "some", rows)
  ch = 0.0 if ref == "log_prob" else 0.01
  got = ops.token_policy_loss(z, actions, old, adv, 0.2, kl_coef=0.1, entropy_coef=ch, ref_log_prob=ref_lp, ref_logits=ref_z, mask=mask)
  check_policy(got, policy_oracle(z, actions, old, adv, 0.2, 0.1, ch, ref_lp, ref_z, mask), vocab, dtype)


@pytest.mark.parametrize("clip,batch,mask", [(None, 0, "none"), (0.1, 64, "some"), (0.0, 0, "some"), (0.2, 0, "all"), (0.2, 5, "all")])
def test_token_policy_loss_arguments(clip, batch, mask):
  """No clipping, a clipping range of nothing, a global batch, a batch that is masked altogether."""
  from derl_amd import ops
  z, actions, old, adv, ref_lp, _ = policy_inputs(40, 333, F32, 5, clip)
  if clip == 0.0:
    old = old + 0.05  # no ratio of exactly 1
  keep = mask_of(40, mask)
  got = ops.token_policy_loss(z, actions, old, adv, clip, kl_coef=0.3, entropy_coef=0.02, ref_log_prob=ref_lp, mask=keep, global_batch=batch)
  check_policy(got, policy_oracle(z, actions, old, adv, clip, 0.3, 0.02, ref_lp, None, keep, batch), 333, F32)
  if mask == "all":
    assert not got[0].any() and not got[1].any() and not got[2].any()


def test_rows_that_have_no_distribution():
  """A banned action, the type's lowest value as a mask, a row of the lowest value alone; rows without a distribution
  (-inf altogether, a NaN, +inf) or with an action outside the vocabulary are NaN and leave the other rows alone."""
  from derl_amd import ops
  for dtype in (F32, BF16, F16):
    for vocab in (40, 3000, 40000):
      z, actions = logits_of(8, vocab, dtype, 3)
      lowest = torch.finfo(dtype).min
      z[0, ::2] = lowest
      z[0, 1] = 1.0
      actions[0] = 1
      z[1] = lowest
      clean = z.clone()
      z[2] = -INF
      z[3, 7] = float("nan")
      z[4, 9] = INF
      actions[5], actions[6] = vocab, -100
      lp, entropy = ops.token_log_prob(z, actions)
      _, _, h64, lp64 = rows64(clean[[0, 1, 7]], actions[[0, 1, 7]])
      within(lp[[0, 1, 7]], lp64, slack(vocab) + 2.0 ** -23 * (lp64.abs() + 16))
      within(entropy[[0, 1, 7]], h64, 2 * slack(vocab) * (1 + math.log(vocab)) + 2.0 ** -22 * (h64 + 1))
      assert torch.isnan(lp[2:7]).all() and torch.isnan(entropy[2:5]).all()
      old, adv = torch.full((8,), -3.0, device=DEV), torch.ones(8, device=DEV)
      loss, dz, _ = ops.token_policy_loss(z, actions, old, adv, 0.2, entropy_coef=0.01)
      assert torch.isnan(loss[0]) and torch.isnan(dz[2:7]).any(1).all() and torch.isfinite(dz[[0, 1, 7]]).all()
      keep = torch.tensor([1, 1, 0, 0, 0, 0, 0, 1], dtype=torch.uint8, device=DEV)
      got = ops.token_policy_loss(z, actions, old, adv, 0.2, entropy_coef=0.01, mask=keep)
      want = policy_oracle(clean[[0, 1, 7]], actions[[0, 1, 7]], old[:3], adv[:3], 0.2, 0.0, 0.01, None, None, None)
      check_policy((got[0], got[1][[0, 1, 7]], got[2][[0, 1, 7]]), want, vocab, dtype)
      assert not got[1][2:7].any() and not got[2][2:7].any()


def test_a_banned_action_has_no_probability():
  from derl_amd import ops
  z, _ = logits_of(3, 100, F32, 1)
  actions = torch.tensor([3, 11, 19], device=DEV)  # all banned
  lp, _ = ops.token_log_prob(z, actions)
  assert (lp == -INF).all()
  loss, dz, _ = ops.token_policy_loss(z, actions, torch.full((3,), -2.0, device=DEV), torch.ones(3, device=DEV), 0.2)
  assert loss[5].item() == 0.0 and not dz.any()  # the ratio is 0 and nothing can move it


def test_exact_divergence_of_unequal_supports():
  """q = 0 where p = 0 costs nothing; q = 0 where p > 0 makes the divergence infinite."""
  from derl_amd import ops
  for vocab in (64, 5000):
    z, actions, old, adv, _, ref = policy_inputs(4, vocab, F32, 11)
    ref[0, 5::8] = -INF
    loss, dz, _ = ops.token_policy_loss(z, actions, old, adv, 0.2, kl_coef=0.1, ref_logits=ref)
    assert loss[3].item() == INF and torch.isfinite(dz[1:]).all()
    z[0, 5::8] = -INF
    keep = actions % 8 != 5
    got = ops.token_policy_loss(z, actions, old, adv, 0.2, kl_coef=0.1, ref_logits=ref, mask=keep)
    check_policy(got, policy_oracle(z, actions, old, adv, 0.2, 0.1, 0.0, None, ref, keep), vocab, F32)


@pytest.mark.parametrize("vocab", [50, 3001, 40001])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strided_rows_in_place_and_the_callers_buffer(dtype, vocab):
  from derl_amd import ops
  z, actions, old, adv, _, ref = policy_inputs(6, vocab, dtype, 21)
  mask = mask_of(6, "some", 4)
  args = dict(kl_coef=0.1, entropy_coef=0.01, mask=mask)
  want = ops.token_policy_loss(z, actions, old, adv, 0.2, ref_logits=ref, **args)
  wide = torch.full((6, vocab + 37), 7.0, dtype=dtype, device=DEV)
  view = wide[:, 5:5 + vocab]
  view.copy_(z)
  wide_ref = torch.zeros((6, vocab + 3), dtype=dtype, device=DEV)
  wide_ref[:, 2:2 + vocab] = ref
  target = torch.full((8, vocab + 1), 3.0, dtype=dtype, device=DEV)
  got = ops.token_policy_loss(view, actions, old, adv, 0.2, ref_logits=wide_ref[:, 2:2 + vocab], dlogits_out=target[1:7, 1:], **args)
  for a, b in zip(got, want):
    assert torch.equal(a, b)
  assert (target[0] == 3).all() and (target[7] == 3).all() and (target[:, 0] == 3).all()
  got = ops.token_policy_loss(view, actions, old, adv, 0.2, ref_logits=ref, dlogits_out=view, **args)
  for a, b in zip(got, want):
    assert torch.equal(a, b)
  assert (wide[:, :5] == 7).all() and (wide[:, 5 + vocab:] == 7).all()
  ref_sum = torch.tensor([-5.0, -6.0], device=DEV)
  offsets = torch.tensor([1, 3, 5], dtype=torch.int32, device=DEV)
  want = ops.preference_loss(z, actions, offsets, ref_sum, 0.3, mask=mask)
  view.copy_(z)
  got = ops.preference_loss(view, actions, offsets, ref_sum, 0.3, mask=mask, dlogits_out=view)
  for a, b in zip(got, want):
    assert torch.equal(a, b)
  assert (wide[:, :5] == 7).all() and (wide[:, 5 + vocab:] == 7).all()


def preference_oracle(z, actions, offsets, ref, beta, s, mask, batch=0):
  p, _, _, lp = rows64(z, actions)
  rows = z.shape[0]
  keep = torch.ones(rows, dtype=torch.bool, device=z.device) if mask is None else mask.bool()
  lp = torch.where(keep, lp, 0.0)
  o = offsets.tolist()
  sums = torch.stack([lp[a:b].sum() for a, b in zip(o[:-1], o[1:])])
  gain = beta * (sums - (0 if ref is None else ref.double()))
  h = gain[0::2] - gain[1::2]
  sig = torch.nn.functional.logsigmoid
  loss = -(1 - s) * sig(h) - s * sig(-h)
  slope = beta * (s * torch.sigmoid(h) - (1 - s) * torch.sigmoid(-h)) / (batch or len(h))
  row = torch.zeros(rows, dtype=torch.float64, device=z.device)
  for k, (a, b) in enumerate(zip(o[:-1], o[1:])):
    row[a:b] = slope[k // 2] * (-1 if k % 2 else 1)
  row = row * keep
  onehot = torch.zeros_like(p).scatter_(1, actions[:, None].clamp(0, z.shape[1] - 1), 1.0)
  terms = torch.stack([loss.mean(), (h > 0).double().mean(), h.mean(), gain[0::2].mean(), gain[1::2].mean(), sums[0::2].mean(),
                       sums[1::2].mean(), torch.tensor(float(len(h)), dtype=torch.float64, device=z.device)])
  return terms, torch.where(row[:, None] != 0, row[:, None] * (onehot - p), 0.0), row.abs()[:, None] * (onehot + p), sums


def check_preference(got, want, vocab, rows, dtype, beta):
  terms, dz, size, sums = want
  loss, dlogits, sequence = got
  each = slack(vocab) + 2.0 ** -23 * 40            # error of one token's log-probability
  within(sequence, sums, rows * each + 2.0 ** -24 * sums.abs(), "sequences")
  # the slope is a smooth function of h, whose error is beta times that of two sequences
  within(dlogits, dz, (8 * slack(vocab) + 4 * beta * rows * each) * size + half_step(dz, dtype), "dlogits")
  within(loss, terms, 4 * (1 + beta) * rows * each + 2.0 ** -22 * terms.abs(), "terms")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("vocab", [3, 18, 1000, 2049, 20011, 65537])
def test_preference_loss(vocab, dtype):
  from derl_amd import ops
  rows, beta = 61, 0.3
  z, actions = logits_of(rows, vocab, dtype, vocab)
  offsets = torch.tensor([2, 9, 9, 10, 31, 31, 31, 50, 58], dtype=torch.int32, device=DEV)  # empty ones, rows before and behind
  ref = -8 * torch.rand(8, generator=gen(1), device=DEV) * 5
  for mask, smooth, r, batch in ((mask_of(rows, "some", 1), 0.1, ref, 0), (None, 0.0, None, 12), (None, 1.0, ref, 0), (mask_of(rows, "all"), 0.0, ref, 0)):
    got = ops.preference_loss(z, actions, offsets, r, beta, label_smoothing=smooth, mask=mask, global_pairs=batch)
    check_preference(got, preference_oracle(z, actions, offsets, r, beta, smooth, mask, batch), vocab, rows, dtype, beta)
  assert torch.equal(ops.sequence_log_prob(z, actions, offsets), ops.preference_loss(z, actions, offsets, ref, beta)[2])


def test_many_pairs_and_extreme_margins():
  """More pairs than workgroups; a margin whose sigmoid underflows; unused rows may hold anything."""
  from derl_amd import ops
  pairs, vocab = 2500, 11
  rows = 2 * pairs * 2 + 7
  z, actions = logits_of(rows, vocab, F32, 3)
  z[-5:] = float("nan")
  actions[-3:] = -1
  offsets = (torch.arange(2 * pairs + 1, device=DEV) * 2).to(torch.int32)
  ref = torch.randn(2 * pairs, generator=gen(4), device=DEV)
  ref[0], ref[3] = 1e4, 1e4
  got = ops.preference_loss(z, actions, offsets, ref, 0.5)
  clean = torch.where(torch.isnan(z), 0.0, z)
  want = preference_oracle(clean, actions.clamp(min=0), offsets, ref, 0.5, 0.0, None)
  assert not got[1][-7:].any()
  check_preference(got, want, vocab, 8, F32, 0.5)


@pytest.mark.parametrize("borders", [[0, 20000, 40000], [3, 17001, 17001, 17050, 39000], [0, 40000, 40000]])
def test_long_sequences(borders):
  """Sequences of tens of thousands of rows, which more threads add up."""
  from derl_amd import ops
  rows, vocab, beta = 40000, 9, 2.0 ** -8
  z, actions = logits_of(rows, vocab, F32, 12, banned=False)
  mask = mask_of(rows, "some", 2)
  offsets = torch.tensor(borders, dtype=torch.int32, device=DEV)
  got = ops.preference_loss(z, actions, offsets, None, beta, mask=mask)
  check_preference(got, preference_oracle(z, actions, offsets, None, beta, 0.0, mask), vocab, rows, F32, beta)
  assert torch.equal(ops.sequence_log_prob(z, actions, offsets, mask), got[2])
  got = ops.preference_loss(z, actions, offsets, None, beta)
  check_preference(got, preference_oracle(z, actions, offsets, None, beta, 0.0, None), vocab, rows, F32, beta)


def test_gradients_against_differences():
  """<dL/dz, v> = (L(z + h v) - L(z - h v)) / 2 h up to h^2 |L'''| / 6 (third derivatives of these losses along a
  direction of length 1 are below 8 here) and the fp32 rounding of L, 2^-22 (1 + |L|) / h."""
  from derl_amd import ops
  z, actions, old, adv, ref_lp, ref_z = policy_inputs(3, 7, F32, 2)
  offsets = torch.tensor([0, 1, 3], dtype=torch.int32, device=DEV)
  h = 2.0 ** -6
  losses = [lambda x: ops.token_policy_loss(x, actions, old, adv, 0.2, kl_coef=0.2, entropy_coef=0.1, ref_log_prob=ref_lp),
            lambda x: ops.token_policy_loss(x, actions, old, adv, None, kl_coef=0.2, entropy_coef=0.1, ref_logits=ref_z),
            lambda x: ops.preference_loss(x, actions, offsets, ref_lp[:2], 0.7, label_smoothing=0.1)]
  for k, f in enumerate(losses):
    for seed in range(4):
      v = torch.randn(z.shape, generator=gen(50 + seed), device=DEV)
      v = v / v.norm()
      up, down, (terms, dz, _) = f(z + h * v)[0], f(z - h * v)[0], f(z)
      slope = (float(up[0]) - float(down[0])) / (2 * h)
      tolerance = 8 * h * h / 6 + 2.0 ** -22 * (1 + abs(float(terms[0]))) / h
      assert abs(slope - float((dz * v).sum())) <= tolerance, (k, seed)


def test_streams_graphs_and_repeats():
  """The same bits on another stream, from two streams at once, and from every replay of a captured graph with eager
  work in between; inputs changed in place are seen by the replay."""
  from derl_amd import ops
  z, actions, old, adv, ref_lp, ref_z = policy_inputs(50, 5003, BF16, 31)
  mask = mask_of(50, "some")
  offsets = torch.tensor([0, 10, 30, 31, 50], dtype=torch.int32, device=DEV)
  update = torch.randn(96, 200, generator=gen(1), device=DEV)

  def work():
    a = ops.token_log_prob(z, actions, mask)
    b = ops.token_policy_loss(z, actions, old, adv, 0.2, kl_coef=0.1, entropy_coef=0.01, ref_logits=ref_z, mask=mask)
    c = ops.preference_loss(z, actions, offsets, None, 0.2, mask=mask)
    return list(a) + list(b) + list(c) + [ops.orthogonalize(update)]

  eager = [t.clone() for t in work()]
  streams = [torch.cuda.Stream(), torch.cuda.Stream()]
  torch.cuda.synchronize()
  results = []
  for s in streams:
    with torch.cuda.stream(s):
      results.append(work())
  torch.cuda.synchronize()
  for got in results:
    assert all(torch.equal(a, b) for a, b in zip(got, eager))
  graphs = []
  for _ in range(2):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
      out = work()
    graphs.append((graph, out))
  for k in range(3):
    for graph, out in graphs:
      graph.replay()
      torch.cuda.synchronize()
      assert all(torch.equal(a, b) for a, b in zip(out, eager)), k
    work()
    adv.mul_(-1.0)
    update.mul_(0.5).add_(0.01)
    eager = [t.clone() for t in work()]
    torch.cuda.synchronize()


def test_long_rows_past_32_bits():
  """Rows whose byte offset passes 2^32 (a (70000, 32768) bf16 view with a wide pitch is not touched in between)."""
  from derl_amd import ops
  rows, vocab, pitch = 3, 129, 1_200_000_000
  if torch.cuda.mem_get_info()[0] < 12e9:
    pytest.skip("needs 8 GB of device memory")
  store = torch.empty(2 * pitch + vocab, dtype=BF16, device=DEV)
  view = store.as_strided((rows, vocab), (pitch, 1))
  z, actions, old, adv, _, _ = policy_inputs(rows, vocab, BF16, 3)
  view.copy_(z)
  want = ops.token_policy_loss(z, actions, old, adv, 0.2, entropy_coef=0.01)
  got = ops.token_policy_loss(view, actions, old, adv, 0.2, entropy_coef=0.01, dlogits_out=view)
  for a, b in zip(got, want):
    assert torch.equal(a, b)


# more rows than a launch has workgroups for them, of every length that is held in registers, and longer ones
MANY = [(2100, 4096), (2100, 8191), (2100, 16001), (600, 20011), (600, 32768), (300, 40003), (300, 65536), (300, 70001), (270, 131072),
        (140, 140001)]


@pytest.mark.parametrize("ref", ["none", "log_prob", "logits"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,vocab", MANY)
def test_many_long_rows(rows, vocab, dtype, ref):
  """The policy loss and the log-probabilities against 64 bits; the same bits in place and on rows at an odd distance; a
  row that is NaN leaves the others alone."""
  from derl_amd import ops
  z, actions, old, adv, ref_lp, ref_z = policy_inputs(rows, vocab, dtype, rows + vocab)
  ref_lp = ref_lp if ref == "log_prob" else None
  ref_z = ref_z if ref == "logits" else None
  mask = mask_of(rows, "some", rows)
  ch = 0.01 if ref == "none" else 0.0
  args = dict(kl_coef=0.1, entropy_coef=ch, ref_log_prob=ref_lp, ref_logits=ref_z, mask=mask)
  got = ops.token_policy_loss(z, actions, old, adv, 0.2, **args)
  want = policy_oracle(z, actions, old, adv, 0.2, 0.1, ch, ref_lp, ref_z, mask)
  check_policy(got, want, vocab, dtype)
  lp, entropy = ops.token_log_prob(z, actions, mask)
  within(lp, want[3], slack(vocab) + 2.0 ** -23 * (want[3].abs() + 16), "log_prob")
  h64 = torch.where(mask, rows64(z, actions)[2], 0.0)
  within(entropy, h64, 2 * slack(vocab) * (1 + math.log(vocab + 1)) + 2.0 ** -22 * (h64 + 1), "entropy")
  del want, h64
  wide = torch.full((rows, vocab + 3), 7.0, dtype=dtype, device=DEV)
  view = wide[:, 1:1 + vocab]
  view.copy_(z)
  again = ops.token_policy_loss(view, actions, old, adv, 0.2, dlogits_out=view, **args)
  for a, b in zip(again, got):
    assert torch.equal(a, b)
  assert (wide[:, 0] == 7).all() and (wide[:, 1 + vocab:] == 7).all()
  keep = torch.nonzero(mask)[:, 0]
  bad = keep[[1, len(keep) // 2, len(keep) - 1]]
  z[bad, vocab // 2] = float("nan")
  again = ops.token_policy_loss(z, actions, old, adv, 0.2, **args)
  assert torch.isnan(again[1][bad]).any(1).all() and torch.isnan(again[2][bad]).all()
  rest = torch.ones(rows, dtype=torch.bool, device=DEV)
  rest[bad] = False
  assert torch.equal(again[1][rest], got[1][rest]) and torch.equal(again[2][rest], got[2][rest])


@pytest.mark.parametrize("rows,vocab,dtype", [(600_000, 5, F32), (540_000, 18, BF16), (140_000, 4100, BF16)])
def test_more_than_64_rows_for_a_workgroup(rows, vocab, dtype):
  """The same bits as when the rows come in parts (a global batch of the whole), and the sums of the parts' terms."""
  from derl_amd import ops
  z, actions = logits_of(rows, vocab, dtype, 5, banned=False)
  old = -math.log(vocab) + 0.1 * torch.randn(rows, generator=gen(6), device=DEV)
  adv = torch.randn(rows, generator=gen(7), device=DEV)
  mask = mask_of(rows, "some", 8)
  count = int(mask.sum())
  loss, dz, lp = ops.token_policy_loss(z, actions, old, adv, 0.2, kl_coef=0.1, entropy_coef=0.01, ref_log_prob=old, mask=mask)
  assert loss[7].item() == count
  full, entropy = ops.token_log_prob(z, actions, mask)
  # (rows that are read once are summed in another order than rows that are kept: each of the two is within its own error)
  within(full, lp, 2 * (slack(vocab) + 2.0 ** -23 * (lp.abs() + 16)), "log_prob")
  sums, parts = torch.zeros(7, dtype=torch.float64, device=DEV), 50_000 if vocab < 100 else 10_000
  for at in range(0, rows, parts):
    s = slice(at, at + parts)
    l, d, p = ops.token_policy_loss(z[s], actions[s], old[s], adv[s], 0.2, kl_coef=0.1, entropy_coef=0.01, ref_log_prob=old[s], mask=mask[s],
                                    global_batch=count)
    assert torch.equal(d, dz[s]) and torch.equal(p, lp[s])
    assert torch.equal(ops.token_log_prob(z[s], actions[s], mask[s])[1], entropy[s])
    sums += l[:7].double() * l[7].double()
  # the parts' means are rounded to fp32 each (2^-24 of values below 16), and so is the whole's
  within(loss[:7], sums / count, torch.full((7,), 2.0 ** -19, dtype=torch.float64, device=DEV), "terms")


def test_more_rows_than_threads_of_a_launch():
  """70 million rows: the preference loss's gradient takes several blocks a workgroup."""
  from derl_amd import ops
  rows = 70_000_000
  if torch.cuda.mem_get_info()[0] < 12e9:
    pytest.skip("needs 8 GB of device memory")
  z = torch.randn(rows, 2, generator=gen(1), device=DEV, dtype=F32).to(BF16)
  actions = torch.randint(0, 2, (rows,), generator=gen(2), device=DEV)
  mask = torch.ones(rows, dtype=torch.uint8, device=DEV)
  mask[::3] = 0
  offsets = torch.tensor([0, 5, 9, rows - 4, rows], dtype=torch.int32, device=DEV)
  loss, dz, seq = ops.preference_loss(z, actions, offsets, None, 1e-6, mask=mask)
  lp, _ = ops.token_log_prob(z, actions, mask)
  want = torch.stack([lp[a:b].double().sum() for a, b in ((0, 5), (5, 9), (9, rows - 4), (rows - 4, rows))])
  within(seq, want, 2.0 ** -23 * want.abs(), "sequences")
  # a row's gradient: c (1 - p) and -c (1 - p), p the action's probability, c = -+ sigmoid(-h) 1e-6 / 2
  h = 1e-6 * (want[0::2] - want[1::2])
  c = torch.sigmoid(-h) * 1e-6 / 2
  row = torch.cat([-c[0].expand(5), c[0].expand(4), -c[1].expand(rows - 13), c[1].expand(4)]) * (mask != 0)
  for at in range(0, rows, 10_000_000):
    s = slice(at, at + 10_000_000)
    first = row[s] * (1 - torch.softmax(z[s].double(), 1).gather(1, actions[s, None])[:, 0])
    got = dz[s].double().gather(1, actions[s, None])[:, 0]
    within(got, first, half_step(first, BF16) + 2.0 ** -18 * row[s].abs(), "dlogits")
    assert torch.equal(dz[s].gather(1, actions[s, None]), -dz[s].gather(1, 1 - actions[s, None])) or \
        float((dz[s].double().sum(1).abs() / (row[s].abs() + 1e-30)).max()) <= 2.0 ** -8


@pytest.mark.parametrize("kind", ["log_prob", "logits"])
@pytest.mark.parametrize("vocab", [40, 5000, 40000])
def test_a_divergence_that_is_only_reported(vocab, kind):
  """kl_coef = 0: the divergence is reported, and where it is infinite neither the loss nor the gradient holds any of it."""
  from derl_amd import ops
  z, actions, old, adv, ref_lp, ref_z = policy_inputs(8, vocab, F32, 3)
  want = ops.token_policy_loss(z, actions, old, adv, 0.2, entropy_coef=0.01)
  ref_lp[2] = 1000.0
  ref_z[2, 5::8] = -INF
  args = dict(ref_log_prob=ref_lp) if kind == "log_prob" else dict(ref_logits=ref_z)
  got = ops.token_policy_loss(z, actions, old, adv, 0.2, entropy_coef=0.01, **args)
  assert got[0][3].item() == INF
  within(got[0][[0, 1, 2, 4, 5, 6, 7]], want[0][[0, 1, 2, 4, 5, 6, 7]], 16 * slack(vocab) * (1 + math.log(vocab)), "terms")
  _, dz, size, lp = policy_oracle(z, actions, old, adv, 0.2, 0.0, 0.01, None, None, None)
  within(got[1], dz, 8 * slack(vocab) * size + half_step(dz, F32), "dlogits")


@pytest.mark.parametrize("rows", [1, 15, 16, 17, 4099, 100_003])
def test_mask_of_any_bytes_and_any_start(rows):
  """A uint8 mask counts what is not 0, wherever it begins."""
  from derl_amd import ops
  z = torch.zeros(rows, 2, device=DEV)
  actions = torch.zeros(rows, dtype=torch.int64, device=DEV)
  one = torch.zeros(rows, device=DEV)
  store = torch.randint(0, 256, (rows + 5,), generator=gen(rows), device=DEV, dtype=torch.uint8)
  store[torch.rand(rows + 5, generator=gen(rows + 1), device=DEV) < 0.4] = 0
  for start in (0, 1, 5):
    mask = store[start:start + rows]
    loss, dz, _ = ops.token_policy_loss(z, actions, one, one, 0.2, mask=mask)
    assert loss[7].item() == int((mask != 0).sum())
    assert not dz[mask == 0].any()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_the_same_index_twice_and_every_action(dtype):
  """Rows that share an action, and each action of a vocabulary once, at widths around a wave's and a vector's."""
  from derl_amd import ops
  for vocab in (1, 7, 8, 9, 63, 64, 65, 515, 2051):
    z, _, old, adv, ref_lp, _ = policy_inputs(vocab, vocab, dtype, vocab, clip=None)
    z = logits_of(vocab, vocab, dtype, vocab, banned=False)[0]
    for actions in (torch.arange(vocab, device=DEV), torch.full((vocab,), vocab - 1, device=DEV)):
      got = ops.token_policy_loss(z, actions, old, adv, None, kl_coef=0.1, entropy_coef=0.01, ref_log_prob=ref_lp)
      dz = policy_oracle(z, actions, old, adv, None, 0.1, 0.01, ref_lp, None, None)
      s = slack(vocab)
      within(got[2], dz[3], s + 2.0 ** -23 * (dz[3].abs() + 16), "log_prob")
      within(got[1], dz[1], 8 * s * (dz[2] + 0.1 / vocab) + half_step(dz[1], dtype), "dlogits")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("vocab", [16, 17, 60, 129, 255, 300, 513, 1030, 2051, 2100, 4090, 4099, 5121, 8190])
def test_rows_of_every_length_in_lanes_and_waves(vocab, dtype):
  """More rows than one turn of the grid takes at the lengths where the threads of a row change, masked and not, from odd
  starts; rows beside each other share cache lines."""
  from derl_amd import ops
  rows = 40003 if vocab < 300 else 9001
  z, actions = logits_of(rows, vocab, dtype, vocab)
  old = -math.log(vocab) - 1 + 0.1 * torch.randn(rows, generator=gen(6), device=DEV)
  adv = torch.randn(rows, generator=gen(7), device=DEV)
  mask = mask_of(rows, "some", 8)
  _, _, h64, lp64 = rows64(z, actions)
  lp, entropy = ops.token_log_prob(z, actions, mask)
  s = slack(vocab)
  within(lp, torch.where(mask, lp64, 0.0), s + 2.0 ** -23 * (lp64.abs() + 16), "log_prob")
  within(entropy, torch.where(mask, h64, 0.0), 2 * s * (1 + math.log(vocab + 1)) + 2.0 ** -22 * (h64 + 1), "entropy")
  got = ops.token_policy_loss(z, actions, old, adv, None, kl_coef=0.1, entropy_coef=0.01, ref_log_prob=old, mask=mask)
  check_policy(got, policy_oracle(z, actions, old, adv, None, 0.1, 0.01, old, None, mask), vocab, dtype)
  wide = torch.zeros((rows, vocab + 1), dtype=dtype, device=DEV)
  view = wide[:, 1:]
  view.copy_(z)
  again = ops.token_policy_loss(view, actions, old, adv, None, kl_coef=0.1, entropy_coef=0.01, ref_log_prob=old, mask=mask, dlogits_out=view)
  for a, b in zip(again, got):
    assert torch.equal(a, b)
  assert not wide[:, 0].any()
  view.copy_(z)
  offsets = torch.tensor([0, rows // 3, rows // 2, rows - 9, rows], dtype=torch.int32, device=DEV)
  want = ops.preference_loss(z, actions, offsets, None, 2.0 ** -10, mask=mask)
  for a, b in zip(ops.preference_loss(view, actions, offsets, None, 2.0 ** -10, mask=mask, dlogits_out=view), want):
    assert torch.equal(a, b)
  check_preference(want, preference_oracle(z, actions, offsets, None, 2.0 ** -10, 0.0, mask), vocab, rows, dtype, 2.0 ** -10)


def test_the_longest_rows():
  """Two rows of 2^30 - 3 columns, nearly 4 GB each.  A thread adds at most 2^15 columns to its sum (128 pieces of 256
  threads a row): 2^15 roundings of 2^-24 each, and the joins' 60."""
  from derl_amd import ops
  rows, vocab = 2, 2 ** 30 - 3
  if torch.cuda.mem_get_info()[0] < 40e9:
    pytest.skip("needs 40 GB of device memory")
  z = torch.empty(rows, vocab, device=DEV)
  z.normal_(generator=gen(1))
  actions = torch.tensor([vocab - 1, vocab // 2 + 5], device=DEV)
  z[0, vocab - 1], z[1, vocab // 2 + 5] = 24.0, 21.0
  total = torch.zeros(rows, dtype=torch.float64, device=DEV)
  for at in range(0, vocab, 1 << 27):
    total += z[:, at:at + (1 << 27)].double().exp().sum(1)
  want = z.gather(1, actions[:, None])[:, 0].double() - total.log()
  s = (2 ** 15 + 60) * 2.0 ** -24
  lp, _ = ops.token_log_prob(z, actions)
  within(lp, want, s + 2.0 ** -23 * (want.abs() + 32), "log_prob")
  old, adv = want.float() - 0.05, torch.tensor([1.0, -2.0], device=DEV)
  _, dz, lp = ops.token_policy_loss(z, actions, old, adv, 0.2)
  within(lp, want, s + 2.0 ** -23 * (want.abs() + 32), "log_prob")
  g = -(want - old.double()).exp() * adv.double() / 2
  offsets = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
  _, dz2, seq = ops.preference_loss(z, actions, offsets, None, 0.5)
  slope = -0.5 * torch.sigmoid(-0.5 * (want[0] - want[1]))
  c = torch.stack([slope, -slope])
  for first in (0, vocab // 2 - 500, vocab - 1000):
    at = torch.arange(first, first + 1000, device=DEV)
    p = z[:, first:first + 1000].double().exp() / total[:, None]
    onehot = (at[None] == actions[:, None]).double()
    for got, k in ((dz, g), (dz2, c)):
      size = k.abs()[:, None] * (onehot + p)
      exact = k[:, None] * (onehot - p)
      within(got[:, first:first + 1000], exact, 8 * s * size + half_step(exact, F32), "dlogits")


# ---- orthogonalisation ---------------------------------------------------------------------------

A, B, C = 3.4445, -4.7750, 2.0315


def newton_schulz64(g, steps, coefficients=(A, B, C), eps=1e-7):
  """(result, Frobenius norms of every step's X) in 64 bits."""
  a, b, c = coefficients
  x = g.double()
  x = x / (torch.linalg.matrix_norm(x) + eps)
  tall = x.shape[0] > x.shape[1]
  x = x.t().contiguous() if tall else x
  norms = [float(x.norm())]
  for _ in range(steps):
    gram = x.mm(x.t())
    x = a * x + (b * gram + c * gram.mm(gram)).mm(x)
    norms.append(float(x.norm()))
  return (x.t().contiguous() if tall else x), norms


def check_orthogonal(got, g, steps, dtype):
  """Each step rounds X, A and B (two fp16 terms: 2^-22 each, one: 2^-12; fp32 accumulation: 2^-24 sqrt(K) each) and
  passes the error on multiplied by the polynomial's slope, a at most.  In Frobenius norm."""
  want, norms = newton_schulz64(g, steps)
  unit = (3 * 2.0 ** -12 if dtype == BF16 else 3 * 2.0 ** -22) + 3 * 2.0 ** -24 * max(g.shape) ** 0.5
  bound = 2 * unit * sum(A ** (steps - k) * n for k, n in enumerate(norms)) + torch.finfo(dtype).eps / 2 * norms[-1]
  assert got.dtype == dtype and got.shape == g.shape
  assert float((got.double() - want).norm()) <= bound, (float((got.double() - want).norm()), bound)


SHAPES = [(1, 1), (1, 9), (9, 1), (3, 5), (17, 16), (64, 64), (64, 11), (64, 576), (65, 63), (128, 128), (129, 300), (300, 129),
          (256, 32), (512, 640), (512, 3136), (700, 1500)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m,n", SHAPES)
def test_orthogonalize(m, n, dtype):
  from derl_amd import ops
  g = (torch.randn(m, n, generator=gen(m + n), device=DEV) * 0.02).to(dtype)
  keep = g.clone()
  for steps in (5, 1, 2):
    check_orthogonal(ops.orthogonalize(g, steps=steps), g, steps, dtype)
  assert torch.equal(g, keep)
  again = ops.orthogonalize(g, steps=5, out=g)
  assert again is g and torch.equal(g, ops.orthogonalize(keep))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m,n", [(64, 256), (100, 417), (300, 1100), (1300, 260)])
def test_orthogonalize_well_conditioned(m, n, dtype):
  """Sides of 1 : 4: the singular values of X0 lie within a factor of 3 of each other, relative errors are not amplified:
  6 roundings a step (2^-22 or 2^-12 each, and fp32 accumulation) and the output's own."""
  from derl_amd import ops
  g = torch.randn(3, m, n, generator=gen(m), device=DEV).to(dtype)
  got = ops.orthogonalize(g)
  for k in range(3):
    want, norms = newton_schulz64(g[k], 5)
    unit = 5 * 6 * (2.0 ** -22 if dtype == F32 else 2.0 ** -12) + 15 * 2.0 ** -24 * n ** 0.5
    assert float((got[k].double() - want).norm()) <= (unit + torch.finfo(dtype).eps / 2) * norms[-1]
    sigma = torch.linalg.svdvals(got[k].double())
    assert sigma.min() > 0.6 and sigma.max() < 1.3


def test_orthogonalize_values():
  """Zeros, norms at the ends of fp32's range, one entry alone, NaN; other coefficients; batches of batches; nothing."""
  from derl_amd import ops
  assert not ops.orthogonalize(torch.zeros(70, 200, device=DEV)).any()
  g = torch.randn(70, 200, generator=gen(1), device=DEV)
  base = ops.orthogonalize(g, eps=0.0)
  for scale in (2.0 ** 100, 2.0 ** -60):
    assert float((ops.orthogonalize(g * scale, eps=0.0) - base).abs().max()) <= 2.0 ** -18
  one = torch.zeros(20, 30, device=DEV)
  one[3, 4] = -5.0
  check_orthogonal(ops.orthogonalize(one), one, 5, F32)
  bad = g.clone()
  bad[3, 4] = float("nan")
  assert torch.isnan(ops.orthogonalize(bad)).all()
  cubic = (1.5, -0.5, 0.0)
  want, _ = newton_schulz64(g, 8, cubic)
  assert float((ops.orthogonalize(g, steps=8, coefficients=cubic).double() - want).norm()) <= 8 * 2.0 ** -18 * float(want.norm())
  nested = torch.randn(2, 3, 33, 20, generator=gen(5), device=DEV)
  got = ops.orthogonalize(nested)
  for i in range(2):
    for j in range(3):
      assert torch.equal(got[i, j], ops.orthogonalize(nested[i, j].contiguous()))
  assert ops.orthogonalize(torch.zeros(0, 4, 5, device=DEV)).shape == (0, 4, 5)
  assert ops.orthogonalize(torch.zeros(4, 0, device=DEV)).shape == (4, 0)


@pytest.mark.parametrize("shape", [(40, 60), (130, 500)])
def test_orthogonalize_at_the_ends_of_the_range(shape):
  """Powers of two change nothing but the smallest entries, which may round to multiples of 2^-149 (2^-29 of entries of
  2^-120); an infinity, like a NaN, leaves nothing."""
  from derl_amd import ops
  g = torch.randn(shape, generator=gen(7), device=DEV)
  base = ops.orthogonalize(g, eps=0.0)
  for scale in (2.0 ** 120, 2.0 ** -120, -1.0):
    got = ops.orthogonalize(g * scale, eps=0.0)
    assert float((got * math.copysign(1.0, scale) - base).abs().max()) <= 2.0 ** -18, scale
  for bad in (INF, -INF, float("nan")):
    broken = g.clone()
    broken[3, 5] = bad
    assert torch.isnan(ops.orthogonalize(broken)).all()
  assert torch.isnan(ops.orthogonalize(torch.zeros(shape, device=DEV), eps=0.0)).all()


# every tile side, split and number of terms: one matrix and batches of them, sides that end inside a tile
BATCHES = [(40, 318, 319), (40, 575, 570), (30, 700, 703), (16, 703, 700), (8, 704, 2111), (3, 700, 1500), (16, 959, 950), (40, 511, 127),
           (16, 384, 1535), (40, 190, 1530), (1, 190, 1530), (1, 701, 5632), (1, 2001, 2100), (1, 4600, 1150), (1, 1150, 9200),
           (1, 2900, 1300), (2, 3600, 3585)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("batch,m,n", BATCHES)
def test_orthogonalize_batches(batch, m, n, dtype):
  from derl_amd import ops
  g = (torch.randn(batch, m, n, generator=gen(batch + m + n), device=DEV) * 0.02).to(dtype)
  got = ops.orthogonalize(g, steps=3)
  for k in {0, batch // 2, batch - 1}:
    check_orthogonal(got[k], g[k], 3, dtype)
  assert torch.equal(ops.orthogonalize(g, steps=3), got)  # split sums are added in one order
  ops.orthogonalize(g, steps=3, out=g)
  assert torch.equal(g, got)


# ---- together ------------------------------------------------------------------------------------

def test_refusals():
  from derl_amd import ops
  z, actions, old, adv, ref_lp, ref_z = policy_inputs(6, 40, F32, 1)
  call = lambda **kw: ops.token_policy_loss(**{**dict(logits=z, actions=actions, old_log_prob=old, advantages=adv, cliprange=0.2), **kw})
  bad = [dict(logits=z.cpu()), dict(logits=z.double()), dict(logits=z[0]), dict(logits=z.t()), dict(logits=z[:, ::2]),
         dict(logits=z[:1].expand(6, 40)), dict(logits=z[:, :0]), dict(actions=actions.int()), dict(actions=actions[:5]),
         dict(actions=actions.cpu()), dict(old_log_prob=old.double()), dict(advantages=adv[None]), dict(mask=adv),
         dict(mask=torch.ones(5, dtype=torch.bool, device=DEV)), dict(ref_log_prob=ref_lp, ref_logits=ref_z),
         dict(ref_logits=ref_z.bfloat16()), dict(ref_logits=ref_z[:5]), dict(cliprange=-0.1), dict(cliprange=float("nan")),
         dict(dlogits_out=torch.empty(6, 41, device=DEV)), dict(dlogits_out=z.bfloat16()), dict(ref_logits=ref_z, dlogits_out=ref_z)]
  for kw in bad:
    with pytest.raises(ValueError):
      call(**kw)
  big = torch.zeros(7, 40, device=DEV)
  with pytest.raises(ValueError, match="overlaps"):
    call(logits=big[:6], dlogits_out=big[1:])
  offsets = torch.tensor([0, 2, 6], dtype=torch.int32, device=DEV)
  for kw in (dict(offsets=offsets[:2]), dict(offsets=offsets.long()), dict(offsets=offsets.cpu()), dict(ref_log_prob=ref_lp),
             dict(label_smoothing=1.5), dict(offsets=offsets[None])):
    with pytest.raises(ValueError):
      ops.preference_loss(**{**dict(logits=z, actions=actions, offsets=offsets, ref_log_prob=None, beta=0.1), **kw})
  g = torch.zeros(4, 6, device=DEV)
  for args in ((g.cpu(),), (g.double(),), (g[0],), (g.t(),), (g, 0), (g, 5, (1.0, float("inf"), 0.0)), (g, 5, (1.0, 0.0, 0.0), -1.0)):
    with pytest.raises(ValueError):
      ops.orthogonalize(*args)
  with pytest.raises(ValueError):
    ops.orthogonalize(g, out=torch.zeros(4, 5, device=DEV))
  with pytest.raises(ValueError):
    ops.orthogonalize(big[:6], out=big[1:])


def test_negative_shares_and_too_many_matrices_are_refused():
  from derl_amd import ops
  z, actions, old, adv, _, _ = policy_inputs(6, 40, F32, 1)
  with pytest.raises(ValueError, match="global_batch"):
    ops.token_policy_loss(z, actions, old, adv, 0.2, global_batch=-1)
  with pytest.raises(ValueError, match="global_pairs"):
    ops.preference_loss(z, actions, torch.tensor([0, 2, 6], dtype=torch.int32, device=DEV), None, 0.1, global_pairs=-1)
  with pytest.raises(RuntimeError, match="batch"):
    ops.orthogonalize(torch.zeros(65536, 2, 2, device=DEV))


def test_no_rows():
  from derl_amd import ops
  z = torch.empty(0, 17, device=DEV)
  none, act = torch.empty(0, device=DEV), torch.empty(0, dtype=torch.int64, device=DEV)
  lp, entropy = ops.token_log_prob(z, act)
  assert lp.shape == entropy.shape == (0,)
  loss, dz, lp = ops.token_policy_loss(z, act, none, none, 0.2)
  assert not loss.any() and dz.shape == (0, 17)
  loss, dz, seq = ops.preference_loss(z, act, torch.zeros(3, dtype=torch.int32, device=DEV), None, 0.1)
  assert abs(loss[0].item() - math.log(2)) < 1e-6 and not seq.any() and dz.shape == (0, 17)


def test_losses_train_a_module_and_muon_steps_its_matrix():
  """The classes on a torch module: gradients of a linear policy from both losses against autograd in 64 bits, the
  summaries' terms, a scaled loss, a second backward; then the update those gradients make orthogonal."""
  import derl_amd as derl
  from derl_amd import ops
  torch.manual_seed(0)
  hidden, vocab, batch, length = 24, 130, 3, 8
  model = torch.nn.Linear(hidden, vocab).to(DEV)
  obs = torch.randn(batch, length, hidden, device=DEV)
  actions = torch.randint(0, vocab, (batch, length), device=DEV)
  mask = torch.rand(batch, length, device=DEV) < 0.8
  with torch.no_grad():
    lp, _ = ops.token_log_prob(model(obs).reshape(-1, vocab), actions.reshape(-1))
  old = (lp + 0.05 * torch.randn_like(lp)).view(batch, length)
  data = dict(observations=obs, actions=actions, log_prob=old, advantages=torch.randn(batch, length, device=DEV),
              ref_log_prob=(lp + 0.1).view(batch, length), mask=mask)
  loss_fn = derl.TokenPolicyLoss(model, cliprange=0.5, kl_coef=0.1, entropy_coef=0.01)
  assert loss_fn.name == "tokenpolicy"

  def reference(kind):
    w, b = model.weight.detach().double().requires_grad_(), model.bias.detach().double().requires_grad_()
    logp = torch.log_softmax(obs.double().reshape(-1, hidden) @ w.t() + b, 1)
    chosen = logp.gather(1, actions.reshape(-1, 1))[:, 0]
    k = mask.reshape(-1).double()
    if kind == "policy":
      r = (chosen - old.reshape(-1).double()).exp()
      a = data["advantages"].reshape(-1).double()
      d = data["ref_log_prob"].reshape(-1).double() - chosen
      each = -torch.min(r * a, r.clamp(0.5, 1.5) * a) + 0.1 * (d.exp() - 1 - d) + 0.01 * (logp.exp() * logp).sum(1)
      loss = (each * k).sum() / k.sum()
    else:
      sums = torch.stack([(chosen * k)[i:j].sum() for i, j in ((0, 4), (4, 10), (10, 17), (17, 20))])
      loss = -torch.nn.functional.logsigmoid(0.1 * (sums[0::2] - sums[1::2])).mean()
    loss.backward()
    return loss.item(), w.grad, b.grad

  pref_fn = derl.PreferenceLoss(model, beta=0.1)
  pref = dict(observations=obs, actions=actions, mask=mask, offsets=torch.tensor([0, 4, 10, 17, 20], device=DEV))
  for kind, fn, d in (("policy", loss_fn, data), ("preference", pref_fn, pref)):
    value, gw, gb = reference(kind)
    for factor in (1.0, 3.0):
      model.zero_grad()
      loss = fn(d)
      (loss * factor).backward(retain_graph=True)
      assert abs(loss.item() - value) < 1e-5 * (1 + abs(value))
      # the library's fp32 products around the loss: a sum of 24 terms each way
      assert float((model.weight.grad.double() - factor * gw).norm()) < 2e-5 * factor * float(gw.norm())
      assert float((model.bias.grad.double() - factor * gb).norm()) < 2e-5 * factor * float(gb.norm())
      with pytest.raises(RuntimeError, match="already handed on"):
        loss.backward()
    assert fn.call_count == 2 and fn.last_terms.shape == (8,)
  step = ops.orthogonalize(model.weight.grad)
  check_orthogonal(step, model.weight.grad, 5, F32)
  with torch.no_grad():
    model.weight -= 0.1 * step
  assert torch.isfinite(pref_fn(pref)).item()
  with pytest.raises(ValueError, match="old|log_prob"):
    loss_fn({k: v for k, v in data.items() if k != "log_prob"})


def test_a_captured_training_step():
  """Loss, backward and the orthogonalised update of a policy captured as one graph: every replay, with the inputs
  changed in place and eager work in between, gives what the eager step gives."""
  import derl_amd as derl
  from derl_amd import ops
  hidden, vocab, rows = 64, 3001, 24
  model = torch.nn.Linear(hidden, vocab, bias=False).to(DEV)
  obs = torch.randn(rows, hidden, generator=gen(1), device=DEV)
  actions = torch.randint(0, vocab, (rows,), generator=gen(2), device=DEV)
  mask = torch.rand(rows, generator=gen(3), device=DEV) < 0.8
  old = torch.full((rows,), -8.0, device=DEV)
  adv = torch.randn(rows, generator=gen(4), device=DEV)
  offsets = torch.tensor([0, 5, 11, 20, 24], dtype=torch.int32, device=DEV)
  policy, preference = derl.TokenPolicyLoss(model, kl_coef=0.1, entropy_coef=0.01), derl.PreferenceLoss(model, beta=0.2)
  data = dict(observations=obs, actions=actions, log_prob=old, advantages=adv, ref_log_prob=old, mask=mask)
  pairs = dict(observations=obs, actions=actions, offsets=offsets, mask=mask)

  def step():
    model.weight.grad = None
    loss = policy(data) + 0.5 * preference(pairs)
    loss.backward()
    return loss.detach(), model.weight.grad, ops.orthogonalize(model.weight.grad)

  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    for _ in range(2):
      step()
  torch.cuda.current_stream().wait_stream(side)
  model.weight.grad = None
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    captured = step()
  kept = model.weight.grad
  for k in range(4):
    graph.replay()
    torch.cuda.synchronize()
    got = [t.clone() for t in captured]
    want = [t.clone() for t in step()]
    for a, b in zip(got, want):
      assert torch.equal(a, b), k
    obs.mul_(-0.9)
    adv.add_(0.1)
    actions.copy_((actions * 7 + 1) % vocab)
    torch.cuda.synchronize()
  assert kept is captured[1]


def muon_reference(params, grads, state, spans, matrices, step, lr, max_norm, mu=0.95, betas=(0.9, 0.999), eps=1e-8, decay=0.0):
  """One step of the flat optimizer in 64 bits; returns the new parameters."""
  norm = float(np.sqrt((grads ** 2).sum()))
  g = grads * min(1.0, max_norm / (norm + 1e-6))
  out = params.copy()
  for begin, end, rows, cols in matrices:
    m = state["m"][begin:end]
    m += (1 - mu) * (g[begin:end] - m)
    u = g[begin:end] + mu * (m - g[begin:end])
    o, _ = newton_schulz64(torch.from_numpy(u.reshape(rows, cols)), 5)
    out[begin:end] = out[begin:end] * (1 - lr * decay) - lr * max(1, rows / cols) ** 0.5 * o.numpy().reshape(-1)
  for begin, end in spans:
    m, v = state["m"][begin:end], state["v"][begin:end]
    m *= betas[0]
    m += (1 - betas[0]) * g[begin:end]
    v *= betas[1]
    v += (1 - betas[1]) * g[begin:end] ** 2
    out[begin:end] -= lr / (1 - betas[0] ** step) * m / (np.sqrt(v) / math.sqrt(1 - betas[1] ** step) + eps)
  return out


@pytest.mark.parametrize("kind", ["cnn", "mlp"])
def test_muon_steps(kind):
  """optim.Muon on both engines: every parameter is stepped once, matrices by the orthogonalised momentum, the rest by
  Adam, against the same step in 64 bits."""
  import derl_amd as derl
  from derl_amd.optim import Muon
  torch.manual_seed(1)
  model = derl.NatureCNNModel([4, 1], max_batch=8) if kind == "cnn" else derl.MuJoCoModel(11, [3, 1])
  opt = Muon(model, lr=0.02, weight_decay=0.1, eps=1e-5)
  names = {name for name, _ in model.named_parameters()}
  assert names == set(model.engine.named_views(model.engine.params))
  covered = sorted([(b, e) for b, e, _, _ in opt._matrices] + opt._spans)
  assert covered[0][0] == 0 and covered[-1][1] == model.engine.params.numel() and all(x[1] == y[0] for x, y in zip(covered, covered[1:]))
  assert len(opt._matrices) == 4
  state = dict(m=np.zeros(model.engine.params.numel()), v=np.zeros(model.engine.params.numel()))
  opt.max_grad_norm = 0.5
  for step in range(1, 4):
    before = model.engine.params.cpu().double().numpy()
    model.engine.grads.copy_(torch.randn(model.engine.grads.numel(), generator=gen(step), device=DEV) * 0.1)
    want = muon_reference(before, model.engine.grads.cpu().double().numpy(), state, opt._spans, opt._matrices, step, 0.02, 0.5, eps=1e-5, decay=0.1)
    opt.reduce_and_norm()
    opt.step()
    got = model.engine.params.cpu().double().numpy()
    # fp32 moments (3 roundings a step), Adam's quotient, an orthogonalised element off by its matrix's error (2^-12 of
    # the largest singular value's worth at most, see check_orthogonal), times the learning rate
    np.testing.assert_allclose(got, want, rtol=1e-6, atol=0.02 * 2e-4)
  assert opt.step_count == 3 and set(opt.state_dict()) == {"step", "exp_avg", "exp_avg_sq"}
  with pytest.raises(ValueError, match="matrices"):
    Muon(model, matrices=["no such weight"])


def test_ppo_factory_with_muon():
  """The trainer's path: PPOFactory(optimizer="muon") on the synthetic device env, two minibatch steps."""
  import derl_amd as derl
  from derl_amd.optim import Muon
  env = derl.env.make("Hopper-v2", nenvs=4)
  factory = derl.PPOFactory.from_default_kwargs("mujoco", num_runner_steps=16, num_minibatches=2, num_epochs=1, num_train_steps=200,
                                                optimizer="muon", lr=1e-3)
  alg = factory.make(env, nlogs=1)
  assert isinstance(alg.trainer.optimizer, Muon)
  before = alg.model.engine.params.clone()
  for k, data in enumerate(alg.runner.run()):
    loss = alg.step(data)
    if k == 1:
      break
  assert torch.isfinite(torch.as_tensor(loss)).all() and torch.isfinite(alg.model.engine.params).all()
  assert not torch.equal(before, alg.model.engine.params)
  with pytest.raises(ValueError, match="optimizer"):
    derl.PPOFactory.from_default_kwargs("mujoco", optimizer="sgd").make(env, nlogs=1)
