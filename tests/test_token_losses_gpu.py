"""Gradients and terms of the token losses where their arithmetic can fail: banned columns, coefficients past the row
count.  Oracles and tolerances are those of tests/test_tokens_gpu.py."""
import pytest
import torch

from tests.test_tokens_gpu import (BF16, DEV, F16, F32, INF, check_policy, gen, half_step, policy_inputs, policy_oracle,
                                   preference_oracle, slack, within)

pytestmark = pytest.mark.gpu

# (rows, columns) for 16 lanes a row, a wave, 256 .. 1024 threads with the row in registers, rows read twice, rows in pieces
KERNELS = [(3, 18), (5, 250), (4, 1000), (3, 4000), (130, 8191), (130, 20011), (130, 40003), (130, 65541), (130, 131100), (2, 20011)]


@pytest.mark.parametrize("coefficient,batch", [(1.5, 0), (-2.0, 0), (3.0, 1), (-40.0, 16)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,vocab", KERNELS)
def test_an_entropy_coefficient_past_the_row_count(rows, vocab, dtype, coefficient, batch):
  """One unmasked row, or a given batch below the coefficient: banned columns (-inf, or the type's lowest value) have a
  gradient of 0, the others theirs."""
  from derl_amd import ops
  z, actions, old, adv, _, _ = policy_inputs(rows, vocab, dtype, 3 * vocab)
  z[:, 6::8] = torch.finfo(dtype).min
  actions = torch.where(actions % 8 == 6, actions - 1, actions)
  mask = torch.zeros(rows, dtype=torch.bool, device=DEV)
  mask[rows // 2] = True
  logp = torch.log_softmax(z.double(), 1).gather(1, actions[:, None])[:, 0]
  old = (logp + 0.05).float()
  got = ops.token_policy_loss(z, actions, old, adv, 0.2, entropy_coef=coefficient, mask=mask, global_batch=batch)
  assert not got[1][:, 3::8].any() and not got[1][:, 6::8].any()
  terms, dz, _, lp = policy_oracle(z, actions, old, adv, 0.2, 0.0, coefficient, None, None, mask, batch)
  size = policy_oracle(z, actions, old, adv, 0.2, 0.0, abs(coefficient), None, None, mask, batch)[2]
  loss = got[0].clone()
  loss[0] = 0  # (a difference of terms that the coefficient scales: looked at below)
  check_policy((loss, got[1], got[2]), ([0.0] + terms[1:], dz, size, lp), vocab, dtype)
  assert abs(float(got[0][0]) - terms[0]) <= 2.0 ** -16 * (1 + abs(coefficient)) * (1 + abs(terms[2]))


def test_an_infinite_ratio_leaves_banned_columns_alone():
  from derl_amd import ops
  for vocab in (40, 3000, 9000):
    z, actions, old, _, _, _ = policy_inputs(4, vocab, F32, 1)
    _, dz, _ = ops.token_policy_loss(z, actions, old - 200.0, torch.full((4,), -1.0, device=DEV), None)
    assert not dz[:, 3::8].any() and not torch.isfinite(dz.gather(1, actions[:, None])).any()
    assert INF in dz.abs()


def losses_of(model, rows, vocab, hidden, seed=0):
  """Both classes on ``model`` with a batch for each: [(loss, data)]."""
  import derl_amd as derl
  g = torch.Generator(device=DEV).manual_seed(seed)
  obs = torch.randn(rows, hidden, generator=g, device=DEV).to(next(model.parameters()).dtype)
  actions = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
  old = -torch.rand(rows, generator=g, device=DEV) - float(torch.tensor(vocab).log())
  adv = torch.randn(rows, generator=g, device=DEV)
  offsets = torch.tensor([0, rows // 4, rows // 2, rows - 1, rows], dtype=torch.int32, device=DEV)
  mask = torch.rand(rows, generator=g, device=DEV) < 0.8
  mask[0] = True
  return [(derl.TokenPolicyLoss(model, cliprange=0.5, kl_coef=0.1, entropy_coef=0.01),
           dict(observations=obs, actions=actions, log_prob=old, advantages=adv, ref_log_prob=old - 0.1, mask=mask)),
          (derl.PreferenceLoss(model, beta=0.2), dict(observations=obs, actions=actions, offsets=offsets, mask=mask))]


def test_second_derivatives_are_refused():
  """Not where a graph of the gradient is only asked for: where it is differentiated, also in part."""
  model = torch.nn.Sequential(torch.nn.Linear(8, 16), torch.nn.Tanh(), torch.nn.Linear(16, 50)).to(DEV)
  for loss_fn, data in losses_of(model, 12, 50, 8):
    once = torch.autograd.grad(loss_fn(data), model.parameters())
    grads = torch.autograd.grad(loss_fn(data), model.parameters(), create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(once, grads))
    for part in (grads, grads[:1], grads[-1:]):
      with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(sum(x.square().sum() for x in part), model.parameters(), retain_graph=True, allow_unused=True)


@pytest.mark.parametrize("apart", [30.0, -3000.0, 30000.0])
@pytest.mark.parametrize("rows,vocab", KERNELS)
def test_exact_divergence_of_logits_at_a_distance(rows, vocab, apart):
  """Logits are defined up to a constant, and two models' have no common one: the divergence and its gradient do not depend on it
  (but for the rounding of the logits themselves, which the oracle reads as they are)."""
  from derl_amd import ops
  z, actions, old, adv, _, ref_z = policy_inputs(rows, vocab, F32, vocab)
  for x, y in ((z, ref_z + apart), (z + apart, ref_z), (z + apart, ref_z - apart)):
    _, _, _, lp = policy_oracle(x, actions, old, adv, 0.2, 0.0, 0.0, None, None, None)
    drift = torch.where(adv > 0, -0.07, 0.07).double()
    old = (lp - drift).float()
    got = ops.token_policy_loss(x, actions, old, adv, 0.2, kl_coef=0.5, entropy_coef=0.01, ref_logits=y)
    want = policy_oracle(x, actions, old, adv, 0.2, 0.5, 0.01, None, y, None)
    check_policy(got, want, vocab, F32)


class Table(torch.nn.Module):
  """Logits that are parameters themselves: their gradient is what the loss hands on."""

  def __init__(self, logits):
    super().__init__()
    self.logits = torch.nn.Parameter(logits)

  def forward(self, observations):
    return self.logits


@pytest.mark.parametrize("factor", [1.0, 3.0, 4096.0])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,vocab", KERNELS + [(17000, 40)])
def test_a_scaled_loss_is_rounded_once(rows, vocab, dtype, factor):
  """loss * factor: the gradient is the factor's multiple in 64 bits, rounded once, also where at scale 1 it would have been
  below f16's smallest step; the same for the preference loss; a graph of both gives the same bits."""
  import derl_amd as derl
  z, actions, old, adv, _, ref_z = policy_inputs(rows, vocab, dtype, 5 * vocab)
  mask = torch.rand(rows, generator=gen(vocab), device=DEV) < 0.7
  mask[0] = True
  model = Table(z.clone())
  policy = derl.TokenPolicyLoss(model, cliprange=0.2, kl_coef=0.1, entropy_coef=0.01)
  data = dict(observations=None, actions=actions, log_prob=old, advantages=adv, ref_logits=ref_z, mask=mask)
  offsets = torch.tensor([0, rows // 3, rows - 1], dtype=torch.int32, device=DEV)
  preference = derl.PreferenceLoss(model, beta=0.3, label_smoothing=0.1)
  pair = dict(observations=None, actions=actions, offsets=offsets, mask=mask)
  s = slack(vocab)
  _, dz, size, _ = policy_oracle(z, actions, old, adv, 0.2, 0.1, 0.01, None, ref_z, mask)
  (policy(data) * factor).backward()
  within(model.logits.grad, factor * dz, 8 * s * factor * size + half_step(factor * dz, dtype), "policy")
  want, model.logits.grad = model.logits.grad, None
  _, dz, size, _ = preference_oracle(z, actions, offsets, None, 0.3, 0.1, mask)
  size = (8 * s + 4 * 0.3 * rows * (s + 2.0 ** -23 * 40)) * size
  (preference(pair) * factor).backward()
  within(model.logits.grad, factor * dz, factor * size + half_step(factor * dz, dtype), "preference")
  want2, model.logits.grad = model.logits.grad, None
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    (a,) = torch.autograd.grad(policy(data) * factor, model.logits)
    (b,) = torch.autograd.grad(preference(pair) * factor, model.logits)
  for _ in range(3):
    graph.replay()
    policy(data)
    torch.cuda.synchronize()
    assert torch.equal(a, want) and torch.equal(b, want2)


def test_what_the_scaled_gradient_depends_on_is_kept():
  """An input that is changed in place between the loss and its gradient is found out, as autograd does for its own."""
  import derl_amd as derl
  z, actions, old, adv, _, _ = policy_inputs(6, 300, F16, 1)
  model = Table(z)
  loss = derl.TokenPolicyLoss(model)(dict(observations=None, actions=actions, log_prob=old, advantages=adv))
  adv.mul_(2.0)
  with pytest.raises(RuntimeError, match="modified by an inplace operation"):
    (loss * 8.0).backward()


def test_refusals_of_the_scaled_gradients():
  from derl_amd import ops
  z, actions, old, adv, _, _ = policy_inputs(6, 40, F16, 1)
  one = torch.ones(1, device=DEV)
  _, dz, _ = ops.token_policy_loss(z, actions, old, adv, 0.2)
  for bad in (dict(dlogits=z), dict(dlogits=dz[:5]), dict(dlogits=dz.float()), dict(factor=one.double()), dict(factor=one.cpu()),
              dict(factor=torch.ones(2, device=DEV)), dict(cliprange=-1.0), dict(actions=actions[:3])):
    with pytest.raises(ValueError):
      ops.token_policy_grad_scaled(**{**dict(dlogits=dz, factor=one, logits=z, actions=actions, old_log_prob=old, advantages=adv, cliprange=0.2), **bad})


@pytest.mark.parametrize("dtype,ref_dtype", [(BF16, F32), (F16, F32), (BF16, F16), (F16, BF16), (F32, BF16), (F16, torch.float64)])
def test_reference_logits_of_another_type_are_not_rounded(dtype, ref_dtype):
  """The divergence is that of the logits as they are given (float64 ones rounded to float32, once)."""
  import derl_amd as derl
  rows, vocab = 5, 700
  z, actions, old, adv, _, _ = policy_inputs(rows, vocab, dtype, 1)
  ref_z = (z.float() + 0.3 * torch.randn(z.shape, generator=gen(5), device=DEV)).to(ref_dtype)
  model = Table(z)
  for given in (ref_z, ref_z.cpu().numpy() if ref_dtype is not BF16 else ref_z.cpu()):
    loss_fn = derl.TokenPolicyLoss(model, cliprange=0.2, kl_coef=0.7)
    model.logits.grad = None
    loss_fn(dict(observations=None, actions=actions, log_prob=old, advantages=adv, ref_logits=given)).backward()
    terms, dz, size, _ = policy_oracle(z, actions, old, adv, 0.2, 0.7, 0.0, None, ref_z, None)
    s = slack(vocab)
    assert model.logits.grad.dtype == dtype
    within(model.logits.grad, dz, 8 * s * size + half_step(dz, dtype), "dlogits")
    assert abs(float(loss_fn.last_terms[3]) - terms[3]) <= 16 * s * (1 + abs(terms[3]))


def test_what_is_written_in_place_is_known_to_autograd():
  """dlogits_out, scale_rows and orthogonalize's out: a backward pass that needs the old values raises, a leaf that requires
  grad is refused, under no_grad it is not."""
  from derl_amd import ops
  z, actions, old, adv, _, _ = policy_inputs(4, 50, F32, 1)
  offsets = torch.tensor([0, 2, 4], dtype=torch.int32, device=DEV)
  one = torch.full((1,), 2.0, device=DEV)
  writes = (lambda x: ops.token_policy_loss(x.detach(), actions, old, adv, 0.2, dlogits_out=x),
            lambda x: ops.preference_loss(x.detach(), actions, offsets, None, 0.1, dlogits_out=x),
            lambda x: ops.scale_rows(x, one), lambda x: ops.orthogonalize(x.detach(), out=x))
  for write in writes:
    w = torch.nan_to_num(z, neginf=-5.0).requires_grad_()
    y = w.sigmoid()  # saves its result
    write(y.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
      y.sum().backward()
    with pytest.raises(ValueError, match="leaf"):
      write(w)
    before = w.detach().clone()
    with torch.no_grad():
      write(w)
    assert not torch.equal(before, w)
    with torch.inference_mode():
      write(torch.nan_to_num(z, neginf=-5.0))


def test_a_gradient_that_lies_over_an_input_is_refused():
  """Other workgroups read masks, actions and scalars while the gradient is being written."""
  from derl_amd import ops
  z, actions, old, adv, ref_lp, _ = policy_inputs(6, 40, F32, 1)
  mask = torch.ones(6, dtype=torch.bool, device=DEV)
  offsets = torch.tensor([0, 2, 6], dtype=torch.int32, device=DEV)
  policy = dict(logits=z, actions=actions, old_log_prob=old, advantages=adv, cliprange=0.2, ref_log_prob=ref_lp, mask=mask)
  preference = dict(logits=z, actions=actions, offsets=offsets, ref_log_prob=ref_lp[:2], beta=0.1, mask=mask)
  for call, given in ((ops.token_policy_loss, policy), (ops.preference_loss, preference)):
    for name, value in given.items():
      if not isinstance(value, torch.Tensor) or name == "logits":
        continue
      store = torch.zeros(6 * 40 + 64, device=DEV)
      inside = store[100:].view(value.dtype)[:value.numel()].view(value.shape)  # (16-byte aligned)
      inside.copy_(value)
      with pytest.raises(ValueError, match="overlaps"):
        call(**{**given, name: inside}, dlogits_out=store[:240].view(6, 40))
      behind = store[240:].view(value.dtype)[:value.numel()].view(value.shape)
      behind.copy_(value)
      got = call(**{**given, name: behind}, dlogits_out=store[:240].view(6, 40))
      assert all(torch.equal(a, b) for a, b in zip(got, call(**given)))
  x = torch.ones(4, 6, device=DEV)
  with pytest.raises(ValueError, match="lies in x"):
    ops.scale_rows(x, x[1, 2:3])


def test_results_without_a_gradient_say_so():
  """token_log_prob, sequence_log_prob and orthogonalize on inputs that require grad: the same values; a gradient through them
  raises, alone or beside other terms; nothing changes under no_grad or for detached inputs."""
  from derl_amd import ops
  z, actions, _, _, _, _ = policy_inputs(6, 300, F32, 1)
  z = torch.nan_to_num(z, neginf=-9.0)
  offsets = torch.tensor([0, 2, 6], dtype=torch.int32, device=DEV)
  calls = (lambda x: ops.token_log_prob(x, actions)[0], lambda x: ops.token_log_prob(x, actions)[1],
           lambda x: ops.sequence_log_prob(x, actions, offsets), lambda x: ops.orthogonalize(x))
  for call in calls:
    want = call(z)
    assert not want.requires_grad
    w = z.clone().requires_grad_()
    got = call(w * 1.0)
    assert torch.equal(got, want)
    with pytest.raises(RuntimeError, match="no gradient"):
      (got.sum() + w.sum()).backward()
    with torch.no_grad():
      assert not call(w).requires_grad
    assert not call(w.detach()).requires_grad
  with pytest.raises(ValueError, match="no gradient"):
    ops.orthogonalize(w * 1.0, out=torch.empty_like(z))


def test_sizes_that_no_int_holds_are_refused():
  """2^32 + 3 columns, sides or matrices are not 3."""
  from derl_amd import ops
  if torch.cuda.mem_get_info()[0] < 40e9:
    pytest.skip("needs 35 GB of device memory")
  size = (1 << 32) + 3
  wide = torch.empty(1, size, dtype=BF16, device=DEV)
  actions = torch.zeros(1, dtype=torch.int64, device=DEV)
  one = torch.ones(1, device=DEV)
  for call in (lambda: ops.token_log_prob(wide, actions), lambda: ops.token_policy_loss(wide, actions, one, one, 0.2),
               lambda: ops.scale_rows(wide, one), lambda: ops.sequence_log_prob(wide, actions, torch.zeros(2, dtype=torch.int32, device=DEV))):
    with pytest.raises(ValueError, match="columns"):
      call()
  for shape in ((1, size), (size, 1)):
    with pytest.raises(RuntimeError, match="sides"):
      ops.orthogonalize(wide.view(shape))
  with pytest.raises(RuntimeError, match="batch"):
    ops.orthogonalize(wide.view(size, 1, 1))
  with pytest.raises(ValueError, match="steps"):
    ops.orthogonalize(torch.ones(2, 2, device=DEV), steps=(1 << 32) + 1)


def test_gradients_of_shards_add_up():
  """global_batch and global_pairs through the classes: the shards' gradients sum to the whole batch's (each of them off by
  ``slack`` of its terms, of which there are eight, and three fp32 roundings of the library's products around them)."""
  model = torch.nn.Linear(16, 120).to(DEV)
  (policy, data), (preference, pairs) = losses_of(model, 24, 120, 16)
  pairs["offsets"] = torch.tensor([0, 5, 12, 17, 24], dtype=torch.int32, device=DEV)
  cut = lambda d, a, b: {k: v[a:b] if k != "offsets" else v for k, v in d.items()}  # noqa: E731
  shards = [(policy, data, [dict(cut(data, 0, 9), global_batch=int(data["mask"].sum())),
                            dict(cut(data, 9, 24), global_batch=int(data["mask"].sum()))]),
            (preference, pairs, [dict(cut(pairs, 0, 12), offsets=pairs["offsets"][:3], global_pairs=2),
                                 dict(cut(pairs, 12, 24), offsets=pairs["offsets"][2:] - 12, global_pairs=2)])]
  for loss_fn, whole, parts in shards:
    want = torch.autograd.grad(loss_fn(whole), model.parameters())
    got = [torch.autograd.grad(loss_fn(part), model.parameters()) for part in parts]
    for w, a, b in zip(want, *got):
      assert float((w - a - b).norm()) <= (16 * slack(120) + 16 * 2.0 ** -24) * float(a.norm() + b.norm())


def test_trainer_steps_a_module_with_the_losses():
  """Trainer and Alg, a torch optimizer and a clipped norm around both losses: the step is that of the same calls by hand."""
  from types import SimpleNamespace
  import derl_amd as derl
  for which in (0, 1):
    models = []
    for by_hand in (False, True):
      torch.manual_seed(0)
      model = torch.nn.Sequential(torch.nn.Linear(16, 32), torch.nn.Tanh(), torch.nn.Linear(32, 120)).to(DEV)
      loss_fn, data = losses_of(model, 24, 120, 16)[which]
      optimizer = torch.optim.SGD(model.parameters(), lr=0.1)
      alg = derl.Alg(SimpleNamespace(policy=SimpleNamespace(model=model), step_count=0), derl.Trainer(optimizer, max_grad_norm=0.05), loss_fn)
      for _ in range(2):
        if by_hand:
          optimizer.zero_grad()
          loss_fn(data).backward()
          torch.nn.utils.clip_grad_norm_(model.parameters(), 0.05)
          optimizer.step()
        else:
          loss = alg.step(data)
          assert loss.shape == () and torch.isfinite(loss)
      models.append(model)
    for a, b in zip(models[0].parameters(), models[1].parameters()):
      assert torch.equal(a, b)


# rows, columns and distance of rows in elements of 2 bytes, the last rows past 2^32 bytes: a wave a row, rows in registers (256 and 1024
# threads), rows read twice, pieces, and 70000 rows of 32768 side by side
FAR = [(3, 4000, 1_200_000_000), (3, 12001, 1_200_000_000), (130, 100_003, 18_000_000), (130, 140_001, 18_000_000), (3, 40003, 1_200_000_000),
       (70_000, 32_768, 32_768)]


@pytest.mark.parametrize("ref", ["none", "logits"])
@pytest.mark.parametrize("rows,vocab,pitch", FAR)
def test_rows_past_32_bits_in_every_row_kernel(rows, vocab, pitch, ref):
  """Rows far apart give what the same rows give side by side (or, 70000 of them, what the last ones give alone)."""
  from derl_amd import ops
  if torch.cuda.mem_get_info()[0] < 40e9:
    pytest.skip("needs 30 GB of device memory")
  few = min(rows, 130)
  z, actions, old, adv, _, ref_z = policy_inputs(few, vocab, BF16, 3)
  views = []
  for source in (z, ref_z):
    store = torch.empty((rows - 1) * pitch + vocab, dtype=BF16, device=DEV)
    view = store.as_strided((rows, vocab), (pitch, 1))
    if rows > few:
      view.fill_(0.5)
    view[rows - few:] = source
    views.append(view)
  view, ref_view = views[0], views[1] if ref == "logits" else None
  wide = lambda x: torch.cat([torch.zeros(rows - few, dtype=x.dtype, device=DEV), x])  # noqa: E731
  mask = wide(torch.ones(few, dtype=torch.bool, device=DEV))
  offsets = torch.tensor([rows - few, rows - 2, rows], dtype=torch.int32, device=DEV)
  near = torch.tensor([0, few - 2, few], dtype=torch.int32, device=DEV)
  want = [ops.token_log_prob(z, actions)[0], ops.preference_loss(z, actions, near, None, 0.1)[1]]
  got = [ops.token_log_prob(view, wide(actions), mask)[0][rows - few:], ops.preference_loss(view, wide(actions), offsets, None, 0.1)[1][rows - few:]]
  _, dz, lp = ops.token_policy_loss(z, actions, old, adv, 0.2, kl_coef=0.1, entropy_coef=0.01, ref_logits=ref_z if ref == "logits" else None)
  _, far, far_lp = ops.token_policy_loss(view, wide(actions), wide(old), wide(adv), 0.2, kl_coef=0.1, entropy_coef=0.01, ref_logits=ref_view,
                                         mask=mask, dlogits_out=view)
  assert far is view
  if rows == few:
    for a, b in zip([dz, lp] + want, [far, far_lp] + got):
      assert torch.equal(a, b)
  else:  # (other kernels, by the number of rows: off by their sums)
    s = slack(vocab)
    within(far_lp[rows - few:], lp, 2 * s + 2.0 ** -22 * (lp.abs() + 16), "log_prob")
    within(got[0], want[0], 2 * s + 2.0 ** -22 * (lp.abs() + 16), "log_prob")
    _, exact, size, _ = policy_oracle(z, actions, old, adv, 0.2, 0.1, 0.01, None, ref_z if ref == "logits" else None, None)
    within(far[rows - few:], exact, 8 * s * size + half_step(exact, BF16), "dlogits")
    _, exact, size, _ = preference_oracle(z, actions, near, None, 0.1, 0.0, None)
    within(got[1], exact, (8 * s + 4 * 0.1 * few * (s + 2.0 ** -23 * 40)) * size + half_step(exact, BF16), "preference")
    assert not far[:rows - few:977].any()


def test_inputs_made_under_inference_mode():
  """What a rollout stores may be inference tensors, which autograd cannot save."""
  import derl_amd as derl
  for dtype in (F32, F16):
    z, actions, old, adv, _, ref_z = policy_inputs(6, 300, dtype, 1)
    offsets = torch.tensor([0, 2, 6], dtype=torch.int32, device=DEV)
    with torch.inference_mode():
      stored = [t.clone() for t in (actions, old, adv, ref_z)]
    model = Table(z)
    grads = []
    for a, o, d, r in ((actions, old, adv, ref_z), stored):
      model.logits.grad = None
      policy = derl.TokenPolicyLoss(model, kl_coef=0.1)(dict(observations=None, actions=a, log_prob=o, advantages=d, ref_logits=r))
      preference = derl.PreferenceLoss(model)(dict(observations=None, actions=a, offsets=offsets))
      (8.0 * (policy + preference)).backward()
      grads.append(model.logits.grad)
    assert torch.equal(*grads)


def test_float32_logits_may_be_overwritten_behind_the_loss():
  """Their gradient exists by then; 16-bit ones may be read again, and autograd says so."""
  import derl_amd as derl
  for dtype in (F32, BF16):
    z, actions, old, adv, _, _ = policy_inputs(6, 300, dtype, 1)
    model = Table(z)
    data = dict(observations=None, actions=actions, log_prob=old, advantages=adv)
    (want,) = torch.autograd.grad(3.0 * derl.TokenPolicyLoss(model)(data), model.logits)
    loss = 3.0 * derl.TokenPolicyLoss(model)(data)
    with torch.no_grad():
      model.logits.mul_(0.5)
    if dtype is F32:
      (got,) = torch.autograd.grad(loss, model.logits)
      assert torch.equal(got, want)
    else:
      with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
