"""Losses of policies over a vocabulary: derl's clipped policy loss (derl/alg/ppo.py:24-64) for logits of any
width, with the KL term such policies are trained with, and the loss of paired log ratios.

The model is any ``torch.nn.Module`` on the GPU that maps ``data["observations"]`` to logits (..., V); the loss
kernels produce the gradient with respect to the logits in the forward pass, autograd carries it through the model."""
import torch

from .common import Loss
from .. import ops, summary


class _NoSecondDerivative(torch.autograd.Function):
  """What is handed on where a graph of the gradient is asked for (``create_graph``): the kernels' gradient is a constant to
  autograd, so whoever differentiates it again, with respect to anything that the logits depend on, is told."""

  @staticmethod
  def forward(ctx, dlogits, logits):
    return dlogits.view_as(dlogits)

  @staticmethod
  def backward(ctx, grad_output):
    raise RuntimeError("the gradient of a token loss cannot be differentiated: it has no second derivative here")


class _LogitsLoss(torch.autograd.Function):
  """A scalar computed from logits together with its gradient.  The gradient is handed on once, times the incoming
  gradient: as it is where that is 1; 16-bit gradients are formed again otherwise, from the logits, so that they are
  rounded once and a loss scale saves what rounding at scale 1 would lose; float32 ones are scaled in place.  A second
  derivative (a gradient's penalty, a product with the Hessian) raises."""

  @staticmethod
  def forward(ctx, logits, evaluate):
    terms, dlogits, ctx.again, inputs = evaluate(logits.detach())
    if dlogits.dtype == torch.float32:  # scaled in place: the logits' values are not needed again, whatever becomes of them
      ctx.logits = logits
    else:
      ctx.save_for_backward(logits)
    # (not saved as the logits are: what was made under inference_mode could not be)
    ctx.inputs = [(t, None if t.is_inference() else t._version) for t in inputs]  # pylint: disable=protected-access
    ctx.dlogits = dlogits
    return terms[0].clone()

  @staticmethod
  def backward(ctx, grad_output):
    dlogits, ctx.dlogits = ctx.dlogits, None
    if dlogits is None:
      raise RuntimeError("the gradient of this loss was already handed on: evaluate the loss again to differentiate it again")
    logits = ctx.logits if dlogits.dtype == torch.float32 else ctx.saved_tensors[0]
    inputs, ctx.inputs, ctx.logits = ctx.inputs, None, None
    with torch.no_grad():
      factor = grad_output.to(torch.float32).contiguous()
      if dlogits.dtype == torch.float32:
        ops.scale_rows(dlogits, factor)
      else:
        if any(version is not None and t._version != version for t, version in inputs):  # pylint: disable=protected-access
          raise RuntimeError("an input of this loss was modified by an inplace operation: its gradient is formed from it")
        ctx.again(dlogits, factor, logits.detach(), *(t for t, _ in inputs))
    if torch.is_grad_enabled():
      dlogits = _NoSecondDerivative.apply(dlogits, logits)
    return dlogits, None


class TokenLoss(Loss):
  """Shared machinery: one model forward, one fused loss on the flattened logits."""
  tags = ()

  def __init__(self, model, name=None):
    super().__init__(model=model, name=name)
    self.last_terms = None  # device float32[8]

  def _logits(self, data):
    logits = self.model(data["observations"])
    if not isinstance(logits, torch.Tensor) or logits.ndim < 2:
      raise ValueError("the model of a token loss must return logits of shape (..., vocab)")
    return logits.reshape(-1, logits.shape[-1])

  def _flat(self, data, key, dtype=None, required=True):
    if data.get(key) is None:
      if required:
        raise ValueError(f"data does not contain '{key}'")
      return None
    return self.to_device(data[key], dtype).reshape(-1)

  def _mask(self, data):
    mask = data.get("mask")
    return None if mask is None else self.to_device(mask, torch.bool).reshape(-1)

  def _evaluate(self, logits, data):
    """(terms, dlogits, function (dlogits, factor, logits, *inputs) that forms the gradient again times a factor, inputs)."""
    raise NotImplementedError

  def _summaries(self, terms):
    for i, tag in enumerate(self.tags):
      summary.add_scalar(f"{self.name}/{tag}", terms[i], global_step=self.call_count)

  def __call__(self, data):
    logits = self._logits(data)

    def evaluate(raw):
      found = self._evaluate(raw, data)
      self.last_terms = found[0]
      return found

    loss = _LogitsLoss.apply(logits, evaluate)
    if summary.should_record():
      self._summaries(self.last_terms)
    self.call_count += 1
    return loss


class TokenPolicyLoss(TokenLoss):
  """Clipped policy loss with a KL term and an entropy bonus (``ops.token_policy_loss``).  ``data``: observations,
  actions, log_prob (of the policy that acted), advantages; optional ref_log_prob or ref_logits (of the reference
  policy), mask, global_batch (unmasked rows over all shards: what the gradient is divided by, so that shards' add
  up).  Reference logits of a wider type than the policy's are not rounded to it: the loss is then taken of
  the policy's logits in the type that holds both (the gradient is rounded to theirs on its way back)."""
  tags = ("loss", "policy_loss", "entropy", "kl", "clip_fraction", "ratio", "log_prob", "tokens")

  def __init__(self, model, cliprange=0.2, kl_coef=0., entropy_coef=0., name=None):
    super().__init__(model, name=name)
    self.cliprange, self.kl_coef, self.entropy_coef = cliprange, kl_coef, entropy_coef

  def _ref_logits(self, data):
    ref_logits = data.get("ref_logits")
    if ref_logits is None:
      return None
    ref_logits = torch.as_tensor(ref_logits)
    return ref_logits if ref_logits.dtype in (torch.bfloat16, torch.float16) else ref_logits.float()

  def _logits(self, data):
    logits, ref_logits = super()._logits(data), self._ref_logits(data)
    return logits if ref_logits is None else logits.to(torch.promote_types(logits.dtype, ref_logits.dtype))

  def _evaluate(self, logits, data):
    f32 = torch.float32
    ref_logits = self._ref_logits(data)
    if ref_logits is not None:
      ref_logits = self.to_device(ref_logits, logits.dtype).reshape(logits.shape)
    given = dict(actions=self._flat(data, "actions", torch.int64), old_log_prob=self._flat(data, "log_prob", f32),
                 advantages=self._flat(data, "advantages", f32), ref_log_prob=self._flat(data, "ref_log_prob", f32, required=False),
                 ref_logits=ref_logits, mask=self._mask(data))
    fixed = dict(cliprange=self.cliprange, kl_coef=self.kl_coef, entropy_coef=self.entropy_coef,
                 global_batch=int(data.get("global_batch") or 0))
    terms, dlogits, _ = ops.token_policy_loss(logits, **given, **fixed)
    names = [name for name, value in given.items() if value is not None]

    def again(dlogits, factor, logits, *inputs):
      ops.token_policy_grad_scaled(dlogits, factor, logits, **dict(zip(names, inputs)), **fixed)

    return terms, dlogits, again, [given[name] for name in names]


class PreferenceLoss(TokenLoss):
  """Loss of paired log ratios (``ops.preference_loss``).  ``data``: observations of the packed sequences (chosen,
  rejected, chosen, ...), actions, offsets (their borders); optional ref_log_prob (per sequence), mask, global_pairs
  (pairs over all shards: what the gradient is divided by, so that shards' add up)."""
  tags = ("loss", "accuracy", "margin", "chosen_reward", "rejected_reward", "chosen_log_prob", "rejected_log_prob", "pairs")

  def __init__(self, model, beta=0.1, label_smoothing=0., name=None):
    super().__init__(model, name=name)
    self.beta, self.label_smoothing = beta, label_smoothing

  def _evaluate(self, logits, data):
    actions = self._flat(data, "actions", torch.int64)
    terms, dlogits, _, workspace = ops._preference_loss(  # pylint: disable=protected-access
        logits, actions, self._flat(data, "offsets", torch.int32), self._flat(data, "ref_log_prob", torch.float32, required=False),
        self.beta, self.label_smoothing, self._mask(data), int(data.get("global_pairs") or 0))
    return terms, dlogits, ops._preference_grad_scaled, [actions, workspace]  # pylint: disable=protected-access
