"""Thin torch-tensor front ends of the C-ABI ops (shape / dtype checks, then one call).

torch supplies device memory and the stream only; all arithmetic happens in
libderl_amd.so.  Every function raises if its inputs are not on a HIP device.
"""
import math

import torch

from . import _lib


def _dev(t, name, dtype=None):
  if not isinstance(t, torch.Tensor) or not t.is_cuda:
    raise ValueError(f"{name} must be a tensor on the GPU (derl_amd has no CPU path)")
  if dtype is not None and t.dtype != dtype:
    raise ValueError(f"{name} must have dtype {dtype}, got {t.dtype}")
  if not t.is_contiguous():
    raise ValueError(f"{name} must be contiguous")
  return t


def gae(rewards, resets, values, last_values, gamma, lambda_, out_advantages=None,
        out_value_targets=None):
  """Device GAE over time-major (T, N) arrays (trajectory_transforms.py:45-65).

  rewards (T,N) f32, resets (T,N) bool/uint8, values (T,N) f32, last_values (N,) f32.
  Returns (advantages (T,N), value_targets (T,N))."""
  _dev(rewards, "rewards", torch.float32)
  _dev(values, "values", torch.float32)
  _dev(last_values, "last_values", torch.float32)
  _dev(resets, "resets")
  if resets.dtype not in (torch.bool, torch.uint8):
    raise ValueError(f"resets must be bool or uint8, got {resets.dtype}")
  if rewards.ndim != 2:
    raise ValueError(f"rewards must be (T, N), got {tuple(rewards.shape)}")
  T, N = rewards.shape
  if tuple(values.shape) != (T, N) or tuple(resets.shape) != (T, N):
    raise ValueError("rewards, resets and values must share the shape (T, N): "
                     f"{tuple(rewards.shape)}, {tuple(resets.shape)}, {tuple(values.shape)}")
  if last_values.numel() != N:
    raise ValueError(f"last_values must have {N} elements, got {tuple(last_values.shape)}")
  adv = out_advantages if out_advantages is not None else torch.empty_like(values)
  vt = out_value_targets if out_value_targets is not None else torch.empty_like(values)
  _dev(adv, "out_advantages", torch.float32)
  _dev(vt, "out_value_targets", torch.float32)
  _lib.call("dx_gae_f32", _lib.ptr(rewards), _lib.ptr(resets), _lib.ptr(values),
            _lib.ptr(last_values), T, N, float(gamma), float(lambda_), _lib.ptr(adv),
            _lib.ptr(vt), _lib.stream_ptr(rewards.device))
  return adv, vt


def adv_normalize(advantages, epsilon=1e-8, out=None, stats=None, stats_ready=False):
  """(a - mean) / (std + eps) on the device (trajectory_transforms.py:89-92).  ``stats`` is a
  float64[3] device tensor {sum, sumsq, count}; pass stats_ready=True to reuse reduced stats."""
  _dev(advantages, "advantages", torch.float32)
  out = torch.empty_like(advantages) if out is None else _dev(out, "out", torch.float32)
  if stats is None:
    stats = torch.empty(3, dtype=torch.float64, device=advantages.device)
  _lib.call("dx_adv_normalize_f32", _lib.ptr(advantages), _lib.ptr(out), advantages.numel(),
            float(epsilon), _lib.ptr(stats), int(stats_ready), _lib.stream_ptr(advantages.device))
  return out


def adv_stats(advantages, stats=None):
  _dev(advantages, "advantages", torch.float32)
  if stats is None:
    stats = torch.empty(3, dtype=torch.float64, device=advantages.device)
  _lib.call("dx_adv_stats_f32", _lib.ptr(advantages), advantages.numel(), _lib.ptr(stats),
            _lib.stream_ptr(advantages.device))
  return stats


def adv_stats_segments(advantages, index, seglen, stats=None):
  """{sum, sumsq, count} of every ``seglen``-long slice of ``advantages[index]`` (the minibatches
  of one epoch; ``index`` int32 or None) -> float64 (ceil(n / seglen), 3)."""
  _dev(advantages, "advantages", torch.float32)
  n = advantages.numel() if index is None else index.numel()
  nseg = -(-n // seglen)
  if index is not None:
    _dev(index, "index", torch.int32)
  if stats is None:
    stats = torch.empty((nseg, 3), dtype=torch.float64, device=advantages.device)
  _lib.call("dx_adv_stats_segments_f32", _lib.ptr(advantages), _lib.ptr(index) if index is not None else None,
            n, seglen, _lib.ptr(stats), _lib.stream_ptr(advantages.device))
  return stats


NORM_PARTIALS = 256


def grad_sumsq(grads, partials=None):
  _dev(grads, "grads", torch.float32)
  if partials is None:
    partials = torch.empty(NORM_PARTIALS, dtype=torch.float64, device=grads.device)
  _lib.call("dx_grad_sumsq_f32", _lib.ptr(grads), grads.numel(), _lib.ptr(partials),
            partials.numel(), _lib.stream_ptr(grads.device))
  return partials


def clip_adam_step(params, grads, exp_avg, exp_avg_sq, partials, max_norm, lr, step,
                   beta1=0.9, beta2=0.999, eps=1e-8, norm_out=None):
  for name, t in (("params", params), ("grads", grads), ("exp_avg", exp_avg),
                  ("exp_avg_sq", exp_avg_sq)):
    _dev(t, name, torch.float32)
  _lib.call("dx_clip_adam_step_f32", _lib.ptr(params), _lib.ptr(grads), _lib.ptr(exp_avg),
            _lib.ptr(exp_avg_sq), params.numel(), _lib.ptr(partials),
            0 if partials is None else partials.numel(),
            float(max_norm) if max_norm is not None else 0.0, float(lr), float(beta1),
            float(beta2), float(eps), int(step), _lib.ptr(norm_out),
            _lib.stream_ptr(params.device))


def clip_rmsprop_step(params, grads, square_avg, partials, max_norm, lr, alpha=0.99, eps=1e-8,
                      norm_out=None):
  for name, t in (("params", params), ("grads", grads), ("square_avg", square_avg)):
    _dev(t, name, torch.float32)
  _lib.call("dx_clip_rmsprop_step_f32", _lib.ptr(params), _lib.ptr(grads), _lib.ptr(square_avg),
            params.numel(), _lib.ptr(partials), 0 if partials is None else partials.numel(),
            float(max_norm) if max_norm is not None else 0.0, float(lr), float(alpha), float(eps),
            _lib.ptr(norm_out), _lib.stream_ptr(params.device))


def gather_rows(src, idx, out=None):
  """out[i] = src[idx[i]] along dim 0 (idx int32 on the device)."""
  _dev(src, "src")
  _dev(idx, "idx", torch.int32)
  n = idx.numel()
  out = torch.empty((n,) + tuple(src.shape[1:]), dtype=src.dtype, device=src.device) if out is None else out
  row_bytes = src.element_size()
  for d in src.shape[1:]:
    row_bytes *= d
  _lib.call("dx_gather_rows", _lib.ptr(src), _lib.ptr(idx), _lib.ptr(out), n, row_bytes,
            _lib.stream_ptr(src.device))
  return out


def gather_rows_multi(sources, idx):
  """[src[idx] for src in sources] along dim 0 with one launch per 16 arrays."""
  _dev(idx, "idx", torch.int32)
  n = idx.numel()
  outs = []
  for start in range(0, len(sources), 16):
    group = sources[start:start + 16]
    k = len(group)
    src_p, dst_p, rb = (_lib.c_void_p * k)(), (_lib.c_void_p * k)(), (_lib.c_longlong * k)()
    for i, src in enumerate(group):
      _dev(src, "src")
      out = torch.empty((n,) + tuple(src.shape[1:]), dtype=src.dtype, device=src.device)
      outs.append(out)
      src_p[i], dst_p[i] = src.data_ptr(), out.data_ptr()
      rb[i] = src.element_size() * math.prod(src.shape[1:])
    _lib.call("dx_gather_rows_multi", src_p, dst_p, rb, k, _lib.ptr(idx), n,
              _lib.stream_ptr(idx.device))
  return outs


def categorical_act(head_out, num_actions, uniforms=None, seed=0, counter=0, out=None):
  """Sample / log_prob / value from the padded head output (B, 32) (policies.py:61-80).
  ``out`` = (actions int64 (B,), log_prob f32 (B,), values f32 (B,)) to write in place."""
  _dev(head_out, "head_out", torch.float32)
  B = head_out.shape[0]
  dev = head_out.device
  if out is not None:
    actions, log_prob, values = out
    _dev(actions, "actions", torch.int64)
    _dev(log_prob, "log_prob", torch.float32)
    _dev(values, "values", torch.float32)
    if actions.numel() != B or log_prob.numel() != B or values.numel() != B:
      raise ValueError("categorical_act: output buffers must hold B elements")
  else:
    actions = torch.empty(B, dtype=torch.int64, device=dev)
    log_prob = torch.empty(B, dtype=torch.float32, device=dev)
    values = torch.empty(B, dtype=torch.float32, device=dev)
  if uniforms is not None:
    _dev(uniforms, "uniforms", torch.float32)
  _lib.call("dx_categorical_act_f32", _lib.ptr(head_out), B, int(num_actions), _lib.ptr(uniforms),
            int(seed), int(counter), _lib.ptr(actions), _lib.ptr(log_prob), _lib.ptr(values),
            _lib.stream_ptr(dev))
  return actions, log_prob, values


def categorical_loss(head_out, actions, old_log_prob, advantages, old_values, value_targets,
                     num_actions, mode, cliprange, value_loss_coef, entropy_coef, dhead_out,
                     global_batch=0, partials=None, loss_out=None):
  """Fused PPO (mode 0) / A2C (mode 1) loss + gradient w.r.t. the head output."""
  _dev(head_out, "head_out", torch.float32)
  B = head_out.shape[0]
  dev = head_out.device
  need = 8 * ((B + 7) // 8)
  if partials is None or partials.numel() < need:
    partials = torch.empty(need, dtype=torch.float64, device=dev)
  if loss_out is None:
    loss_out = torch.empty(8, dtype=torch.float32, device=dev)
  _lib.call("dx_categorical_loss_f32", _lib.ptr(head_out), _lib.ptr(actions),
            _lib.ptr(old_log_prob), _lib.ptr(advantages), _lib.ptr(old_values),
            _lib.ptr(value_targets), B, int(num_actions), int(mode),
            -1.0 if cliprange is None else float(cliprange), float(value_loss_coef),
            float(entropy_coef), int(global_batch), _lib.ptr(dhead_out), _lib.ptr(partials),
            partials.numel(), _lib.ptr(loss_out), _lib.stream_ptr(dev))
  return loss_out


def normal_act(head_out, logstd, normals=None, seed=0, counter=0, out=None):
  """Diagonal-Gaussian sample / log_prob / value from the padded head (policies.py:66,76-77)."""
  _dev(head_out, "head_out", torch.float32)
  _dev(logstd, "logstd", torch.float32)
  B, P = head_out.shape[0], logstd.numel()
  dev = head_out.device
  if out is not None:
    actions, log_prob, values = out
  else:
    actions = torch.empty(B, P, dtype=torch.float32, device=dev)
    log_prob = torch.empty(B, dtype=torch.float32, device=dev)
    values = torch.empty(B, dtype=torch.float32, device=dev)
  _lib.call("dx_normal_act_f32", _lib.ptr(head_out), _lib.ptr(logstd), B, P, _lib.ptr(normals),
            int(seed), int(counter), _lib.ptr(actions), _lib.ptr(log_prob), _lib.ptr(values),
            _lib.stream_ptr(dev))
  return actions, log_prob, values


def normal_loss(head_out, logstd, actions, old_log_prob, advantages, old_values, value_targets,
                mode, cliprange, value_loss_coef, entropy_coef, dhead_out, dlogstd_out,
                global_batch=0, partials=None, loss_out=None):
  """Fused PPO / A2C loss + gradients for the diagonal-Gaussian head."""
  _dev(head_out, "head_out", torch.float32)
  _dev(actions, "actions", torch.float32)
  B, P = head_out.shape[0], logstd.numel()
  dev = head_out.device
  need = 40 * ((B + 255) // 256)
  if partials is None or partials.numel() < need:
    partials = torch.empty(need, dtype=torch.float64, device=dev)
  if loss_out is None:
    loss_out = torch.empty(8, dtype=torch.float32, device=dev)
  _lib.call("dx_normal_loss_f32", _lib.ptr(head_out), _lib.ptr(logstd), _lib.ptr(actions),
            _lib.ptr(old_log_prob), _lib.ptr(advantages), _lib.ptr(old_values),
            _lib.ptr(value_targets), B, P, int(mode),
            -1.0 if cliprange is None else float(cliprange), float(value_loss_coef),
            float(entropy_coef), int(global_batch), _lib.ptr(dhead_out), _lib.ptr(dlogstd_out),
            _lib.ptr(partials), partials.numel(), _lib.ptr(loss_out), _lib.stream_ptr(dev))
  return loss_out


# ---- policies over a vocabulary -----------------------------------------------------------------

_INT_MAX = (1 << 31) - 1  # ctypes would wrap what is larger around
_ELEMENT_TYPES = {torch.float32: _lib.DX_F32, torch.bfloat16: _lib.DX_BF16, torch.float16: _lib.DX_F16}


class _NoGradient(torch.autograd.Function):
  """Results of a call that has no gradient, on inputs that require one: they belong to the graph, and whoever
  differentiates them is told (detached, their terms would be missing from a gradient without a word)."""

  @staticmethod
  def forward(ctx, source, name, *results):
    ctx.name = name
    return tuple(t.view_as(t) for t in results)

  @staticmethod
  def backward(ctx, *grads):
    raise RuntimeError(f"{ctx.name} has no gradient: call it under torch.no_grad() or on detached inputs; "
                       "TokenPolicyLoss and PreferenceLoss are the losses to differentiate")


def _constants(source, name, *results):
  """``results``, tied to ``source`` where autograd would expect a gradient to it."""
  if source.requires_grad and torch.is_grad_enabled():
    results = _NoGradient.apply(source, name, *results)
  return results


def _call_on(device, name, *args):
  """One native call with ``device`` current (kernels launch on the current device)."""
  if device.index == torch.cuda.current_device():
    _lib.check(getattr(_lib.load(), name)(*args), name)
  else:
    with torch.cuda.device(device):
      _lib.call(name, *args)


def _rows_of(t, name, like=None):
  """(rows, columns, pitch) of a 2-D tensor whose rows are contiguous; any distance between rows."""
  if not isinstance(t, torch.Tensor) or not t.is_cuda:
    raise ValueError(f"{name} must be a tensor on the GPU (derl_amd has no CPU path)")
  if t.dtype not in _ELEMENT_TYPES:
    raise ValueError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
  if t.ndim != 2 or t.shape[1] < 1:
    raise ValueError(f"{name} must be (rows, vocab) with vocab >= 1, got {tuple(t.shape)}")
  rows, columns = t.shape
  if columns > 1 << 30:
    raise ValueError(f"{name} must have 2^30 columns at most, got {columns}")
  pitch = t.stride(0) if rows > 1 else columns
  if (columns > 1 and t.stride(1) != 1) or pitch < columns:
    raise ValueError(f"the rows of {name} must be contiguous and must not overlap: strides {t.stride()}")
  if like is not None and (t.dtype != like.dtype or t.shape != like.shape or t.device != like.device):
    raise ValueError(f"{name} must match logits ({like.dtype}, {tuple(like.shape)}, {like.device}): "
                     f"{t.dtype}, {tuple(t.shape)}, {t.device}")
  return rows, columns, pitch


def _vector(t, name, n, device, dtype):
  """Address of a contiguous vector of ``n`` on the logits' device (None stays None)."""
  if t is None:
    return None
  if (isinstance(t, torch.Tensor) and t.dtype in dtype and t.shape == (n,) and t.get_device() == device.index
      and t.is_contiguous()):
    return t.data_ptr()
  _dev(t, name)
  if t.dtype not in dtype:
    raise ValueError(f"{name} must have dtype {' or '.join(map(str, dtype))}, got {t.dtype}")
  raise ValueError(f"{name} must be ({n},) on {device}, got {tuple(t.shape)} on {t.device}")


_INDEX, _FLAG, _FLOAT = (torch.int64,), (torch.bool, torch.uint8), (torch.float32,)


def _span(t):
  """First and last byte address of a tensor with non-negative strides."""
  if t.numel() == 0:
    return 0, 0
  last = sum((size - 1) * stride for size, stride in zip(t.shape, t.stride()))
  return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _writable(t, name):
  """A tensor of the caller's that a kernel overwrites: as torch's own operations in place, autograd learns of it (a backward
  pass that has kept the old values raises), and a leaf that requires grad is refused."""
  if t.requires_grad and t.is_leaf and torch.is_grad_enabled():
    raise ValueError(f"{name} is a leaf that requires grad: it cannot be written in place")
  if not t.is_inference():
    torch.autograd.graph.increment_version(t)
  return t


def _gradient_buffer(dlogits_out, logits, *others, in_place=True):
  """The tensor the gradient goes to: new, the caller's, or (``in_place``) ``logits`` itself."""
  if dlogits_out is None:
    return torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
  _rows_of(dlogits_out, "dlogits_out", like=logits)
  same = in_place and dlogits_out.data_ptr() == logits.data_ptr() and (logits.shape[0] <= 1 or dlogits_out.stride(0) == logits.stride(0))
  begin, end = _span(dlogits_out)
  for other in others + (() if same else (logits,)):
    if other is not None:
      b, e = _span(other)
      if b < end and begin < e:
        raise ValueError("dlogits_out overlaps an input (it may only be logits itself)")
  return _writable(dlogits_out, "dlogits_out")


def token_log_prob(logits, actions, mask=None):
  """Log-probability of each row's action and the entropy of its distribution.

  logits (N, V) float32 / bfloat16 / float16 with contiguous rows (any row stride >= V), actions (N,)
  int64, mask (N,) bool or uint8: rows that are False are not read and give 0.  Returns (log_prob,
  entropy), float32 (N,).  A logit of -inf is an action that cannot be chosen; a row without any
  distribution (all -inf, NaN, +inf) or an action outside [0, V) gives NaN.  N = 1 .. is the form for
  single tokens of sequences being generated.  They have no gradient: differentiating them raises."""
  return _constants(logits, "token_log_prob", *_token_log_prob(logits, actions, mask))


def _token_log_prob(logits, actions, mask, entropies=True):
  rows, vocab, pitch = _rows_of(logits, "logits")
  dev = logits.device
  log_prob = torch.empty(rows, dtype=torch.float32, device=dev)
  entropy = torch.empty(rows, dtype=torch.float32, device=dev) if entropies else None
  workspace = torch.empty(_lib.DX_TOKEN_WORKSPACE, dtype=torch.float64, device=dev)
  act = _vector(actions, "actions", rows, dev, _INDEX)
  keep = _vector(mask, "mask", rows, dev, _FLAG)
  _call_on(dev, "dx_token_log_prob", logits.data_ptr(), _ELEMENT_TYPES[logits.dtype], rows, vocab, pitch, act, keep,
           log_prob.data_ptr(), entropy.data_ptr() if entropies else None, workspace.data_ptr(), workspace.numel(), _lib.stream_ptr(dev))
  return log_prob, entropy


def _check_offsets(offsets, device):
  _dev(offsets, "offsets", torch.int32)
  if offsets.ndim != 1 or offsets.numel() < 1 or offsets.device != device:
    raise ValueError(f"offsets must be a vector of sequence borders on {device}, got {tuple(offsets.shape)} on {offsets.device}")
  if offsets.numel() > _INT_MAX:
    raise ValueError(f"offsets must have fewer than 2^31 entries, got {offsets.numel()}")
  return offsets.numel() - 1


def sequence_log_prob(logits, actions, offsets, mask=None):
  """Summed log-probabilities of packed sequences: sequence s holds the rows offsets[s] .. offsets[s + 1]
  of ``logits`` (offsets int32 (S + 1,), non-decreasing; empty sequences give 0).  float32 (S,): what
  ``preference_loss`` takes as ``ref_log_prob`` when the logits are the reference's.  Differentiating them raises."""
  rows, _, _ = _rows_of(logits, "logits")
  dev = logits.device
  sequences = _check_offsets(offsets, dev)
  log_prob, _ = _token_log_prob(logits, actions, mask, entropies=False)
  out = torch.empty(sequences, dtype=torch.float32, device=dev)
  _call_on(dev, "dx_sequence_log_prob", log_prob.data_ptr(), offsets.data_ptr(), rows, sequences, out.data_ptr(),
           _lib.stream_ptr(dev))
  return _constants(logits, "sequence_log_prob", out)[0]


def token_policy_loss(logits, actions, old_log_prob, advantages, cliprange, kl_coef=0., entropy_coef=0.,
                      ref_log_prob=None, ref_logits=None, mask=None, global_batch=0, dlogits_out=None):
  """Clipped policy loss with a KL term and an entropy bonus over wide logits, and its gradient.

  Per unmasked row: ratio = exp(log p(action) - old_log_prob); ``-min(ratio A, clip(ratio, 1 - cliprange,
  1 + cliprange) A) - entropy_coef H + kl_coef KL`` (cliprange None: not clipped).  The divergence from
  the reference policy is estimated from the action alone, ``e^d - 1 - d`` with ``d = ref_log_prob - log p``,
  or summed over the vocabulary where ``ref_logits`` are given (at most one of the two); with kl_coef 0 it is
  reported and takes no part, also where it is infinite.  The loss is the mean over the unmasked rows; ``global_batch`` > 0 divides the gradient by that instead (shards add up).

  logits (N, V) float32 / bfloat16 / float16 (rows contiguous, any row stride), actions (N,) int64,
  old_log_prob / advantages / ref_log_prob (N,) float32, ref_logits like logits, mask (N,) bool / uint8.
  Returns (loss float32 (8,), dlogits (N, V), log_prob float32 (N,)); loss = {loss, policy loss, entropy, KL,
  share of ratios outside the range, mean ratio, mean log-probability, unmasked rows}.  ``dlogits_out`` may
  be ``logits``.  Masked rows have gradient and log_prob 0; without an unmasked row the loss is 0."""
  given = _policy_arguments(logits, actions, old_log_prob, advantages, cliprange, kl_coef, entropy_coef, ref_log_prob, ref_logits, mask,
                            global_batch)
  dev, rows, vocab = logits.device, given[2], given[3]
  dlogits = _gradient_buffer(dlogits_out, logits, actions, old_log_prob, advantages, ref_log_prob, ref_logits, mask)
  log_prob = torch.empty(rows, dtype=torch.float32, device=dev)
  loss_out = torch.empty(8, dtype=torch.float32, device=dev)
  workspace = torch.empty(_lib.DX_TOKEN_WORKSPACE, dtype=torch.float64, device=dev)
  _call_on(dev, "dx_token_policy_loss", *given, dlogits.data_ptr(), dlogits.stride(0) if rows > 1 else vocab, log_prob.data_ptr(),
           workspace.data_ptr(), workspace.numel(), loss_out.data_ptr(), _lib.stream_ptr(dev))
  return loss_out, dlogits, log_prob


def _policy_arguments(logits, actions, old_log_prob, advantages, cliprange, kl_coef, entropy_coef, ref_log_prob, ref_logits, mask, global_batch):
  """The checked inputs of the native policy loss, in its order."""
  rows, vocab, pitch = _rows_of(logits, "logits")
  dev = logits.device
  if ref_log_prob is not None and ref_logits is not None:
    raise ValueError("give ref_log_prob or ref_logits, not both")
  if cliprange is not None and not cliprange >= 0:
    raise ValueError(f"cliprange must be None or >= 0, got {cliprange}")
  if global_batch < 0:
    raise ValueError(f"global_batch must be >= 0, got {global_batch}")
  ref_pitch = vocab
  if ref_logits is not None:
    _, _, ref_pitch = _rows_of(ref_logits, "ref_logits", like=logits)
  return (logits.data_ptr(), _ELEMENT_TYPES[logits.dtype], rows, vocab, pitch, _vector(actions, "actions", rows, dev, _INDEX),
          _vector(old_log_prob, "old_log_prob", rows, dev, _FLOAT), _vector(advantages, "advantages", rows, dev, _FLOAT),
          _vector(ref_log_prob, "ref_log_prob", rows, dev, _FLOAT), None if ref_logits is None else ref_logits.data_ptr(), ref_pitch,
          _vector(mask, "mask", rows, dev, _FLAG), -1.0 if cliprange is None else float(cliprange), float(kl_coef), float(entropy_coef),
          int(global_batch))


def _factor(factor, device):
  _dev(factor, "factor", torch.float32)
  if factor.numel() != 1 or factor.device != device:
    raise ValueError(f"factor must be one float32 on {device}, got {tuple(factor.shape)} on {factor.device}")
  return factor.data_ptr()


def token_policy_grad_scaled(dlogits, factor, logits, actions, old_log_prob, advantages, cliprange, kl_coef=0., entropy_coef=0.,
                             ref_log_prob=None, ref_logits=None, mask=None, global_batch=0):
  """``dlogits``, the gradient that ``token_policy_loss`` gave for these arguments, becomes ``factor`` (float32 device scalar)
  times the gradient, multiplied before it is rounded: formed again from the logits, left alone where the factor is 1."""
  given = _policy_arguments(logits, actions, old_log_prob, advantages, cliprange, kl_coef, entropy_coef, ref_log_prob, ref_logits, mask,
                            global_batch)
  dev, rows, vocab = logits.device, given[2], given[3]
  _gradient_buffer(dlogits, logits, actions, old_log_prob, advantages, ref_log_prob, ref_logits, mask, in_place=False)
  workspace = torch.empty(_lib.DX_TOKEN_WORKSPACE, dtype=torch.float64, device=dev)
  _call_on(dev, "dx_token_policy_grad_scaled", *given, dlogits.data_ptr(), dlogits.stride(0) if rows > 1 else vocab, workspace.data_ptr(),
           workspace.numel(), _factor(factor, dev), _lib.stream_ptr(dev))
  return dlogits


def preference_loss(logits, actions, offsets, ref_log_prob, beta, label_smoothing=0., mask=None, global_pairs=0,
                    dlogits_out=None):
  """Loss of paired log ratios over packed sequences, and its gradient.

  Sequences 2 p (chosen) and 2 p + 1 (rejected) are the rows offsets[s] .. offsets[s + 1] of logits (N, V);
  offsets int32 (2 P + 1,), non-decreasing.  With a sequence's log-probability summed over its unmasked
  rows, ``h = beta ((chosen - ref_chosen) - (rejected - ref_rejected))`` and the loss is the mean over the
  pairs of ``-(1 - s) log sigmoid(h) - s log sigmoid(-h)``, s = label_smoothing.  ref_log_prob float32 (2 P,)
  (``sequence_log_prob`` of the reference policy) or None for 0.  ``global_pairs`` > 0 divides the gradient
  by that instead of P.

  Returns (loss float32 (8,), dlogits (N, V), sequence log-probabilities float32 (2 P,)); loss = {loss, share of
  pairs with h > 0, h, beta (chosen - ref), beta (rejected - ref), chosen, rejected, P}.  Rows that are masked
  or belong to no sequence have gradient 0.  ``dlogits_out`` may be ``logits``."""
  return _preference_loss(logits, actions, offsets, ref_log_prob, beta, label_smoothing, mask, global_pairs, dlogits_out)[:3]


def _preference_loss(logits, actions, offsets, ref_log_prob, beta, label_smoothing, mask, global_pairs, dlogits_out=None):
  """``preference_loss`` and its workspace, with the rows' statistics that its gradient is made of."""
  rows, vocab, pitch = _rows_of(logits, "logits")
  dev = logits.device
  sequences = _check_offsets(offsets, dev)
  if sequences < 2 or sequences % 2:
    raise ValueError(f"offsets must have 2 pairs + 1 entries, got {offsets.numel()}")
  if not 0 <= label_smoothing <= 1:
    raise ValueError(f"label_smoothing must lie in [0, 1], got {label_smoothing}")
  if global_pairs < 0:
    raise ValueError(f"global_pairs must be >= 0, got {global_pairs}")
  act = _vector(actions, "actions", rows, dev, _INDEX)
  ref = _vector(ref_log_prob, "ref_log_prob", sequences, dev, _FLOAT)
  keep = _vector(mask, "mask", rows, dev, _FLAG)
  dlogits = _gradient_buffer(dlogits_out, logits, actions, offsets, ref_log_prob, mask)
  sequence = torch.empty(sequences, dtype=torch.float32, device=dev)
  loss_out = torch.empty(8, dtype=torch.float32, device=dev)
  # the library's scratch and behind it four floats a row
  workspace = torch.empty(_lib.DX_TOKEN_WORKSPACE + 2 * rows, dtype=torch.float64, device=dev)
  _call_on(dev, "dx_preference_loss", logits.data_ptr(), _ELEMENT_TYPES[logits.dtype], rows, vocab, pitch, act,
           offsets.data_ptr(), sequences // 2, ref, keep, float(beta), float(label_smoothing), int(global_pairs),
           dlogits.data_ptr(), dlogits.stride(0) if rows > 1 else vocab, sequence.data_ptr(),
           workspace.data_ptr() + 8 * _lib.DX_TOKEN_WORKSPACE, workspace.data_ptr(), _lib.DX_TOKEN_WORKSPACE, loss_out.data_ptr(),
           _lib.stream_ptr(dev))
  return loss_out, dlogits, sequence, workspace


def _preference_grad_scaled(dlogits, factor, logits, actions, workspace):
  """As ``token_policy_grad_scaled``, from the workspace that ``_preference_loss`` gave."""
  rows, vocab, pitch = _rows_of(logits, "logits")
  dev = logits.device
  _gradient_buffer(dlogits, logits, actions, workspace, in_place=False)
  _vector(workspace, "workspace", _lib.DX_TOKEN_WORKSPACE + 2 * rows, dev, (torch.float64,))
  _call_on(dev, "dx_preference_grad_scaled", logits.data_ptr(), _ELEMENT_TYPES[logits.dtype], rows, vocab, pitch,
           _vector(actions, "actions", rows, dev, _INDEX), workspace.data_ptr() + 8 * _lib.DX_TOKEN_WORKSPACE, dlogits.data_ptr(),
           dlogits.stride(0) if rows > 1 else vocab, _factor(factor, dev), _lib.stream_ptr(dev))
  return dlogits


def scale_rows(x, factor):
  """x *= factor in place, ``factor`` a float32 device scalar; nothing but the factor is read when it is 1."""
  rows, columns, pitch = _rows_of(x, "x")
  by = _factor(factor, x.device)
  begin, end = _span(x)
  if begin <= by < end:
    raise ValueError("factor lies in x")
  _writable(x, "x")
  _call_on(x.device, "dx_scale_rows", x.data_ptr(), _ELEMENT_TYPES[x.dtype], rows, columns, pitch, by, _lib.stream_ptr(x.device))
  return x


# ---- matrix optimizer ---------------------------------------------------------------------------

NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def orthogonalize(update, steps=5, coefficients=NS_COEFFICIENTS, eps=1e-7, out=None):
  """Newton-Schulz orthogonalisation of (..., m, n) matrices: X = G / (|G|_F + eps), then ``steps`` times
  X <- a X + (b A + c A A) X with A = X X^T (of the shorter side).  The singular vectors stay, the singular
  values approach 1.  float32, float16 or bfloat16, computed alike (22-bit operands, fp32 sums and
  copies) and rounded to the type once; every row and column keeps the digits its own size allows, however small it is
  against the others.  Contiguous; the result has update's type and shape.  ``out`` may be ``update``.  With eps > 0 a
  zero matrix gives zeros; a matrix with a NaN or an infinity gives NaN.  Coefficients that let a singular value pass
  8, and what `a` alone makes of 1, leave fp16's range.  Differentiating the result raises."""
  if not isinstance(update, torch.Tensor) or not update.is_cuda:
    raise ValueError("update must be a tensor on the GPU (derl_amd has no CPU path)")
  if update.dtype not in _ELEMENT_TYPES:
    raise ValueError(f"update must be float32, bfloat16 or float16, got {update.dtype}")
  if update.ndim < 2 or not update.is_contiguous():
    raise ValueError(f"update must be contiguous (..., m, n), got {tuple(update.shape)}, strides {update.stride()}")
  if not 1 <= int(steps) <= _INT_MAX:
    raise ValueError(f"steps must be >= 1 (and below 2^31), got {steps}")
  a, b, c = (float(v) for v in coefficients)
  if not all(math.isfinite(v) for v in (a, b, c, eps)) or eps < 0:
    raise ValueError(f"coefficients and eps must be finite, eps >= 0: {coefficients}, {eps}")
  given = out is not None
  if not given:
    out = torch.empty_like(update)
  else:
    if update.requires_grad and torch.is_grad_enabled():
      raise ValueError("out is given and update requires grad: orthogonalize has no gradient")
    _dev(out, "out", update.dtype)
    if out.shape != update.shape or out.device != update.device:
      raise ValueError(f"out must match update: {tuple(out.shape)} on {out.device}")
    (b0, e0), (b1, e1) = _span(update), _span(out)
    if b0 != b1 and b0 < e1 and b1 < e0:
      raise ValueError("out overlaps update (it may only be update itself)")
    _writable(out, "out")
  m, n = update.shape[-2:]
  if update.numel() == 0:
    return out
  batch, m, n = (min(size, _INT_MAX) for size in (update.numel() // (m * n), m, n))  # (the library says what it takes)
  kind = _ELEMENT_TYPES[update.dtype]
  need = _lib.load().dx_orthogonalize_workspace(kind, batch, m, n)
  _lib.check(min(need, 0), "dx_orthogonalize_workspace")
  workspace = torch.empty(need, dtype=torch.uint8, device=update.device)
  _call_on(update.device, "dx_orthogonalize", update.data_ptr(), kind, batch, m, n, int(steps), a, b, c, float(eps),
           out.data_ptr(), workspace.data_ptr(), need, _lib.stream_ptr(update.device))
  return out if given else _constants(update, "orthogonalize", out)[0]


def muon_momentum(grads, momentum, update, partials, max_norm, mu, nesterov=True, norm_out=None):
  """First half of a Muon step on flat float32 buffers: clips ``grads`` in place, advances ``momentum`` and
  writes the direction to orthogonalise to ``update``."""
  for name, t in (("grads", grads), ("momentum", momentum), ("update", update)):
    _dev(t, name, torch.float32)
    if t.numel() != grads.numel():
      raise ValueError(f"{name} must have {grads.numel()} elements, got {t.numel()}")
  _call_on(grads.device, "dx_muon_momentum_f32", _lib.ptr(grads), _lib.ptr(momentum), _lib.ptr(update), grads.numel(),
           _lib.ptr(partials), 0 if partials is None else partials.numel(),
           float(max_norm) if max_norm is not None else 0.0, float(mu), int(bool(nesterov)), _lib.ptr(norm_out),
           _lib.stream_ptr(grads.device))


def muon_apply(params, update, decay, step):
  """params <- params * decay - step * update (flat float32 buffers)."""
  for name, t in (("params", params), ("update", update)):
    _dev(t, name, torch.float32)
  if params.numel() != update.numel():
    raise ValueError(f"update must have {params.numel()} elements, got {update.numel()}")
  _call_on(params.device, "dx_muon_apply_f32", _lib.ptr(params), _lib.ptr(update), params.numel(), float(decay), float(step),
           _lib.stream_ptr(params.device))
