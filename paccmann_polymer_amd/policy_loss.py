"""Log-probabilities of taken tokens and the clipped policy loss on them: the objectives that train a generator of token
sequences from rewards, beside the cross-entropy K2 (`stack_gru_vae._CrossEntropy`) and on the same packed logits.  The
reference trains by likelihood only (paccmann_polymer/models/paccmann_encoder.py:168); these have no counterpart in it.

Rows of logits are in whatever order the caller's targets are (the framework's own paths use packed order).  A row whose
target is `ignore_index` counts nowhere.  Logits are fp32 or bf16; everything per row is fp32, and sums over rows are held
in 64 bits.  Kernels: csrc/ppk_policy.hip.
"""
import torch
from torch.autograd.function import once_differentiable

from . import _C

_lib = _C.lib


def _check_logits(what, logits, targets, temperature):
    if not torch.is_tensor(logits) or logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f'{what}: logits must be [rows, vocabulary]')
    if not torch.is_tensor(targets) or tuple(targets.shape) != (logits.shape[0],):
        raise ValueError(f'{what}: targets must be [rows]')
    if targets.dtype != torch.int64:
        raise TypeError(f'{what}: targets must be int64')
    if not 1e-30 <= float(temperature) <= 1e30:
        raise ValueError(f'{what}: the temperature must be positive and finite (1e-30 to 1e30)')
    return _C.dtype_code(logits, what)


def _row_values(what, name, t, rows):
    if not torch.is_tensor(t) or tuple(t.shape) != (rows,):
        raise ValueError(f'{what}: {name} must be [rows]')
    if t.dtype != torch.float32:
        raise TypeError(f'{what}: {name} must be float32')
    return t.detach().contiguous()


def _rows_of(logits):
    """The logits with elements of a row next to each other (a row stride is taken as it is)."""
    if (logits.stride(1) == 1 or logits.shape[1] == 1) and (logits.shape[0] <= 1 or logits.stride(0) >= logits.shape[1]):
        return logits
    return logits.contiguous()


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _ld(logits):
    return max(logits.stride(0), logits.shape[1])


class _TokenLogProbs(torch.autograd.Function):

    @staticmethod
    def forward(ctx, logits, targets, ignore_index, temperature, want_grad):
        code = _check_logits('token_log_probs', logits, targets, temperature)
        dev = _C.one_device(logits, targets)
        x, t = _rows_of(logits), targets.contiguous()
        rows, V = x.shape
        with _C.on_device(dev):
            logp = torch.empty(rows, dtype=torch.float32, device=dev)
            saved = torch.empty(rows, 2, dtype=torch.float32, device=dev) if want_grad else None
            _C.check(_lib.ppk_token_logp_fwd(code, _C.addr(x), _ld(x), _C.addr(t), rows, V, ignore_index, temperature, _C.addr(logp), _C.addr(saved), _C.stream_on(x.device)))
        if saved is not None:
            ctx.save_for_backward(x, t, saved)
            ctx.args = (code, ignore_index, temperature)
        return logp

    @staticmethod
    @once_differentiable
    def backward(ctx, dlogp):
        x, t, saved = ctx.saved_tensors
        code, ignore_index, temperature = ctx.args
        rows, V = x.shape
        with _C.on_device(x.device):
            d = torch.empty(rows, V, dtype=x.dtype, device=x.device)
            g = dlogp.to(torch.float32).contiguous()
            _C.check(_lib.ppk_token_logp_bwd(code, _C.addr(x), _ld(x), _C.addr(t), rows, V, ignore_index, temperature, _C.addr(saved), _C.addr(g), _C.addr(d), V, _C.stream_on(x.device)))
        return d, None, None, None, None


def token_log_probs(logits, targets, ignore_index=0, temperature=1.0):
    """log softmax(logits / temperature) at each row's target, [rows] fp32; 0 where the target is `ignore_index`.

    logits [rows, V] fp32 or bf16 (rows may be strided), targets [rows] int64.  Differentiable in the logits.  A target that is
    neither `ignore_index` nor in [0, V) gives NaN (nothing is read through it, and nothing synchronises)."""
    return _TokenLogProbs.apply(logits, targets, int(ignore_index), float(temperature), _wants_grad(logits))


def _policy_call(code, x, t, old, adv, ref, args, want_grad):
    rows, V = x.shape
    clip_low, clip_high, kl_coef, ignore_index, temperature = args
    dev = x.device
    with _C.on_device(dev):
        loss, stats = torch.empty((), dtype=torch.float32, device=dev), torch.empty(3, dtype=torch.float32, device=dev)     # no views: callers change them in place
        d = torch.empty(rows, V, dtype=x.dtype, device=dev) if want_grad else None
        wsb = _lib.ppk_policy_loss_workspace_bytes(rows)
        ws = torch.empty(max(int(wsb), 256), dtype=torch.uint8, device=dev)
        _C.check(_lib.ppk_policy_loss(code, _C.addr(x), _ld(x), _C.addr(t), rows, V, ignore_index, temperature, _C.addr(old), _C.addr(adv), _C.addr(ref),
                                      clip_low, clip_high, kl_coef, _C.addr(loss), _C.addr(stats), _C.addr(d), V, _C.addr(ws), wsb, _C.stream_on(x.device)))
    return loss, stats, d


class _PolicyLoss(torch.autograd.Function):
    """The forward pass writes the gradient of the loss while it holds the logits; the backward pass multiplies it by the upstream
    gradient, which costs nothing but a look where that is 1."""

    @staticmethod
    def forward(ctx, logits, targets, old, adv, ref, args, want_grad):
        code = _C.dtype_code(logits, 'policy_loss')
        x = _rows_of(logits)
        loss, stats, d = _policy_call(code, x, targets, old, adv, ref, args, want_grad)
        if d is not None:
            ctx.save_for_backward(x, targets, old, adv, ref)
            ctx.grad, ctx.code, ctx.args, ctx.captured = d, code, args, torch.cuda.is_current_stream_capturing()
        ctx.mark_non_differentiable(stats)
        return loss, stats

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, _dstats):
        d, ctx.grad = ctx.grad, None                        # it is handed on and may be changed: a second backward pass makes its own
        # so does one that is captured behind an eager forward pass: each replay would multiply the same memory once more
        if d is None or (not ctx.captured and torch.cuda.is_current_stream_capturing()):
            x, targets, old, adv, ref = ctx.saved_tensors
            d = _policy_call(ctx.code, x, targets, old, adv, ref, ctx.args, True)[2]
        dev = d.device
        with _C.on_device(dev):
            s = dloss if dloss.dtype == torch.float32 else dloss.to(torch.float32)
            _C.check(_lib.ppk_scale_unless_one(ctx.code, _C.addr(d), d.numel(), _C.addr(s), _C.stream_on(dev)))
        return d, None, None, None, None, None, None


def policy_loss(logits, targets, old_log_probs, advantages, ref_log_probs=None, clip_low=0.2, clip_high=0.2, kl_coef=0.0,
                ignore_index=0, temperature=1.0):
    """Clipped policy loss with a KL term, and its means: (loss, stats).

    Per row that counts, with lp = log softmax(logits / temperature) at the target, ratio = exp(lp - old), d = ref - lp:
      -min(ratio A, clip(ratio, 1 - clip_low, 1 + clip_high) A) + kl_coef (exp(d) - d - 1)
    loss: 0-dim fp32, the mean of that over the rows whose target is not `ignore_index` (0 where there is none), differentiable
    in the logits.  stats: [3] fp32 on the device, not differentiable: the means of the policy term, of the KL term (0 without a
    reference) and of the rows that the clip holds.
    logits [rows, V] fp32 or bf16; targets [rows] int64; old_log_probs, advantages, ref_log_probs [rows] fp32 (constants: what
    `token_log_probs` gave under the sampling and under the reference parameters, at the same temperature).
    A call whose logits want a gradient writes it in the same pass and holds it, a tensor of the logits' size and type, until the
    backward pass."""
    what = 'policy_loss'
    _check_logits(what, logits, targets, temperature)
    rows = logits.shape[0]
    if not (0.0 <= float(clip_low) <= 1.0 and 0.0 <= float(clip_high) < float('inf')):
        raise ValueError(f'{what}: the clip range must be 0 <= clip_low <= 1, clip_high >= 0')
    if float(kl_coef) != 0.0 and ref_log_probs is None:
        raise ValueError(f'{what}: a KL term needs ref_log_probs')
    if not abs(float(kl_coef)) < float('inf'):
        raise ValueError(f'{what}: kl_coef must be finite')
    old = _row_values(what, 'old_log_probs', old_log_probs, rows)
    adv = _row_values(what, 'advantages', advantages, rows)
    ref = None if ref_log_probs is None else _row_values(what, 'ref_log_probs', ref_log_probs, rows)
    _C.one_device(logits, targets, old, adv, ref)
    args = (float(clip_low), float(clip_high), float(kl_coef), int(ignore_index), float(temperature))
    return _PolicyLoss.apply(logits, targets.contiguous(), old, adv, ref, args, _wants_grad(logits))
