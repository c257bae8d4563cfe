"""panvram_b200.train - the operators of a training step around a model that is fed from a cohort: log-probabilities of
the windows' tokens, two losses made of them, and the gradients' norm and clipping. The reference hands its batch out and
has none of these.

They take the batch as the cohort gives it, with no copy to labels: uint8 tokens 0..4 (Cohort.sample / windows with
tokens=True) or int64 ids (token_ids=..., or the Megatron adapter's labels with its loss mask). Position t of a window is
scored against the token at t + shift, and only where that token is counted:
  * t + shift < W (shift 1, the default, is next-token prediction; 0 takes labels that are shifted already, or a model
    that fills in masked tokens);
  * mask (bool, uint8 or float32 [n, W], at the tokens' positions), if given, is not zero there;
  * it is in [0, V) and not `ignore` (None: 4, any base that is not A C G T, for uint8 tokens; -100 for ids).
What lies at other positions, NaN and infinities included, is not read into any result, and their gradient is zero.

Kernels run on torch's current stream of the logits' (gradients') device, without a wait; scratch comes from torch's
allocator on that stream. Logits are bf16, fp16 or fp32 [n, W, V] with any strides between windows and positions; their
gradient has their type. Arguments other than the logits are constants. A loss keeps the logits, tokens and mask for its
backward pass: with Cohort.sampler, run it before the sampler's next call overwrites its windows."""
import ctypes
import math

import torch

from . import _C

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_ready = set()


def _failed(what):
    return RuntimeError(f"panvram_b200 {what}: " + (_C._lib.pv_kernels_last_error() or b"").decode())


def _device(t, what):
    if t.device.type != "cuda":
        raise RuntimeError(f"panvram_b200 runs on the GPU only: {what} on {t.device}")
    if t.device not in _ready:
        if torch.cuda.get_device_capability(t.device) < (10, 0):
            raise RuntimeError(f"panvram_b200 is built for sm_100a (B200); {torch.cuda.get_device_name(t.device)} is not one")
        _ready.add(t.device)
    return t.device


def _batch(logits, tokens, mask, shift, ignore):
    """The arguments that all operators share, checked -> pv_scored without a gradient."""
    if not isinstance(logits, torch.Tensor) or logits.dim() != 3 or logits.dtype not in _TYPES:
        raise ValueError("logits: a bf16, fp16 or fp32 tensor [n, W, V]")
    n, W, V = logits.shape
    sn, sw, sv = logits.stride()
    if V < 1 or (V > 1 and sv != 1):
        raise ValueError("logits: at least one word, and a position's words contiguous")
    if W >= 1 << 31 or V >= 1 << 30:
        raise ValueError("logits: W below 2^31 and V below 2^30")
    if not isinstance(tokens, torch.Tensor) or tokens.shape != (n, W) or tokens.dtype not in (torch.uint8, torch.int64):
        raise ValueError("tokens: a uint8 or int64 tensor [n, W]")
    ids = tokens.dtype == torch.int64
    kind = 0
    if mask is not None:
        if not isinstance(mask, torch.Tensor) or mask.shape != (n, W) or mask.dtype not in (torch.bool, torch.uint8, torch.float32):
            raise ValueError("mask: a bool, uint8 or float32 tensor [n, W]")
        kind = mask.element_size()
    shift = int(shift)
    if not 0 <= shift < 1 << 31:
        raise ValueError("shift: 0 or more")
    dev = _device(logits, "logits")
    for t, name in ((tokens, "tokens"), (mask, "mask")):
        if t is not None and t.device != dev:
            raise ValueError(f"{name}: on {t.device}, the logits on {dev}")
    tn, tw = tokens.stride()
    mn, mw = mask.stride() if mask is not None else (0, 0)
    ignore = (-100 if ids else 4) if ignore is None else int(ignore)
    return _C.Scored(logits.data_ptr(), None, tokens.data_ptr(), mask.data_ptr() if mask is not None else None, n, W, V, sn, sw, 0, 0, tn, tw,
                     mn, mw, ignore, shift, _TYPES[logits.dtype], 8 if ids else 1, kind)


def _floats(t, name, shapes, dev):
    """a float32 tensor of one of these shapes on dev"""
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or tuple(t.shape) not in shapes:
        raise ValueError(f"{name}: a float32 tensor {' or '.join(str(list(s)) for s in shapes)}")
    if t.device != dev:
        raise ValueError(f"{name}: on {t.device}, the logits on {dev}")
    return t.detach()


def _number(v, name, low, high=math.inf):
    v = float(v)
    if not (low <= v <= high) or math.isinf(v):
        raise ValueError(f"{name}: from {low} to {high}" if high < math.inf else f"{name}: finite, {low} or more")
    return v


def _work(b, dev):
    need = _C._lib.pv_score_work_bytes(ctypes.byref(b))
    return torch.empty(need, dtype=torch.uint8, device=dev), need


def _stream(dev):
    return torch.cuda.current_stream(dev).cuda_stream


def _grad_into(b, logits):
    """a new gradient of the logits, entered in b"""
    g = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    b.grad, b.grad_n, b.grad_w = g.data_ptr(), g.stride(0), g.stride(1)
    return g


def _scale(g):
    """a loss's upstream gradient as a device float"""
    return g if g.dtype == torch.float32 else g.float()


class _Saved:
    """what a backward pass reads again: the batch's tensors go through autograd's saved tensors (which refuse one that
    was changed in place meanwhile), the rest stays here"""

    def __init__(self, ctx, logits, tokens, mask, shift, ignore):
        ctx.save_for_backward(logits, tokens, mask)
        self.shift, self.ignore = shift, ignore

    def batch(self, ctx):
        logits, tokens, mask = ctx.saved_tensors
        return logits, _batch(logits, tokens, mask, self.shift, self.ignore)


# ---------------------------------------------------------------------- log-probabilities
def _logprobs(logits, tokens, mask, shift, ignore, window):
    b = _batch(logits, tokens, mask, shift, ignore)
    dev = logits.device
    with torch.cuda.device(dev):
        out = torch.empty((b.n,) if window else (b.n, b.W), dtype=torch.float32, device=dev)
        work, need = _work(b, dev) if window else (None, 0)
        if _C._lib.pv_logprobs(ctypes.byref(b), None if window else out.data_ptr(), out.data_ptr() if window else None,
                               work.data_ptr() if window else None, need, _stream(dev)):
            raise _failed("log-probabilities")
    return out


class _LogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, mask, shift, ignore, window):
        out = _logprobs(logits, tokens, mask, shift, ignore, window)
        ctx.saved = _Saved(ctx, logits, tokens, mask, shift, ignore)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, up):
        logits, b = ctx.saved.batch(ctx)
        up_n, up_w = (up.stride(0), 0) if up.dim() == 1 else up.stride()
        with torch.cuda.device(logits.device):
            g = _grad_into(b, logits)
            if _C._lib.pv_logprobs_grad(ctypes.byref(b), up.data_ptr(), up_n, up_w, None, 0, _stream(logits.device)):
                raise _failed("log-probabilities' gradient")
        return g, None, None, None, None, None


def window_logprobs(logits, tokens, mask=None, shift=1, ignore=None, reduce="token"):
    """Log-probabilities of the windows' tokens under a model's logits -> float32 [n, W] (position t: the token at
    t + shift; 0 where it is not counted), or with reduce="window" their sums, float32 [n] (0 for a window with none).
    Differentiable by the logits."""
    if reduce not in ("token", "window"):
        raise ValueError('reduce: "token" or "window"')
    f = _LogProbs.apply if torch.is_grad_enabled() and isinstance(logits, torch.Tensor) and logits.requires_grad else _logprobs
    return f(logits, tokens, mask, shift, ignore, reduce == "window")


# ---------------------------------------------------------------------- preference
def _preference(logits, tokens, mask, shift, ignore, ref, beta, smoothing):
    """-> (loss, margins, each window's derivative)"""
    b = _batch(logits, tokens, mask, shift, ignore)
    dev = logits.device
    if b.n % 2:
        raise ValueError("logits: an even number of windows, the preferred ones first")
    ref = _floats(ref, "ref_logp", ((b.n,),), dev)
    with torch.cuda.device(dev):
        loss = torch.empty((), dtype=torch.float32, device=dev)
        margins = torch.empty(b.n // 2, dtype=torch.float32, device=dev)
        coef = torch.empty(b.n, dtype=torch.float32, device=dev)
        work, need = _work(b, dev)
        if _C._lib.pv_preference(ctypes.byref(b), ref.data_ptr(), ref.stride(0), beta, smoothing, loss.data_ptr(), margins.data_ptr(),
                                 coef.data_ptr(), work.data_ptr(), need, _stream(dev)):
            raise _failed("preference loss")
    return loss, margins, coef


class _Preference(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, mask, shift, ignore, ref, beta, smoothing):
        loss, margins, ctx.coef = _preference(logits, tokens, mask, shift, ignore, ref, beta, smoothing)
        ctx.saved = _Saved(ctx, logits, tokens, mask, shift, ignore)
        ctx.mark_non_differentiable(margins)
        return loss, margins

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, up, _):
        logits, b = ctx.saved.batch(ctx)
        with torch.cuda.device(logits.device):
            up = _scale(up)
            g = _grad_into(b, logits)
            if _C._lib.pv_logprobs_grad(ctypes.byref(b), ctx.coef.data_ptr(), 1, 0, up.data_ptr(), 0, _stream(logits.device)):
                raise _failed("preference loss's gradient")
        return (g,) + (None,) * 7


def preference_loss(logits, tokens, ref_logp, beta=0.1, label_smoothing=0.0, mask=None, shift=1, ignore=None, return_margins=False):
    """The preference loss over pairs of windows, a float32 scalar: windows 0 .. n/2 - 1 are preferred over windows
    n/2 .. n - 1. With each window's sum of log-probabilities S (window_logprobs(reduce="window")) and the same sum under
    the reference model R = ref_logp (float32 [n]), a pair's margin is (S - R) of the preferred less (S - R) of the other,
    and its loss -(1 - label_smoothing) log sigmoid(beta margin) - label_smoothing log sigmoid(-beta margin); the mean over
    pairs (0 without any). return_margins: also the margins, float32 [n/2], which carry no gradient."""
    beta, smoothing = _number(beta, "beta", 0.0), _number(label_smoothing, "label_smoothing", 0.0, 1.0)
    f = _Preference.apply if torch.is_grad_enabled() and isinstance(logits, torch.Tensor) and logits.requires_grad else _preference
    r = f(logits, tokens, mask, shift, ignore, ref_logp, beta, smoothing)
    return (r[0], r[1]) if return_margins else r[0]


# ---------------------------------------------------------------------- policy
def _policy_args(b, old, adv, ref, clip, kl, by_window, dev):
    """-> (pv_policy_args, the tensors it points to)"""
    each = ((b.n, b.W),)
    old = _floats(old, "old_logp", each, dev)
    adv = _floats(adv, "advantages", ((b.n,),) + each, dev)
    ref = _floats(ref, "ref_logp", each, dev) if ref is not None else None
    av = adv.stride() if adv.dim() == 2 else (adv.stride(0), 0)
    rv = ref.stride() if ref is not None else (0, 0)
    return _C.PolicyArgs(old.data_ptr(), adv.data_ptr(), ref.data_ptr() if ref is not None else None, *old.stride(), *av, *rv, clip[0], clip[1], kl,
                         by_window), (old, adv, ref)


def _policy(logits, tokens, mask, shift, ignore, old, adv, ref, clip, kl, by_window):
    """-> (loss, the arguments and weights that the gradient takes)"""
    b = _batch(logits, tokens, mask, shift, ignore)
    dev = logits.device
    a, kept = _policy_args(b, old, adv, ref, clip, kl, by_window, dev)
    with torch.cuda.device(dev):
        loss = torch.empty((), dtype=torch.float32, device=dev)
        weight = torch.empty(b.n, dtype=torch.float64, device=dev)
        work, need = _work(b, dev)
        if _C._lib.pv_policy(ctypes.byref(b), ctypes.byref(a), loss.data_ptr(), weight.data_ptr(), work.data_ptr(), need, _stream(dev)):
            raise _failed("policy loss")
    return loss, (a, kept, weight)


class _Policy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, mask, shift, ignore, old, adv, ref, clip, kl, by_window):
        loss, ctx.rest = _policy(logits, tokens, mask, shift, ignore, old, adv, ref, clip, kl, by_window)
        ctx.saved = _Saved(ctx, logits, tokens, mask, shift, ignore)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, up):
        logits, b = ctx.saved.batch(ctx)
        a, _, weight = ctx.rest
        with torch.cuda.device(logits.device):
            up = _scale(up)
            g = _grad_into(b, logits)
            if _C._lib.pv_policy_grad(ctypes.byref(b), ctypes.byref(a), weight.data_ptr(), up.data_ptr(), 0, _stream(logits.device)):
                raise _failed("policy loss's gradient")
        return (g,) + (None,) * 10


def policy_loss(logits, tokens, old_logp, advantages, ref_logp=None, clip=0.2, kl=0.0, mask=None, shift=1, ignore=None, reduce="token"):
    """The clipped policy loss with a KL term, a float32 scalar. With logp the log-probabilities of window_logprobs, and
    old_logp (of the policy that drew the tokens) and ref_logp (of the reference model) laid out the same, float32 [n, W]:
    r = exp(logp - old_logp), and per counted position
        -min(r A, clamp(r, 1 - clip, 1 + clip) A) + kl (exp(d) - d - 1),    d = ref_logp - logp.
    advantages A: float32 [n], or [n, W] at the logits' positions. clip: a number, or (below, above). kl > 0 needs ref_logp.
    reduce: "token", the mean over all counted positions; "window", the mean over the windows that have any of their own
    means. 0 where nothing is counted."""
    if reduce not in ("token", "window"):
        raise ValueError('reduce: "token" or "window"')
    lo, hi = clip if isinstance(clip, (tuple, list)) else (clip, clip)
    clip, kl = (_number(lo, "clip", 0.0), _number(hi, "clip", 0.0)), _number(kl, "kl", 0.0)
    if kl and ref_logp is None:
        raise ValueError("kl: a KL term needs ref_logp")
    args = (logits, tokens, mask, shift, ignore, old_logp, advantages, ref_logp if kl else None, clip, kl, reduce == "window")
    if torch.is_grad_enabled() and isinstance(logits, torch.Tensor) and logits.requires_grad:
        return _Policy.apply(*args)
    return _policy(*args)[0]


# ---------------------------------------------------------------------- gradients
def _dense(t):
    """contiguous in memory, in whatever order of dimensions"""
    if t.is_contiguous():
        return True
    at = 1
    for size, stride in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n != 1), key=lambda x: x[1]):
        if stride != at:
            return False
        at *= size
    return True


def _tensors(ts, name):
    """-> (pv_tensors, what it points to, the tensors as a list)"""
    if isinstance(ts, torch.Tensor):
        ts = [ts]
    ts = list(ts)
    try:
        types = bytes([_TYPES[t.dtype] for t in ts])
    except (KeyError, AttributeError):
        raise ValueError(f"{name}: bf16, fp16 or fp32 tensors") from None
    dense = [t.is_contiguous() for t in ts]
    if not all(dense) and not all(_dense(t) for t in ts):
        raise ValueError(f"{name}: tensors that are dense in memory (no gaps, no expanded dimensions)")
    if len({t.device for t in ts}) > 1:
        raise ValueError(f"{name}: on one device")
    n = len(ts)
    ptr, numel = (ctypes.c_uint64 * n)(*[t.data_ptr() for t in ts]), (ctypes.c_int64 * n)(*[t.numel() for t in ts])
    kept = (ptr, numel, ctypes.c_char_p(types))
    return _C.Tensors(ctypes.cast(ptr, ctypes.c_void_p), ctypes.cast(numel, ctypes.c_void_p), ctypes.cast(kept[2], ctypes.c_void_p), n), kept, ts


def _norm_buffers(g, ts):
    dev = _device(ts[0], "gradients")
    need = _C._lib.pv_grads_work_bytes(ctypes.byref(g))
    return dev, torch.empty((), dtype=torch.float32, device=dev), torch.empty(need, dtype=torch.uint8, device=dev), need


def grad_norm(grads):
    """The 2-norm over all elements of all tensors (a tensor, or bf16 / fp16 / fp32 tensors of any shapes on one device,
    each dense in memory) -> float32 scalar on their device, summed in 64 bits. An empty list is refused: it has no
    device."""
    g, kept, ts = _tensors(grads, "grads")
    if not ts:
        raise ValueError("grads: no tensors")
    with torch.cuda.device(_device(ts[0], "gradients")):
        dev, norm, work, need = _norm_buffers(g, ts)
        if _C._lib.pv_grad_norm(ctypes.byref(g), norm.data_ptr(), work.data_ptr(), need, _stream(dev)):
            raise _failed("gradient norm")
    return norm


def clip_grads(grads, max_norm, out=None):
    """Scale the gradients by min(1, max_norm / (norm + 1e-6)) -> their norm before it (grad_norm), no wait for the device.
    In place; or into `out`, one tensor per gradient of its shape and strides, of its type or float32 (an optimizer's
    full-precision gradients), then always written. A tensor that is written may not share memory with another. A norm of
    infinity scales finite elements to 0, NaN makes every element NaN, as the formula says."""
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError("max_norm: 0 or more")
    g, kept, ts = _tensors(grads, "grads")
    if not ts:
        raise ValueError("grads: no tensors")
    o = okept = None
    if out is not None:
        o, okept, outs = _tensors(out, "out")
        if len(outs) != len(ts) or any(a.shape != b.shape or a.stride() != b.stride() for a, b in zip(ts, outs)):
            raise ValueError("out: one tensor per gradient, of its shape and strides")
        if any(b.dtype != a.dtype and b.dtype != torch.float32 for a, b in zip(ts, outs)):
            raise ValueError("out: of the gradient's type, or float32")
        if outs[0].device != ts[0].device:
            raise ValueError("out: on the gradients' device")
    written = ts if out is None else outs
    if any(t.requires_grad and t.is_leaf and torch.is_grad_enabled() for t in written):
        raise ValueError("clip_grads: pass the gradients (p.grad), not parameters")
    with torch.cuda.device(_device(ts[0], "gradients")):
        dev, norm, work, need = _norm_buffers(g, ts)
        code = _C._lib.pv_clip_grads(ctypes.byref(g), ctypes.byref(o) if o is not None else None, max_norm, norm.data_ptr(), work.data_ptr(), need,
                                     _stream(dev))
    if code == _C.PV_EARG:
        raise ValueError((_C._lib.pv_kernels_last_error() or b"").decode())
    if code:
        raise _failed("gradient clipping")
    return norm
