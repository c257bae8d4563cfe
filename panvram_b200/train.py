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
gradient has their type, and no second derivative. Arguments other than the logits are constants. A loss keeps the logits, tokens and mask for its
backward pass: with Cohort.sampler, run it before the sampler's next call overwrites its windows."""
import ctypes
import math
from array import array
from contextlib import nullcontext

import torch

from . import _C

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_ready = set()
_here = nullcontext()


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


def _on(dev):
    """the device made current for a launch (nothing to do where it is)"""
    return _here if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


def _stream(dev):
    return torch._C._cuda_getCurrentRawStream(dev.index)


def _work(b, dev, more=0):
    """scratch for b, and `more` bytes in front of it (rounded up to 16) -> (tensor, address of the scratch, its bytes)"""
    need, more = _C._lib.pv_score_work_bytes(ctypes.byref(b)), (more + 15) // 16 * 16
    t = torch.empty(more + need, dtype=torch.uint8, device=dev)
    return t, t.data_ptr() + more, need


def _with_grad(b, logits, g=None):
    """b with a gradient of the logits to be written, a new one if none is given -> (b, gradient)"""
    if g is None:
        g = logits.new_empty(logits.shape)
    b = _C.Scored.from_buffer_copy(b)
    b.grad, (b.grad_n, b.grad_w, _) = g.data_ptr(), g.stride()
    return b, g


class _NoSecond(torch.autograd.Function):
    """a gradient that may be used, but not differentiated by the logits"""

    @staticmethod
    def forward(ctx, g, logits):
        return g.view_as(g)

    @staticmethod
    def backward(ctx, up):
        raise RuntimeError("panvram_b200: no second derivative")


def _once(backward):
    """a backward pass whose gradient refuses a second one (which only a pass that makes a graph could ask for)"""
    def run(ctx, up):
        if not torch.is_grad_enabled():
            return backward(ctx, up)
        with torch.no_grad():
            out = backward(ctx, up)
        return (_NoSecond.apply(out[0], ctx.saved_tensors[0]),) + out[1:]
    return run


def _wants_grad(logits):
    return isinstance(logits, torch.Tensor) and logits.requires_grad and torch.is_grad_enabled()


# ---------------------------------------------------------------------- log-probabilities
def _logprobs(b, dev, window, keep=False):
    """-> (log-probabilities, with `keep` a buffer that starts with the rows' statistics)"""
    with _on(dev):
        out = torch.empty((b.n,) if window else (b.n, b.W), dtype=torch.float32, device=dev)
        more = _C._lib.pv_score_stat_bytes(ctypes.byref(b)) if keep else 0
        buf, work, need = _work(b, dev, more) if window or more else (None, None, 0)
        if _C._lib.pv_logprobs(ctypes.byref(b), None if window else out.data_ptr(), out.data_ptr() if window else None,
                               buf.data_ptr() if more else None, work, need, _stream(dev)):
            raise _failed("log-probabilities")
    return out, buf if more else None


class _LogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, mask, b, window):
        # autograd's saved tensors refuse one that is changed in place before the backward pass; b points into them
        ctx.save_for_backward(logits, tokens, mask)
        ctx.b = b
        out, ctx.stat = _logprobs(b, logits.device, window, True)
        return out

    @staticmethod
    @_once
    def backward(ctx, up):
        logits = ctx.saved_tensors[0]
        up_n, up_w = (up.stride(0), 0) if up.dim() == 1 else up.stride()
        with _on(logits.device):
            b, g = _with_grad(ctx.b, logits)
            if _C._lib.pv_logprobs_grad(ctypes.byref(b), up.data_ptr(), up_n, up_w,
                                        ctx.stat.data_ptr() if ctx.stat is not None else None, None, _stream(logits.device)):
                raise _failed("log-probabilities' gradient")
        return g, None, None, None, None


def window_logprobs(logits, tokens, mask=None, shift=1, ignore=None, reduce="token"):
    """Log-probabilities of the windows' tokens under a model's logits -> float32 [n, W] (position t: the token at
    t + shift; 0 where it is not counted), or with reduce="window" their sums, float32 [n] (0 for a window with none).
    Differentiable by the logits."""
    if reduce not in ("token", "window"):
        raise ValueError('reduce: "token" or "window"')
    b = _batch(logits, tokens, mask, shift, ignore)
    if _wants_grad(logits):
        return _LogProbs.apply(logits, tokens, mask, b, reduce == "window")
    return _logprobs(b, logits.device, reduce == "window")[0]


# ---------------------------------------------------------------------- preference
def _preference(b, dev, ref, beta, smoothing, margins, keep=False):
    """-> (loss, a buffer of the rows' statistics (with `keep`) and each window's derivative, those' address)"""
    with _on(dev):
        loss = torch.empty((), dtype=torch.float32, device=dev)
        more = _C._lib.pv_score_stat_bytes(ctypes.byref(b)) if keep else 0
        buf, work, need = _work(b, dev, more + 4 * b.n)
        coef = buf.data_ptr() + more
        if _C._lib.pv_preference(ctypes.byref(b), ref.data_ptr(), ref.stride(0), beta, smoothing, loss.data_ptr(),
                                 margins.data_ptr() if margins is not None else None, coef, buf.data_ptr() if more else None, work, need,
                                 _stream(dev)):
            raise _failed("preference loss")
    return loss, buf, coef


class _Preference(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, mask, b, ref, beta, smoothing, margins):
        ctx.save_for_backward(logits, tokens, mask)
        ctx.b = b
        loss, ctx.buf, ctx.coef = _preference(b, logits.device, ref, beta, smoothing, margins, True)
        return loss

    @staticmethod
    @_once
    def backward(ctx, up):
        logits = ctx.saved_tensors[0]
        with _on(logits.device):
            b, g = _with_grad(ctx.b, logits)
            stat = ctx.buf.data_ptr() if ctx.buf.data_ptr() != ctx.coef else None
            if _C._lib.pv_logprobs_grad(ctypes.byref(b), ctx.coef, 1, 0, stat, up.data_ptr(), _stream(logits.device)):
                raise _failed("preference loss's gradient")
        return g, None, None, None, None, None, None, None


def preference_loss(logits, tokens, ref_logp, beta=0.1, label_smoothing=0.0, mask=None, shift=1, ignore=None, return_margins=False):
    """The preference loss over pairs of windows, a float32 scalar: windows 0 .. n/2 - 1 are preferred over windows
    n/2 .. n - 1. With each window's sum of log-probabilities S (window_logprobs(reduce="window")) and the same sum under
    the reference model R = ref_logp (float32 [n]), a pair's margin is (S - R) of the preferred less (S - R) of the other,
    and its loss -(1 - label_smoothing) log sigmoid(beta margin) - label_smoothing log sigmoid(-beta margin); the mean over
    pairs (0 without any). return_margins: also the margins, float32 [n/2], which carry no gradient."""
    beta, smoothing = _number(beta, "beta", 0.0), _number(label_smoothing, "label_smoothing", 0.0, 1.0)
    b = _batch(logits, tokens, mask, shift, ignore)
    dev = logits.device
    if b.n % 2:
        raise ValueError("logits: an even number of windows, the preferred ones first")
    ref = _floats(ref_logp, "ref_logp", ((b.n,),), dev)
    margins = torch.empty(b.n // 2, dtype=torch.float32, device=dev) if return_margins else None
    if _wants_grad(logits):
        loss = _Preference.apply(logits, tokens, mask, b, ref, beta, smoothing, margins)
    else:
        loss = _preference(b, dev, ref, beta, smoothing, margins)[0]
    return (loss, margins) if return_margins else loss


# ---------------------------------------------------------------------- policy
def _policy_args(b, old, adv, ref, clip, kl, by_window, scale, dev):
    """-> (pv_policy_args, the tensors it points to)"""
    each = ((b.n, b.W),)
    old = _floats(old, "old_logp", each, dev)
    adv = _floats(adv, "advantages", ((b.n,),) + each, dev)
    ref = _floats(ref, "ref_logp", each, dev) if ref is not None else None
    av = adv.stride() if adv.dim() == 2 else (adv.stride(0), 0)
    rv = ref.stride() if ref is not None else (0, 0)
    return _C.PolicyArgs(old.data_ptr(), adv.data_ptr(), ref.data_ptr() if ref is not None else None, *old.stride(), *av, *rv, clip[0], clip[1], kl,
                         scale, by_window), (old, adv, ref)


def _policy(b, dev, a):
    """-> (loss, (a buffer that starts with the windows' weights, its scratch's address and bytes)); b's gradient too, if it
    names one"""
    with _on(dev):
        loss = torch.empty((), dtype=torch.float32, device=dev)
        buf, work, need = _work(b, dev, 8 * b.n)
        if _C._lib.pv_policy(ctypes.byref(b), ctypes.byref(a), loss.data_ptr(), buf.data_ptr(), work, need, _stream(dev)):
            raise _failed("policy loss")
    return loss, (buf, work, need)


class _Policy(torch.autograd.Function):
    # A position's weight is known from the tokens alone, so the loss's pass over the logits forms their gradient too and
    # the logits are read once: backward finds it made where its upstream gradient is 1, and forms it again where it is not
    # (found out on the device, without a wait). Half-precision logits come with a loss scale that keeps their gradient in
    # range, so theirs is left to backward.
    @staticmethod
    def forward(ctx, logits, tokens, mask, b, a, kept):
        ctx.save_for_backward(logits, tokens, mask, *kept)
        ctx.b, ctx.a, ctx.grad = b, a, None
        if logits.dtype != torch.float16:
            b, ctx.grad = _with_grad(b, logits)
        loss, ctx.work = _policy(b, logits.device, a)
        return loss

    @staticmethod
    @_once
    def backward(ctx, up):
        logits = ctx.saved_tensors[0]
        made, ctx.grad = ctx.grad, None
        with _on(logits.device):
            b, g = _with_grad(ctx.b, logits, made)
            # the loss's scratch again: it is done with, and long rows need some
            buf, work, need = ctx.work
            if _C._lib.pv_policy_grad(ctypes.byref(b), ctypes.byref(ctx.a), buf.data_ptr(), up.data_ptr(), made is not None, work, need,
                                      _stream(logits.device)):
                raise _failed("policy loss's gradient")
        return g, None, None, None, None, None


def policy_loss(logits, tokens, old_logp, advantages, ref_logp=None, clip=0.2, kl=0.0, mask=None, shift=1, ignore=None, reduce="token", scale=1.0):
    """The clipped policy loss with a KL term, a float32 scalar. With logp the log-probabilities of window_logprobs, and
    old_logp (of the policy that drew the tokens) and ref_logp (of the reference model) laid out the same, float32 [n, W]:
    r = exp(logp - old_logp), and per counted position
        -min(r A, clamp(r, 1 - clip, 1 + clip) A) + kl (exp(d) - d - 1),    d = ref_logp - logp.
    advantages A: float32 [n], or [n, W] at the logits' positions. clip: a number, or (below, above). kl > 0 needs ref_logp.
    reduce: "token", the mean over all counted positions; "window", the mean over the windows that have any of their own
    means. 0 where nothing is counted. The result is multiplied by `scale`: with 1 / (batches a step) there, and not on the
    loss, the gradient is made in the loss's own pass over bf16 or fp32 logits (whose memory it takes from then on); an
    upstream gradient other than 1 makes it once more."""
    if reduce not in ("token", "window"):
        raise ValueError('reduce: "token" or "window"')
    lo, hi = clip if isinstance(clip, (tuple, list)) else (clip, clip)
    clip, kl, scale = (_number(lo, "clip", 0.0), _number(hi, "clip", 0.0)), _number(kl, "kl", 0.0), _number(scale, "scale", 0.0)
    if kl and ref_logp is None:
        raise ValueError("kl: a KL term needs ref_logp")
    b = _batch(logits, tokens, mask, shift, ignore)
    dev = logits.device
    a, kept = _policy_args(b, old_logp, advantages, ref_logp if kl else None, clip, kl, reduce == "window", scale, dev)
    if _wants_grad(logits):
        return _Policy.apply(logits, tokens, mask, b, a, kept)
    return _policy(b, dev, a)[0]


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
    """-> (pv_tensors, the arrays it points to, the tensors as a list, their types, whether all are contiguous)"""
    ts = [ts] if isinstance(ts, torch.Tensor) else list(ts)
    try:
        types = [t.dtype for t in ts]
        same = bool(ts) and types.count(types[0]) == len(ts)
        types = array("B", [_TYPES[types[0]]]) * len(ts) if same else array("B", [_TYPES[t] for t in types])
    except (KeyError, AttributeError):
        raise ValueError(f"{name}: bf16, fp16 or fp32 tensors") from None
    plain = all([t.is_contiguous() for t in ts])
    if not plain and not all(_dense(t) for t in ts):
        raise ValueError(f"{name}: tensors that are dense in memory (no gaps, no expanded dimensions)")
    if len(set([t.get_device() for t in ts])) > 1:
        raise ValueError(f"{name}: on one device")
    if not ts:
        raise ValueError(f"{name}: no tensors")
    kept = array("Q", [t.data_ptr() for t in ts]), array("q", [t.numel() for t in ts]), types
    return _C.Tensors(*(a.buffer_info()[0] for a in kept), len(ts)), kept, ts, types, plain


def _norm_buffers(g, dev):
    need = _C._lib.pv_grads_work_bytes(ctypes.byref(g))
    return torch.empty((), dtype=torch.float32, device=dev), torch.empty(need, dtype=torch.uint8, device=dev), need


def grad_norm(grads):
    """The 2-norm over all elements of all tensors (a tensor, or bf16 / fp16 / fp32 tensors of any shapes on one device,
    each dense in memory) -> float32 scalar on their device, summed in 64 bits. An empty list is refused: it has no
    device."""
    g, kept, ts, _, _ = _tensors(grads, "grads")
    dev = _device(ts[0], "gradients")
    with _on(dev):
        norm, work, need = _norm_buffers(g, dev)
        if _C._lib.pv_grad_norm(ctypes.byref(g), norm.data_ptr(), work.data_ptr(), need, _stream(dev)):
            raise _failed("gradient norm")
    return norm


def clip_grads(grads, max_norm, out=None):
    """Scale the gradients by min(1, max_norm / (norm + 1e-6)) -> their norm before it (grad_norm), no wait for the device.
    In place; or into `out`, one tensor per gradient, of its type or float32 (an optimizer's full-precision gradients) and as
    many elements, contiguous as it is (else of its shape and strides); then always written. A tensor that is written may not share memory with another. A norm of
    infinity scales finite elements to 0, NaN makes every element NaN, as the formula says."""
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError("max_norm: 0 or more")
    g, kept, ts, types, plain = _tensors(grads, "grads")
    o, written = None, ts
    if out is not None:
        o, okept, written, otypes, oplain = _tensors(out, "out")
        if plain and oplain:
            alike = kept[1] == okept[1]
        else:
            alike = len(ts) == len(written) and all(a.shape == b.shape and a.stride() == b.stride() for a, b in zip(ts, written))
        if not alike:
            raise ValueError("out: one tensor per gradient, of its size and laid out alike")
        if types != otypes and any([b != 2 and a != b for a, b in zip(types, otypes)]):
            raise ValueError("out: of the gradient's type, or float32")
        if written[0].device != ts[0].device:
            raise ValueError("out: on the gradients' device")
    if True in [t.requires_grad for t in written]:
        raise ValueError("clip_grads: pass gradients (p.grad), not parameters, and none that autograd has a graph for")
    dev = _device(ts[0], "gradients")
    with _on(dev):
        norm, work, need = _norm_buffers(g, dev)
        code = _C._lib.pv_clip_grads(ctypes.byref(g), ctypes.byref(o) if o is not None else None, max_norm, norm.data_ptr(), work.data_ptr(), need,
                                     _stream(dev))
    if code == _C.PV_EARG:
        raise ValueError((_C._lib.pv_kernels_last_error() or b"").decode())
    if code:
        raise _failed("gradient clipping")
    return norm
