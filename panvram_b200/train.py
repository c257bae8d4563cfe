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
gradient has their type, and no second derivative. Arguments other than the logits are constants. A loss keeps the logits,
tokens and mask for its backward pass (hooks on saved tensors apply): with Cohort.sampler, run it before the sampler's next
call overwrites its windows (autograd refuses it afterwards). A clipped list counts as changed in place."""
import os

import torch

from . import _C

_train = None               # torch_ext/pv_torch.cpp, loaded by the first call: the data path does without it


def _ext():
    """the compiled side (bound to one torch release, unlike the library that it calls and _C has loaded)"""
    global _train
    if _train is None:
        try:
            from . import _train as ext
        except ImportError as e:
            path = os.path.join(os.path.dirname(_C.LIB_PATH), "_train.so")
            why = "is missing" if not os.path.exists(path) else f"does not load under torch {torch.__version__}"
            raise ImportError(f"panvram_b200: the training step's operators are in {path}, which {why}; build it: "
                              "python panvram_b200/build.py") from e
        _train = ext
    return _train


def _shared(logits, tokens, mask, shift, ignore):
    """what the compiled side cannot take at all, refused in the words it has for the rest; -> its last arguments"""
    if not isinstance(logits, torch.Tensor):
        raise ValueError("logits: a bf16, fp16 or fp32 tensor [n, W, V]")
    if not isinstance(tokens, torch.Tensor):
        raise ValueError("tokens: a uint8 or int64 tensor [n, W]")
    if mask is not None and not isinstance(mask, torch.Tensor):
        raise ValueError("mask: a bool, uint8 or float32 tensor [n, W]")
    shift, ignore = int(shift), None if ignore is None else int(ignore)
    if not 0 <= shift < 1 << 31:
        raise ValueError("shift: 0 or more")
    if ignore is not None and not -1 << 63 <= ignore < 1 << 63:
        raise ValueError("ignore: a 64-bit integer")
    return mask, shift, ignore


def _floats(**tensors):
    for name, t in tensors.items():
        if not isinstance(t, torch.Tensor):
            raise ValueError(f"{name}: a float32 tensor")


def _by_window(reduce):
    if reduce not in ("token", "window"):
        raise ValueError('reduce: "token" or "window"')
    return reduce == "window"


def window_logprobs(logits, tokens, mask=None, shift=1, ignore=None, reduce="token"):
    """Log-probabilities of the windows' tokens under a model's logits -> float32 [n, W] (position t: the token at
    t + shift; 0 where it is not counted), or with reduce="window" their sums, float32 [n] (0 for a window with none).
    Differentiable by the logits."""
    window = _by_window(reduce)
    return _ext().window_logprobs(logits, tokens, *_shared(logits, tokens, mask, shift, ignore), window)


def preference_loss(logits, tokens, ref_logp, beta=0.1, label_smoothing=0.0, mask=None, shift=1, ignore=None, return_margins=False):
    """The preference loss over pairs of windows, a float32 scalar: windows 0 .. n/2 - 1 are preferred over windows
    n/2 .. n - 1. With each window's sum of log-probabilities S (window_logprobs(reduce="window")) and the same sum under
    the reference model R = ref_logp (float32 [n]), a pair's margin is (S - R) of the preferred less (S - R) of the other,
    and its loss -(1 - label_smoothing) log sigmoid(beta margin) - label_smoothing log sigmoid(-beta margin); the mean over
    pairs (0 without any). return_margins: also the margins, float32 [n/2], which carry no gradient."""
    rest = _shared(logits, tokens, mask, shift, ignore)
    _floats(ref_logp=ref_logp)
    out = _ext().preference_loss(logits, tokens, ref_logp, float(beta), float(label_smoothing), *rest, bool(return_margins))
    return out if return_margins else out[0]


def policy_loss(logits, tokens, old_logp, advantages, ref_logp=None, clip=0.2, kl=0.0, mask=None, shift=1, ignore=None, reduce="token", scale=1.0):
    """The clipped policy loss with a KL term, a float32 scalar. With logp the log-probabilities of window_logprobs, and
    old_logp (of the policy that drew the tokens) and ref_logp (of the reference model) laid out the same, float32 [n, W]:
    r = exp(logp - old_logp), and per counted position
        -min(r A, clamp(r, 1 - clip, 1 + clip) A) + kl (exp(d) - d - 1),    d = ref_logp - logp.
    advantages A: float32 [n], or [n, W] at the logits' positions; where A is 0 an r that overflows counts as 0. clip: a number, or (below, above). kl > 0 needs ref_logp.
    reduce: "token", the mean over all counted positions; "window", the mean over the windows that have any of their own
    means. 0 where nothing is counted. The result is multiplied by `scale`: with 1 / (batches a step) there, and not on the
    loss, the gradient is made in the loss's own pass over bf16 or fp32 logits (whose memory it takes from then on); an
    upstream gradient other than 1 makes it once more."""
    by_window = _by_window(reduce)
    rest = _shared(logits, tokens, mask, shift, ignore)
    _floats(old_logp=old_logp, advantages=advantages)
    if ref_logp is not None:
        _floats(ref_logp=ref_logp)
    low, high = clip if isinstance(clip, (tuple, list)) else (clip, clip)
    return _ext().policy_loss(logits, tokens, old_logp, advantages, ref_logp, float(low), float(high), float(kl), *rest, by_window, float(scale))


def _list(ts):
    return [ts] if isinstance(ts, torch.Tensor) else list(ts)


def grad_norm(grads):
    """The 2-norm over all elements of all tensors (a tensor, or bf16 / fp16 / fp32 tensors of any shapes on one device,
    each dense in memory) -> float32 scalar on their device, summed in 64 bits. An empty list is refused: it has no
    device."""
    try:
        return _ext().grad_norm(_list(grads))
    except TypeError:
        raise ValueError("grads: bf16, fp16 or fp32 tensors") from None


def clip_grads(grads, max_norm, out=None):
    """Scale the gradients by min(1, max_norm / (norm + 1e-6)) -> their norm before it (grad_norm), no wait for the device.
    In place; or into `out`, one tensor per gradient, of its type or float32 (an optimizer's full-precision gradients) and as
    many elements, contiguous as it is (else of its shape and strides); then always written. A tensor that is written may not share memory with another. A norm of
    infinity scales finite elements to 0, NaN makes every element NaN, as the formula says."""
    try:
        return _ext().clip_grads(_list(grads), float(max_norm), None if out is None else _list(out))
    except TypeError:
        raise ValueError("grads, out: bf16, fp16 or fp32 tensors") from None
