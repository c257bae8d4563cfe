"""panvram_b200 - a B200-native drop-in for panvram's refrel3 v1 random-access window path: a pangenome cohort
resident on the GPU as refrel3 v1 archives (edits against one decoded reference); random windows and coordinate
slices decoded on the card by one sm_100a kernel.

    c = panvram_b200.Cohort.open(dir, device="cuda")  # reference + assemblies resident
    x = c.sample(n, W, generator=g)                    # uint8 [n, W] (bytes or tokens) on the device
    y = c.fetch(assembly, contig, start, length)       # a slice by coordinates

and the operators of a training step around a model fed from it (panvram_b200.train):

    lp = window_logprobs(logits, x)                    # the windows' tokens under a model; c.score(model, ...) per window
    loss = preference_loss(logits, x, ref_logp)        # or policy_loss(logits, x, old_logp, advantages, ref_logp, ...)
    norm = clip_grads([p.grad for p in parameters], 1.0)
"""
import torch  # noqa: F401  (CUDA context and caching allocator come from torch)

from . import _C
from .cohort import DATASETS, Cohort, global_batch
from .train import clip_grads, grad_norm, policy_loss, preference_loss, window_logprobs

FormatError = _C.FormatError
with_cuda = _C.with_cuda
__version__ = "0.1.0"
__all__ = ["Cohort", "DATASETS", "FormatError", "with_cuda", "global_batch", "window_logprobs", "preference_loss",
           "policy_loss", "grad_norm", "clip_grads"]
