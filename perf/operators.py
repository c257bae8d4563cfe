"""The training-step operators that stand around a model fed from a cohort, as cases to be timed: log-probabilities of
the windows' tokens, the preference loss over pairs of windows, the clipped policy loss with a KL term, and the gradient
norm over many tensors with clipping.

`run` computes a case in its plain form (elementary torch operations, in 32 bits, long sums in 64), or, where `own` is
true, by the calls of panvram_b200. `exact` computes it in 64 bits from the definitions.

The rule shared by the first three: position t of window i is scored against the token at t + shift, and only where that
token is counted: inside the window, its mask not zero, in [0, V), and not the ignored code (4, any base that is not
A C G T, for the cohort's uint8 tokens; -100 for ids)."""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
TOKEN_IDS = (8, 5, 6, 7, 9)             # ids of A C G T and anything else, as the Megatron adapter's tokenizer has them
BETA, SMOOTH = 0.1, 0.05
CLIP, KL = (0.2, 0.28), 0.04


def listed():
    return [
        # one short window scored by a single-nucleotide model (vocabulary padded to 16): latency
        {"name": "score-512", "op": "logprobs", "n": 1, "W": 512, "V": 16, "type": "bf16", "tokens": "bases", "shift": 1, "reduce": "window",
         "grad": False, "mask": False},
        # the Megatron adapter's batch: labels already shifted, ids, a float loss mask, the vocabulary padded to 128
        {"name": "score-labels-8k", "op": "logprobs", "n": 32, "W": 8192, "V": 128, "type": "bf16", "tokens": "ids", "shift": 0, "reduce": "token",
         "grad": False, "mask": True},
        # a 6-mer model (4^6 words and 5 specials: odd rows), a user's own loss on the tokens' log-probabilities, with its gradient
        {"name": "logprobs-6mer", "op": "logprobs", "n": 4, "W": 4095, "V": 4101, "type": "bf16", "tokens": "words", "shift": 1, "reduce": "token",
         "grad": True, "mask": False},
        # two pairs of short windows in full precision: a test run's step
        {"name": "preference-512", "op": "preference", "n": 4, "W": 512, "V": 16, "type": "fp32", "tokens": "bases", "shift": 1, "mask": False},
        # eight pairs of 8 kb windows at the padded single-nucleotide vocabulary
        {"name": "preference-8k", "op": "preference", "n": 16, "W": 8192, "V": 128, "type": "bf16", "tokens": "ids", "shift": 1, "mask": True},
        # four pairs under a 7-mer model: a gigabyte of logits
        {"name": "preference-7mer", "op": "preference", "n": 8, "W": 4096, "V": 16384, "type": "bf16", "tokens": "words", "shift": 1, "mask": False},
        # eight short windows, half precision, a vocabulary of nine (rows of 18 bytes)
        {"name": "policy-509", "op": "policy", "n": 8, "W": 509, "V": 9, "type": "fp16", "tokens": "bases", "shift": 1, "mask": False, "kl": True,
         "reduce": "token", "each": False},
        # a batch of 8 kb windows, the first part of each a prompt that the mask leaves out, one advantage a window
        {"name": "policy-8k", "op": "policy", "n": 64, "W": 8192, "V": 128, "type": "bf16", "tokens": "ids", "shift": 1, "mask": True, "kl": True,
         "reduce": "window", "each": False},
        # an 8-mer model (4^8 words and 5 specials), an advantage for each token: two gigabytes of logits
        {"name": "policy-8mer", "op": "policy", "n": 8, "W": 2048, "V": 65541, "type": "bf16", "tokens": "words", "shift": 1, "mask": False, "kl": False,
         "reduce": "token", "each": True},
        # a tiny convolutional model's gradients, clipped into the optimizer's own buffer: latency
        {"name": "clip-tiny", "op": "clip", "layers": 3, "width": 64, "type": "fp32", "into": True, "bound": 0.5},
        # a model of 100 million weights, bf16 gradients with fp32 ones for its norms, clipped into fp32 gradients
        {"name": "clip-into-fp32", "op": "clip", "layers": 24, "width": 592, "type": "bf16", "into": True, "bound": 0.5},
        # a model of a billion weights in place, its norm below the bound (most steps of a run that goes well)
        {"name": "clip-in-place", "op": "clip", "layers": 20, "width": 2048, "type": "bf16", "into": False, "bound": 0.5},
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(("logprobs", "preference", "policy", "clip"))
    t = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if op == "clip":
        return {"op": op, "layers": rng.randint(2, 24), "width": log(48, 1600), "type": t, "into": rng.random() < 0.6, "bound": rng.choice((0.3, 0.9))}
    kind = rng.choice(("bases", "ids", "words"))
    V = log(5, 200) if kind == "bases" else log(13, 1024) if kind == "ids" else log(64, 66000)
    W = log(300, 9000)
    most = 4e8 / (W * V)
    n = max(1, min(256, int(most)))
    n = 2 * max(1, log(1, max(1, n // 2 + 1)) if n > 3 else 1) if op == "preference" else log(1, n)
    if n * W * V > 9e8:
        W = max(1, int(9e8 / (n * V)))
    case = {"op": op, "n": n, "W": W, "V": V, "type": t, "tokens": kind, "shift": rng.choice((0, 1, 1)), "mask": rng.random() < 0.5}
    if op == "logprobs":
        case.update(reduce=rng.choice(("token", "window")), grad=rng.random() < 0.6)
    if op == "policy":
        case.update(kl=rng.random() < 0.6, reduce=rng.choice(("token", "window")), each=rng.random() < 0.5)
    if case.get("reduce") == "window" and op == "logprobs":
        case["grad"] = rng.random() < 0.5
    return case


def shapes(case):
    """the tensors of a model of so many layers: per layer two square matrices, one of four times the width and back, and
    two vectors; an embedding; one odd-sized bias"""
    w = case["width"]
    out = [(w, 16), (w + 1,)]
    for _ in range(case["layers"]):
        out += [(w, w), (w, w), (4 * w, w), (w, 4 * w), (w,), (w,)]
    return out


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    if case["op"] == "clip":
        return prepare_clip(case, g)
    n, W, V, s = case["n"], case["W"], case["V"], case["shift"]
    st = dict(case, kind=case["tokens"])
    if case["tokens"] == "words":
        tokens = torch.randint(0, V, (n, W), generator=g, device=DEV)
        tokens[torch.rand(n, W, generator=g, device=DEV) < 0.01] = -100
    else:
        tokens = torch.randint(0, 4, (n, W), generator=g, device=DEV, dtype=torch.uint8)
        tokens[(torch.rand(n, (W + 31) // 32, generator=g, device=DEV) < 0.02).repeat_interleave(32, 1)[:, :W]] = 4
        if case["tokens"] == "ids":
            tokens = torch.tensor(TOKEN_IDS, device=DEV)[tokens.long()]
    st["tokens"] = tokens
    # a model that has learnt something: the right token is raised at most places
    x = torch.empty(n, W, V, dtype=TYPES[case["type"]], device=DEV)
    for i in range(n):
        r = torch.randn(W, V, generator=g, device=DEV) * 1.5
        up = 4 * torch.rand(W, 1, generator=g, device=DEV)
        y = torch.zeros(W, dtype=torch.int64, device=DEV)
        y[:W - s] = tokens[i, s:].long()
        r.scatter_add_(1, y.clamp(0, V - 1)[:, None], up)
        x[i] = r
    st["logits"] = x.requires_grad_(case.get("grad", True))
    st["weights"] = None
    if case["mask"]:
        keep = torch.arange(W, device=DEV)[None] >= torch.randint(0, W // 3 + 1, (n, 1), generator=g, device=DEV)
        st["weights"] = keep.float() if case["tokens"] == "ids" and s == 0 else keep
    if case["op"] == "logprobs":
        st["upstream"] = torch.randn(n, *([W] if case["reduce"] == "token" else []), generator=g, device=DEV) / (n * W)
        return st
    with torch.no_grad():
        lp = torch.cat([log_probs(x[i:i + 1], tokens[i:i + 1], st["weights"][i:i + 1] if case["mask"] else None, s, ignored(st))[0] for i in range(n)])
    if case["op"] == "preference":
        # the reference model's sums over the windows: near this model's, as early in such a run
        st["ref"] = (lp.double().sum(1) + 8 * torch.randn(n, generator=g, device=DEV)).float()
        return st
    st["old"] = lp + 0.15 * torch.randn(n, W, generator=g, device=DEV)
    st["ref"] = lp + 0.3 * torch.randn(n, W, generator=g, device=DEV) if case["kl"] else None
    st["advantages"] = torch.randn(*([n, W] if case["each"] else [n]), generator=g, device=DEV)
    return st


def prepare_clip(case, g):
    """the gradients as views of one flat buffer a type, one after another, as a trainer's gradient buckets hold them"""
    t = TYPES[case["type"]]
    mats = [s for s in shapes(case) if len(s) > 1]
    vecs = [s for s in shapes(case) if len(s) == 1]
    if t == torch.float32:
        mats, vecs = shapes(case), []
    st = {"op": "clip", "into": case["into"]}
    flat, grads, square = [], [], 0.0
    for these, kind in ((mats, t), (vecs, torch.float32)):
        if these:
            buf = (torch.randn(sum(math.prod(s) for s in these), generator=g, device=DEV) * 1e-3).to(kind)
            flat.append(buf)
            square += float(buf.double().square().sum())
            grads += [v.view(s) for v, s in zip(buf.split([math.prod(s) for s in these]), these)]
    # in place the norm is below the bound, so that a pass leaves what it found and can be taken again
    st["flat"], st["grads"], st["max_norm"] = flat, grads, (case["bound"] if case["into"] else 1 + case["bound"]) * math.sqrt(square)
    st["out_flat"] = [torch.empty(b.numel(), device=DEV) for b in flat] if case["into"] else None
    st["out"] = None
    if case["into"]:
        st["out"] = [v.view(s) for b, these in zip(st["out_flat"], (mats, vecs)) for v, s in zip(b.split([math.prod(s) for s in these]), these)]
    return st


def ignored(case):
    return 4 if case["kind"] == "bases" else -100


def counted(tokens, weights, V, shift, ignore):
    W = tokens.shape[1]
    y = tokens[:, shift:].long()
    c = (y >= 0) & (y < V) & (y != ignore)
    if weights is not None:
        c = c & (weights[:, shift:] != 0)
    pad = torch.zeros(tokens.shape[0], W - c.shape[1], dtype=torch.int64, device=y.device)
    return torch.cat([y.clamp(0, V - 1), pad], 1), torch.cat([c, pad.bool()], 1)


def log_probs(logits, tokens, weights, shift, ignore):
    """(log-probabilities [n, W], 0 where not counted; probabilities [n, W, V]; targets; which are counted)"""
    y, c = counted(tokens, weights, logits.shape[2], shift, ignore)
    x = logits.float()
    m = x.amax(2, keepdim=True)
    x = x - m
    e = torch.exp(x)
    z = e.sum(2)
    lp = x.gather(2, y[..., None])[..., 0] - torch.log(z)
    return torch.where(c, lp, torch.zeros_like(lp)), e.div_(z[..., None]), y, c


def grad_of(p, y, c, g, kind):
    """g (one value a position) times (one at the target minus the probabilities), none where not counted; p is used up"""
    g = torch.where(c, g, torch.zeros_like(g)).float()
    p.scatter_add_(2, y[..., None], torch.full_like(g, -1.0)[..., None])
    return p.mul_(-g[..., None]).to(kind)


def run(st):
    return run_own(st) if own else run_plain(st)


def run_plain(st):
    if st["op"] == "clip":
        # over the flat buffers that the gradients are views of: one per type
        norm = torch.sqrt(sum(b.float().square().sum(dtype=torch.float64) for b in st["flat"])).float()
        scale = (st["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
        for b, o in zip(st["flat"], st["out_flat"] or st["flat"]):
            o.copy_(b.float() * scale)
        return [norm] + (st["out_flat"] or st["flat"])
    with torch.no_grad():
        lp, p, y, c = log_probs(st["logits"], st["tokens"], st["weights"], st["shift"], ignored(st))
        kind = st["logits"].dtype
        if st["op"] == "logprobs":
            out = lp if st["reduce"] == "token" else lp.double().sum(1).float()
            if not st["grad"]:
                return [out]
            g = st["upstream"] if st["reduce"] == "token" else st["upstream"][:, None].expand_as(lp)
            return [out, grad_of(p, y, c, g, kind)]
        if st["op"] == "preference":
            d = lp.double().sum(1) - st["ref"].double()
            m = st["n"] // 2
            h = BETA * (d[:m] - d[m:])
            loss = ((1 - SMOOTH) * torch.log1p(torch.exp(-h)) + SMOOTH * torch.log1p(torch.exp(h))).mean()
            k = BETA / m * (SMOOTH - 1 / (1 + torch.exp(h)))          # the loss by each chosen window's sum
            g = torch.cat([k, -k])[:, None].expand_as(lp)
            return [loss.float(), grad_of(p, y, c, g, kind)]
        a = st["advantages"] if st["each"] else st["advantages"][:, None].expand_as(lp)
        r = torch.exp(lp - st["old"])
        one, two = r * a, r.clamp(1 - CLIP[0], 1 + CLIP[1]) * a
        each = -torch.minimum(one, two)
        g = torch.where(one <= two, -one, torch.zeros_like(one))
        if st["ref"] is not None:
            d = (st["ref"] - lp).double()
            each = each + KL * (torch.expm1(d) - d).float()
            g = g - KL * torch.expm1(d).float()
        each = torch.where(c, each, torch.zeros_like(each))
        if st["reduce"] == "token":
            w = 1.0 / c.sum().clamp(min=1).double()
        else:
            k = c.sum(1, keepdim=True)
            w = 1.0 / (k.clamp(min=1) * (k > 0).sum().clamp(min=1)).double()
        loss = (each.double() * w).sum().float()
        return [loss, grad_of(p, y, c, g * w.float(), kind)]


def run_own(st):
    import panvram_b200 as P
    if st["op"] == "clip":
        norm = P.clip_grads(st["grads"], st["max_norm"], out=st["out"])
        return [norm] + (st["out_flat"] if st["into"] else st["flat"])
    x, tokens, kw = st["logits"], st["tokens"], {"mask": st["weights"], "shift": st["shift"]}
    if st["op"] == "logprobs":
        out = P.window_logprobs(x, tokens, reduce=st["reduce"], **kw)
        if not st["grad"]:
            return [out]
        return [out.detach(), torch.autograd.grad(out, x, st["upstream"])[0]]
    if st["op"] == "preference":
        loss = P.preference_loss(x, tokens, st["ref"], beta=BETA, label_smoothing=SMOOTH, **kw)
    else:
        loss = P.policy_loss(x, tokens, st["old"], st["advantages"], ref_logp=st["ref"], clip=CLIP, kl=KL if st["kl"] else 0.0, reduce=st["reduce"], **kw)
    return [loss.detach(), torch.autograd.grad(loss, x)[0]]


def work(case):
    if case["op"] == "clip":
        k = sum(math.prod(s) for s in shapes(case))
        vec = 0 if case["type"] == "fp32" else sum(math.prod(s) for s in shapes(case) if len(s) == 1)
        read = (k - vec) * SIZE[case["type"]] + vec * 4
        return {"bytes": read + (4 * k if case["into"] else 0), "flops": 3 * k if case["into"] else 2 * k}
    n, W, V = case["n"], case["W"], case["V"]
    rows = n * W
    grad = case.get("grad", True)
    small = rows * (1 if case["tokens"] == "bases" else 8)
    if case["mask"]:
        small += rows * (4 if case["tokens"] == "ids" and case["shift"] == 0 else 1)
    if case["op"] == "logprobs":
        small += (4 * rows if case["reduce"] == "token" else 4 * n) * (2 if grad else 1)
    elif case["op"] == "preference":
        small += 4 * n
    else:
        small += rows * (4 + (4 if case["kl"] else 0) + (4 if case["each"] else 0))
    big = rows * V * SIZE[case["type"]]
    return {"bytes": small + big * (2 if grad else 1), "flops": rows * V * (6 if grad else 4)}


def exact(case, seed):
    """from the definitions, in 64 bits: the log-softmax and its derivative window by window, the losses' derivatives by
    autograd over the log-probabilities"""
    st = prepare(case, seed)
    if case["op"] == "clip":
        norm = math.sqrt(sum(float((b.to(torch.float64) ** 2).sum()) for b in st["flat"]))
        f = min(1.0, st["max_norm"] / (norm + 1e-6))
        return [torch.tensor(norm, dtype=torch.float64)] + [b.to(torch.float64) * f for b in st["flat"]]
    x, tok, s, V = st["logits"].detach(), st["tokens"], st["shift"], case["V"]
    n, W, _ = x.shape
    aim = torch.full((n, W), -1, dtype=torch.int64, device=x.device)
    if W > s:
        aim[:, :W - s] = tok[:, s:].to(torch.int64)
    ok = (aim >= 0) & (aim < V) & (aim != ignored(st))
    if st["weights"] is not None:
        seen = torch.zeros_like(ok)
        seen[:, :W - s] = st["weights"][:, s:] > 0
        ok &= seen
    at = aim.clamp(0, V - 1).unsqueeze(2)
    lp = torch.zeros(n, W, dtype=torch.float64, device=x.device)
    for i in range(n):
        lp[i] = torch.log_softmax(x[i].to(torch.float64), 1).gather(1, at[i])[:, 0]
    lp = lp.masked_fill(~ok, 0.0).requires_grad_(True)
    if case["op"] == "logprobs":
        value = lp if case["reduce"] == "token" else lp.sum(1)
        if not case["grad"]:
            return [value.detach()]
        up = torch.autograd.grad(value, lp, st["upstream"].to(torch.float64))[0]
    elif case["op"] == "preference":
        gap = lp.sum(1) - st["ref"].to(torch.float64)
        h = BETA * (gap[:n // 2] - gap[n // 2:])
        value = -((1 - SMOOTH) * torch.nn.functional.logsigmoid(h) + SMOOTH * torch.nn.functional.logsigmoid(-h)).mean()
        up = torch.autograd.grad(value, lp)[0]
    else:
        adv = st["advantages"].to(torch.float64)
        adv = adv if case["each"] else adv[:, None]
        ratio = (lp - st["old"].to(torch.float64)).exp()
        term = -torch.min(ratio * adv, ratio.clamp(1 - CLIP[0], 1 + CLIP[1]) * adv)
        if st["ref"] is not None:
            d = st["ref"].to(torch.float64) - lp
            term = term + KL * (d.expm1() - d)
        term = term.masked_fill(~ok, 0.0)
        if case["reduce"] == "token":
            value = term.sum() / max(1, int(ok.sum()))
        else:
            k = ok.sum(1)
            value = (term.sum(1) / k.clamp(min=1)).sum() / max(1, int((k > 0).sum()))
        up = torch.autograd.grad(value, lp)[0]
    up = up.masked_fill(~ok, 0.0)
    d = torch.empty(n, W, V, dtype=torch.float64, device=x.device)
    for i in range(n):
        p = torch.softmax(x[i].to(torch.float64), 1)
        d[i] = -up[i][:, None] * p
        d[i].scatter_add_(1, at[i], up[i][:, None])
    return [value.detach(), d]
