"""Log-probabilities of windows' tokens, the preference loss and the clipped policy loss against plain 64-bit forms.

Tolerances, per row of V logits (eps32 = 2^-24, half a step of float relative to the value):
  * the sum of the numerators adds at most V positive terms one after another and a few partial sums: (V + 8) eps32
    relative at the very worst, and the approximate 2^x adds 2^-22 = 4 eps32, the rounding of its argument |x - max| eps32
    (counted with the term's weight, below 1): S = (V + 16) eps32. V is replaced by the longest run of additions that one
    thread makes, at most V / 32 + 64 (rows of any length are spread over 32 threads or more, those up to 64 words may
    be one thread's).
  * log p: S absolute, and the rounding of the logarithm and of the target's argument, 4 eps32 |log p|.
  * p and 1 - p: S + 4 eps32 + eps32 * |x - max| relative, at most 100 |x - max| here.
  * a gradient: g times that, one rounding to the logits' type (finfo.eps / 2 relative; half the smallest subnormal).
"""
import itertools
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

E32 = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
IDS = (8, 5, 6, 7, 9)


@pytest.fixture(scope="module")
def P(cuda):
    import panvram_b200 as P
    return P


def run_of(V):
    return (min(V, V / 32 + 64) + 16) * E32


def tol_lp(V, lp):
    return run_of(V) + 4 * E32 * lp.abs()


def make(cuda, n, W, V, kind, tokens="bases", mask=None, shift=1, seed=0, pad=0, spread=2.0):
    """logits (with `pad` words behind each position's that belong to nobody), tokens, mask"""
    g = torch.Generator(device=cuda).manual_seed(seed * 7919 + n * 31 + W * 17 + V)
    x = (torch.randn(n, W, V + pad, generator=g, device=cuda) * spread).to(TYPES[kind])[..., :V]
    if tokens == "bases":
        t = torch.randint(0, 6, (n, W), generator=g, device=cuda).to(torch.uint8)       # 4: ignored, 5: a word where V > 5
    else:
        t = torch.randint(0, V, (n, W), generator=g, device=cuda)
        t[torch.rand(n, W, generator=g, device=cuda) < 0.1] = -100
        t[torch.rand(n, W, generator=g, device=cuda) < 0.05] = V                        # outside the vocabulary
    m = None
    if mask:
        m = (torch.rand(n, W, generator=g, device=cuda) < 0.7).to({"bool": torch.bool, "uint8": torch.uint8, "float": torch.float32}[mask])
    return x, t, m


def targets(t, m, V, shift, ignore=None):
    """(target, counted) [n, W]"""
    n, W = t.shape
    ignore = ignore if ignore is not None else 4 if t.dtype == torch.uint8 else -100
    y = torch.full((n, W), -1, dtype=torch.int64, device=t.device)
    if shift < W:
        y[:, :W - shift] = t[:, shift:].long()
    ok = (y >= 0) & (y < V) & (y != ignore)
    if m is not None and shift < W:
        ok[:, :W - shift] &= m[:, shift:] != 0
    return y.clamp(0, V - 1), ok


def oracle(x, t, m, shift, ignore=None):
    """log-probabilities in 64 bits [n, W] (a leaf), softmax, targets, counted"""
    y, ok = targets(t, m, x.shape[2], shift, ignore)
    p = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    lp = torch.zeros(t.shape, dtype=torch.float64, device=x.device)
    for i in range(x.shape[0]):                                       # rows that are not counted may hold anything
        z = torch.where(ok[i][:, None], x[i].double(), 0.0)
        l = torch.log_softmax(z, 1)
        p[i] = l.exp()
        lp[i] = torch.where(ok[i], l.gather(1, y[i][:, None])[:, 0], 0.0)
    return lp.requires_grad_(True), p, y, ok


def grad_of(x, p, y, ok, g, err=0.0):
    """g (onehot - p), and its tolerance where each g is off by at most `err` relative (or absolute per row)"""
    g = torch.where(ok, g, 0.0)
    # 1 - p of the target as the sum of the others, which keeps its digits where the model is sure
    others = p.scatter(2, y[..., None], 0.0).sum(2, keepdim=True)
    d = (-p).scatter(2, y[..., None], others)
    want = d * g[..., None]
    V = x.shape[2]
    step = torch.finfo(x.dtype).eps / 2
    rel = run_of(V) + 100 * E32
    tol = want.abs() * (rel + step * 1.01) + torch.as_tensor(err, device=x.device).expand_as(g)[..., None] * d.abs()
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -126}[x.dtype]
    return want, tol + tiny * 1.01


def close(got, want, tol, what=""):
    bad = (got.double() - want).abs() > tol
    bad |= got.isnan() != want.isnan()
    assert not bad.any(), (what, int(bad.sum()), float(((got.detach().double() - want).abs() / tol).max()))


SHAPES = [(1, 1, 1, 0), (1, 1, 5, 1), (1, 2, 5, 1), (3, 7, 5, 1), (2, 33, 9, 1), (5, 64, 16, 0), (2, 130, 31, 1), (2, 65, 32, 3), (2, 40, 33, 1),
          (3, 37, 64, 1), (2, 50, 65, 0), (4, 100, 128, 1), (2, 17, 129, 1), (2, 33, 255, 1), (2, 20, 512, 1), (2, 19, 1000, 1), (2, 11, 1024, 0),
          (2, 9, 1025, 1), (2, 9, 2048, 1), (3, 5, 2049, 0), (2, 5, 4101, 1), (1, 4, 8192, 1), (2, 3, 16384, 1), (1, 3, 16391, 1), (1, 3, 33000, 0),
          (1, 3, 65541, 1), (1, 2, 70001, 1), (1, 3, 140007, 1), (2, 5, 7, 9),
          (2, 40, 96, 1), (2, 35, 192, 1), (2, 21, 282, 1), (2, 19, 384, 0), (2, 19, 577, 1), (2, 17, 768, 1), (2, 9, 1500, 0), (2, 9, 1536, 1),
          (2, 75, 21, 1), (3, 41, 45, 1), (2, 37, 85, 0), (2, 35, 171, 1)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n, W, V, shift", SHAPES)
def test_logprobs(P, cuda, n, W, V, shift, kind):
    for tokens, mask in (("ids", "bool"), ("bases", None), ("ids", "float")):
        x, t, m = make(cuda, n, W, V, kind, tokens, mask, shift)
        lp, p, y, ok = oracle(x, t, m, shift)
        x.requires_grad_(True)
        got = P.window_logprobs(x, t, m, shift)
        close(got, lp.detach(), tol_lp(V, lp.detach()), "token")
        assert (got[~ok] == 0).all()
        up = torch.randn(n, W, device=cuda, generator=torch.Generator(device=cuda).manual_seed(3))
        (d,) = torch.autograd.grad(got, x, up)
        assert d.dtype == x.dtype and d.shape == x.shape
        close(d, *grad_of(x, p, y, ok, up.double()), "gradient")
        assert (d[~ok] == 0).all()
        s = P.window_logprobs(x, t, m, shift, reduce="window")
        want = lp.detach().sum(1)
        close(s, want, tol_lp(V, lp.detach()).sum(1) + E32 * want.abs(), "window")
        (d,) = torch.autograd.grad(s, x, up[:, 0])
        close(d, *grad_of(x, p, y, ok, up[:, :1].double().expand(n, W)), "window's gradient")
        with torch.no_grad():
            assert torch.equal(P.window_logprobs(x, t, m, shift), got)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("V, pad", [(5, 1), (5, 3), (16, 8), (16, 16), (100, 28), (125, 3), (128, 1), (4101, 3), (5000, 120), (65541, 1)])
def test_strides(P, cuda, V, pad, kind):
    """rows of a padded vocabulary, rows out of order, windows and positions exchanged, tokens and masks with strides"""
    n, W = 3, 21
    x, t, m = make(cuda, n, W, V, kind, "ids", "uint8", pad=pad)
    forms = [(x, t, m),
             (x[:, 1:], t[:, :-1], m[:, 1:]),
             (x.transpose(0, 1).contiguous().transpose(0, 1), t.t().contiguous().t(), m.t().contiguous().t()),
             (x[::2], t[::2], m[::2]), (x[:, ::3], t[:, ::3], m[:, ::3]),
             (x[:1].expand(n, W, V), t, m)]
    for k, (a, b, c) in enumerate(forms):
        lp, p, y, ok = oracle(a, b, c, 1)
        a = a.detach().requires_grad_(True)
        got = P.window_logprobs(a, b, c)
        close(got, lp.detach(), tol_lp(V, lp.detach()), k)
        up = torch.randn(b.shape[1], b.shape[0], device=cuda).t()               # an upstream gradient with strides
        (d,) = torch.autograd.grad(got, a, up)
        close(d, *grad_of(a, p, y, ok, up.double()), k)
        (d,) = torch.autograd.grad(P.window_logprobs(a, b, c).sum(), a)         # an expanded one
        close(d, *grad_of(a, p, y, ok, torch.ones_like(up).double()), k)


@pytest.mark.parametrize("off", [1, 2, 3, 5, 7])
@pytest.mark.parametrize("V", [5, 16, 128, 257, 4096, 20000])
def test_unaligned_base_leaves_neighbours_alone(P, cuda, V, off):
    """logits that start anywhere in a buffer whose other values are NaN; the gradient written by the C entry point into
    a buffer of its own, whose other values stay"""
    import ctypes
    from panvram_b200 import _C
    for kind in TYPES:
        n, W = 2, 9
        x, t, _ = make(cuda, n, W, V, kind, "ids")
        buf = torch.full((n * W * V + 64,), math.nan, dtype=x.dtype, device=cuda)
        a = buf[off:off + n * W * V].view(n, W, V)
        a.copy_(x)
        lp, p, y, ok = oracle(x, t, None, 1)
        close(P.window_logprobs(a, t), lp.detach(), tol_lp(V, lp.detach()))
        up = torch.randn(n, W, device=cuda)
        for goff in (off, 0, 4):
            gbuf = torch.full((n * W * V + 64,), 7.0, dtype=x.dtype, device=cuda)
            d = gbuf[goff:goff + n * W * V].view(n, W, V)
            st = torch.cuda.current_stream().cuda_stream
            b = _C.Scored(a.data_ptr(), None, t.data_ptr(), None, n, W, V, *a.stride()[:2], 0, 0, *t.stride(), 0, 0, -100, 1,
                          list(TYPES).index(kind), 8, 0)
            stat = torch.empty(_C._lib.pv_score_stat_bytes(ctypes.byref(b)), dtype=torch.uint8, device=cuda)
            logp = torch.empty(n, W, device=cuda)
            assert _C._lib.pv_logprobs(ctypes.byref(b), logp.data_ptr(), None, stat.data_ptr() or None, None, 0, st) == 0
            b.grad, b.grad_n, b.grad_w = d.data_ptr(), d.stride(0), d.stride(1)
            assert _C._lib.pv_logprobs_grad(ctypes.byref(b), up.data_ptr(), W, 1, stat.data_ptr() or None, None, st) == 0
            close(d, *grad_of(x, p, y, ok, up.double()))
            assert (gbuf[:goff] == 7).all() and (gbuf[goff + n * W * V:] == 7).all()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("V", [5, 16, 40, 128, 1000, 4101, 17000, 70000])
def test_values(P, cuda, V, kind):
    """what must not be read (NaN, infinities at positions that are not counted), -inf and the lowest value among the
    logits, sure and hopeless targets, a row of nothing but -inf"""
    n, W = 2, 12
    x, t, m = make(cuda, n, W, V, kind, "ids", "bool", shift=0)
    t = t.clamp(0, V - 1)
    m[:] = True
    low = torch.finfo(x.dtype).min
    m[0, 0] = m[0, 3] = False
    x[0, 0] = math.nan
    x[0, 3] = math.inf
    t[1, 0] = -100
    x[1, 0, ::2] = math.nan
    x[0, 1, 0] = -math.inf
    x[0, 2, : V // 2 + 1] = low
    t[0, 1] = 0                                            # a target that cannot be
    t[0, 2] = V - 1
    x[0, 4, V - 1], t[0, 4] = 60.0, V - 1                  # sure
    x[0, 5, V - 1], t[0, 5] = 60.0, 0                      # hopeless
    x[0, 6] = low                                          # all alike
    x[0, 7] = torch.finfo(x.dtype).max
    x[0, 8] = 30000.0                                      # far from 0, alike but for one
    x[0, 8, 0], t[0, 8] = 30016.0, V - 1
    lp, p, y, ok = oracle(x, t, m, 0)
    x.requires_grad_(True)
    got = P.window_logprobs(x, t, m, 0)
    assert got[0, 1] == -math.inf
    fin = lp.detach().isfinite()
    assert int((~fin).sum()) == 1
    close(got.detach()[fin], lp.detach()[fin], tol_lp(V, lp.detach()[fin]))
    up = torch.ones(n, W, device=cuda)
    (d,) = torch.autograd.grad(got, x, up)
    close(d, *grad_of(x, p, y, ok, up.double()))
    assert (d[0, 0] == 0).all() and (d[0, 3] == 0).all() and (d[1, 0] == 0).all()
    # sure: 1 - p is about V e^-60, far below the rounding of p itself
    sure = d[0, 4, V - 1].double()
    assert 0 < sure < V * math.exp(-50) or kind == "fp16"
    with torch.no_grad():                                  # NaN where there is nothing to normalise by, and where a counted row holds NaN
        z = x.clone()
        z[0, 4] = -math.inf
        z[0, 5, 1] = math.nan
        z[0, 6, 2] = math.inf
        got2 = P.window_logprobs(z, t, m, 0)
        assert got2[0, 4:7].isnan().all()
        keep = torch.ones(n, W, dtype=torch.bool, device=cuda)
        keep[0, 4:7] = False
        assert torch.equal(got2[keep], got.detach()[keep])


def test_ignore_and_uint8_words(P, cuda):
    x, t, _ = make(cuda, 3, 40, 6, "fp32")
    for ignore in (None, -1, 0, 5, 77):
        lp, _, _, ok = oracle(x, t, None, 1, ignore)
        close(P.window_logprobs(x, t, ignore=ignore), lp.detach(), tol_lp(6, lp.detach()))
    assert (t == 4).any() and (t == 5).any()


def pref_oracle(x, t, m, ref, beta, eps, shift=1):
    lp, p, y, ok = oracle(x, t, m, shift)
    n = x.shape[0]
    gap = lp.sum(1) - ref.double()
    margin = gap[:n // 2] - gap[n // 2:]
    h = beta * margin
    loss = -((1 - eps) * torch.nn.functional.logsigmoid(h) + eps * torch.nn.functional.logsigmoid(-h)).mean()
    (g,) = torch.autograd.grad(loss, lp)
    err = tol_lp(x.shape[2], lp.detach()).sum(1)
    return loss.detach(), margin.detach(), g, p, y, ok, float(err[:n // 2].max() + err[n // 2:].max())


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n, W, V", [(2, 1, 5), (2, 40, 5), (4, 100, 16), (6, 257, 33), (2, 300, 128), (10, 33, 128), (4, 20, 1000), (2, 30, 4101), (2, 4, 20000),
                                     (2, 3, 70001), (600, 3, 8)])
def test_preference(P, cuda, n, W, V, kind):
    for beta, eps, mask in ((0.1, 0.0, None), (0.5, 0.1, "bool"), (0.0, 0.0, None)):
        x, t, m = make(cuda, n, W, V, kind, "ids", mask, seed=5)
        lp, _, _, _ = oracle(x, t, m, 1)
        ref = (lp.detach().sum(1) + torch.randn(n, device=cuda).double() * 3).float()
        loss, margin, g, p, y, ok, err = pref_oracle(x, t, m, ref, beta, eps)
        x.requires_grad_(True)
        got, got_margin = P.preference_loss(x, t, ref, beta, eps, m, return_margins=True)
        assert got.shape == () and got.dtype == torch.float32 and not got_margin.requires_grad
        close(got_margin, margin, err + E32 * margin.abs(), "margin")
        close(got, loss, beta * err + 2 * E32 * loss.abs() + 1e-12, "loss")
        # d coef / d margin <= beta^2 / (4 pairs)
        g_err = beta * beta / (2 * n) * err + 2 * E32 * g.abs()
        (d,) = torch.autograd.grad(got, x, retain_graph=True)
        close(d, *grad_of(x, p, y, ok, g, g_err), "gradient")
        (d3,) = torch.autograd.grad(got, x, torch.tensor(3.0, device=cuda), retain_graph=True)      # a loss scale, after a pass without one
        close(d3, *grad_of(x, p, y, ok, 3 * g, 3 * g_err), "scaled")
        (again,) = torch.autograd.grad(got, x)
        assert torch.equal(again, d)
        with torch.no_grad():
            assert torch.equal(P.preference_loss(x, t, ref, beta, eps, m), got)


def policy_oracle(x, t, m, old, adv, ref, clip, kl, reduce, shift):
    lp, p, y, ok = oracle(x, t, m, shift)
    a = adv.double() if adv.dim() == 2 else adv.double()[:, None].expand_as(lp)
    r = (lp - old.double()).exp()
    edge = torch.minimum((r - (1 - clip[0])).abs(), (r - (1 + clip[1])).abs())
    assert (edge[ok] > 1e-3).all()                          # nothing so near a bound that rounding decides its gradient
    each = -torch.min(r * a, r.clamp(1 - clip[0], 1 + clip[1]) * a)
    if ref is not None:
        d = ref.double() - lp
        each = each + kl * (d.expm1() - d)
    each = torch.where(ok, each, 0.0)
    k = ok.sum(1)
    if reduce == "token":
        w = torch.full_like(lp, 1.0 / max(1, int(ok.sum())))
    else:
        w = (1.0 / (k.clamp(min=1) * max(1, int((k > 0).sum()))))[:, None].expand_as(lp).double()
    loss = (each * w).sum()
    (g,) = torch.autograd.grad(loss, lp)
    g = torch.where(ok, g, 0.0)
    l = lp.detach()
    el = tol_lp(x.shape[2], l) + E32 * (l.abs() + old.abs()) + (E32 * ref.abs() if ref is not None else 0)
    mag = (r * a).detach().abs() * 4 + (kl * 4 * (d.detach().abs() + d.detach().exp()) if ref is not None else 0)
    term_err = torch.where(ok, (el + 4 * E32) * mag * w.abs(), 0.0)
    return loss.detach(), g, p, y, ok, term_err.sum(), term_err


def policy_inputs(lp, clip, cuda, seed, far=False):
    """old log-probabilities whose ratios are not within a thousandth of the bounds, reference ones, advantages"""
    gen = torch.Generator(device=cuda).manual_seed(seed)
    n, W = lp.shape
    choices = torch.tensor([0.0, 0.05, -0.05, 0.11, -0.12, 0.31, -0.4, 0.6, -0.7], device=cuda, dtype=torch.float64)
    delta = choices[torch.randint(0, len(choices), (n, W), generator=gen, device=cuda)]
    old = (lp.detach() - delta).float()
    ref = (lp.detach() + torch.randn(n, W, generator=gen, device=cuda) * (0.01 if not far else 1.0)).float()
    adv = torch.randn(n, W, generator=gen, device=cuda)
    adv[torch.rand(n, W, generator=gen, device=cuda) < 0.1] = 0
    return old, ref, adv


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n, W, V, shift", [(1, 1, 5, 1), (1, 2, 5, 1), (3, 50, 5, 1), (8, 61, 9, 1), (4, 100, 16, 0), (3, 300, 33, 1), (3, 200, 128, 1), (2, 77, 130, 1),
                                            (2, 30, 1000, 1), (3, 12, 4101, 1), (2, 5, 20000, 0), (1, 4, 65541, 1), (1, 3, 90000, 1), (700, 4, 8, 1)])
def test_policy(P, cuda, n, W, V, shift, kind):
    clip = (0.2, 0.28)
    for reduce, kl, each, mask in (("token", 0.0, False, None), ("window", 0.04, True, "bool"), ("token", 0.5, True, "uint8")):
        x, t, m = make(cuda, n, W, V, kind, "ids", mask, shift, seed=11)
        if m is not None:
            m[-1] = 0                                       # a window with nothing to count
        lp, _, _, _ = oracle(x, t, m, shift)
        old, ref, adv = policy_inputs(lp, clip, cuda, V, far=kl == 0.5)
        adv = adv if each else adv[:, 0]
        ref = ref if kl else None
        loss, g, p, y, ok, l_err, g_err = policy_oracle(x, t, m, old, adv, ref, clip, kl, reduce, shift)
        x.requires_grad_(True)
        got = P.policy_loss(x, t, old, adv, ref, clip, kl, m, shift, reduce=reduce)
        assert got.shape == () and got.dtype == torch.float32
        close(got, loss, l_err + 2 * E32 * loss.abs() + 1e-12, "loss")
        (d,) = torch.autograd.grad(got, x, retain_graph=True)
        close(d, *grad_of(x, p, y, ok, g, g_err), "gradient")
        assert (d[~ok] == 0).all()
        (d2,) = torch.autograd.grad(got, x, torch.tensor(-2.5, device=cuda), retain_graph=True)
        close(d2, *grad_of(x, p, y, ok, -2.5 * g, 2.5 * g_err), "scaled")
        (again,) = torch.autograd.grad(got, x)
        assert torch.equal(again, d)
        half = P.policy_loss(x, t, old, adv, ref, clip, kl, m, shift, reduce=reduce, scale=0.5)           # exact in every step
        assert torch.equal(half, 0.5 * got) and (kind == "fp16" or torch.equal(torch.autograd.grad(half, x)[0], 0.5 * d))
        with torch.no_grad():                                # without a gradient rows may be split otherwise: another order of the same sums
            close(P.policy_loss(x, t, old, adv, ref, clip, kl, m, shift, reduce=reduce), loss, l_err + 2 * E32 * loss.abs() + 1e-12, "no gradient")


def test_policy_does_not_read_what_is_not_counted(P, cuda):
    n, W, V = 3, 40, 16
    x, t, m = make(cuda, n, W, V, "fp32", "ids", "bool", seed=2)
    lp, _, _, ok = oracle(x, t, m, 1)
    old, ref, adv = policy_inputs(lp, (0.2, 0.2), cuda, 1)
    a = P.policy_loss(x.requires_grad_(True), t, old, adv, ref, 0.2, 0.1, m)
    (da,) = torch.autograd.grad(a, x)
    z = x.detach().clone()
    for q in (z, old, ref, adv):
        q[~ok] = math.nan
    z[~ok] = -math.inf
    b = P.policy_loss(z.requires_grad_(True), t, old, adv, ref, 0.2, 0.1, m)
    (db,) = torch.autograd.grad(b, z)
    assert torch.equal(a, b) and torch.equal(da, db)


def test_policy_extremes(P, cuda):
    """a ratio that overflows with an advantage of 0 or one that clips it; nothing counted at all"""
    x, t, _ = make(cuda, 2, 4, 16, "fp32", "ids", shift=0)
    t = t.clamp(0, 15)
    old = torch.full((2, 4), -300.0, device=cuda)
    for adv, want in ((torch.zeros(2, device=cuda), 0.0), (torch.ones(2, device=cuda), -1.2)):
        got = P.policy_loss(x.requires_grad_(True), t, old, adv, shift=0)
        assert abs(float(got) - want) < 4 * E32 * 1.2
        assert (torch.autograd.grad(got, x)[0] == 0).all()
    none = torch.zeros(2, 4, dtype=torch.bool, device=cuda)
    for reduce in ("token", "window"):
        got = P.policy_loss(x, t, old, adv, mask=none, reduce=reduce)
        assert float(got) == 0 and (torch.autograd.grad(got, x)[0] == 0).all()
    assert float(P.preference_loss(x, t, torch.zeros(2, device=cuda), mask=none)) == pytest.approx(math.log(2), abs=2 * E32)


@pytest.mark.parametrize("n, W", [(0, 5), (2, 0), (0, 0)])
def test_empty(P, cuda, n, W):
    x = torch.zeros(n, W, 7, device=cuda, requires_grad=True)
    t = torch.zeros(n, W, dtype=torch.uint8, device=cuda)
    f, s = torch.zeros(n, W, device=cuda), torch.zeros(n, device=cuda)
    for out in (P.window_logprobs(x, t), P.window_logprobs(x, t, reduce="window"), P.policy_loss(x, t, f, s, f, kl=0.1), P.preference_loss(x, t, s)):
        assert torch.isfinite(out).all()
        (d,) = torch.autograd.grad(out, x, torch.ones_like(out))
        assert d.shape == x.shape
    assert P.window_logprobs(x, t, reduce="window").tolist() == [0.0] * n


def test_offsets_beyond_32_bits(P, cuda):
    """windows and positions that lie more than 2^32 elements apart"""
    for V, far_w in ((40, False), (41, True), (3000, False), (70001, False)):
        n, W = 2, 3
        buf = torch.empty(2 * 2_200_000_001 + 3 * V, dtype=torch.bfloat16, device=cuda)
        sn, sw = (2 * 2_200_000_001, V) if not far_w else (V, 2_200_000_001)
        x = buf.as_strided((n, W, V), (sn, sw, 1))
        x.copy_(torch.randn(n, W, V, device=cuda))
        t = torch.randint(0, V, (n, W), device=cuda)
        lp, p, y, ok = oracle(x, t, None, 0)
        a = x.detach().requires_grad_(True)
        got = P.window_logprobs(a, t, shift=0)
        close(got, lp.detach(), tol_lp(V, lp.detach()))
        close(torch.autograd.grad(got.sum(), a)[0], *grad_of(x, p, y, ok, torch.ones(n, W, device=cuda).double()))
        old, adv = lp.detach().float() + 0.01, torch.ones(n, device=cuda)
        d = torch.autograd.grad(P.policy_loss(a, t, old, adv, shift=0), a)[0]
        r = (lp.detach() - old.double()).exp()
        el = tol_lp(V, lp.detach()) + E32 * 2 * old.abs()
        close(d, *grad_of(x, p, y, ok, -r / 6, r / 6 * (el + 4 * E32)))


@pytest.mark.parametrize("n, W, V", [(20, 8000, 2057), (2, 4000, 40001), (3, 1 << 19, 5), (40, 8192, 24)])
def test_more_rows_than_the_blocks_look_up_at_once(P, cuda, n, W, V):
    """every row of a batch that keeps each block busy for many rows, a stretch of them not counted"""
    x, t, m = make(cuda, n, W, V, "bf16", "ids", "bool", seed=1)
    m[1, W // 3:2 * W // 3] = False
    up = torch.randn(n, W, device=cuda, generator=torch.Generator(device=cuda).manual_seed(2))
    a = x.requires_grad_(True)
    got = P.window_logprobs(a, t, m)
    (d,) = torch.autograd.grad(got, a, up)
    x = x.detach()
    old = torch.empty_like(up)
    lps = []
    for i in range(n):
        lp, p, y, ok = oracle(x[i:i + 1], t[i:i + 1], m[i:i + 1], 1)
        close(got[i:i + 1], lp.detach(), tol_lp(V, lp.detach()), i)
        close(d[i:i + 1], *grad_of(x[i:i + 1], p, y, ok, up[i:i + 1].double()), i)
        old[i] = lp.detach()[0].float() + 0.01
        lps.append((lp.detach(), ok))
    del d
    count = sum(int(ok.sum()) for _, ok in lps)
    loss = P.policy_loss(a, t, old, up[:, 0], mask=m)
    (d,) = torch.autograd.grad(loss, a)
    total, err = 0.0, 0.0
    for i in range(n):
        lp, ok = lps[i]
        _, p, y, _ = oracle(x[i:i + 1], t[i:i + 1], m[i:i + 1], 1)
        r = torch.where(ok, (lp - old[i:i + 1].double()).exp() * up[i, 0].double(), 0.0)
        el = tol_lp(V, lp) + 2 * E32 * old[i:i + 1].abs()
        close(d[i:i + 1], *grad_of(x[i:i + 1], p, y, ok, -r / count, r.abs() / count * (el + 4 * E32)), i)
        total -= float(r.sum())
        err += float((r.abs() * (el + 4 * E32)).sum())
    assert abs(float(loss) - total / count) <= err / count + 2 * E32 * abs(total / count)


def test_shapes_at_random(P, cuda):
    import random
    rng = random.Random(7)
    for _ in range(60):
        V = int(round(math.exp(rng.uniform(0, math.log(40000)))))
        W = rng.randint(1, max(2, min(400, 600000 // V)))
        n = 2 * rng.randint(1, 3)
        kind, shift = rng.choice(list(TYPES)), rng.choice((0, 1, 2))
        tokens, mask, pad = rng.choice(("ids", "bases")), rng.choice((None, "bool", "uint8", "float")), rng.choice((0, 0, 0, 1, 5, 8))
        x, t, m = make(cuda, n, W, V, kind, tokens, mask, shift, seed=rng.randint(0, 1 << 20), pad=pad)
        what = (n, W, V, kind, shift, tokens, mask, pad)
        lp, p, y, ok = oracle(x, t, m, shift)
        a = x.detach().requires_grad_(True)
        got = P.window_logprobs(a, t, m, shift)
        close(got, lp.detach(), tol_lp(V, lp.detach()), what)
        up = torch.randn(n, W, device=cuda)
        close(torch.autograd.grad(got, a, up)[0], *grad_of(x, p, y, ok, up.double()), what)
        old, ref, adv = policy_inputs(lp, (0.2, 0.2), cuda, V)
        reduce = rng.choice(("token", "window"))
        loss, g, p, y, ok, l_err, g_err = policy_oracle(x, t, m, old, adv, ref, (0.2, 0.2), 0.1, reduce, shift)
        got = P.policy_loss(a, t, old, adv, ref, 0.2, 0.1, m, shift, reduce=reduce)
        close(got, loss, l_err + 2 * E32 * loss.abs() + 1e-12, what)
        close(torch.autograd.grad(got, a)[0], *grad_of(x, p, y, ok, g, g_err), what)


def test_second_derivatives_are_refused(P, cuda):
    x, t, _ = make(cuda, 2, 8, 16, "fp32", "ids")
    x.requires_grad_(True)
    f = torch.zeros(2, 8, device=cuda)
    for loss in (P.window_logprobs(x, t).sum(), P.preference_loss(x, t, f[:, 0]), P.policy_loss(x, t, f, f)):
        (want,) = torch.autograd.grad(loss, x, retain_graph=True)
        (d,) = torch.autograd.grad(loss, x, create_graph=True)
        assert torch.equal(d, want)
        with pytest.raises(RuntimeError, match="no second derivative"):
            torch.autograd.grad((d * d).sum(), x)


def test_gradients_against_differences(P, cuda):
    """the kernels' gradients along a direction, against central differences of the 64-bit losses: h^2 times the third
    derivative (below 10 here) and the gradients' own rounding"""
    n, W, V = 4, 30, 21
    x, t, m = make(cuda, n, W, V, "fp32", "ids", "bool", seed=9)
    lp, _, _, _ = oracle(x, t, m, 1)
    old, ref, adv = policy_inputs(lp, (0.2, 0.2), cuda, 4)
    sums = lp.detach().sum(1).float()
    way = torch.randn(n, W, V, device=cuda, generator=torch.Generator(device=cuda).manual_seed(1), dtype=torch.float64)
    h = 1e-4
    for f, o in ((lambda a: P.policy_loss(a, t, old, adv, ref, 0.2, 0.3, m), lambda a: policy_oracle(a, t, m, old, adv, ref, (0.2, 0.2), 0.3, "token", 1)[0]),
                 (lambda a: P.preference_loss(a, t, sums, 0.3, 0.1, m), lambda a: pref_oracle(a, t, m, sums, 0.3, 0.1)[0])):
        a = x.detach().requires_grad_(True)
        (d,) = torch.autograd.grad(f(a), a)
        slope = (o(x.detach().double() + h * way) - o(x.detach().double() - h * way)) / (2 * h)
        size = (d.double() * way).abs().sum()
        assert abs(float((d.double() * way).sum() - slope)) < float(size) * (run_of(V) + 100 * E32) + 1e-6 * float(size) + 10 * h * h


def test_saved_logits_changed_in_place_are_refused(P, cuda):
    x, t, _ = make(cuda, 2, 8, 16, "fp32", "ids")
    y = x.requires_grad_(True) * 1
    loss = P.window_logprobs(y, t).sum()
    y.mul_(2)
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()


def test_threads_on_streams_of_their_own(P, cuda):
    """calls leave the interpreter's lock: four threads at once, each on its stream, give what one gives alone"""
    import threading
    cases = []
    for V in (5, 128, 577, 9001):
        x, t, _ = make(cuda, 4, 50, V, "bf16", "ids")
        cases.append((x, t, torch.randn(4, device=cuda), torch.full((4, 50), -3.0, device=cuda)))

    def step(x, t, a, old):
        x = x.detach().requires_grad_()
        pair = P.preference_loss(x, t, a)
        pol = P.policy_loss(x, t, old, a)
        g = torch.autograd.grad(pair, x)[0], torch.autograd.grad(pol, x)[0]
        return pair.detach(), pol.detach(), *g, P.clip_grads(list(g), 0.1)
    want = [step(*c) for c in cases]
    torch.cuda.synchronize()
    got, errors = {}, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    out = step(*cases[i])
                torch.cuda.current_stream().synchronize()
                got[i] = out
        except Exception as e:                                       # noqa: BLE001  (raised again below)
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join(60)
    assert not errors and len(got) == 4, errors
    for i in range(4):
        assert all(torch.equal(a, b) for a, b in zip(got[i], want[i])), i


def test_negations_that_torch_put_off(P, cuda):
    """a real view of a conjugate holds the sign beside its memory: refused as a constant, applied to an upstream gradient"""
    x, t, _ = make(cuda, 2, 6, 16, "fp32")
    x.requires_grad_()
    old = torch.complex(torch.zeros(2, 6, device=cuda), torch.rand(2, 6, device=cuda)).conj().imag
    assert old.is_neg()
    with pytest.raises(ValueError, match="old_logp.*negation"):
        P.policy_loss(x, t, old, torch.ones(2, device=cuda))
    one = torch.complex(torch.zeros(1, device=cuda), torch.ones(1, device=cuda)).conj().imag
    with pytest.raises(ValueError, match="negation"):
        P.clip_grads([one], 0.5)
    a, = torch.autograd.grad(P.window_logprobs(x, t), x, old)
    b, = torch.autograd.grad(P.window_logprobs(x, t), x, old.clone())
    assert torch.equal(a, b) and a.abs().max() > 0
    loss = P.policy_loss(x, t, old.clone(), torch.ones(2, device=cuda))
    assert "PolicyLoss" in loss.grad_fn.name() and loss.grad_fn.next_functions[0][0].variable is x


@pytest.mark.parametrize("V", [5, 128, 2045, 2048, 4096, 70000])
@pytest.mark.parametrize("how", ["host", "unaligned", "recomputed"])
def test_saved_tensors_brought_back_elsewhere(P, cuda, V, how):
    """hooks on saved tensors bring the logits, tokens and the rest back in other memory, at another alignment and laid out
    otherwise; what lay at the old addresses is overwritten meanwhile"""
    n, W = 4, 6
    x0, t0, m0 = make(cuda, n, W, V, "bf16", "ids")
    m0 = (torch.rand(n, W, device=cuda) < 0.8).float() if m0 is None else m0
    ref = torch.randn(n, device=cuda)
    adv, old = torch.randn(n, device=cuda), torch.randn(n, W, device=cuda) * 0.1 - 3
    losses = {"logp": lambda x, t, m, o, a: P.window_logprobs(x, t, mask=m).mul(o).sum(),
              "pair": lambda x, t, m, o, a: P.preference_loss(x, t, ref, mask=m),
              "policy": lambda x, t, m, o, a: P.policy_loss(x, t, o, a, o * 0.9, kl=0.1, mask=m)}

    def unaligned(t):
        if t.numel() == 0:
            return t
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=cuda)[1:]
        return buf.view(t.shape).copy_(t)
    for name, f in losses.items():
        for up in (1.0, 0.5):
            leaf = x0.clone().requires_grad_()
            (f(leaf * 1, t0, m0, old, adv) * up).backward()
            want = leaf.grad
            leaf = x0.clone().requires_grad_()
            fresh = [z.clone() for z in (t0, m0, old, adv)]
            if how == "recomputed":
                from torch.utils.checkpoint import checkpoint
                loss = checkpoint(lambda z, *r: f(z * 1, *r), leaf, *fresh, use_reentrant=False)
            else:
                pack = (lambda z: z.cpu()) if how == "host" else (lambda z: z.clone())
                back = (lambda z: z.to(cuda)) if how == "host" else unaligned
                with torch.autograd.graph.saved_tensors_hooks(pack, back):
                    x = leaf * 1
                    loss = f(x, *fresh)
                x.detach().fill_(math.nan)
                for z in fresh:
                    z.zero_()
            junk = [torch.full_like(x0, math.nan) for _ in range(4)]
            (loss * up).backward()
            del junk
            # another form of the kernels may have run. Either's log-probabilities are off by run_of(V) < 2^-12, a position's
            # weight by that times what its terms add up to (their sum may cancel: the absolute part), probabilities by that
            # again; then each rounds to bf16 once
            tol = want.float().abs() * (2.0 ** -7 + 2.0 ** -9) + want.float().abs().max() * 2.0 ** -11
            assert ((leaf.grad.float() - want.float()).abs() <= tol).all(), (name, up)


def test_streams_and_graph(P, cuda):
    """two streams at once, and a step captured into a graph and replayed on new inputs"""
    sets = []
    for k in range(2):
        x, t, m = make(cuda, 4, 200, 128, "bf16", "ids", "bool", seed=20 + k)
        lp, _, _, _ = oracle(x, t, m, 1)
        sets.append((x.requires_grad_(True), t, m) + policy_inputs(lp, (0.2, 0.2), cuda, k))

    def step(x, t, m, old, ref, adv):
        a = P.policy_loss(x, t, old, adv, ref, 0.2, 0.05, m)
        b = P.preference_loss(x, t, old[:, 0].contiguous(), mask=m)
        return a, b, torch.autograd.grad(a + b, x)[0]
    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        got = []
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(step(*s))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(g, w))
    static = [q.detach().clone() for q in sets[0]]
    static[0].requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*static)
    for k in (1, 0, 1):
        with torch.no_grad():
            for a, b in zip(static, sets[k]):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want[k]))


def test_same_result_every_time(P, cuda):
    x, t, m = make(cuda, 6, 1000, 40, "bf16", "ids", "bool", seed=3)
    lp, _, _, _ = oracle(x, t, m, 1)
    old, ref, adv = policy_inputs(lp, (0.2, 0.2), cuda, 4)
    x.requires_grad_(True)
    a = [P.policy_loss(x, t, old, adv, ref, 0.2, 0.05, m) for _ in range(4)]
    assert all(torch.equal(a[0], b) for b in a)
    b = [P.window_logprobs(x, t, m, reduce="window") for _ in range(4)]
    assert all(torch.equal(b[0], c) for c in b)


# ---------------------------------------------------------------------- together with the cohort
class Model(torch.nn.Module):
    """a small convolutional model over tokens"""

    def __init__(self, V, width=24):
        super().__init__()
        self.emb = torch.nn.Embedding(V, width)
        self.conv = torch.nn.Conv1d(width, width, 5)
        self.head = torch.nn.Linear(width, V)

    def forward(self, x):
        h = self.emb(x.long()).transpose(1, 2)
        h = torch.relu(self.conv(torch.nn.functional.pad(h, (4, 0))))
        return self.head(h.transpose(1, 2))


@pytest.fixture(scope="module")
def cohort(P, golden, cuda):
    return P.Cohort.open(golden["dirs"]["q4k"], device=cuda, dataset="q4k", reference=golden["ref"])


@pytest.mark.parametrize("ids", [None, IDS])
def test_score(P, cohort, cuda, ids):
    torch.manual_seed(0)
    model = Model(13).to(cuda)
    x, c = cohort.sample(6, 700, generator=torch.Generator(device=cuda).manual_seed(1), reverse_complement=0.5, return_coords=True)
    asm = c[:, 0]
    start = torch.tensor([cohort.contigs(int(a))[int(k)][3] + int(s) for a, k, s, _ in c.tolist()], device=cuda)
    got = cohort.score(model, asm, start, 700, reverse_complement=c[:, 3].bool(), token_ids=ids)
    with torch.no_grad():
        t = cohort.windows(asm, start, 700, c[:, 3].bool(), tokens=True, token_ids=ids)
        lp, _, _, _ = oracle(model(t), t, None, 1, 4 if ids is None else ids[4])
    close(got, lp.detach().sum(1), tol_lp(13, lp.detach()).sum(1) + E32 * lp.detach().sum(1).abs())


def test_training_step_from_the_sampler(P, cohort, cuda):
    """windows from a sampler's graph, a reference model's sums, the loss, its gradient through the model, the clipped
    step: the parameters' gradients against the same step in 64 bits"""
    torch.manual_seed(1)
    model, ref_model = Model(8).to(cuda), Model(8).to(cuda)
    for _ in range(2):
        s = cohort.sampler(8, 300, torch.Generator(device=cuda).manual_seed(5), tokens=True)
        x = s()
        with torch.no_grad():
            ref = P.window_logprobs(ref_model(x), x, reduce="window")
        loss = P.preference_loss(model(x), x, ref, 0.2)
        model.zero_grad()
        loss.backward()
        grads = [p.grad for p in model.parameters()]
        want = [g.clone() for g in grads]
        norm = P.clip_grads(grads, 0.01)
        big = torch.cat([w.double().flatten() for w in want]).norm()
        assert abs(float(norm) - float(big)) <= 4 * E32 * float(big)
        f = min(1.0, 0.01 / (float(big) + 1e-6))
        for g, w in zip(grads, want):
            assert ((g.double() - w.double() * f).abs() <= 4 * E32 * w.double().abs() * f).all()
    double = Model(8).to(cuda).double()
    double.load_state_dict({k: v.double() for k, v in model.state_dict().items()})
    logits = double(x)
    lp = torch.log_softmax(logits[:, :-1], 2).gather(2, x[:, 1:].long().clamp(max=7)[..., None])[..., 0]
    lp = torch.where(x[:, 1:] != 4, lp, 0.0)
    gap = lp.sum(1) - ref.double()
    torch.nn.functional.softplus(-0.2 * (gap[:4] - gap[4:])).mean().backward()
    for w, p in zip(want, double.parameters()):
        # the model's own 32-bit (TF32 off) products bound this, not the loss: sums of 2,400 rows
        assert (w.double() - p.grad).norm() <= 1e-3 * p.grad.norm() + 1e-7


def test_a_sampler_marks_its_windows_as_changed(P, cohort, cuda):
    """a backward pass behind the sampler's next call would pair that call's tokens with this one's logits: refused"""
    s = cohort.sampler(4, 200, torch.Generator(device=cuda).manual_seed(3), tokens=True, return_coords=True)
    table = torch.randn(5, 8, device=cuda, requires_grad=True)
    a, old = torch.ones(4, device=cuda), torch.full((4, 200), -2.0, device=cuda)
    for f in (lambda x: P.window_logprobs(table[x.long()], x).sum(), lambda x: P.preference_loss(table[x.long()], x, a),
              lambda x: P.policy_loss(table[x.long()], x, old, a), lambda x: P.policy_loss(table[x.long()].half(), x, old, a) * 2):
        f(s()[0]).backward()                                         # before the next call: as ever
        loss = f(s()[0])
        x, c = s()
        with pytest.raises(RuntimeError, match="inplace"):
            loss.backward()
        versions = x._version, c._version
        s()
        assert x._version > versions[0] and c._version > versions[1]
    with torch.inference_mode():                                     # its tensors have no versions
        s = cohort.sampler(4, 200, torch.Generator(device=cuda).manual_seed(3), tokens=True)
        assert s().shape == (4, 200)


@pytest.mark.parametrize("V", [2049, 4101, 16384, 65541])
def test_maxima_on_both_sides_of_the_far_border(P, cuda, V):
    """threads (and steps) of a row whose maxima lie just below and just above 2^29, where the reference changes its form:
    floats there are 32 and 64 apart, so the words below weigh e^-32 and e^-64 (and more where there are many)"""
    top = 2.0 ** 29
    x = torch.full((1, 6, V), -top, device=cuda)
    x[0, :, ::3] = top - 32
    x[0, 1] = top - 32
    x[0, 2, :64] = top - 64
    x[0, 3:5] = -top + 32                                    # the same around -2^29
    x[0, 3, 1::2] = -top - 64
    x[0, 4, : V // 2] = -top
    x[0, 5, ::7] = top + 64
    t = torch.zeros(1, 6, dtype=torch.int64, device=cuda)
    for i, at in enumerate((V - 1, V // 2, 5, 0, V - 1, 7)):
        t[0, i] = at
        if i < 3:
            x[0, i, at] = top
    lp, p, y, ok = oracle(x, t, None, 0)
    x.requires_grad_(True)
    got = P.window_logprobs(x, t, shift=0)
    close(got, lp.detach(), tol_lp(V, lp.detach()))
    (d,) = torch.autograd.grad(got.sum(), x)
    want, tol = grad_of(x, p, y, ok, torch.ones(1, 6, device=cuda).double())
    close(d, want, tol + 1e-9)
    old = lp.detach().float()
    (d,) = torch.autograd.grad(P.policy_loss(x, t, old, torch.ones(1, device=cuda), shift=0), x)
    r = (lp.detach() - old.double()).exp()
    close(d, *grad_of(x, p, y, ok, -r / 6, r / 6 * (tol_lp(V, lp.detach()) + 2 * E32 * (1 + old.abs()))))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("V", [4, 16, 128, 1024, 4096])
def test_equal_logits_have_no_offset(P, cuda, V, kind):
    """a fresh head: logits of 0, V a power of two, so numerators and their sums are exact and a row's log-probability is
    -log V to the bits of the 64-bit constant it is made from. A margin is formed in 64 bits from a window's sum and a
    reference sum that cancels it, so it shows an offset of 1e-12 a position (a few 64-bit roundings of W log V), beside its
    own rounding to 32 bits."""
    n, W = 2, 4000
    x = torch.zeros(n, W, V, dtype=TYPES[kind], device=cuda)
    t = torch.randint(0, V, (n, W), device=cuda)
    m = torch.ones(n, W, device=cuda)
    m[1] = 0
    want = -W * math.log(V)
    ref = torch.tensor([want, 0.0], device=cuda)
    _, margin = P.preference_loss(x, t, ref, mask=m, shift=0, return_margins=True)
    rest = want - float(ref[0])
    assert abs(float(margin) - rest) <= W * 1e-12 + E32 * abs(rest)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("V, pad", [(5, 0), (8, 0), (16, 0), (33, 0), (128, 0), (282, 0), (1024, 0), (4101, 0), (5000, 120)])
def test_log_probabilities_have_no_mean_error(P, cuda, V, pad, kind):
    """Targets drawn from the model, so that what a scale of the logits (log2 e is rounded to 32 bits) does to log p is nothing
    on average. A numerator's error has a standard deviation of 3e-8 about its mean, and the same logit at the same reference
    the same error; where a handful of values (bf16 has 32 between 4 and 8) make up most of every sum, no fewer than four, it
    leaves 3e-8 / 2 of them, and its mean is known to 2e-9: below 2e-8. A mean error that nothing takes out is 5e-8."""
    W = 32768 if V < 4000 else 8192
    gen = torch.Generator(device=cuda).manual_seed(V)
    total, count = 0.0, 0
    for _ in range(65536 // W):
        x = (torch.randn(1, W, V + pad, generator=gen, device=cuda) * 1.5).to(TYPES[kind])[..., :V]
        t = torch.multinomial(torch.softmax(x[0].double(), 1), 1, generator=gen)[:, 0][None]
        want = float(torch.log_softmax(x[0].double(), 1).gather(1, t[0][:, None]).sum())
        x2, t2 = x.expand(2, W, V), t.expand(2, W)
        m = torch.ones(2, W, device=cuda)
        m[1] = 0
        ref = torch.tensor([want, 0.0], device=cuda)
        _, margin = P.preference_loss(x2, t2, ref, mask=m, shift=0, return_margins=True)
        total += float(margin) - (want - float(ref[0]))
        count += W
    assert abs(total / count) <= 2e-8


@pytest.mark.parametrize("d", [s * v for v in (1e-3, 0.1, 0.2499, 0.25, 0.26, 0.3, 0.4, 0.5, 0.7, 0.9, 0.99, 1.0, 1.01, 1.3, 2.0, 3.0, 8.0, 20.0) for s in (1, -1)])
def test_policy_kl_term_keeps_its_digits(P, cuda, d):
    """exp(d) - d - 1 by itself (one word: log p is 0, d the reference's; advantage 0). Below 1 a series: its last step's
    rounding, the steps' before it (at -1 1.2 of the sum's), d d and the product: 5 eps32. From 1 on expm1 (1 ulp = 2 eps32) less
    d: 2 * 2.39 + 1 at 1, less elsewhere. 6, and 1 for the loss. Its derivative expm1(d), times 1 - p = 1/2 (two equal words, whose
    log p is log1p(1) to 1 ulp: an error of d, as is d's own rounding): 4 eps32, the reciprocal's 2 and three products."""
    x, t, z = torch.zeros(1, 1, 1, device=cuda), torch.zeros(1, 1, dtype=torch.int64, device=cuda), torch.zeros(1, 1, device=cuda)
    ref = torch.full((1, 1), d, device=cuda)
    v = ref.double().item()
    want = math.expm1(v) - v if abs(v) > 0.1 else sum(v ** k / math.factorial(k) for k in range(2, 18))
    got = float(P.policy_loss(x, t, z, z[:, 0], ref, kl=1.0, shift=0))
    assert abs(got - want) <= 7 * E32 * want
    x = torch.zeros(1, 1, 2, device=cuda, requires_grad=True)
    ref = torch.full((1, 1), d - math.log(2), device=cuda)
    v = ref.double().item() + math.log(2)
    (g,) = torch.autograd.grad(P.policy_loss(x, t, z, z[:, 0], ref, kl=1.0, shift=0), x)
    want = -math.expm1(v) * 0.5
    tol = 9 * E32 * abs(want) + 0.5 * math.exp(v) * E32 * (abs(v) + 2 * math.log(2))
    assert abs(float(g[0, 0, 0]) - want) <= tol and abs(float(g[0, 0, 1]) + want) <= tol


@pytest.mark.parametrize("V", [8, 9, 128, 4096])
def test_policy_nan_is_not_hidden_by_an_advantage_of_0(P, cuda, V):
    """a counted position whose logits or old_logp are NaN gives NaN whatever its advantage, in the loss as in the gradient;
    beside it positions with an overflowing ratio give 0"""
    t = torch.zeros(1, 3, dtype=torch.int64, device=cuda)
    adv = torch.zeros(1, device=cuda)
    for where in ("logits", "old"):
        x, old = torch.zeros(1, 3, V, device=cuda), torch.full((1, 3), -300.0, device=cuda)
        if where == "logits":
            x[0, 1, 2] = math.nan
        else:
            old[0, 1] = math.nan
        loss = P.policy_loss(x.requires_grad_(), t, old, adv, shift=0)
        (g,) = torch.autograd.grad(loss, x)
        assert loss.isnan() and g[0, 1].isnan().all() and (g[0, ::2] == 0).all()
        with torch.no_grad():
            assert P.policy_loss(x, t, old, adv, shift=0).isnan()
            m = torch.tensor([[1.0, 0.0, 1.0]], device=cuda)                 # not counted: not read
            assert P.policy_loss(x, t, old, adv, shift=0, mask=m) == 0


def test_preference_smoothing_at_its_ends_with_infinite_margins(P, cuda):
    """label_smoothing 0 and 1 each leave out one of the two terms, also where it is infinite (a window that cannot be)"""
    x = torch.zeros(2, 2, 8, device=cuda)
    x[0, 0, 0] = -math.inf
    t, r = torch.zeros(2, 2, dtype=torch.int64, device=cuda), torch.zeros(2, device=cuda)
    for first, smoothing, want in ((x, 0.0, math.inf), (x, 1.0, 0.0), (x.flip(0), 0.0, 0.0), (x.flip(0), 1.0, math.inf)):
        loss, margin = P.preference_loss(first, t, r, label_smoothing=smoothing, shift=0, return_margins=True)
        assert float(loss) == want and float(margin) == (-math.inf if first is x else math.inf)


def test_transforms_and_tensors_without_memory_are_refused(P, cuda):
    """as on the CPU (test_train.py), and several upstream gradients at once"""
    from test_train import Wrapped
    x, t, _ = make(cuda, 2, 6, 16, "fp32")
    a = torch.zeros(2, device=cuda)
    for call, name in ((lambda: P.window_logprobs(Wrapped(x), t), "logits"), (lambda: P.preference_loss(x, t, Wrapped(a)), "ref_logp"),
                       (lambda: torch.vmap(lambda z: P.window_logprobs(z, t))(x[None].repeat(3, 1, 1, 1)), "logits"),
                       (lambda: torch.func.grad(lambda z: P.preference_loss(z, t, a))(x), "logits"),
                       (lambda: P.clip_grads([Wrapped(x)], 1.0), "grads")):
        with pytest.raises(ValueError, match=name + ": a tensor without memory"):
            call()
    with pytest.raises(ValueError, match="logits.*negation"):
        P.window_logprobs(torch._neg_view(x), t)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            P.window_logprobs(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)), t)
    x.requires_grad_()
    out = P.window_logprobs(x, t)
    with pytest.raises(RuntimeError, match="storage|memory"):
        torch.autograd.grad(out, x, torch.ones(3, 2, 6, device=cuda), is_grads_batched=True)


@pytest.mark.parametrize("how", ["host", "unaligned", "recomputed"])
def test_saved_tensors_brought_back_to_a_form_that_reads_twice(P, cuda, how):
    """9,216 pieces fit the policy loss's ring; brought back astride one more they are read twice, with scratch of their own"""
    test_saved_tensors_brought_back_elsewhere(P, cuda, 73728, how)
