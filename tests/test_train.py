"""The training-step operators' refusals and argument checks, without a GPU (nothing is launched: every call here is
refused before its first CUDA call)."""
import ctypes

import pytest
import torch

import panvram_b200 as P
from panvram_b200 import _C

X = torch.zeros(2, 3, 4)
T = torch.zeros(2, 3, dtype=torch.uint8)
L = torch.zeros(2, 3)
A = torch.zeros(2)


def _calls(logits=X, tokens=T, **kw):
    return (lambda: P.window_logprobs(logits, tokens, **kw), lambda: P.preference_loss(logits, tokens, A, **kw),
            lambda: P.policy_loss(logits, tokens, L, A, **kw))


@pytest.mark.parametrize("kw, what", [
    ({"logits": X.double()}, "logits"), ({"logits": X[0]}, "logits"), ({"logits": torch.zeros(2, 3, 0)}, "logits"),
    ({"logits": torch.zeros(2, 4, 3).transpose(1, 2)}, "logits"), ({"logits": [[[0.0]]]}, "logits"), ({"logits": X.int()}, "logits"),
    ({"logits": torch.zeros(2, 3, 1).expand(2, 3, 4)}, "logits"),
    ({"tokens": T[:, :2]}, "tokens"), ({"tokens": T.int()}, "tokens"), ({"tokens": T.bool()}, "tokens"), ({"tokens": None}, "tokens"),
    ({"mask": T[:1]}, "mask"), ({"mask": T.long()}, "mask"), ({"mask": X.half()[..., 0]}, "mask"), ({"mask": True}, "mask"),
    ({"shift": -1}, "shift"), ({"shift": 1 << 31}, "shift"), ({"shift": 1 << 70}, "shift"), ({"ignore": 1 << 63}, "ignore"),
])
def test_shared_refusals(kw, what):
    for call in _calls(**kw):
        with pytest.raises(ValueError, match=what):
            call()


def test_cpu_tensors_are_refused():
    for call in _calls():
        with pytest.raises(RuntimeError, match="GPU only"):
            call()
    for call in (lambda: P.grad_norm([A]), lambda: P.clip_grads([A], 1.0), lambda: P.clip_grads(A, 1.0, out=[torch.zeros(2)])):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()


def test_refusals_of_numbers_and_names():
    for bad in (-0.1, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="beta"):
            P.preference_loss(X, T, A, beta=bad)
        with pytest.raises(ValueError, match="clip"):
            P.policy_loss(X, T, L, A, clip=bad)
        with pytest.raises(ValueError, match="clip"):
            P.policy_loss(X, T, L, A, clip=(0.2, bad))
        with pytest.raises(ValueError, match="scale"):
            P.policy_loss(X, T, L, A, scale=bad)
        with pytest.raises(ValueError, match="kl"):
            P.policy_loss(X, T, L, A, ref_logp=L, kl=bad)
    for bad in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="label_smoothing"):
            P.preference_loss(X, T, A, label_smoothing=bad)
    with pytest.raises(ValueError, match="ref_logp"):
        P.policy_loss(X, T, L, A, kl=0.1)
    with pytest.raises(ValueError, match="reduce"):
        P.policy_loss(X, T, L, A, reduce="sum")
    with pytest.raises(ValueError, match="reduce"):
        P.window_logprobs(X, T, reduce="mean")
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            P.clip_grads([A], bad)


def test_refusals_of_gradient_lists():
    for fn in (P.grad_norm, lambda g: P.clip_grads(g, 1.0)):
        with pytest.raises(ValueError, match="no tensors"):
            fn([])
        with pytest.raises(ValueError, match="bf16, fp16 or fp32"):
            fn([A, A.double()])
        with pytest.raises(ValueError, match="bf16, fp16 or fp32"):
            fn([None])
        with pytest.raises(ValueError, match="dense"):
            fn([torch.zeros(4, 4)[:, :2]])
        with pytest.raises(ValueError, match="dense"):
            fn([torch.zeros(1).expand(4)])
    with pytest.raises(ValueError, match="out"):
        P.clip_grads([A], 1.0, out=[A, A])
    with pytest.raises(ValueError, match="out"):
        P.clip_grads([A], 1.0, out=[torch.zeros(3)])
    with pytest.raises(ValueError, match="out"):
        P.clip_grads([torch.zeros(2, 3)], 1.0, out=[torch.zeros(3, 2).t()])
    with pytest.raises(ValueError, match="out"):
        P.clip_grads([A], 1.0, out=[A.half()])
    with pytest.raises(ValueError, match="not parameters"):
        P.clip_grads([torch.nn.Parameter(A.clone())], 1.0)


def test_refusals_of_what_is_no_tensor():
    for call in (lambda: P.preference_loss(X, T, None), lambda: P.policy_loss(X, T, [0.0], A), lambda: P.policy_loss(X, T, L, 1.0),
                 lambda: P.policy_loss(X, T, L, A, ref_logp=0.5, kl=0.1), lambda: P.clip_grads([A], 1.0, out=[None]),
                 lambda: P.grad_norm(["A"]), lambda: P.window_logprobs(X, T, mask=[[1, 1, 1], [1, 1, 1]])):
        with pytest.raises(ValueError):
            call()


def _scored(**kw):
    b = _C.Scored(64, None, 64, None, 2, 3, 4, 12, 4, 0, 0, 3, 1, 0, 0, 4, 1, 2, 1, 0)
    for k, v in kw.items():
        setattr(b, k, v)
    return ctypes.byref(b)


def _message():
    return (_C._lib.pv_kernels_last_error() or b"").decode()


@pytest.mark.parametrize("kw", [{"n": -1}, {"W": -1}, {"W": 1 << 31}, {"V": 0}, {"V": 1 << 31}, {"shift": -1}, {"type": 3}, {"type": -1},
                                {"token_bytes": 4}, {"mask_bytes": 2}, {"mask_bytes": 1}, {"logits": None}, {"tokens": None},
                                {"n": 1 << 40, "W": 1 << 30}])
def test_entry_points_refuse_a_bad_batch(kw):
    lib, b = _C._lib, _scored(**kw)
    a = _C.PolicyArgs(64, 64, None, 3, 1, 1, 0, 0, 0, 0.2, 0.2, 0.0, 1.0, 0)
    assert lib.pv_score_work_bytes(b) == 0
    assert lib.pv_logprobs(b, 64, None, None, None, 0, None) == _C.PV_EARG and _message().startswith("batch")
    assert lib.pv_logprobs_grad(b, 64, 0, 0, None, None, None) == _C.PV_EARG
    assert lib.pv_preference(b, 64, 1, 0.1, 0.0, 64, None, 64, None, 64, 1 << 40, None) == _C.PV_EARG
    assert lib.pv_policy(b, ctypes.byref(a), 64, 64, 64, 1 << 40, None) == _C.PV_EARG
    assert lib.pv_policy_grad(b, ctypes.byref(a), 64, None, 0, None, 0, None) == _C.PV_EARG


def test_entry_points_refuse_missing_arguments():
    lib, b = _C._lib, _scored()
    good = dict(old=64, adv=64, ref=None, clip_low=0.2, clip_high=0.2, kl=0.0, scale=1.0)
    assert lib.pv_logprobs(b, None, 64, None, None, 0, None) == _C.PV_EARG and "scratch" in _message()
    assert lib.pv_logprobs(b, None, 64, None, 72, 1 << 30, None) == _C.PV_EARG and "scratch" in _message()      # not 16-byte aligned
    assert lib.pv_logprobs_grad(b, 64, 0, 0, None, None, None) == _C.PV_EARG                                  # no gradient to write
    long = _scored(V=100000, logits_w=100000, logits_n=300000, grad=64)
    assert lib.pv_score_stat_bytes(b) == 0 and lib.pv_score_stat_bytes(long) == 16 * 2 * 3
    for stat in (None, 72):                                                                                # missing, not aligned
        assert lib.pv_logprobs_grad(long, 64, 0, 0, stat, None, None) == _C.PV_EARG and "statistics" in _message()
    assert lib.pv_preference(_scored(n=3), 64, 1, 0.1, 0.0, 64, None, 64, None, 64, 1 << 30, None) == _C.PV_EARG and "odd" in _message()
    assert lib.pv_preference(b, None, 1, 0.1, 0.0, 64, None, 64, None, 64, 1 << 30, None) == _C.PV_EARG
    assert lib.pv_preference(b, 64, 1, 0.1, 0.0, 64, None, 64, None, 64, 1, None) == _C.PV_EARG and "scratch" in _message()
    for kw in ({"old": None}, {"adv": None}, {"clip_low": -1.0}, {"clip_high": float("nan")}, {"kl": 0.1}, {"scale": -1.0}):
        assert lib.pv_policy(b, ctypes.byref(_C.PolicyArgs(**{**good, **kw})), 64, 64, 64, 1 << 30, None) == _C.PV_EARG
        assert lib.pv_policy_grad(_scored(grad=64), ctypes.byref(_C.PolicyArgs(**{**good, **kw})), 64, None, 0, None, 0, None) == _C.PV_EARG
    assert lib.pv_policy_grad(long, ctypes.byref(_C.PolicyArgs(**good)), 64, None, 0, None, 0, None) == _C.PV_EARG and "scratch" in _message()
    assert lib.pv_policy(b, None, 64, 64, 64, 1 << 30, None) == _C.PV_EARG
    assert lib.pv_policy(b, ctypes.byref(_C.PolicyArgs(**good)), 64, 64, 64, 8, None) == _C.PV_EARG


def _list(ptrs, numels, types):
    n = len(ptrs)
    p, k, t = (ctypes.c_uint64 * n)(*ptrs), (ctypes.c_int64 * n)(*numels), (ctypes.c_uint8 * n)(*types)
    g = _C.Tensors(ctypes.cast(p, ctypes.c_void_p), ctypes.cast(k, ctypes.c_void_p), ctypes.cast(t, ctypes.c_void_p), n)
    g.kept = (p, k, t)
    return g


def test_entry_points_refuse_bad_lists_and_shared_memory():
    lib = _C._lib

    def clip(g, out=None, max_norm=1.0, work=64, need=1 << 20):
        return lib.pv_clip_grads(ctypes.byref(g), ctypes.byref(out) if out is not None else None, max_norm, 64, work, need, None)
    f = 2                                                                       # float
    for g in (_list([0], [4], [f]), _list([66], [4], [f]), _list([65], [4], [0]), _list([64], [-1], [f]), _list([64], [4], [3]),
              _list([64], [1 << 50], [f])):
        assert clip(g) == _C.PV_EARG and _message().startswith("tensors")
        assert lib.pv_grad_norm(ctypes.byref(g), 64, 64, 1 << 20, None) == _C.PV_EARG
    g = _list([256, 512], [4, 8], [f, f])
    assert clip(g, max_norm=float("nan")) == _C.PV_EARG and clip(g, max_norm=-1.0) == _C.PV_EARG
    assert clip(g, need=8) == _C.PV_EARG and "scratch" in _message()
    assert clip(g, work=None) == _C.PV_EARG and clip(g, work=72) == _C.PV_EARG
    for out in (_list([256], [4], [f]), _list([256, 512], [4, 7], [f, f]), _list([256, 512], [4, 8], [f, 0])):
        assert clip(g, out) == _C.PV_EARG and _message().startswith("out")
    shared = "shares memory"
    for g, out in ((_list([256, 256], [4, 4], [f, f]), None),                    # the same tensor twice, in place
                   (_list([256, 268], [4, 8], [f, f]), None),                    # one behind the other's start
                   (_list([268, 256], [8, 4], [f, f]), None),
                   (_list([256, 512], [4, 8], [f, f]), _list([1024, 1024], [4, 8], [f, f])),     # into the same place
                   (_list([256, 512], [4, 8], [f, f]), _list([512, 1024], [4, 8], [f, f])),      # over another gradient
                   (_list([256], [8], [f]), _list([272], [8], [f])),                             # over part of itself
                   (_list([256], [8], [0]), _list([256], [8], [f]))):                            # wider, over itself
        assert clip(g, out) == _C.PV_EARG and shared in _message()


@pytest.mark.parametrize("how", ["missing", "another torch"])
def test_the_package_needs_its_torch_extension_only_for_the_operators(tmp_path, how):
    """a copy of the package without _train.so, or with one that does not load: it imports, and a call names the build"""
    import os
    import shutil
    import subprocess
    import sys
    copy = tmp_path / "panvram_b200"
    shutil.copytree(os.path.dirname(P.__file__), copy, ignore=shutil.ignore_patterns("__pycache__", "_train.so", "csrc", "torch_ext"))
    if how != "missing":
        (copy / "_train.so").write_bytes(b"not a library")
    code = ("import torch, panvram_b200 as P\n"
            "assert P.__file__.startswith(%r) and P.Cohort and P._C.with_cuda\n"
            "x = torch.zeros(2, 3, 4)\n"
            "for f in (lambda: P.window_logprobs(x, x[..., 0].byte()), lambda: P.grad_norm([x]), lambda: P.clip_grads([x], 1.0)):\n"
            "    try:\n"
            "        f()\n"
            "    except ImportError as e:\n"
            "        assert 'build.py' in str(e) and %r in str(e), e\n"
            "    else:\n"
            "        raise AssertionError('no error')\n" % (str(tmp_path), "missing" if how == "missing" else "does not load"))
    r = subprocess.run([sys.executable, "-c", code], cwd=tmp_path, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr


def test_the_torch_extension_is_linked_again_for_another_torch(tmp_path, monkeypatch):
    """built under one torch, another, and the first again: each time its own object is what _train.so is linked from"""
    import os
    import sysconfig
    from panvram_b200 import build as B
    monkeypatch.setattr(B, "BUILD", str(tmp_path))
    monkeypatch.setattr(B, "LIB", str(tmp_path / "lib.so"))
    monkeypatch.setattr(B, "TRAIN_LIB", str(tmp_path / "_train.so"))
    monkeypatch.setattr(B, "SYNTH_LIB", str(tmp_path / "synth.so"))
    clock = [2_000_000_000]                                              # later than every source

    def run(cmd, verbose):
        out = cmd[cmd.index("-o") + 1]
        with open(out, "w") as f:
            f.write(" ".join(c for c in cmd if c.endswith(".o") and c != out))
        clock[0] += 10
        os.utime(out, (clock[0], clock[0]))
        ran.append(out)
        return ""
    monkeypatch.setattr(B, "_run", run)
    real = sysconfig.get_config_var
    for torch_version, soabi in (("2.11.0", "cpython-312"), ("2.12.0", "cpython-312"), ("2.11.0", "cpython-312"), ("2.11.0", "cpython-313")):
        monkeypatch.setattr(torch, "__version__", torch_version)
        monkeypatch.setattr(sysconfig, "get_config_var", lambda k: soabi if k == "SOABI" else real(k))
        ran = []
        B.build()
        with open(tmp_path / "_train.so") as f:
            linked = os.path.basename(f.read())
        assert torch_version in linked and soabi in linked, linked
        ran = []
        B.build()
        assert ran == []                                                 # nothing changed


def test_refusals_of_numbers_that_32_bits_cannot_hold():
    """1e39 is finite, but infinity to the kernels"""
    for call, name in ((lambda: P.preference_loss(X, T, A, beta=1e39), "beta"), (lambda: P.policy_loss(X, T, L, A, clip=1e39), "clip"),
                       (lambda: P.policy_loss(X, T, L, A, clip=(0.2, 1e39)), "clip"), (lambda: P.policy_loss(X, T, L, A, scale=1e39), "scale"),
                       (lambda: P.policy_loss(X, T, L, A, ref_logp=L, kl=1e39), "kl"), (lambda: P.clip_grads([A], 1e39), "max_norm")):
        with pytest.raises(ValueError, match=name):
            call()
    for call in (lambda: P.preference_loss(X, T, A, beta=3e38), lambda: P.clip_grads([A], float("inf"))):
        with pytest.raises(RuntimeError, match="GPU only"):                      # accepted as far as the device
            call()


def test_entry_points_refuse_bad_numbers():
    lib, b = _C._lib, _scored()
    good = dict(old=64, adv=64, ref=64, clip_low=0.2, clip_high=0.2, kl=0.1, scale=1.0)
    for k in ("clip_low", "clip_high", "kl", "scale"):
        for bad in (-1.0, float("nan"), float("inf")):
            a = _C.PolicyArgs(**{**good, k: bad})
            assert lib.pv_policy(b, ctypes.byref(a), 64, 64, 64, 1 << 30, None) == _C.PV_EARG and k.split("_")[0] in _message()
            assert lib.pv_policy_grad(_scored(grad=64), ctypes.byref(a), 64, None, 0, None, 0, None) == _C.PV_EARG
    for beta, smoothing, what in ((-1.0, 0.0, "beta"), (float("nan"), 0.0, "beta"), (float("inf"), 0.0, "beta"), (0.1, -0.1, "smoothing"),
                                  (0.1, 1.5, "smoothing"), (0.1, float("nan"), "smoothing")):
        assert lib.pv_preference(b, 64, 1, beta, smoothing, 64, None, 64, None, 64, 1 << 30, None) == _C.PV_EARG and what in _message()


def test_entry_points_refuse_addresses_that_are_not_aligned():
    """a misaligned access ends the CUDA context, so none is launched: host addresses, nothing is read"""
    lib, ok = _C._lib, (64, 1 << 30, None)
    for kw in ({"logits": 66}, {"grad": 66}, {"logits": 65, "type": 0}, {"tokens": 68, "token_bytes": 8}, {"mask": 66, "mask_bytes": 4}):
        assert lib.pv_logprobs(_scored(**kw), 64, None, None, *ok) == _C.PV_EARG and "aligned" in _message()
    assert lib.pv_score_work_bytes(_scored(logits=66, type=0)) > 0                              # 2-byte logits there are fine
    b, g = _scored(), _scored(grad=64)
    long = _scored(V=100000, logits_w=100000, logits_n=300000, grad=64)
    for args in ((66, None, None), (None, 66, None), (64, None, 72)):
        assert lib.pv_logprobs(long, *args, *ok) == _C.PV_EARG and "aligned" in _message()
    for up, scale in ((66, None), (64, 66)):
        assert lib.pv_logprobs_grad(g, up, 3, 1, None, scale, None) == _C.PV_EARG and "aligned" in _message()
    for k in range(5):
        ref, loss, margins, coef, stat = [64 + (2 if i == k else 0) for i in range(4)] + [72 if k == 4 else 64]
        assert lib.pv_preference(long, ref, 1, 0.1, 0.0, loss, margins, coef, stat, *ok) == _C.PV_EARG and "aligned" in _message()
    good = dict(old=64, adv=64, ref=64, clip_low=0.2, clip_high=0.2, kl=0.1, scale=1.0)
    for k in ("old", "adv", "ref"):
        a = ctypes.byref(_C.PolicyArgs(**{**good, k: 66}))
        assert lib.pv_policy(b, a, 64, 64, *ok) == _C.PV_EARG and "aligned" in _message()
        assert lib.pv_policy_grad(g, a, 64, None, 0, *ok) == _C.PV_EARG and "aligned" in _message()
    a = ctypes.byref(_C.PolicyArgs(**good))
    assert lib.pv_policy(b, a, 66, 64, *ok) == _C.PV_EARG and lib.pv_policy(b, a, 64, 68, *ok) == _C.PV_EARG and "aligned" in _message()
    assert lib.pv_policy_grad(g, a, 68, None, 0, *ok) == _C.PV_EARG and lib.pv_policy_grad(g, a, 64, 66, 0, *ok) == _C.PV_EARG
    grads = _list([64], [4], [2])
    assert lib.pv_grad_norm(ctypes.byref(grads), 66, 64, 1 << 20, None) == _C.PV_EARG and "aligned" in _message()
    assert lib.pv_clip_grads(ctypes.byref(grads), None, 1.0, 66, 64, 1 << 20, None) == _C.PV_EARG and "aligned" in _message()


@pytest.mark.parametrize("n, W", [(1 << 62, 0), (1 << 61, 0), (1 << 61, 1), (1 << 31, (1 << 31) - 1)])
def test_sizes_whose_bytes_wrap_round_are_refused(n, W):
    """expanded tensors may have such shapes; scratch of n W doubles would come out as few bytes or none"""
    lib, b = _C._lib, _scored(n=n, W=W, V=1 << 20)
    assert lib.pv_score_work_bytes(b) == 0 and lib.pv_score_stat_bytes(b) == 0
    for call in (lambda: lib.pv_logprobs(b, None, 64, None, 64, 1 << 40, None),
                 lambda: lib.pv_preference(b, 64, 0, 0.1, 0.0, 64, None, 64, None, 64, 1 << 40, None)):
        assert call() == _C.PV_EARG and _message().startswith("batch")
    x = torch.zeros(1, 1, 1).expand(n, W, 1) if W else torch.zeros(n, 0, 1)
    t = torch.zeros(1, 1, dtype=torch.uint8).expand(n, W) if W else torch.zeros(n, 0, dtype=torch.uint8)
    for call in _calls(x, t):
        with pytest.raises(ValueError, match="n W"):
            call()


class Wrapped(torch.Tensor):
    """a tensor class that holds another one and has no memory itself"""

    @staticmethod
    def __new__(cls, inside):
        return torch.Tensor._make_wrapper_subclass(cls, inside.size(), strides=inside.stride(), dtype=inside.dtype, device=inside.device)

    @classmethod
    def __torch_dispatch__(cls, f, types, args=(), kwargs=None):
        raise NotImplementedError(str(f))


def test_tensors_without_memory_are_refused_by_name():
    for call, name in ((lambda: P.window_logprobs(Wrapped(X), T), "logits"), (lambda: P.window_logprobs(X, Wrapped(T)), "tokens"),
                       (lambda: P.window_logprobs(X, T, Wrapped(T)), "mask"), (lambda: P.grad_norm([Wrapped(X)]), "grads"),
                       (lambda: P.clip_grads([A, Wrapped(X)], 1.0), "grads"), (lambda: P.clip_grads([X], 1.0, out=[Wrapped(X)]), "out"),
                       (lambda: torch.vmap(lambda z: P.window_logprobs(z, T))(X[None].repeat(3, 1, 1, 1)), "logits"),
                       (lambda: torch.vmap(lambda z: P.policy_loss(X, z, L, A))(T[None].repeat(3, 1, 1)), "tokens"),
                       (lambda: torch.func.grad(lambda z: P.window_logprobs(z, T).sum())(X), "logits"),
                       (lambda: torch.vmap(lambda z: P.grad_norm([z]))(X), "grads")):
        with pytest.raises(ValueError, match=name + ": a tensor without memory"):
            call()


def test_negated_logits_and_forward_mode_are_refused():
    for call in _calls(torch._neg_view(X)):
        with pytest.raises(ValueError, match="logits.*negation"):
            call()
    with torch.autograd.forward_ad.dual_level():
        for call in _calls(torch.autograd.forward_ad.make_dual(X, torch.ones_like(X))):
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                call()
