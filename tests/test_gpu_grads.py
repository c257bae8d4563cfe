"""The gradients' norm and clipping against 64 bits. The norm: squares are summed eight at a time in 32 bits (8 roundings of
eps32 = 2^-24 relative at most), else in 64, so the square is within 9 eps32 and the norm within 5 with its own rounding.
A clipped element: the factor's rounding, the product's, and that to the element's type (finfo.eps / 2, or half its
smallest subnormal)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E32 = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}


@pytest.fixture(scope="module")
def P(cuda):
    import panvram_b200 as P
    return P


def norm_of(ts):
    return math.sqrt(sum(float((t.double() ** 2).sum()) for t in ts))


def check(P, grads, max_norm, out=None):
    want = [t.clone() for t in grads]
    big = norm_of(want)
    norm = P.clip_grads(grads, max_norm, out=out)
    assert norm.shape == () and norm.dtype == torch.float32
    assert abs(float(norm) - big) <= 5 * E32 * big
    f = min(1.0, max_norm / (big + 1e-6))
    for g, w in zip(out if out is not None else grads, want):
        tol = w.double().abs() * f * (7 * E32 + (torch.finfo(g.dtype).eps / 2 * 1.01 if g.dtype != torch.float32 else E32)) + TINY[g.dtype]
        assert ((g.double() - w.double() * f).abs() <= tol).all()
    if out is not None:
        assert all(torch.equal(a, b) for a, b in zip(grads, want))
    elif f == 1.0:
        assert all(torch.equal(a, b) for a, b in zip(grads, want))


SIZES = [[1], [0, 3], [7], [8, 0, 9, 1], [255, 256, 257], [16383, 16384, 16385], [1 << 20, 5, 40001], [(64, 64, 3), (5,), (1, 1)]]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("sizes", SIZES, ids=str)
def test_norm_and_clip(P, cuda, sizes, kind):
    gen = torch.Generator(device=cuda).manual_seed(1)
    make = lambda: [torch.randn(s, generator=gen, device=cuda).to(TYPES[kind]) for s in sizes]
    grads = make()
    big = norm_of(grads)
    assert abs(float(P.grad_norm(grads)) - big) <= 5 * E32 * big
    for part in (0.1, 0.999, 1.5, math.inf):
        check(P, make(), part * big)
        check(P, make(), part * big, [torch.empty(t.shape, device=cuda) for t in grads])
        check(P, make(), part * big, [torch.empty_like(t) for t in grads])
    assert all((t == 0).all() for t in (lambda g: (P.clip_grads(g, 0.0), g)[1])(make()))


@pytest.mark.parametrize("kind", list(TYPES))
def test_views_at_any_offset_leave_the_rest_alone(P, cuda, kind):
    for off in range(9):
        buf = torch.randn(70000, device=cuda).to(TYPES[kind])
        keep = buf.clone()
        spans = [(off, 33), (off + 40, 20000), (off + 20041, 1), (off + 20050, 40000)]
        grads = [buf[a:a + k] for a, k in spans]
        check(P, grads, 0.5 * norm_of(grads))
        inside = torch.zeros(70000, dtype=torch.bool, device=cuda)
        for a, k in spans:
            inside[a:a + k] = True
        assert torch.equal(buf[~inside], keep[~inside])
        for ooff in (off, 0, 3):
            grads = [keep[a:a + k] for a, k in spans]
            obuf = torch.full((70010,), 7.0, device=cuda)
            out = [obuf[ooff + a:ooff + a + k] for a, k in spans]
            check(P, grads, 0.5 * norm_of(grads), out)
            seen = torch.zeros(70010, dtype=torch.bool, device=cuda)
            for a, k in spans:
                seen[ooff + a:ooff + a + k] = True
            assert (obuf[~seen] == 7).all()


@pytest.mark.parametrize("count", [1, 96, 97, 700, 1024, 1025, 2500])
def test_many_tensors_of_mixed_types(P, cuda, count):
    gen = torch.Generator(device=cuda).manual_seed(count)
    kinds = list(TYPES.values())
    grads = [torch.randn(int(k) % 61, generator=gen, device=cuda).to(kinds[i % 3]) for i, k in enumerate(torch.randint(0, 1 << 20, (count,)))]
    if norm_of(grads) == 0:
        grads[0] = torch.ones(5, device=cuda)
    assert abs(float(P.grad_norm(grads)) - norm_of(grads)) <= 5 * E32 * norm_of(grads)
    check(P, grads, 0.3 * norm_of(grads))
    check(P, grads, 0.3 * norm_of(grads), [torch.empty(t.shape, device=cuda) for t in grads])


def test_out_may_name_the_gradient_itself(P, cuda):
    a, b = torch.randn(1000, device=cuda), torch.randn(50, device=cuda).bfloat16()
    want = [a.double(), b.double()]
    big = norm_of([a, b])
    fresh = torch.empty(50, device=cuda)
    P.clip_grads([a, b], 0.5 * big, out=[a, fresh])
    f = 0.5 * big / (big + 1e-6)
    assert ((a.double() - want[0] * f).abs() <= 8 * E32 * want[0].abs()).all()
    assert ((fresh.double() - want[1] * f).abs() <= 8 * E32 * want[1].abs()).all() and torch.equal(b.double(), want[1])


def test_any_order_of_dimensions(P, cuda):
    x = torch.randn(8, 6, 5, 4, device=cuda)
    for t in (x.to(memory_format=torch.channels_last), x.transpose(0, 3), x.permute(2, 0, 3, 1)):
        check(P, [t.clone(memory_format=torch.preserve_format)], 1.0)
        check(P, [t], 1.0, [torch.empty_like(t, memory_format=torch.preserve_format)])


@pytest.mark.parametrize("kind, values", [("fp32", [3e38, 3e38, 1.0]), ("fp32", [1e-40, 3e-42]), ("fp32", [1e-30] * 9), ("bf16", [3e38, -3e38]),
                                          ("bf16", [1e-39] * 20), ("fp16", [65504.0] * 30), ("fp16", [6e-8] * 30), ("fp32", [1e20] * 17 + [1e-20]),
                                          ("fp32", [0.0] * 40), ("fp32", [2e18] * 16), ("fp32", [1e-13] * 16)])
def test_range(P, cuda, kind, values):
    t = torch.tensor(values, device=cuda).to(TYPES[kind])
    big = math.sqrt(sum(float(v) ** 2 for v in t.double().cpu()))
    got = float(P.grad_norm([t]))
    if big > torch.finfo(torch.float32).max:
        assert got == math.inf
    else:
        assert abs(got - big) <= 5 * E32 * big + 2.0 ** -150
    w = t.double()
    P.clip_grads([t], 1.0)
    f = min(1.0, 1.0 / (big + 1e-6))
    # the factor itself may be subnormal in float: half its smallest step
    tol = w.abs() * f * (7 * E32 + torch.finfo(t.dtype).eps / 2 * 1.01) + TINY[t.dtype] + (w.abs() * 2.0 ** -150 if f < 2.0 ** -120 else 0)
    assert ((t.double() - w * f).abs() <= tol).all()


def test_infinity_and_nan(P, cuda):
    a, b = torch.tensor([1.0, math.inf], device=cuda), torch.ones(40, device=cuda).half()
    assert float(P.clip_grads([a, b], 1.0)) == math.inf
    assert a[0] == 0 and a[1].isnan() and (b == 0).all()
    a, b = torch.tensor([1.0, math.nan], device=cuda), torch.ones(40, device=cuda).half()
    assert math.isnan(float(P.clip_grads([a, b], 1.0)))
    assert a.isnan().all() and b.isnan().all()


def test_shared_memory_is_refused(P, cuda):
    x = torch.ones(100, device=cuda)
    for grads, out in (([x, x], None), ([x[:50], x[40:]], None), ([x[:50]], [x[25:75]]), ([x[:50], x[50:]], [torch.empty(50, device=cuda), x[:50]])):
        with pytest.raises(ValueError, match="shares memory"):
            P.clip_grads(grads, 1.0, out=out)
    assert (x == 1).all()
    assert abs(float(P.grad_norm([x, x])) - math.sqrt(200)) < 1e-5


def test_streams_and_graph(P, cuda):
    gen = torch.Generator(device=cuda).manual_seed(4)
    sets = [[torch.randn(s, generator=gen, device=cuda) for s in (30000, 7, 100000)] for _ in range(2)]
    outs = [[torch.empty_like(t) for t in s] for s in sets]
    want = []
    for s, o in zip(sets, outs):
        n = P.clip_grads(s, 1.0, out=o)
        want.append((n.clone(), [t.clone() for t in o]))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        norms = []
        for st, s, o in zip(streams, sets, outs):
            with torch.cuda.stream(st):
                norms.append(P.clip_grads(s, 1.0, out=o))
        torch.cuda.synchronize()
        for n, o, (wn, wo) in zip(norms, outs, want):
            assert torch.equal(n, wn) and all(torch.equal(a, b) for a, b in zip(o, wo))
    static = [t.clone() for t in sets[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n = P.clip_grads(static, 1.0)
    for k in (1, 0, 1):
        for a, b in zip(static, sets[k]):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(n, want[k][0]) and all(torch.equal(a, b) for a, b in zip(static, want[k][1]))


def test_parameters_are_refused_and_no_grad_parameters_work(P, cuda):
    p = torch.nn.Parameter(torch.ones(5, device=cuda))
    with pytest.raises(ValueError, match="not parameters"):
        P.clip_grads([p], 1.0)
    (p * 3).sum().backward()
    assert float(P.clip_grads([p.grad], 1.0)) == pytest.approx(3 * math.sqrt(5), rel=5 * E32)


def test_a_clipped_tensor_counts_as_changed(P, cuda):
    """autograd refuses a saved tensor that clipping has written since"""
    a, w = torch.ones(4, device=cuda), torch.ones(4, device=cuda, requires_grad=True)
    y = (a * w).sum()
    P.clip_grads([a], 0.5)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        b = torch.ones(4, device=cuda)
        P.clip_grads([b], 1.0)
        assert b.max() < 0.51
