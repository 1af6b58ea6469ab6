"""GPU tests of the norm and clipping of gradient lists, against float64.

Bounds. e = 2^-24. A thread adds at most 8 squares in fp32 (8 e of the sum,
half of that in its root), everything after is double, and the norm is rounded
to fp32: 5 e. The coefficient rounds once more, the product once, then the
result's type: |out - ref| <= |ref| (8 e + u), u = eps / 2 of the type.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E32 = 2.0 ** -24


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)


def _grads(shapes, dtypes, seed=0, std=1.0):
    gen = torch.Generator(device=_dev()).manual_seed(seed)
    return [(torch.randn(s, device=_dev(), generator=gen) * std).to(d) for s, d in zip(shapes, dtypes)]


def _norm(grads, p):
    return float(torch.linalg.vector_norm(torch.cat([g.double().reshape(-1) for g in grads]), p))


def _coef(total, max_norm):
    return min(max_norm / (total + 1e-6), 1.0)


def _check(out, ref_grads, factor):
    for o, g in zip(out, ref_grads):
        ref = g.double() * factor
        bound = ref.abs() * (8 * E32 + torch.finfo(o.dtype).eps / 2) * (1 + 2 ** -10) + 2.0 ** -126
        assert not ((o.double() - ref).abs() > bound).any()


B, F = torch.bfloat16, torch.float32
SHAPES = [(300, 77), (2048,), (1,), (64, 64), (0,), (7,), (16384,), (16385,), (5, 3, 11), (1000, 130)]


@pytest.mark.parametrize("norm", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("kind", ["bf16", "fp32", "mixed"])
@pytest.mark.parametrize("max_norm", [0.5, 1e9, 0.0])
def test_clip_matches_formula(norm, kind, max_norm):
    from opendm_b200.optimizer import clip_grads, get_total_norm

    dts = {"bf16": [B], "fp32": [F], "mixed": [B, F, F]}[kind] * len(SHAPES)
    grads = _grads(SHAPES, dts, 1)
    total = _norm(grads, norm)
    got = get_total_norm(grads, norm)
    assert got.dtype == torch.float32 and got.shape == ()
    assert abs(float(got) - total) <= 9 * E32 * total
    for odts in ([B] * len(SHAPES), [F] * len(SHAPES), None):
        src = [g.clone() for g in grads]
        out = None if odts is None else [torch.full(g.shape, 7.0, device=g.device, dtype=d) for g, d in
                                         zip(src, odts)]
        ret = clip_grads(src, max_norm, norm_type=norm, out=out)
        assert torch.equal(ret, got)
        _check(src if out is None else out, grads, _coef(total, max_norm))
        if out is not None:
            assert all(torch.equal(s, g) for s, g in zip(src, grads))
        elif max_norm == 1e9:
            assert all(torch.equal(s, g) for s, g in zip(src, grads))


@pytest.mark.parametrize("count", [1, 64, 65, 1024, 1025, 2500])
def test_list_lengths(count):
    """Lists around the number of tensors one launch takes."""
    from opendm_b200.optimizer import clip_grads

    shapes = [(1 + (37 * i) % 300,) for i in range(count)]
    grads = _grads(shapes, [B if i % 3 else F for i in range(count)], 2)
    ref = [g.clone() for g in grads]
    total = _norm(ref, 2.0)
    got = clip_grads(grads, 1.0)
    assert abs(float(got) - total) <= 9 * E32 * total
    _check(grads, ref, _coef(total, 1.0))


@pytest.mark.parametrize("std", [1e-30, 1e-22, 1e25, 1e30])
@pytest.mark.parametrize("norm", [2.0, 1.0])
def test_values_whose_squares_leave_fp32(std, norm):
    from opendm_b200.optimizer import clip_grads, get_total_norm

    grads = _grads([(1000,), (33,), (50, 64)], [F, B, F], 3, std)
    total = _norm(grads, norm)
    got = get_total_norm(grads, norm)
    assert abs(float(got) - total) <= 9 * E32 * total
    ref = [g.clone() for g in grads]
    clip_grads(grads, 1.0, norm_type=norm)
    _check(grads, ref, _coef(total, 1.0))


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("norm", [2.0, 1.0, math.inf])
def test_nonfinite_gradients(bad, norm):
    """As torch: a NaN norm makes every gradient NaN; an infinite one makes the
    finite ones 0 and the infinite ones NaN."""
    from opendm_b200.optimizer import clip_grad_norm_

    shapes = [(100,), (17, 9), (40000,)]
    params = [torch.nn.Parameter(torch.zeros(s, device=_dev())) for s in shapes]
    other = [torch.nn.Parameter(torch.zeros(s, device=_dev())) for s in shapes]
    for p, q, g in zip(params, other, _grads(shapes, [F] * 3, 4)):
        p.grad, q.grad = g.clone(), g.clone()
    params[1].grad[3, 3] = other[1].grad[3, 3] = bad
    keep = [p.grad.clone() for p in params]
    with pytest.raises(RuntimeError, match="non-finite"):
        clip_grad_norm_(params, 1.0, norm, error_if_nonfinite=True)
    for p, k in zip(params, keep):  # raised before anything is scaled
        assert torch.equal(p.grad.nan_to_num(), k.nan_to_num())
    got = clip_grad_norm_(params, 1.0, norm)
    want = torch.nn.utils.clip_grad_norm_(other, 1.0, norm)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
    for p, q in zip(params, other):
        assert torch.equal(p.grad.isnan(), q.grad.isnan())
        assert torch.equal(p.grad.nan_to_num(), q.grad.nan_to_num())


def test_layouts_duplicates_and_refusals():
    from opendm_b200.optimizer import clip_grad_norm_, clip_grads, clip_grads_with_norm_, get_total_norm

    dev = _dev()
    base = _grads([(64, 48)], [F], 5)[0]
    flat = _grads([(1001,)], [B], 6)[0]
    views = [base.t(), base.clone()[:, ::2], base.clone()[3:50, 5:17], flat[1:], flat.clone()[7:500],
             torch.randn(2, 3, 4, 5, device=dev).to(memory_format=torch.channels_last)]
    for g in views:
        ref, total = g.clone(), _norm([g], 2.0)
        whole = g._base.clone() if g._base is not None else None
        got = clip_grads([g], 0.5)
        assert abs(float(got) - total) <= 9 * E32 * total
        _check([g], [ref], _coef(total, 0.5))
        if whole is not None and g.stride() == base[:, ::2].stride():
            assert torch.equal(g._base[:, 1::2], whole[:, 1::2])  # the columns between stay
    # into an output of other strides
    src = _grads([(20, 30)], [F], 7)
    out = [torch.zeros(30, 20, device=dev, dtype=B).t()]
    total = _norm(src, 2.0)
    clip_grads(src, 1.0, out=out)
    _check(out, src, _coef(total, 1.0))
    # the same tensor twice counts and is scaled once
    g = _grads([(100,)], [F], 8)[0]
    ref, total = g.clone(), _norm([g], 2.0)
    clip_grads([g, g], 1.0)
    _check([g], [ref], _coef(total, 1.0))
    p = torch.nn.Parameter(torch.zeros(100, device=dev))
    p.grad = ref.clone()
    clip_grad_norm_([p, p], 1.0)
    assert torch.equal(p.grad, g)
    clip_grad_norm_(p, 1e9)
    # parts of one buffer that overlap, or outputs that cover another's input
    buf = torch.randn(200, device=dev)
    for grads, out in (([buf[:120], buf[100:]], None), ([buf[:50], buf[50:100]], [buf[50:100], buf[:50]]),
                       ([buf[:50]], [buf[10:60]])):
        with pytest.raises(RuntimeError, match="overlap"):
            clip_grads(grads, 1.0, out=out)
    with pytest.raises(RuntimeError, match="expanded"):
        clip_grads([torch.ones(1, device=dev).expand(5)], 1.0)
    assert float(get_total_norm([torch.ones(1, device=dev).expand(9)])) == 3.0
    assert float(get_total_norm(torch.full((4,), 2.0, device=dev))) == 4.0
    for bad in ([buf.half()], [buf, torch.zeros(3)], [buf.to_sparse()], [buf.double()]):
        with pytest.raises(RuntimeError):
            clip_grads(bad, 1.0)
    for total in (torch.ones(2, device=dev), torch.ones(1), torch.ones((), device=dev, dtype=torch.float64)):
        with pytest.raises(RuntimeError, match="total_norm"):
            clip_grads_with_norm_([p], 1.0, total)
    # empty tensors only
    assert float(clip_grads([torch.zeros(0, device=dev)], 1.0)) == 0.0


def test_known_norm_and_sparse_gradients():
    from opendm_b200.optimizer import clip_grad_norm_, clip_grads_with_norm_, get_total_norm

    dev = _dev()
    p = torch.nn.Parameter(torch.zeros(50, 8, device=dev))
    q = torch.nn.Parameter(torch.zeros(33, device=dev))
    ids = torch.tensor([[3, 7, 3, 49, 3]], device=dev)
    vals, g = _grads([(5, 8), (33,)], [F, F], 9)
    p.grad, q.grad = torch.sparse_coo_tensor(ids, vals.clone(), (50, 8)), g.clone()  # (the values are scaled in place)
    dense = torch.sparse_coo_tensor(ids, vals.double(), (50, 8)).to_dense()
    total = math.hypot(float(dense.norm()), float(g.double().norm()))
    got = clip_grad_norm_([p, q], 0.25)
    assert abs(float(got) - total) <= 12 * E32 * total  # two more fp32 additions in the merged rows
    _check([q.grad], [g], _coef(total, 0.25))
    _check([p.grad._values()], [vals], _coef(total, 0.25))
    # a norm known already
    q.grad = g.clone()
    clip_grads_with_norm_([q], 1.0, torch.tensor(40.0, device=dev))
    _check([q.grad], [g], 1.0 / (40.0 + 1e-6))
    clip_grads_with_norm_([torch.nn.Parameter(torch.zeros(3, device=dev))], 1.0, torch.tensor(1.0, device=dev))
    assert float(get_total_norm([q.grad, q.grad])) > float(get_total_norm([q.grad]))


def test_known_norm_among_the_gradients_is_refused():
    from opendm_b200.optimizer import clip_grads_with_norm_

    p = torch.nn.Parameter(torch.zeros(10, device=_dev()))
    p.grad = torch.ones(10, device=_dev())
    with pytest.raises(RuntimeError, match="overlap"):
        clip_grads_with_norm_([p], 1.0, p.grad[3])
    assert torch.equal(p.grad, torch.ones_like(p.grad))
    clip_grads_with_norm_([p], 0.5, p.grad[3].clone())
    assert float((p.grad - 0.5).abs().max()) <= 1e-6


def test_streams_graphs_and_repeat():
    from opendm_b200.optimizer import clip_grads

    dev = _dev()
    shapes = [(300, 77), (2048,), (100000,)] * 30
    grads = _grads(shapes, [B, F, F] * 30, 10)
    out = [torch.empty_like(g) for g in grads]
    total = clip_grads(grads, 1.0, out=out)
    again = [torch.empty_like(g) for g in grads]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        total2 = clip_grads(grads, 1.0, out=again)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(total, total2) and all(torch.equal(a, b) for a, b in zip(out, again))
    graphs, results = [], []
    for _ in range(2):
        src, dst = [g.clone() for g in grads], [torch.empty_like(g) for g in grads]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            t = clip_grads(src, 1.0, out=dst)
        graphs.append(graph)
        results.append((src, dst, t))
    for s in results[1][0]:
        s.mul_(0.5)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(results[0][2], total) and all(torch.equal(a, b) for a, b in zip(results[0][1], out))
    half = clip_grads(results[1][0], 1.0, out=again)
    assert torch.equal(results[1][2], half) and all(torch.equal(a, b) for a, b in zip(results[1][1], again))


def test_offsets_past_32_bits():
    """A list whose one tensor has more than 2^31 elements."""
    from opendm_b200.optimizer import clip_grads

    n = 2 ** 31 + 12345
    g = torch.full((n,), 2.0 ** -10, device=_dev(), dtype=B)
    g[-1] = 3.0
    total = math.sqrt((n - 1) * 2.0 ** -20 + 9.0)
    got = clip_grads([g], 1.0)
    assert abs(float(got) - total) <= 9 * E32 * total
    assert abs(float(g[-1]) - 3.0 / total) <= 3.0 / total * (8 * E32 + 2.0 ** -8)
    first = g[0].item()
    assert abs(first - 2.0 ** -10 / total) <= 2.0 ** -10 / total * (8 * E32 + 2.0 ** -8)
    assert bool((g[:-1] == first).all())
