"""GPU tests of calls around the embedding, clipping and row-gradient AdamW kernels: errors, aliases, modes."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)


def _gen(seed):
    return torch.Generator(device=_dev()).manual_seed(seed)


def _model_and_optimizer(**options):
    from opendm_b200.embedding import ScaledEmbedding
    from opendm_b200.optimizer import MuonAdamW, mark_muon_parameters

    model = torch.nn.Module()
    model.embed = ScaledEmbedding(500, 64, sparse=True, device=_dev())
    model.layer = torch.nn.Linear(64, 128, bias=False, device=_dev())
    mark_muon_parameters(model, predicate=lambda n, p: "layer" in n)
    return model, MuonAdamW(model, lr=0.01, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.0, sparse_grads=True, **options)


def _backward(model, ids, scale=1.0):
    (model.layer(model.embed(ids.to(_dev()))) * scale).square().mean().backward()


def test_a_token_id_error_is_raised_once():
    model, opt = _model_and_optimizer()
    _backward(model, torch.tensor([1, 500, 2]))
    opt.step()  # queues a copy of the error word
    with pytest.raises(RuntimeError, match="token id out of range"):
        opt.check_device_errors()
    opt.check_device_errors()
    for _ in range(2):  # the error was raised; these are healthy steps
        opt.zero_grad(set_to_none=True)
        _backward(model, torch.tensor([1, 2, 3]))
        opt.step()
    opt.check_device_errors()
    _backward(model, torch.tensor([-1]))
    opt.step()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="token id out of range"):
        opt.clip_grad_norm_(1.0)
    opt.step()
    opt.check_device_errors()


def test_the_clip_of_an_abandoned_step_is_not_used_later():
    model, opt = _model_and_optimizer(max_grad_norm=1e-3)
    _backward(model, torch.tensor([-1]))
    opt.step()
    torch.cuda.synchronize()
    # a clip that leaves the pending coefficient behind: the late error is raised by the step
    opt._pending_clip = torch.tensor([1.0, 0.0], device=_dev())
    with pytest.raises(RuntimeError, match="token id out of range"):
        opt.step()
    opt.zero_grad(set_to_none=True)
    _backward(model, torch.tensor([1, 2, 3]), 100.0)
    total = sum(float(p.grad.to_dense().double().square().sum()) for p in model.parameters()) ** 0.5
    opt.step()  # with a coefficient of 0 the norm would not be taken and the moments would stay as they were
    assert abs(float(opt.last_grad_norm) - total) <= 1e-5 * total
    assert bool(opt.state[model.embed.weight]["exp_avg"][1:4].any())


@pytest.mark.parametrize("sparse", [False, True])
def test_forward_mode_of_the_lookup(sparse):
    from torch.autograd import forward_ad as fw

    from opendm_b200.embedding import ScaledEmbedding, embedding

    w = torch.randn(20, 12, device=_dev(), generator=_gen(1))
    t = torch.randn(20, 12, device=_dev(), generator=_gen(2))
    ids = torch.randint(20, (4, 9), device=_dev(), generator=_gen(3))
    for weight in (w, w.clone().requires_grad_()):
        with fw.dual_level():
            out = embedding(ids, fw.make_dual(weight, t), scale=0.5, padding_idx=3, sparse=sparse)
            primal, tangent = fw.unpack_dual(out)
            assert torch.equal(primal, w[ids] * 0.5) and torch.equal(tangent, t[ids] * 0.5)
    # as torch's own module has it, the padding row's tangent included
    mod = ScaledEmbedding.from_pretrained(w, padding_idx=3, sparse=sparse)
    ref = torch.nn.Embedding.from_pretrained(w, padding_idx=3)
    with fw.dual_level():
        tangents = []
        for m in (mod, ref):
            out = torch.func.functional_call(m, {"weight": fw.make_dual(w, t)}, (ids,))
            tangents.append(fw.unpack_dual(out).tangent)
        assert torch.equal(*tangents)
    # the derivative of a gradient along a tangent is refused, not dropped
    p = w.clone().requires_grad_()
    with fw.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        loss = embedding(ids, fw.make_dual(p, t), sparse=sparse).square().sum()
        torch.autograd.grad(loss, p)
    # function transforms are refused
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: embedding(ids, x), (w,), (t,))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda x: embedding(ids, x).sum())(w)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda x: embedding(ids, x))(w[None])


def test_second_derivatives_are_refused():
    from opendm_b200.embedding import embedding

    p = torch.randn(20, 12, device=_dev(), generator=_gen(1), requires_grad=True)
    ids = torch.randint(20, (9,), device=_dev(), generator=_gen(3))
    g, = torch.autograd.grad(embedding(ids, p).square().sum(), p, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def test_autograd_sees_what_clipping_and_adamw_write():
    from opendm_b200.optimizer import adamw, clip_grads

    x = torch.ones(300, device=_dev(), requires_grad=True)
    g, = torch.autograd.grad((x ** 3).sum(), x, create_graph=True)
    y = (g ** 2).sum()
    with torch.no_grad():
        clip_grads([g], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    y = (x ** 2).sum()
    m, v = torch.zeros(300, device=_dev()), torch.zeros(300, device=_dev())
    adamw([x], [torch.ones(300, device=_dev())], [m], [v], [1], lr=0.1, beta1=0.9, beta2=0.95, eps=1e-8,
          weight_decay=0.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    # a loop of forward, backward, clip and update stays as it is; so do inference tensors
    w = torch.nn.Parameter(torch.ones(8, 8, device=_dev()))
    m, v = torch.zeros_like(w), torch.zeros_like(w)
    for step in (1, 2):
        w.grad = None
        (w @ w).sum().backward()
        clip_grads([w.grad], 1.0)
        adamw([w], [w.grad], [m], [v], [step], lr=0.1, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.0)
    with torch.inference_mode():
        t = torch.full((4,), 2.0, device=_dev())
        assert float(clip_grads([t], 1.0)) == 4.0 and float((t - 0.5).abs().max()) <= 1e-6


def test_adamw_beside_a_clipped_step_of_another_thread():
    """The engine is shared by the process; the coefficient of one thread's step is not another's."""
    import threading

    from opendm_b200.engine import engine_for
    from opendm_b200.optimizer import adamw

    dev = _dev()
    kw = dict(lr=0.02, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.0)
    g = torch.randn(64, 8, device=dev, generator=_gen(1))
    results = []

    def update():
        p, m, v = (torch.zeros(64, 8, device=dev) for _ in range(3))
        adamw([p], [g], [m], [v], [1], **kw)
        results.append((p, m, v))

    update()
    engine = engine_for(dev, "fp16")
    engine.grad_scale = torch.zeros(1, device=dev)
    try:
        torch.cuda.synchronize()
        other = threading.Thread(target=update)
        other.start()
        other.join()
    finally:
        engine.grad_scale = None
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(*results)) and bool(results[0][1].any())


def test_adamw_takes_empty_parameters_and_refuses_shared_memory():
    from opendm_b200.embedding import RowGrad
    from opendm_b200.optimizer import adamw

    dev = _dev()
    kw = dict(lr=0.02, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.0)
    p, m, v, g = (torch.ones(40, 8, device=dev) for _ in range(4))
    e = [torch.zeros(0, 8, device=dev) for _ in range(2)]
    rows = RowGrad(0, torch.zeros(0, dtype=torch.long, device=dev), e[0])
    adamw([e[0], p, e[1], e[0]], [e[0], g, e[1], rows], [e[0], m, e[1], e[1]], [e[0], v, e[1], e[1]], [1] * 4, **kw)
    assert bool((p < 1).all())
    with pytest.raises(ValueError, match="share memory"):
        adamw([p[:20], p[10:30]], [g[:20], g[:20]], [m[:20], m[20:]], [v[:20], v[20:]], [1, 1], **kw)


def test_strided_gradients_that_overlap_are_refused_and_others_clipped():
    from opendm_b200.optimizer import clip_grads

    buf = torch.randn(64, 48, device=_dev(), generator=_gen(1))
    ref = buf.clone()
    with pytest.raises(RuntimeError, match="overlap"):
        clip_grads([buf[:, :20], buf[:, 10:30]], 1.0)
    assert torch.equal(buf, ref)
    total = clip_grads([buf[:, :20], buf[:, 20:30], buf[:, 30:].t()], 1.0)
    want = ref.double().norm()
    # five half steps of fp32 in the norm, one each in the coefficient and the product
    assert abs(float(total) - float(want)) <= 9 * 2.0 ** -24 * float(want)
    assert ((buf.double() - ref.double() / (want + 1e-6)).abs() <= ref.double().abs() / want * 11 * 2.0 ** -24).all()


@pytest.mark.parametrize("scale", [float("inf"), float("nan"), -2.0])
def test_rows_of_bad_ids_are_zeros_for_every_scale(scale):
    from opendm_b200.embedding import check_errors, embedding

    for dim in (16, 20, 33):  # in groups of eight, four and single elements
        w = torch.ones(10, dim, device=_dev())
        got = embedding(torch.tensor([3, 10, -1, 9], device=_dev()), w, scale=scale)
        with pytest.raises(RuntimeError, match="token id out of range"):
            check_errors()
        assert not got[1:3].any() and not got[1:3].isnan().any()
        assert torch.equal(got[[0, 3]].isnan(), torch.full((2, dim), scale != scale, device=_dev()))
        assert scale != scale or bool((got[[0, 3]] == scale).all())


def test_adamw_rows_in_a_captured_graph():
    from opendm_b200.embedding import embedding_row_grad
    from opendm_b200.optimizer import adamw

    dev = _dev()
    kw = dict(lr=0.02, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.01)
    start = torch.randn(300, 24, device=dev, generator=_gen(1))
    ids, grad = torch.randint(300, (50,), device=dev, generator=_gen(2)), torch.randn(50, 24, device=dev)
    p, m, v = start.clone(), torch.zeros_like(start), torch.zeros_like(start)
    adamw([p], [embedding_row_grad(grad, ids, 300)], [m], [v], [1], **kw)  # makes the engine and the error word
    want = [t.clone() for t in (p, m, v)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        adamw([p], [embedding_row_grad(grad, ids, 300)], [m], [v], [1], **kw)
    p.copy_(start), m.zero_(), v.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((p, m, v), want))
    ids.copy_(torch.randint(300, (50,), device=dev, generator=_gen(3)))
    for t, u in zip(want, (p, m, v)):
        t.copy_(u)
    graph.replay()
    adamw([want[0]], [embedding_row_grad(grad, ids, 300)], [want[1]], [want[2]], [1], **kw)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((p, m, v), want))


def test_neighbours_in_one_buffer_are_updated():
    """Parameter, moments and rows that touch, as views of one buffer, and one element of overlap."""
    from opendm_b200.embedding import RowGrad
    from opendm_b200.optimizer import adamw

    dev = _dev()
    kw = dict(lr=0.02, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.0)
    buf = torch.ones(7, 4, 8, device=dev)
    p, m, v, values = buf[1], buf[2], buf[3], buf[4, :2]
    ids = torch.tensor([0, 3], device=dev)
    want = [t.clone() for t in (p, m, v)]
    adamw([want[0]], [RowGrad(4, ids, values)], [want[1]], [want[2]], [1], **kw)
    adamw([p], [RowGrad(4, ids, values)], [m], [v], [1], **kw)
    assert all(torch.equal(a, b) for a, b in zip((p, m, v), want))
    assert bool((buf[[0, 4, 5, 6]] == 1).all())
    flat = buf.view(-1)
    for k in (1, 31):
        with pytest.raises(RuntimeError, match="share memory"):
            adamw([p], [RowGrad(4, ids, values)], [flat[32 + k:64 + k].view(4, 8)], [buf[6]], [1], **kw)


def test_sparse_backward_captured_into_a_graph():
    """Forward and sparse backward, captured with the AdamW of its rows and replayed with other tokens."""
    from opendm_b200.embedding import check_errors, embedding
    from opendm_b200.optimizer import adamw
    from opendm_b200.optimizer.functional import rows_of

    dev = _dev()
    kw = dict(lr=0.02, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.0)
    ids = torch.randint(300, (600,), device=dev, generator=_gen(1))
    coef = torch.randn(600, 24, device=dev, generator=_gen(2))
    weight = torch.nn.Parameter(torch.randn(300, 24, device=dev, generator=_gen(3)))
    m, v = torch.zeros_like(weight), torch.zeros_like(weight)

    def step(w, m, v):
        w.grad = None
        (embedding(ids, w, sparse=True) * coef).sum().backward()
        adamw([w], [rows_of(w.grad)], [m], [v], [1], **kw)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(weight, m, v)
        weight.grad = None
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(weight, m, v)
    for seed in (4, 5):
        ids.copy_(torch.randint(300, (600,), device=dev, generator=_gen(seed)))
        want = [torch.nn.Parameter(weight.detach().clone()), m.clone(), v.clone()]
        graph.replay()
        torch.cuda.synchronize()
        step(*want)
        assert torch.equal(weight, want[0]) and torch.equal(m, want[1]) and torch.equal(v, want[2])
    check_errors()
