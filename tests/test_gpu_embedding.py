"""GPU tests of the embedding lookup, its gradient by sorted tokens and AdamW
over row gradients, against the formulas in float64.

Bounds. u = half a step of the result's type (bf16 2^-8 / 2 relative to the
value's power of two, taken as eps / 2), e = 2^-24 for each fp32 operation.
Lookup: the scale is an fp32 number, the product one fp32 rounding, then u.
Gradient: a sum of L fp32 terms in any order is off by at most
(L - 1) e sum|x| (1 + small), then the product and u.
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


def _u(dtype):
    return torch.finfo(dtype).eps / 2


def _gen(seed):
    return torch.Generator(device=_dev()).manual_seed(seed)


def _f32(x):
    return float(torch.tensor(x, dtype=torch.float32))


def _zipf(n, rows, seed):
    u = torch.rand(n, device=_dev(), generator=_gen(seed), dtype=torch.float64)
    return ((torch.pow(float(rows + 1), u).long().clamp_(1, rows) - 1) * 1000003) % rows


def _close(got, ref, bound):
    """|got - ref| <= bound elementwise, with room for the smallest fp32 normals."""
    err = (got.double() - ref).abs() - bound - 2.0 ** -126
    assert not (err > 0).any() and not err.isnan().any(), float(err.max())


# ------------------------------------------------------------------ lookup
@pytest.mark.parametrize("wdt,odt", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.bfloat16),
                                     (torch.bfloat16, torch.float32), (torch.float32, torch.float32)])
@pytest.mark.parametrize("n,rows,dim", [(1, 1, 1), (1, 100, 2048), (7, 5, 8), (33, 1000, 257), (1000, 77, 24),
                                        (513, 50, 1001), (3, 40, 70000),
                                        (300, 60, 36), (300, 60, 250), (90, 60, 2052)])
def test_lookup_matches_formula(wdt, odt, n, rows, dim):
    from opendm_b200.embedding import check_errors, embedding

    w = torch.randn(rows, dim, device=_dev(), generator=_gen(1)).to(wdt)
    ids = torch.randint(rows, (n,), device=_dev(), generator=_gen(2))
    for scale, id_dtype in ((1.0, torch.int64), (math.sqrt(dim), torch.int32)):
        got = embedding(ids.to(id_dtype), w, scale=scale, out_dtype=odt)
        ref = w.double()[ids] * _f32(scale)
        assert got.shape == (n, dim) and got.dtype == odt
        _close(got, ref, ref.abs() * (_u(odt) + E32) * (1 + 2 ** -10))
    check_errors()


def test_lookup_layouts_and_empty_sizes():
    from opendm_b200.embedding import embedding

    dev = _dev()
    base = torch.randn(50, 96, device=dev, generator=_gen(3))
    ids = torch.randint(50, (4, 6), device=dev, generator=_gen(4))
    for w in (base[:, :64], base[:, 3:67], base[:, :33], base.t()[:50, :40], base[::2], base[:, ::2], base[:1]):
        got = embedding(ids % w.shape[0], w)
        assert torch.equal(got, w[ids % w.shape[0]])
    assert torch.equal(embedding(ids.t(), base), base[ids.t()])  # strided ids
    assert torch.equal(embedding(ids[0, 0], base), base[ids[0, 0]])  # a single token
    assert embedding(ids[:0], base).shape == (0, 6, 96)
    assert embedding(ids, base[:, :0]).shape == (4, 6, 0)
    flat = torch.randn(50 * 64 + 1, device=dev, generator=_gen(5))
    w = flat[1:].view(50, 64)  # rows that start between 16-byte boundaries
    assert torch.equal(embedding(ids, w), w[ids])


def test_out_of_range_ids_are_reported_not_read():
    from opendm_b200.embedding import check_errors, embedding, embedding_grad, embedding_row_grad

    dev = _dev()
    w = torch.randn(10, 16, device=dev, generator=_gen(6))
    good = torch.tensor([3, 9, 0, 3], device=dev)
    ids = torch.tensor([3, 10, 9, -1, 0, 3, 2 ** 40], device=dev)
    got = embedding(ids, w)
    with pytest.raises(RuntimeError, match="token id out of range"):
        check_errors()
    check_errors()  # cleared
    assert torch.equal(got[[0, 2, 4, 5]], w[good]) and not got[[1, 3, 6]].any()
    g = torch.randn(7, 16, device=dev, generator=_gen(7))
    want = embedding_grad(g[[0, 2, 4, 5]], good, 10)
    for fn in (embedding_grad, embedding_row_grad):
        res = fn(g, ids, 10)
        with pytest.raises(RuntimeError, match="token id out of range"):
            check_errors(dev)
        if fn is embedding_grad:
            assert torch.equal(res, want)
        else:
            assert res.count.item() == 3 and res.ids.tolist() == [0, 3, 9, 0, 0, 0, 0]
            assert torch.equal(res.values[:3], want[[0, 3, 9]]) and not res.values[3:].any()
    # every id out of range, as int32
    res = embedding_row_grad(g, torch.full((7,), -5, device=dev, dtype=torch.int32), 10)
    with pytest.raises(RuntimeError, match="token id out of range"):
        check_errors()
    assert res.count.item() == 0 and not res.ids.any() and not res.values.any()


# ---------------------------------------------------------------- gradient
def _check_gradient(grad, ids, rows, *, scale=1.0, padding_idx=None, dtype=None):
    from opendm_b200.embedding import check_errors, embedding_grad, embedding_row_grad

    dtype = dtype or grad.dtype
    kw = dict(scale=scale, padding_idx=padding_idx, dtype=dtype)
    flat, key = grad.reshape(-1, grad.shape[-1]).double(), ids.reshape(-1).long()
    use = torch.ones_like(key, dtype=torch.bool) if padding_idx is None else key != padding_idx
    seen, back, counts = torch.unique(key[use], return_inverse=True, return_counts=True)
    ref = torch.zeros(seen.numel(), flat.shape[1], dtype=torch.float64, device=grad.device)
    mag = ref.clone().index_add_(0, back, flat[use].abs()) * abs(scale)
    ref.index_add_(0, back, flat[use]).mul_(_f32(scale))
    # float64's own error in the reference is 2^-53 L sum|x|: absorbed by the 1 + 2^-10
    bound = (mag * (counts[:, None] * E32) + ref.abs() * (E32 + _u(dtype))) * (1 + 2 ** -10)
    got = embedding_row_grad(grad, ids, rows, **kw)
    again = embedding_row_grad(grad, ids, rows, **kw)
    check_errors()
    n = seen.numel()
    assert got.ids.numel() == min(key.numel(), rows) == got.values.shape[0]
    assert got.count.item() == n and torch.equal(got.ids[:n], seen)
    assert not got.ids[n:].any() and not got.values[n:].any()
    assert got.values.dtype == dtype
    _close(got.values[:n], ref, bound)
    assert torch.equal(got.values, again.values)
    if rows <= 1 << 20:
        dense = embedding_grad(grad, ids, rows, **kw)
        assert dense.shape == (rows, grad.shape[-1])
        assert torch.equal(dense[seen], got.values[:n])
        rest = torch.ones(rows, dtype=torch.bool, device=grad.device)
        rest[seen] = False
        assert not dense[rest].any()


GRAD_SIZES = [(1, 1, 1), (1, 100, 8), (2, 1, 16), (31, 7, 8), (32, 1, 8), (33, 1, 24), (64, 1, 257), (65, 2, 8),
              (500, 3, 40), (512, 32003, 1024), (2048, 1, 64), (2049, 5, 8), (5000, 151936, 256), (8191, 100, 33),
              (8193, 100, 32), (3000, 700, 36), (3001, 700, 250), (1500, 90, 1002), (40000, 60000, 4), (33000, 300, 2),
              (20000, 50000, 72), (70000, 262144, 8), (40000, 9, 520)]


@pytest.mark.parametrize("gdt,odt", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32)])
@pytest.mark.parametrize("n,rows,dim", GRAD_SIZES)
def test_gradient_matches_formula(n, rows, dim, gdt, odt):
    grad = torch.randn(n, dim, device=_dev(), generator=_gen(n)).to(gdt)
    _check_gradient(grad, _zipf(n, rows, n + 1), rows, dtype=odt)


@pytest.mark.parametrize("kind", ["same", "distinct", "reversed", "runs", "two"])
@pytest.mark.parametrize("n", [96, 1000, 12345])
def test_gradient_id_patterns(kind, n):
    dev = _dev()
    if kind == "same":
        rows, ids = 40000, torch.full((n,), 39999, device=dev)
    elif kind == "distinct":
        rows, ids = n, torch.randperm(n, device=dev, generator=_gen(1))
    elif kind == "reversed":
        rows, ids = n, torch.arange(n - 1, -1, -1, device=dev)
    elif kind == "two":
        rows, ids = 2, torch.arange(n, device=dev) % 2
    else:  # runs of every length around the kernels' chunk sizes, tokens shuffled
        lengths = [1, 7, 8, 9, 15, 16, 17, 24, 31, 32, 33, 47, 48, 49, 63, 64, 65, 95, 96, 97, 128, 200, 500, 1, 1]
        rows = n
        ids = torch.repeat_interleave(torch.arange(len(lengths), device=dev), torch.tensor(lengths, device=dev))
        ids = ids.repeat(n // ids.numel() + 1)[:n] * 3 % rows
        ids = ids[torch.randperm(n, device=dev, generator=_gen(2))]
    grad = torch.randn(n, 72, device=dev, generator=_gen(3)).bfloat16()
    _check_gradient(grad, ids, rows, dtype=torch.float32)
    _check_gradient(grad, ids.int(), rows, scale=0.3, padding_idx=int(ids[0]))


@pytest.mark.parametrize("chunk_runs", [8, 16, 32])
@pytest.mark.parametrize("shift", [0, 1, 5])
def test_gradient_runs_on_chunk_boundaries(chunk_runs, shift):
    """Sorted runs that start, end and span at every offset of a chunk."""
    dev = _dev()
    lengths = [shift] if shift else []
    for k in range(60):
        lengths += [chunk_runs * (k % 4) + (k % 3 - 1) if k % 4 else 1 + k % 5]
    lengths = [x for x in lengths if x > 0]
    ids = torch.repeat_interleave(torch.arange(len(lengths), device=dev), torch.tensor(lengths, device=dev))
    grad = torch.randn(ids.numel(), 2056, device=dev, generator=_gen(chunk_runs))
    _check_gradient(grad, ids, len(lengths))
    _check_gradient(grad, ids, len(lengths), padding_idx=len(lengths) - 1)


def test_gradient_large_vocabularies():
    """Keys of one to four radix digits."""
    dev = _dev()
    for rows in (2, 500, 513, 2 ** 18 - 1, 2 ** 18, 2 ** 27 + 5, 2 ** 30, 2 ** 31 - 3):
        n = 9001
        ids = (torch.rand(n, device=dev, generator=_gen(5), dtype=torch.float64) * rows).long()
        ids[::3] = ids[0]
        ids[1], ids[2] = 0, rows - 1
        grad = torch.randn(n, 8, device=dev, generator=_gen(6))
        _check_gradient(grad, ids, rows)


def test_gradient_padding_scale_shapes_and_strides():
    dev = _dev()
    ids = _zipf(6 * 50, 200, 9).view(6, 50)
    ids[:, 40:] = 0
    grad = torch.randn(6, 50, 48, device=dev, generator=_gen(10))
    _check_gradient(grad, ids, 200, padding_idx=0, scale=math.sqrt(48))
    _check_gradient(grad, ids, 200, padding_idx=199, scale=-2.0, dtype=torch.bfloat16)
    _check_gradient(grad.transpose(0, 1), ids.t(), 200)
    _check_gradient(grad[..., ::2], ids, 200)
    _check_gradient(torch.ones(1, device=dev).expand(6, 50, 40), ids, 200)
    flat = torch.randn(300 * 48 + 1, device=dev, generator=_gen(11))
    _check_gradient(flat[1:].view(6, 50, 48), ids, 200)
    # only padding
    from opendm_b200.embedding import embedding_grad, embedding_row_grad

    res = embedding_row_grad(grad, torch.full_like(ids, 7), 200, padding_idx=7)
    assert res.count.item() == 0 and not res.values.any() and not res.ids.any()
    # no tokens, no columns
    none = embedding_row_grad(grad[:0], ids[:0], 200)
    assert none.count.item() == 0 and none.values.shape == (0, 48)
    assert not embedding_grad(grad[:0], ids[:0], 5).any()
    assert embedding_grad(grad[..., :0], ids, 5 + 200).shape == (205, 0)
    assert embedding_row_grad(grad[..., :0], ids, 205).count.item() in (0, int(torch.unique(ids).numel()))


def test_gradient_keeps_nonfinite_values_in_their_rows():
    from opendm_b200.embedding import embedding_grad

    dev = _dev()
    ids = torch.arange(100, device=dev) % 10
    grad = torch.ones(100, 16, device=dev)
    grad[3, 5], grad[14, 0], grad[7, 1], grad[17, 1] = math.nan, math.inf, math.inf, -math.inf
    got = embedding_grad(grad, ids, 10)
    want = torch.zeros(10, 16, device=dev).index_add_(0, ids, grad)
    assert torch.equal(got.isnan(), want.isnan()) and got[4, 0] == math.inf
    fine = want.isfinite()
    assert torch.equal(got[fine], want[fine])  # small whole numbers: exact


def test_padding_gradients_are_never_read():
    """NaN and infinities in the rows of dropped tokens stay out of every sum."""
    dev = _dev()
    for n, rows in ((300, 40), (5000, 40), (40000, 3)):
        ids = torch.randint(rows, (n,), device=dev, generator=_gen(n))
        grad = torch.randn(n, 40, device=dev, generator=_gen(n + 1))
        grad[ids == 2] = torch.tensor([math.nan, math.inf, -math.inf, 1e38], device=dev).repeat(10)
        _check_gradient(torch.where((ids == 2)[:, None], 0.0, grad), ids, rows, padding_idx=2)
        from opendm_b200.embedding import embedding_grad

        got = embedding_grad(grad, ids, rows, padding_idx=2)
        want = embedding_grad(torch.where((ids == 2)[:, None], 0.0, grad), ids, rows, padding_idx=2)
        assert torch.equal(got, want) and got.isfinite().all()


def test_offsets_past_32_bits():
    """More than 2^31 elements in the weight, the output, the gradient and the dense result."""
    from opendm_b200.embedding import RowGrad, check_errors, embedding, embedding_grad
    from opendm_b200.optimizer import adamw

    dev, big, dim = _dev(), 1_100_000, 2048
    w = torch.zeros(big, dim, device=dev, dtype=torch.bfloat16)
    w[-1], w[-2] = 3.0, 5.0
    got = embedding(torch.tensor([big - 1, 0, big - 2], device=dev), w)
    assert bool((got[0] == 3).all()) and not got[1].any() and bool((got[2] == 5).all())
    ids = torch.arange(big, device=dev) % 50
    out = embedding(ids, (torch.arange(50, device=dev)[:, None] + torch.zeros(dim, device=dev)).bfloat16())
    assert torch.equal(out[:, 0].float(), ids.float()) and torch.equal(out[:, -1].float(), ids.float())
    out.fill_(1.0)
    sums = embedding_grad(out, ids, 50, dtype=torch.float32)
    assert bool((sums == big / 50).all())  # whole numbers below 2^24: exact
    del out
    g = torch.ones(3, dim, device=dev, dtype=torch.bfloat16)
    dense = embedding_grad(g, torch.tensor([big - 1, 7, big - 1], device=dev), big)
    assert bool((dense[-1] == 2).all()) and bool((dense[7] == 1).all())
    assert not dense[:7].any() and not dense[8:-1].any()
    del dense
    # AdamW of the same size: the last row and one without a gradient, against a small parameter's
    m, v = torch.zeros(big, dim, device=dev), torch.full((big, dim), 1e-4, device=dev)
    kw = dict(lr=0.02, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.0)
    small = [t[-3:].clone() for t in (w, m, v)]
    adamw([w], [RowGrad(big, torch.tensor([big - 1], device=dev), g[:1])], [m], [v], [2], **kw)
    adamw([small[0]], [RowGrad(3, torch.tensor([2], device=dev), g[:1])], [small[1]], [small[2]], [2], **kw)
    for a, b in zip((w, m, v), small):
        assert torch.equal(a[-3:], b)
    check_errors()


# ---------------------------------------------------------------- autograd
@pytest.mark.parametrize("sparse", [False, True])
def test_autograd_matches_formula_and_differences(sparse):
    from opendm_b200.embedding import ScaledEmbedding

    dev = _dev()
    mod = ScaledEmbedding(20, 12, padding_idx=3, scale=2.5, sparse=sparse, device=dev)
    ids = torch.randint(20, (4, 9), device=dev, generator=_gen(12))
    coef = torch.randn(4, 9, 12, device=dev, generator=_gen(13))

    def loss():
        return (mod(ids) * coef).sum()

    loss().backward()
    grad = mod.weight.grad
    assert grad.is_sparse == sparse
    grad = grad.to_dense() if sparse else grad
    use = (ids != 3).reshape(-1)
    ref = torch.zeros(20, 12, dtype=torch.float64, device=dev).index_add_(
        0, ids.reshape(-1)[use], coef.reshape(-1, 12)[use].double()) * 2.5
    # at most 36 fp32 terms of a row, then the product
    mag = torch.zeros_like(ref).index_add_(0, ids.reshape(-1)[use], coef.reshape(-1, 12)[use].double().abs()) * 2.5
    _close(grad, ref, mag * 38 * E32)
    # the loss is linear in the weight: a central difference with step h has only rounding error,
    # of the two losses' fp32 sums of 432 terms
    with torch.no_grad():
        for row, col in ((int(ids[0, 0]), 0), (int(ids[2, 5]), 7)):
            if row == 3:
                continue
            h = 0.5
            keep = mod.weight[row, col].item()
            mod.weight[row, col] = keep + h
            up = (mod(ids) * coef).double().sum()
            mod.weight[row, col] = keep - h
            down = (mod(ids) * coef).double().sum()
            mod.weight[row, col] = keep
            diff = float((up - down) / (2 * h))
            terms = float((mod(ids).abs().double() + 2.5) .mul(coef.double().abs()).sum())
            assert abs(diff - float(grad[row, col])) <= terms * 4 * E32 / h + 38 * E32 * float(mag[row, col])


def test_autograd_accumulates_and_mixes():
    from opendm_b200.embedding import embedding

    dev = _dev()
    a = torch.randint(30, (50,), device=dev, generator=_gen(14))
    b = torch.randint(30, (20,), device=dev, generator=_gen(15))
    w = torch.randn(30, 8, device=dev, generator=_gen(16))
    grads = []
    for sparse in (False, True):
        p = torch.nn.Parameter(w.clone())
        embedding(a, p, sparse=sparse).square().sum().backward()
        embedding(b, p, sparse=sparse, scale=0.5).square().sum().backward()
        grads.append(p.grad.to_dense() if sparse else p.grad)
    assert torch.allclose(grads[0], grads[1], rtol=1e-5, atol=1e-5)
    # a weight used for the lookup (sparse) and in a product (dense), as tied output layers are
    p = torch.nn.Parameter(w.clone())
    x = embedding(a, p, sparse=True)
    (x @ p.t()).sum().backward()
    q = torch.nn.Parameter(w.clone())
    (q[a] @ q.t()).sum().backward()
    assert not p.grad.is_sparse and torch.allclose(p.grad, q.grad, rtol=1e-4, atol=1e-4)
    # frozen weight and no_grad: no graph
    assert not embedding(a, w).requires_grad
    with torch.no_grad():
        assert not embedding(a, p).requires_grad


# ------------------------------------------------------- streams and graphs
@pytest.mark.parametrize("n", [300, 1500, 9000, 20000, 40000])
def test_other_stream_and_graph_replay(n):
    """Each of the token sorts (one block, a cluster, tiles) on another stream and in two graphs at once."""
    from opendm_b200.embedding import check_errors, embedding, embedding_grad, embedding_row_grad

    dev = _dev()
    w = torch.randn(3000, 64, device=dev, generator=_gen(17))
    ids = _zipf(n, 3000, 18)
    grad = torch.randn(n, 64, device=dev, generator=_gen(19))
    want = (embedding(ids, w), embedding_grad(grad, ids, 3000), embedding_row_grad(grad, ids, 3000))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = (embedding(ids, w), embedding_grad(grad, ids, 3000))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # two captured graphs with buffers of their own, replayed at the same time
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    inputs = [(ids.clone(), grad.clone()), (ids.clone(), grad.clone())]
    for graph, (i, g) in zip(graphs, inputs):
        with torch.cuda.graph(graph):
            outs.append((embedding(i, w), embedding_grad(g, i, 3000), embedding_row_grad(g, i, 3000)))
    other_ids, other_grad = _zipf(n, 3000, 20), torch.randn(n, 64, device=dev, generator=_gen(21))
    inputs[1][0].copy_(other_ids)
    inputs[1][1].copy_(other_grad)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    new = (embedding(other_ids, w), embedding_grad(other_grad, other_ids, 3000),
           embedding_row_grad(other_grad, other_ids, 3000))
    for out, ref in zip(outs, (want, new)):
        assert torch.equal(out[0], ref[0]) and torch.equal(out[1], ref[1])
        assert torch.equal(out[2].ids, ref[2].ids) and torch.equal(out[2].values, ref[2].values)
        assert torch.equal(out[2].count, ref[2].count)
    check_errors()


def test_backward_captured_into_a_graph():
    """Forward and backward of the embedding, captured once and replayed with other tokens and weights."""
    from opendm_b200.embedding import check_errors, embedding

    dev = _dev()
    ids = _zipf(600, 300, 22)
    coef = torch.randn(600, 24, device=dev, generator=_gen(23))
    weight = torch.nn.Parameter(torch.randn(300, 24, device=dev, generator=_gen(24)))

    def step():
        (embedding(ids, weight, scale=3.0, padding_idx=5) * coef).sum().backward()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # warm up on the stream kind that captures; its autograd graph ends with it
        step()
        weight.grad = None
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in (25, 26):
        ids.copy_(_zipf(600, 300, seed))
        coef.copy_(torch.randn(600, 24, device=dev, generator=_gen(seed)))
        graph.replay()
        torch.cuda.synchronize()
        use = ids != 5
        ref = torch.zeros(300, 24, dtype=torch.float64, device=dev).index_add_(0, ids[use], coef[use].double()) * 3
        mag = torch.zeros_like(ref).index_add_(0, ids[use], coef[use].double().abs()) * 3
        _close(weight.grad, ref, mag * 602 * E32)
    check_errors()


# -------------------------------------------------------------- AdamW rows
def _moments(shape, seed):
    dev = _dev()
    return (torch.randn(shape, device=dev, generator=_gen(seed)) * 1e-3,
            (torch.randn(shape, device=dev, generator=_gen(seed + 1)) * 1e-3).square())


@pytest.mark.parametrize("pdt,gdt", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32),
                                     (torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("rows,dim,n", [(1, 1, 1), (9000, 1, 500), (5, 8192, 3), (3, 20000, 2), (100, 257, 30),
                                        (1000, 64, 0), (1000, 64, 5000), (4097, 132, 700), (40000, 24, 9000)])
def test_adamw_rows_equals_dense(rows, dim, n, pdt, gdt):
    from opendm_b200.embedding import RowGrad, embedding_grad, embedding_row_grad
    from opendm_b200.optimizer import adamw

    dev = _dev()
    p = torch.randn(rows, dim, device=dev, generator=_gen(30)).to(pdt)
    m, v = _moments((rows, dim), 31)
    ids = _zipf(n, rows, 33)
    g = torch.randn(n, dim, device=dev, generator=_gen(34)).to(gdt)
    row_grad = embedding_row_grad(g, ids, rows)
    count = int(row_grad.count)
    dense = embedding_grad(g, ids, rows)
    kw = dict(lr=0.02, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.01)
    want = [t.clone() for t in (p, m, v)]
    adamw([want[0]], [dense], [want[1]], [want[2]], [7], **kw)
    for rg in (row_grad, RowGrad(rows, row_grad.ids[:count], row_grad.values[:count])):
        got = [t.clone() for t in (p, m, v)]
        adamw([got[0]], [rg], [got[1]], [got[2]], [7], **kw)
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("eps", [1e-8, 0.0])
@pytest.mark.parametrize("decay", [0.0, 0.1])
@pytest.mark.parametrize("coef", [None, 0.5, math.inf])
@pytest.mark.parametrize("dim,dtype", [(64, torch.float32), (33, torch.float32), (64, torch.bfloat16)])
def test_adamw_rows_with_untouched_rows(eps, decay, coef, dim, dtype):
    """Rows whose moments are (signed) zeros, denormal or tiny, alone and beside others, bit for bit as in the
    dense form."""
    from opendm_b200.embedding import embedding_grad, embedding_row_grad
    from opendm_b200.optimizer import adamw
    from opendm_b200.optimizer.muon_adamw import _engine_for

    dev = _dev()
    p = torch.randn(3000, dim, device=dev, generator=_gen(75))
    p[::5] = torch.tensor([0.0, -0.0, 1e-42, math.inf], device=dev).repeat(dim)[:dim]
    m, v = _moments((3000, dim), 76)
    m[100:2900], v[100:2900] = 0.0, 0.0
    m[200:300], m[400:500, ::3], v[600:700, ::7] = -0.0, 1e-40, 1e-42
    m[800:900], m[1000:1100], m[1200:1300], v[1000:1100] = 2.0 ** -90, -(2.0 ** -89), 2.0 ** -95, 1e-4
    m[1400:1500, 1::2], v[1400:1500], v[1600:1610] = 1e-44, 1e-44, math.inf
    v[1620:1630] = math.nan
    p[1200:1300:2] = 2.0 ** -20
    p[1201:1300:2] = 2.0 ** -21
    p[1640:1650] = math.nan
    p = p.to(dtype)
    ids = torch.randint(3000, (400,), device=dev, generator=_gen(78))
    g = torch.randn(400, dim, device=dev, generator=_gen(79)).to(dtype)
    kw = dict(lr=0.02, beta1=0.9, beta2=0.95, eps=eps, weight_decay=decay)
    engine = _engine_for(dev, "fp16")
    engine.grad_scale = None if coef is None else torch.full((1,), coef, device=dev)
    try:
        results = []
        for grad in (embedding_row_grad(g, ids, 3000), embedding_grad(g, ids, 3000)):
            t = [x.clone() for x in (p, m, v)]
            adamw([t[0]], [grad], [t[1]], [t[2]], [4], **kw)
            results.append(t)
    finally:
        engine.grad_scale = None
    for a, b in zip(*results):
        nan = b.isnan()
        assert torch.equal(a.isnan(), nan)
        bits = torch.int32 if a.dtype == torch.float32 else torch.int16
        assert torch.equal(a.view(bits)[~nan], b.view(bits)[~nan])  # signs of zeros too


def test_adamw_rows_mixed_lists_clip_and_refusals():
    from opendm_b200.embedding import RowGrad, embedding_grad, embedding_row_grad
    from opendm_b200.optimizer.muon_adamw import _engine_for
    from opendm_b200.optimizer import adamw

    dev = _dev()
    shapes = [(300, 40), (77,), (128, 16)]
    p = [torch.randn(s, device=dev, generator=_gen(40 + i)) for i, s in enumerate(shapes)]
    ms, vs = zip(*[_moments(s, 50 + 2 * i) for i, s in enumerate(shapes)])
    ids = _zipf(100, 300, 60)
    g0 = torch.randn(100, 40, device=dev, generator=_gen(61))
    rest = [torch.randn(s, device=dev, generator=_gen(62)) for s in shapes[1:]]
    kw = dict(lr=0.02, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.0)
    engine = _engine_for(dev, "fp16")
    results = []
    for coef in (0.25, math.nan, 0.0):
        engine.grad_scale = torch.full((1,), coef, device=dev)
        try:
            for first in (embedding_row_grad(g0, ids, 300), embedding_grad(g0, ids, 300)):
                q, m, v = ([t.clone() for t in x] for x in (p, ms, vs))
                adamw(q, [first, *rest], m, v, [3, 3, 9], **kw)
                results.append(q + m + v)
        finally:
            engine.grad_scale = None
    for a, b in zip(results[0::2], results[1::2]):
        for x, y in zip(a, b):
            assert torch.equal(x.isnan(), y.isnan()) and torch.equal(x.nan_to_num(), y.nan_to_num())
    rg = embedding_row_grad(g0, ids, 300)
    q, m, v = p[0].clone(), ms[0].clone(), vs[0].clone()

    def call(param=q, grad=rg, exp_avg=m, exp_avg_sq=v):
        adamw([param], [grad], [exp_avg], [exp_avg_sq], [1], **kw)

    for bad in ({"grad": RowGrad(299, rg.ids, rg.values, rg.count)}, {"grad": RowGrad(300, rg.ids[:5], rg.values)},
                {"grad": RowGrad(300, rg.ids.int(), rg.values)}, {"grad": RowGrad(300, rg.ids, rg.values[:, :39])},
                {"grad": RowGrad(300, rg.ids, rg.values, rg.count.int())}, {"param": q.t().contiguous().t()},
                {"exp_avg": m.bfloat16()}, {"exp_avg_sq": v[:299]}, {"param": q.half()},
                {"grad": RowGrad(300, rg.ids, rg.values.half(), rg.count)}, {"grad": rg.ids.cpu()},
                {"grad": RowGrad(300, rg.ids.cpu(), rg.values, rg.count)}, {"grad": rg.to_sparse()}):
        with pytest.raises(RuntimeError):
            call(**bad)
    with pytest.raises(ValueError, match="distinct"):
        adamw([q, q], [rg, rg], [m, m], [v, v], [1, 1], **kw)
    with pytest.raises(ValueError, match="count from 1"):
        adamw([q], [rg], [m], [v], [0], **kw)


def test_adamw_rows_ignores_ids_outside_the_parameter():
    """A row list that lies about its ids changes no memory outside the parameter."""
    from opendm_b200.embedding import RowGrad
    from opendm_b200.optimizer import adamw

    dev = _dev()
    p, (m, v) = torch.randn(50, 16, device=dev, generator=_gen(70)), _moments((50, 16), 71)
    ids = torch.tensor([-7, 3, 49, 50, 2 ** 40], device=dev)
    vals = torch.randn(5, 16, device=dev, generator=_gen(72))
    dense = torch.zeros(50, 16, device=dev)
    dense[3], dense[49] = vals[1], vals[2]
    kw = dict(lr=0.02, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.0)
    want = [t.clone() for t in (p, m, v)]
    adamw([want[0]], [dense], [want[1]], [want[2]], [1], **kw)
    for count in (None, torch.tensor([5], device=dev), torch.tensor([2 ** 50], device=dev)):
        got = [t.clone() for t in (p, m, v)]
        adamw([got[0]], [RowGrad(50, ids, vals, count)], [got[1]], [got[2]], [1], **kw)
        for a, b in zip(got, want):
            assert torch.equal(a, b)


# --------------------------------------------------------------- optimizer
class _Model(torch.nn.Module):
    def __init__(self, sparse, kind, dtype):
        super().__init__()
        from opendm_b200.embedding import ScaledEmbedding

        dev = _dev()
        if kind == "scaled":
            self.embed = ScaledEmbedding(500, 64, scale=8.0, padding_idx=0, sparse=sparse, device=dev, dtype=dtype)
        else:
            self.embed = torch.nn.Embedding(500, 64, sparse=sparse, device=dev, dtype=dtype)
        self.layer = torch.nn.Linear(64, 128, bias=False, device=dev, dtype=dtype)
        self.norm = torch.nn.Parameter(torch.ones(128, device=dev, dtype=dtype))
        with torch.no_grad():
            for i, p in enumerate((self.embed.weight, self.layer.weight)):
                p.copy_(torch.randn(p.shape, device=dev, generator=_gen(80 + i)) * 0.1)

    def forward(self, ids):
        return (self.layer(self.embed(ids)) * self.norm).float().square().mean()


@pytest.mark.parametrize("kind,dtype,clip,passes", [("scaled", torch.float32, None, 1),
                                                    ("scaled", torch.bfloat16, None, 1),
                                                    ("scaled", torch.float32, 1e-4, 1),
                                                    ("scaled", torch.float32, 1e-4, 3),
                                                    ("torch", torch.float32, 1e-4, 2)])
def test_optimizer_sparse_grads_match_dense(kind, dtype, clip, passes):
    """MuonAdamW with sparse embedding gradients against the same steps with dense ones."""
    from opendm_b200.optimizer import MuonAdamW, mark_muon_parameters

    results = []
    for sparse in (False, True):
        model = _Model(sparse, kind, dtype)
        mark_muon_parameters(model, predicate=lambda n, p: "layer" in n)
        opt = MuonAdamW(model, lr=0.01, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.01, sparse_grads=sparse)
        for step in range(3):
            for k in range(passes):
                model(torch.randint(500, (4, 30), device=_dev(), generator=_gen(90 + 10 * step + k))).backward()
            assert model.embed.weight.grad.is_sparse == sparse
            if clip is not None:
                opt.clip_grad_norm_(clip)
            opt.step()
            opt.zero_grad(set_to_none=True)
        opt.check_device_errors()
        results.append([p.detach().clone() for p in model.parameters()])
    for (name, _), a, b in zip(model.named_parameters(), *results):
        if clip is None and passes == 1:
            assert torch.equal(a, b)
        elif "layer" in name:
            # a last-bit change of the clip coefficient moves the fp16 Newton-Schulz operands by a rounding, and
            # each run's update is within 2e-3 of the fp32 one: 2 x 2e-3 x ||eff U|| a step, with ||U|| <= 1.2
            # sqrt(64) and eff = 0.01 x 0.2 x sqrt(128)
            assert (a.double() - b.double()).norm() <= 3 * 2 * 2e-3 * 1.2 * 8 * 0.01 * 0.2 * math.sqrt(128)
        else:  # the norm adds, and accumulated passes round, in another order: a few fp32 roundings of the
            # gradient, which an update of lr = 0.01 per step passes on relative to itself. Elements whose
            # second moment is tiny against eps are bounded by the update itself.
            assert (a.double() - b.double()).abs().max() <= 3 * 0.01 * 1e-3
            assert ((a.double() - b.double()).norm() / b.double().norm()) <= 1e-5


def test_optimizer_max_grad_norm_and_coalesced_gradients():
    from opendm_b200.optimizer import MuonAdamW, mark_muon_parameters

    results = []
    for mode in ("dense", "sparse", "coalesced"):
        model = _Model(mode != "dense", "torch", torch.float32)
        mark_muon_parameters(model, predicate=lambda n, p: "layer" in n)
        opt = MuonAdamW(model, lr=0.01, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.0, max_grad_norm=1e-4,
                        sparse_grads=mode != "dense")
        model(torch.randint(500, (4, 30), device=_dev(), generator=_gen(99))).backward()
        if mode == "coalesced":
            model.embed.weight.grad = model.embed.weight.grad.coalesce()
        opt.step()
        results.append([opt.last_grad_norm] + [p.detach().clone() for p in model.parameters()])
    for other in results[1:]:
        for name, a, b in zip(["total"] + [n for n, _ in model.named_parameters()], results[0], other):
            if "layer" in name:  # as above, one step
                assert (a.double() - b.double()).norm() <= 2 * 2e-3 * 1.2 * 8 * 0.01 * 0.2 * math.sqrt(128)
                continue
            assert ((a.double() - b.double()).norm() / b.double().norm()) <= 1e-5
    # a gradient without entries still decays the moments, as a dense zero gradient does
    model = _Model(True, "torch", torch.float32)
    mark_muon_parameters(model, predicate=lambda n, p: "layer" in n)
    opt = MuonAdamW(model, lr=0.01, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.0, sparse_grads=True)
    w = model.embed.weight
    w.grad = torch.sparse_coo_tensor(torch.zeros(1, 0, dtype=torch.long, device=_dev()),
                                     torch.zeros(0, 64, device=_dev()), (500, 64))
    before = w.detach().clone()
    opt.step()
    assert torch.equal(w, before) and opt.state[w]["step"].item() == 1


def test_optimizer_clips_other_norms_of_sparse_gradients():
    """Norm types that are not folded into the step clip in place, sparse gradients included."""
    from opendm_b200.optimizer import MuonAdamW, mark_muon_parameters

    model = _Model(True, "torch", torch.float32)
    mark_muon_parameters(model, predicate=lambda n, p: "layer" in n)
    opt = MuonAdamW(model, lr=0.01, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.0, sparse_grads=True)
    model(torch.randint(500, (4, 30), device=_dev(), generator=_gen(98))).backward()
    dense = [(p.grad.to_dense() if p.grad.is_sparse else p.grad).double() for p in model.parameters()]
    total = max(float(g.abs().max()) for g in dense)
    got = opt.clip_grad_norm_(total / 4, norm_type=math.inf)
    # merged rows add at most 120 entries in fp32, in another order than to_dense()
    assert abs(float(got) - total) <= 120 * E32 * 4 * total
    factor = total / 4 / (total + 1e-6)
    for p, g in zip(model.parameters(), dense):
        now = (p.grad.to_dense() if p.grad.is_sparse else p.grad).double()
        assert (now - g * factor).abs().max() <= 600 * E32 * total
    opt.step()
    opt.check_device_errors()


def test_optimizer_reports_a_bad_token_id():
    from opendm_b200.embedding import embedding
    from opendm_b200.optimizer import MuonAdamW, mark_muon_parameters

    model = _Model(True, "scaled", torch.float32)
    mark_muon_parameters(model, predicate=lambda n, p: "layer" in n)
    opt = MuonAdamW(model, lr=0.01, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.0, sparse_grads=True)
    model(torch.tensor([[1, 500, 2]], device=_dev())).backward()
    with pytest.raises(RuntimeError, match="token id out of range"):
        opt.check_device_errors()
    embedding(torch.tensor([-1], device=_dev()), model.embed.weight)
    opt.step()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="token id out of range"):
        opt.step()
