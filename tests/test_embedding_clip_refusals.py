"""Argument checks of the embedding, list-clipping and row-gradient AdamW entry
points. None of these calls reaches a launch, so they run without a GPU."""

import ctypes
import math

import pytest
import torch

from opendm_b200 import _native as N
from opendm_b200 import embedding as E
from opendm_b200 import optimizer as O
from opendm_b200.build import build
from opendm_b200.optimizer import MuonAdamW, mark_muon_parameters


@pytest.fixture(scope="module")
def lib():
    build()
    return N.lib()


P = ctypes.c_void_p(4096)  # aligned, never dereferenced


def _lookup(lib, weight=P, wd=N.MUON_BF16, rows=10, dim=8, ld=8, ids=P, idt=N.MUON_I64, tokens=4, out=P,
            od=N.MUON_BF16, err=P):
    return lib.muon_embedding(weight, wd, rows, dim, ld, ids, idt, tokens, ctypes.c_float(1.0), out, od, err, None)


def test_lookup_arguments(lib):
    for bad in ({"wd": N.MUON_F16}, {"od": N.MUON_TF32}, {"idt": 0}, {"rows": -1}, {"tokens": -1}, {"dim": -8},
                {"ld": 7}, {"weight": None}, {"ids": None}, {"out": None}, {"err": None},
                {"rows": 1 << 40, "ld": 1 << 40}, {"tokens": 1 << 40, "dim": 1 << 30, "ld": 1 << 30}):
        assert _lookup(lib, **bad) == N.MUON_ERR_ARG, bad
    assert _lookup(lib, tokens=0) == N.MUON_OK
    assert _lookup(lib, dim=0, ld=0) == N.MUON_OK


def _grad(lib, grad=P, gd=N.MUON_BF16, ids=P, idt=N.MUON_I64, tokens=4, rows=10, dim=8, pad=-1, out=P,
          od=N.MUON_BF16, out_ids=None, count=None, work=P, size=1 << 40, err=P):
    return lib.muon_embedding_grad(grad, gd, ids, idt, tokens, rows, dim, pad, ctypes.c_float(1.0), out, od, out_ids,
                                   count, work, size, err, None)


def test_gradient_arguments(lib):
    for bad in ({"gd": N.MUON_F16}, {"od": 7}, {"idt": 3}, {"tokens": -1}, {"rows": -1}, {"dim": -1}, {"pad": 10},
                {"pad": -2}, {"grad": None}, {"ids": None}, {"out": None}, {"err": None}, {"work": None},
                {"work": ctypes.c_void_p(4096 + 16)}, {"size": 8}, {"out_ids": P}, {"tokens": 1 << 31},
                {"rows": 1 << 31}, {"tokens": 1 << 30, "dim": 1 << 30}):
        assert _grad(lib, **bad) == N.MUON_ERR_ARG, bad
    assert lib.muon_embedding_grad_workspace_bytes(-1, 2, 3) == -1
    assert lib.muon_embedding_grad_workspace_bytes(1 << 31, 2, 3) == -1
    small, large = (lib.muon_embedding_grad_workspace_bytes(n, 1000, 64) for n in (10, 100000))
    assert 0 < small < large


def _segs(*items):
    arr = (N.ClipSeg * max(len(items), 1))()
    for s, it in zip(arr, items):
        s.grad, s.out, s.numel, s.grad_dtype, s.out_dtype = it
    return ctypes.cast(arr, ctypes.c_void_p), len(items)


def test_clip_arguments(lib):
    bf, f32 = N.MUON_BF16, N.MUON_F32
    good = (4096, 8192, 16, bf, f32)
    for item in ((None, 8192, 16, bf, bf), (4096, None, 16, bf, bf), (4096, 8192, -1, bf, bf),
                 (4096, 8192, 16, N.MUON_F16, bf), (4096, 8192, 16, bf, 9), (4097, 8192, 16, bf, bf),
                 (4098, 8192, 16, f32, f32), (4096, 8194, 16, f32, f32), (4096, 4096, 16, bf, f32),
                 (4096, 8192, 1 << 50, bf, bf)):
        segs, n = _segs(good, item)
        assert lib.muon_clip_grads(segs, n, N.MUON_NORM_2, 1.0, P, P, None) == N.MUON_ERR_ARG, item
        assert lib.muon_scale_grads(segs, n, 1.0, P, None) == N.MUON_ERR_ARG, item
    segs, n = _segs(good)
    assert lib.muon_clip_grads(segs, n, 3, 1.0, P, P, None) == N.MUON_ERR_ARG
    assert lib.muon_clip_grads(segs, n, 0, 1.0, None, P, None) == N.MUON_ERR_ARG
    assert lib.muon_clip_grads(segs, n, 0, 1.0, ctypes.c_void_p(4100), P, None) == N.MUON_ERR_ARG
    assert lib.muon_clip_grads(segs, n, 0, 1.0, P, None, None) == N.MUON_ERR_ARG
    assert lib.muon_clip_grads(segs, -1, 0, 1.0, P, P, None) == N.MUON_ERR_ARG
    assert lib.muon_clip_grads(None, 1, 0, 1.0, P, P, None) == N.MUON_ERR_ARG
    assert lib.muon_total_norm(segs, n, -1, P, P, None) == N.MUON_ERR_ARG
    assert lib.muon_scale_grads(segs, n, 1.0, None, None) == N.MUON_ERR_ARG
    assert lib.muon_clip_workspace_bytes(-1) == -1
    assert lib.muon_clip_workspace_bytes(5000) > lib.muon_clip_workspace_bytes(5) > 0


def test_adamw_rows_arguments(lib):
    def call(**kw):
        s = N.AdamwRowsSeg()
        vals = {"param": 4096, "exp_avg": 4096, "exp_avg_sq": 4096, "ids": 4096, "values": 4096, "rows": 4, "dim": 8,
                "cap": 2, "param_dtype": N.MUON_BF16, "grad_dtype": N.MUON_BF16} | kw
        for k, v in vals.items():
            setattr(s, k, v)
        return lib.muon_adamw_rows(ctypes.byref(s), 0.9, 0.95, 1e-8, 1.0, None, None)

    for bad in ({"param": None}, {"exp_avg": None}, {"exp_avg_sq": None}, {"ids": None}, {"values": None},
                {"rows": -1}, {"dim": -1}, {"cap": -1}, {"cap": 1 << 31}, {"param_dtype": N.MUON_F16},
                {"grad_dtype": 9}, {"rows": 1 << 40, "dim": 1 << 20}):
        assert call(**bad) == N.MUON_ERR_ARG, bad
    assert call(rows=0) == N.MUON_OK and call(dim=0) == N.MUON_OK
    assert lib.muon_adamw_rows(None, 0.9, 0.95, 1e-8, 1.0, None, None) == N.MUON_ERR_ARG


def test_cpu_tensors_have_no_fallback():
    w, ids, g = torch.zeros(4, 8), torch.zeros(3, dtype=torch.long), torch.zeros(3, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        E.embedding(ids, w)
    with pytest.raises(RuntimeError, match="CUDA"):
        E.embedding_grad(g, ids, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        E.embedding_row_grad(g, ids, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        O.clip_grads([g], 1.0)
    with pytest.raises(RuntimeError, match="CUDA"):
        O.get_total_norm([g])
    with pytest.raises(RuntimeError, match="CUDA"):
        O.adamw([w], [w], [w], [w], [1], lr=0.1, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.0)


def test_python_argument_checks():
    g = torch.zeros(3, 8)
    for norm in (0.0, 3.0, -math.inf):
        with pytest.raises(ValueError, match="norm_type"):
            O.clip_grads([g], 1.0, norm_type=norm)
        with pytest.raises(ValueError, match="norm_type"):
            O.get_total_norm([g], norm)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            O.clip_grads([g], bad)
    with pytest.raises(ValueError, match="match the gradients"):
        O.clip_grads([g], 1.0, out=[])
    with pytest.raises(ValueError, match="match the gradients"):
        O.clip_grads([g], 1.0, out=[torch.zeros(8, 3)])
    with pytest.raises(ValueError, match="one entry"):
        O.adamw([g], [], [g], [g], [1], lr=0.1, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.0)
    with pytest.raises(ValueError, match="padding_idx"):
        E.embedding(torch.zeros(3, dtype=torch.long), torch.zeros(4, 8), padding_idx=4)
    # lists without a gradient have norm 0, as torch's
    assert float(O.clip_grad_norm_([torch.nn.Parameter(g)], 1.0)) == 0.0
    assert float(O.clip_grads([], 1.0)) == 0.0 and float(O.get_total_norm([])) == 0.0


def test_sparse_grads_option():
    class Tiny(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.embed = torch.nn.Embedding(10, 4, sparse=True)
            self.layer = torch.nn.Linear(4, 4, bias=False)

    m = Tiny()
    mark_muon_parameters(m, predicate=lambda n, p: "layer" in n)
    kw = dict(lr=1e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.0)
    with pytest.raises(ValueError, match="adamw_sharding"):
        MuonAdamW(m, state_sharding=True, adamw_sharding=True, sparse_grads=True, **kw)
    opt = MuonAdamW(m, sparse_grads=True, **kw)
    m.embed(torch.tensor([1, 2, 1])).sum().backward()
    with pytest.raises(RuntimeError, match="CUDA"):  # no CPU path for the merge
        opt.step()
    m.embed.weight.grad = None
    m.layer.weight.grad = torch.zeros(4, 4).to_sparse(1)
    with pytest.raises(RuntimeError, match="sparse"):  # Muon matrices stay dense
        opt._engine = object()
        opt.step()


def test_scaled_embedding_is_a_torch_embedding():
    e = E.ScaledEmbedding(7, 4, padding_idx=2, scale=3.0, sparse=True)
    ref = torch.nn.Embedding(7, 4, padding_idx=2)
    ref.load_state_dict(e.state_dict())
    assert not e.weight[2].any() and "scale=3.0" in repr(e) and e.sparse
    table = torch.randn(6, 3)
    f = E.ScaledEmbedding.from_pretrained(table, padding_idx=1, scale=2.0, sparse=True)
    assert f.weight.data_ptr() == table.data_ptr() and not f.weight.requires_grad
    assert (f.num_embeddings, f.embedding_dim, f.padding_idx, f.scale, f.sparse) == (6, 3, 1, 2.0, True)
    with pytest.raises(ValueError, match="2-D"):
        E.ScaledEmbedding.from_pretrained(table[0])


def test_a_norm_inside_the_clipped_memory_is_refused(lib):
    segs, n = _segs((4096, 8192, 16, N.MUON_F32, N.MUON_F32))
    for inside in (8192, 8200, 8252):
        total = ctypes.c_void_p(inside)
        assert lib.muon_scale_grads(segs, n, 1.0, total, None) == N.MUON_ERR_ARG
        assert "norm" in N.last_error()
        assert lib.muon_clip_grads(segs, n, N.MUON_NORM_2, 1.0, P, total, None) == N.MUON_ERR_ARG
        assert "norm" in N.last_error()


def test_misaligned_pointers_are_refused(lib):
    """Pointers that are no multiple of their element's size would fault in a kernel."""
    odd, two, four = ctypes.c_void_p(4097), ctypes.c_void_p(4098), ctypes.c_void_p(4100)
    f32 = {"wd": N.MUON_F32, "od": N.MUON_F32}
    for bad in ({"weight": odd}, {"out": odd}, {"ids": four}, {"ids": two, "idt": N.MUON_I32}, {"err": two},
                {"weight": two} | f32, {"out": two} | f32):
        assert _lookup(lib, **bad) == N.MUON_ERR_ARG, bad
        assert "aligned" in N.last_error()
    f32 = {"gd": N.MUON_F32, "od": N.MUON_F32}
    rows = {"out_ids": P, "count": P}
    for bad in ({"grad": odd}, {"out": odd}, {"ids": four}, {"ids": two, "idt": N.MUON_I32}, {"err": two},
                {"grad": two} | f32, {"out": two} | f32, rows | {"out_ids": four}, rows | {"count": four}):
        assert _grad(lib, **bad) == N.MUON_ERR_ARG, bad
        assert "aligned" in N.last_error()
    segs, n = _segs((4096, 8192, 16, N.MUON_F32, N.MUON_F32))
    assert lib.muon_scale_grads(segs, n, 1.0, two, None) == N.MUON_ERR_ARG
    assert lib.muon_clip_grads(segs, n, N.MUON_NORM_2, 1.0, P, two, None) == N.MUON_ERR_ARG
    assert lib.muon_total_norm(segs, n, N.MUON_NORM_2, P, two, None) == N.MUON_ERR_ARG
    good = {"param": 4096, "exp_avg": 4096, "exp_avg_sq": 4096, "ids": 4096, "values": 4096, "count": 4096, "rows": 4,
            "dim": 8, "cap": 2, "param_dtype": N.MUON_F32, "grad_dtype": N.MUON_F32}
    for key, at in (("param", 4098), ("exp_avg", 4098), ("exp_avg_sq", 4098), ("ids", 4100), ("values", 4098),
                    ("count", 4100)):
        s = N.AdamwRowsSeg(**(good | {key: at}))
        assert lib.muon_adamw_rows(ctypes.byref(s), 0.9, 0.95, 1e-8, 1.0, None, None) == N.MUON_ERR_ARG, key
        assert "aligned" in N.last_error()
    s = N.AdamwRowsSeg(**good)
    assert lib.muon_adamw_rows(ctypes.byref(s), 0.9, 0.95, 1e-8, 1.0, two, None) == N.MUON_ERR_ARG
