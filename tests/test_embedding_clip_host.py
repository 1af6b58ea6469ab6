"""Host logic of the embedding, list-clipping and row-gradient AdamW entry points, with the device faked."""

import contextlib
import ctypes
import random
import threading
import time

import pytest
import torch
from torch.autograd import forward_ad as fw

from opendm_b200 import embedding as E
from opendm_b200 import optimizer as O
from opendm_b200.build import build
from opendm_b200.engine import CudaMuonEngine
from opendm_b200.optimizer import functional
from opendm_b200.optimizer import MuonAdamW, mark_muon_parameters


class _Word:
    """E._ErrorWord without a GPU: the device's word is a host tensor, a queued copy is there at once."""

    class Event:
        def query(self):
            return True

    def __init__(self, code=0):
        self.word, self.host, self.event = torch.tensor([code]), torch.zeros(1, dtype=torch.int32), None
        self.pointer = 0

    def queue_copy(self):
        self.host.copy_(self.word)
        self.event = self.Event()


class _Library:
    def __init__(self, word):
        self.word = word

    def muon_read_error(self, pointer, code, stream):
        found = int(self.word.word)
        ctypes.cast(code, ctypes.POINTER(ctypes.c_int))[0] = found
        self.word.word.zero_()
        return E.N.MUON_ERR_KERNEL if found else E.N.MUON_OK

    def muon_last_error(self):
        return b"token id out of range"


@pytest.fixture
def word(monkeypatch):
    w = _Word(E.N.MUON_DEV_BAD_INDEX)
    lib = _Library(w)
    monkeypatch.setattr(E.N, "lib", lambda: lib)
    monkeypatch.setattr(E, "_WORDS", {0: w})
    monkeypatch.setattr(E, "raw_stream", lambda index: 0)
    monkeypatch.setattr(torch.cuda, "device", lambda index: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "synchronize", lambda: None)
    return w


def test_a_reported_token_id_error_is_not_raised_again(word):
    device = torch.device("cuda", 0)
    word.queue_copy()
    with pytest.raises(RuntimeError, match="out of range"):
        E.check_errors(0)
    E.check_errors(0)
    E.poll_errors(device)  # the copy queued before is of the error already raised
    word.word.fill_(E.N.MUON_DEV_BAD_INDEX)  # the next one is raised once too
    word.queue_copy()
    with pytest.raises(RuntimeError, match="out of range"):
        E.poll_errors(device)
    E.poll_errors(device)
    E.check_errors(0)


def _sparse_model():
    m = torch.nn.Module()
    m.embed = torch.nn.Embedding(10, 4, sparse=True)
    m.layer = torch.nn.Linear(4, 4, bias=False)
    mark_muon_parameters(m, predicate=lambda n, p: "layer" in n)
    return m, MuonAdamW(m, lr=1e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.0, sparse_grads=True)


@pytest.mark.parametrize("closure", [False, True])
def test_a_step_that_raises_drops_its_clip(closure):
    m, opt = _sparse_model()
    opt._pending_clip = torch.tensor([2.0, 0.5])

    def fail():
        raise RuntimeError("CUDA")

    m.embed(torch.tensor([1, 2])).sum().backward()
    with pytest.raises(RuntimeError, match="CUDA"):  # in the closure, or in the merge, which has no CPU path
        opt.step(fail) if closure else opt.step()
    assert opt._pending_clip is None


def _formula(ids, weight, scale, out_dtype):
    with torch.no_grad():
        return (weight.detach()[ids].float() * scale).to(out_dtype)


def test_the_lookup_has_a_forward_mode_derivative(monkeypatch):
    monkeypatch.setattr(E, "_lookup", _formula)
    w, t = torch.randn(7, 3), torch.randn(7, 3)
    ids = torch.tensor([[1, 6], [1, 0]])
    for requires in (False, True):
        w.requires_grad_(requires)
        with fw.dual_level():
            primal, tangent = fw.unpack_dual(E.embedding(ids, fw.make_dual(w, t), scale=2.0, padding_idx=1))
            assert torch.equal(primal, w[ids] * 2) and torch.equal(tangent, t[ids] * 2)
            assert fw.unpack_dual(E.embedding(ids, w)).tangent is None
    # a tangent that requires grad keeps its graph
    t.requires_grad_()
    with fw.dual_level():
        tangent = fw.unpack_dual(E.embedding(ids, fw.make_dual(w.detach(), t))).tangent
        assert tangent.requires_grad
        with torch.no_grad():
            assert torch.equal(fw.unpack_dual(E.embedding(ids, fw.make_dual(w.detach(), t.detach()))).tangent, t[ids])


def test_gradients_record_no_derivatives():
    g, ids = torch.zeros(3, 8, requires_grad=True), torch.zeros(3, dtype=torch.long)
    for call in (E.embedding_grad, E.embedding_row_grad):
        with pytest.raises(RuntimeError, match="no derivatives"):
            call(g, ids, 4)
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):  # gets as far as the device check
            call(g, ids, 4)
        with fw.dual_level(), torch.no_grad(), pytest.raises(RuntimeError, match="no derivatives"):
            call(fw.make_dual(g.detach(), torch.ones(3, 8)), ids, 4)
    with fw.dual_level(), pytest.raises(RuntimeError, match="no forward-mode"):  # as a backward pass asks for it
        E._gradient(fw.make_dual(g.detach(), torch.ones(3, 8)), ids, 4, 1.0, None, None, as_rows=False)


def test_writes_by_pointer_bump_version_counters(monkeypatch):
    monkeypatch.setattr(functional, "_apply", lambda grads, *_: torch.tensor(1.0))
    a, b, out = torch.ones(3, 4), torch.ones(4, 6)[:, ::2], torch.ones(3, 4)
    O.clip_grads([a, b], 1.0)
    assert a._version == 1 and b._version >= 1 and b._base._version == b._version
    O.clip_grads([a], 1.0, out=[out])
    assert a._version == 1 and out._version == 1
    p = torch.nn.Parameter(torch.ones(3, 4))
    p.grad = a
    O.clip_grad_norm_([p], 1.0)
    O.clip_grads_with_norm_(p, 1.0, torch.tensor(2.0))
    assert a._version == 3 and p._version == 0
    p.grad = torch.sparse_coo_tensor([[0, 2]], torch.ones(2, 4), (3, 4))
    O.clip_grads_with_norm_(p, 1.0, torch.tensor(2.0))
    assert p.grad._version == 1
    x = torch.ones(3, requires_grad=True)
    g, = torch.autograd.grad((x ** 3).sum(), x, create_graph=True)
    y = (g ** 2).sum()
    with torch.no_grad():
        O.clip_grads([g], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.fixture
def adam_items(monkeypatch):
    """The items that adamw hands to its engine."""
    seen = []

    class Engine:
        def adamw(self, items, **_):
            seen.extend(items)

    monkeypatch.setattr(functional, "device_index", lambda t: 0)
    monkeypatch.setattr(functional, "on_device", lambda index, call: call())
    monkeypatch.setattr(functional, "engine_for", lambda *_: Engine())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return seen


ADAM = dict(lr=0.1, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.0)


def test_adamw_bumps_version_counters(adam_items):
    p, g, m, v = torch.nn.Parameter(torch.ones(3)), torch.ones(3), torch.zeros(3), torch.zeros(3)
    y = (p ** 2).sum()
    O.adamw([p], [g], [m], [v], [1], lr=0.1, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.0)
    assert [t._version for t in (p, g, m, v)] == [1, 0, 1, 1]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_clipping_refuses_derivatives(monkeypatch):
    monkeypatch.setattr(functional, "_apply", lambda grads, *_: torch.tensor(1.0))
    g, r, out = torch.ones(3), torch.ones(3, requires_grad=True), torch.ones(3)
    for grads, outs in (([g, r], None), ([r], [out]), ([g], [r]), ([r * 2], None)):
        with pytest.raises(RuntimeError, match="no derivatives"):
            O.clip_grads(grads, 1.0, out=outs)
        with torch.no_grad():
            O.clip_grads(grads, 1.0, out=outs)
    p = torch.nn.Parameter(torch.ones(3))
    p.grad = r * 2  # as backward(create_graph=True) leaves it: torch clips it too
    O.clip_grad_norm_(p, 1.0)
    with fw.dual_level():
        dual = fw.make_dual(torch.ones(3), torch.ones(3))
        O.clip_grads([g], 1.0)
        for call in (lambda: O.clip_grads([g, dual], 1.0), lambda: O.clip_grads([g], 1.0, out=[dual]),
                     lambda: O.get_total_norm([g, dual]),
                     lambda: O.adamw([dual], [g], [g], [g], [1], lr=0.1, beta1=0.9, beta2=0.95, eps=1e-8,
                                     weight_decay=0.0),
                     lambda: O.adamw([p], [E.RowGrad(3, g, dual)], [g], [g], [1], lr=0.1, beta1=0.9, beta2=0.95,
                                     eps=1e-8, weight_decay=0.0)):
            with pytest.raises(RuntimeError, match="derivative"):
                call()


def test_a_step_keeps_its_clip_coefficient_to_its_thread():
    engine = object.__new__(CudaMuonEngine)
    engine._local = threading.local()
    seen = []
    engine.grad_scale = 0.5
    other = threading.Thread(target=lambda: seen.append(engine.grad_scale))
    other.start()
    other.join()
    assert seen == [None] and engine.grad_scale == 0.5


def test_threads_that_make_the_first_call_share_one_error_word(monkeypatch):
    class Library:
        def muon_device_check(self, index):
            return E.N.MUON_OK

    class Stream:
        def synchronize(self):
            time.sleep(0.05)

    class Slow:
        def __init__(self, device):
            time.sleep(0.05)

    monkeypatch.setattr(E.N, "lib", lambda: Library())
    monkeypatch.setattr(E, "_WORDS", {})
    monkeypatch.setattr(E, "_ErrorWord", Slow)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda index: Stream())
    words = []
    threads = [threading.Thread(target=lambda: words.append(E._error_word(0))) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(words) == 4 and len(set(map(id, words))) == 1 and E._WORDS[0] is words[0]


def test_adamw_lists_may_not_share_memory(adam_items):
    empty = [torch.zeros(0) for _ in range(2)]
    O.adamw(empty, empty, empty, empty, [1, 1], **ADAM)
    O.adamw([empty[0], empty[0]], empty, empty, empty, [1, 1], **ADAM)
    assert len(adam_items) == 4
    buf = torch.zeros(12 * 6)
    p, q, m, n, v, w, g, h = buf.view(12, 6)[:8]
    ids = torch.zeros(1, dtype=torch.long)

    def call(params=(p, q), grads=(g, h), exp_avgs=(m, n), exp_avg_sqs=(v, w)):
        O.adamw(list(params), list(grads), list(exp_avgs), list(exp_avg_sqs), [1, 1], **ADAM)

    call()  # neighbours in one buffer
    call(grads=(g, g))  # what is only read may be shared
    call(grads=(buf[36:48].view(6, 2)[:, 0], buf[0:12].view(6, 2)[:, 1]))  # read through a copy
    del adam_items[:]
    for bad in ({"params": (p, p)}, {"params": (p, buf[3:9])}, {"params": (buf[3:9], p)}, {"exp_avgs": (m, m)},
                {"exp_avgs": (m, v)}, {"exp_avg_sqs": (v, buf[31:37])}, {"grads": (g, q)}, {"grads": (buf[3:9], h)},
                {"grads": (g, E.RowGrad(1, ids, buf[2:8].view(1, 6)))},
                {"params": (p, torch.zeros(6).view(2, 3)), "grads": (g, E.RowGrad(2, ids, buf[1:4].view(1, 3)))}):
        with pytest.raises(ValueError, match="share memory"):
            call(**({"params": (p, q)} | bad))
    assert not adam_items


def _addresses(t):
    at = torch.zeros((), dtype=torch.long)
    for size, stride in zip(t.shape, t.stride()):
        at = at[..., None] + torch.arange(size) * stride
    at = t.data_ptr() + at.reshape(-1) * t.element_size()
    return (at[:, None] + torch.arange(t.element_size())).reshape(-1)


def test_overlaps_of_strided_tensors_are_found_exactly():
    """Against all addresses, over random views of one buffer."""
    rng = random.Random(1)
    raw = torch.zeros(4000, dtype=torch.uint8)
    met = 0
    for _ in range(3000):
        a, b = (torch.as_strided(raw.view(rng.choice([torch.bfloat16, torch.float32])), shape, stride, offset)
                for shape, stride, offset in
                [([rng.randint(1, 5) for _ in range(d)], [rng.choice([1, 2, 3, 5, 8, 40]) for _ in range(d)],
                  rng.randint(0, 60)) for d in (rng.randint(0, 3), rng.randint(0, 3))])
        want = bool(torch.isin(_addresses(a), _addresses(b)).any())
        assert functional._meet(a, b) == want == functional._meet(b, a)
        assert functional._meet(a) == (_addresses(a).unique().numel() < _addresses(a).numel())
        met += want
    assert 300 < met < 2700


def test_overlapping_strided_gradients_are_refused(monkeypatch):
    monkeypatch.setattr(functional, "_apply", lambda grads, *_: torch.tensor(1.0))
    buf = torch.ones(20, 12)
    O.clip_grads([buf[:, :4], buf[:, 4:7], buf[:, 7:]], 1.0)
    O.clip_grads([buf[::2], buf[1::2]], 1.0)
    O.clip_grads([buf[:, ::2].t(), buf[:, 1::2]], 1.0)
    O.clip_grads([buf[:, :0], buf[:, :4]], 1.0)
    out = torch.ones(20, 12)
    for grads, outs in (([buf[:, :4], buf[:, 2:6]], None), ([buf[:, :4], buf[3]], None), ([buf, buf[:, 3:5]], None),
                        ([buf[:, :4].t(), buf[:, 3:]], None), ([buf[::2], buf[4]], None),
                        ([torch.ones(20, 4)] * 2, [out[:, :4], out[:, 3:7]]),
                        ([torch.ones(20, 4)] * 2, [out[:, :4]] * 2),
                        ([torch.ones(8, 3)], [out.view(-1).as_strided((8, 3), (2, 1))])):
        with pytest.raises(RuntimeError, match="overlap"):
            O.clip_grads(grads, 1.0, out=outs)
    p = torch.nn.Parameter(torch.ones(20, 4))
    p.grad = buf[:, :4]
    O.clip_grads_with_norm_(p, 1.0, buf[0, 4])
    with pytest.raises(RuntimeError, match="overlap"):
        O.clip_grads_with_norm_(p, 1.0, buf[0, 3])
    with pytest.raises(RuntimeError, match="expanded"):
        O.clip_grads([torch.ones(1).expand(5)], 1.0)


def test_adamw_of_dense_gradients_is_not_captured(adam_items, monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    p, q, g, m, n, v, w = (torch.zeros(4, 2) for _ in range(7))
    rows = E.RowGrad(4, torch.zeros(1, dtype=torch.long), torch.zeros(1, 2))
    O.adamw([p], [rows], [m], [v], [1], **ADAM)
    assert len(adam_items) == 1
    with pytest.raises(RuntimeError, match="captured"):
        O.adamw([p, q], [rows, g], [m, n], [v, w], [1, 1], **ADAM)
    assert len(adam_items) == 1


def test_row_update_buffers_may_not_share_memory():
    build()
    lib = E.N.lib()
    at = {"param": 1 << 20, "exp_avg": 2 << 20, "exp_avg_sq": 3 << 20, "ids": 4 << 20, "values": 5 << 20,
          "count": 6 << 20}

    def refused(scale=7 << 20, **moved):
        seg = E.N.AdamwRowsSeg(**(at | {"rows": 4, "dim": 8, "cap": 2, "param_dtype": E.N.MUON_F32,
                                        "grad_dtype": E.N.MUON_F32} | moved))
        code = lib.muon_adamw_rows(ctypes.byref(seg), 0.9, 0.95, 1e-8, 1.0, scale, None)
        return code == E.N.MUON_ERR_ARG and "share memory" in E.N.last_error()

    for written in ("param", "exp_avg", "exp_avg_sq"):  # 4 x 8 fp32 each
        for other, size in (("param", 128), ("exp_avg", 128), ("exp_avg_sq", 128), ("ids", 16), ("values", 64),
                            ("count", 8)):
            if other != written:
                assert refused(**{other: at[written] + 120}) and refused(**{other: at[written] - size + 8})
        assert refused(scale=at[written] + 124)
    seg = E.N.AdamwRowsSeg(**(at | {"rows": 4, "dim": 1 << 30, "cap": (1 << 31) - 1, "param_dtype": E.N.MUON_F32,
                                    "grad_dtype": E.N.MUON_F32}))
    assert lib.muon_adamw_rows(ctypes.byref(seg), 0.9, 0.95, 1e-8, 1.0, None, None) == E.N.MUON_ERR_ARG


def test_an_engine_is_not_made_inside_a_capture(monkeypatch):
    from opendm_b200 import engine

    monkeypatch.setattr(engine, "_ENGINES", {})
    monkeypatch.setattr(engine, "CudaMuonEngine", lambda *_: "engine")
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="before capturing"):
        engine.engine_for(torch.device("cuda", 0), "fp16")
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    assert engine.engine_for(torch.device("cuda", 0), "fp16") == "engine"
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    assert engine.engine_for(torch.device("cuda", 0), "fp16") == "engine"
