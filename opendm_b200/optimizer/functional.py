"""Gradient norm, clipping and AdamW over lists of tensors.

``clip_grad_norm_``, ``get_total_norm`` and ``clip_grads_with_norm_`` take the
arguments of their ``torch.nn.utils`` namesakes; ``clip_grads`` is the form
over the gradients themselves, in place or into other tensors (fp32
accumulators into bf16 gradients, say). Norms of type 1, 2 and inf; the norm is
returned in fp32 whatever the gradients' dtype, sums are held in fp32 and
double, and a clipped gradient is rounded once. (``MuonAdamW.clip_grad_norm_``
is the form that folds the clip into the optimizer's step, with torch's
roundings.) ``adamw`` is the optimizer's fused AdamW over lists, for dense
gradients and for row gradients (``opendm_b200.embedding.RowGrad``).

All run sm_100a kernels on the current stream of the tensors' device; CPU
tensors raise. Nothing is read back unless asked for (``error_if_nonfinite``),
and the norm and clipping calls can be captured into a CUDA graph. What a call
writes counts as changed in place for autograd: a backward pass that saved the
old values raises.
"""

from __future__ import annotations

import math
from array import array
from collections.abc import Iterable
from itertools import chain
from operator import attrgetter, or_

import torch
from torch.autograd.graph import increment_version

from .. import _native as N
from ..embedding import (RowGrad, device_index, embedding_row_grad, has_tangent, in_dual_level, on_device, raw_stream,
                         refuse_derivatives)
from ..engine import AdamItem, engine_for

_CODE = {torch.bfloat16: N.MUON_BF16, torch.float32: N.MUON_F32}
# The lists are long and each call is short: what is asked of every tensor goes through map.
_POINTER, _NUMEL, _DEVICE = torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.get_device
_CONTIGUOUS, _SIZE = torch.Tensor.is_contiguous, torch.Tensor.size
_DTYPE, _NBYTES = attrgetter("dtype"), attrgetter("nbytes")
_NORMS = {2.0: N.MUON_NORM_2, 1.0: N.MUON_NORM_1, math.inf: N.MUON_NORM_INF}


def _norm_kind(norm_type: float) -> int:
    kind = _NORMS.get(float(norm_type))
    if kind is None:
        raise ValueError(f"norm_type must be 1, 2 or inf, got {norm_type}")
    return kind


def _dense_storage(t: torch.Tensor) -> bool:
    """True when the tensor's elements fill one block of memory, in any order."""
    if t.layout is not torch.strided:
        raise RuntimeError(f"gradients must be dense tensors, got layout {t.layout}")
    if t.is_contiguous():
        return True
    expect = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != expect:
            return False
        expect *= size
    return True


def _steps(a: torch.Tensor, b: torch.Tensor) -> list[tuple[int, int, int]]:
    """Per stride in bytes, descending, the least and greatest step between an element of ``a`` and one of ``b``."""
    reach: dict[int, list[int]] = {}
    for t, side in ((a, 0), (b, 1)):
        for stride, size in zip(t.stride(), t.shape):
            if size > 1:
                ends = reach.setdefault(stride * t.element_size(), [0, 0])
                ends[side] += (size - 1) * (1 if side else -1)
    return [(stride, *reach[stride]) for stride in sorted(reach, reverse=True)]


def _meet(a: torch.Tensor, b: torch.Tensor | None = None) -> bool:
    """Whether elements of two strided tensors share memory, or, of one alone, two different elements.

    Elements i of a and j of b do where the distance of their addresses,
    b - a + sum of (steps x stride), lies in (-size of b's, size of a's): a
    search over the steps of each stride, widest first, that drops what the
    narrower ones cannot bring back. Views of one buffer leave it two or three
    choices a stride; past 10000 it gives up and answers yes."""
    same = b is None
    b = a if same else b
    steps, left = _steps(a, b), 10000
    if same and (sum(n > 1 for n in a.shape) > len(steps) or steps and steps[-1][0] == 0):
        return True  # two dimensions of one stride, or one that does not move
    narrower = [(0, 0)]  # what the strides behind each one reach
    for stride, low, high in reversed(steps):
        narrower.append((narrower[-1][0] + stride * low, narrower[-1][1] + stride * high))
    narrower.reverse()

    def search(k: int, low: int, high: int, moved: bool) -> bool:  # can steps k on sum to [low, high]?
        nonlocal left
        left -= 1
        if left < 0:
            return True
        if k == len(steps):
            return low <= 0 <= high and moved
        stride, least, most = steps[k]
        if stride == 0:
            return search(k + 1, low, high, moved)
        down, up = narrower[k + 1]
        first, last = max(least, -((up - low) // stride)), min(most, (high - down) // stride)
        return any(search(k + 1, low - x * stride, high - x * stride, moved or x != 0) for x in range(first, last + 1))

    apart = b.data_ptr() - a.data_ptr()
    return search(0, 1 - b.element_size() - apart, a.element_size() - 1 - apart, not same)


def _check_overlap(outs: list[torch.Tensor]) -> None:
    """Raise where two of the tensors share memory, or two elements of one do."""
    spans = []  # address behind the last byte, tensor; of those before that may still be met
    for t in sorted((t for t in outs if t.numel()), key=_POINTER):
        begin = t.data_ptr()
        if not t.is_contiguous() and _meet(t):
            raise RuntimeError("a tensor whose elements overlap in memory cannot be clipped into")
        spans = [(end, other) for end, other in spans if end > begin]
        if any(_meet(other, t) for _, other in spans):
            raise RuntimeError("clipped gradients overlap in memory")
        reach = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
        spans.append((begin + (reach + 1) * t.element_size(), t))


def _check_grads(grads: list[torch.Tensor], what: str) -> int:
    """Device index of the list; raises where a tensor is on another."""
    index = device_index(grads[0])
    if set(map(_DEVICE, grads)) != {index}:
        raise RuntimeError(f"{what} must be on one device")
    return index


def _codes(grads: list[torch.Tensor]) -> list[int]:
    kinds = list(map(_DTYPE, grads))
    if kinds.count(kinds[0]) == len(kinds) and kinds[0] in _CODE:  # one dtype, the usual case
        return [_CODE[kinds[0]]] * len(kinds)
    codes = list(map(_CODE.get, kinds))
    if None in codes:
        raise RuntimeError(f"unsupported dtype {kinds[codes.index(None)]}: the kernels take bfloat16 or float32")
    return codes


def _table(src: list[torch.Tensor], dst: list[torch.Tensor] | None) -> array:
    """The list as muon_clip_seg structures: two pointers, the size and the two 32-bit dtypes of each."""
    flat = [0] * (4 * len(src))
    pointers, codes = list(map(_POINTER, src)), _codes(src)
    flat[0::4] = pointers
    flat[2::4] = map(_NUMEL, src)
    flat[3::4] = codes
    if dst is not None:
        flat[1::4] = pointers if dst is src else map(_POINTER, dst)
        out_codes = codes if dst is src else _codes(dst)
        flat[3::4] = map(or_, codes, [c << 32 for c in out_codes])
    return array("q", flat)


def _unique(tensors: Iterable[torch.Tensor]) -> list[torch.Tensor]:
    seen: set[int] = set()
    return [t for t in tensors if not (id(t) in seen or seen.add(id(t)))]


def _workspace(grads: list[torch.Tensor]) -> torch.Tensor:
    return grads[0].new_empty(N.lib().muon_clip_workspace_bytes(len(grads)), dtype=torch.uint8)


def _raise_nonfinite(total: torch.Tensor, norm_type: float) -> None:
    if not torch.isfinite(total).item():
        raise RuntimeError(f"The total norm of order {float(norm_type)} for gradients from `parameters` is "
                           "non-finite, so it cannot be clipped. To disable this error and scale the "
                           "gradients by the non-finite norm anyway, set `error_if_nonfinite=False`")


def get_total_norm(tensors: torch.Tensor | Iterable[torch.Tensor], norm_type: float = 2.0,
                   error_if_nonfinite: bool = False, foreach: bool | None = None) -> torch.Tensor:
    """Norm of all elements of ``tensors`` together, a 0-d fp32 tensor.
    ``foreach`` is accepted for torch's signature and changes nothing."""
    kind = _norm_kind(norm_type)
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if has_tangent(tensors):
        raise RuntimeError("the norm of a list has no forward-mode derivative")
    if not tensors:
        return torch.tensor(0.0)
    index = _check_grads(tensors, "tensors")
    if not all(map(_CONTIGUOUS, tensors)):
        tensors = [t if _dense_storage(t) else t.contiguous() for t in tensors]

    def call():
        total = tensors[0].new_empty((), dtype=torch.float32)
        table, work = _table(tensors, None), _workspace(tensors)
        N.check(N.lib().muon_total_norm(table.buffer_info()[0], len(tensors), kind, work.data_ptr(), total.data_ptr(),
                                        raw_stream(index)), "muon_total_norm")
        return total

    total = on_device(index, call)
    if error_if_nonfinite:
        _raise_nonfinite(total, norm_type)
    return total


def _apply(grads: list[torch.Tensor], outs: list[torch.Tensor], max_norm: float, norm_type: float | None,
           total: torch.Tensor | None) -> torch.Tensor:
    """Norm (unless given) and scaling of dense-storage tensors."""
    index = _check_grads(grads, "gradients")
    if outs is not grads and _check_grads(outs, "outputs") != index:
        raise RuntimeError("gradients and outputs must be on one device")

    def call():
        lib, stream = N.lib(), raw_stream(index)
        table = _table(grads, outs)
        if total is not None:
            N.check(lib.muon_scale_grads(table.buffer_info()[0], len(grads), max_norm, total.data_ptr(), stream),
                    "muon_scale_grads")
            return total
        norm = grads[0].new_empty((), dtype=torch.float32)
        work = _workspace(grads)
        N.check(lib.muon_clip_grads(table.buffer_info()[0], len(grads), _norm_kind(norm_type), max_norm,
                                    work.data_ptr(), norm.data_ptr(), stream), "muon_clip_grads")
        return norm

    return on_device(index, call)


def _max_norm(max_norm: float) -> float:
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"max_norm must be >= 0, got {max_norm}")
    return max_norm


def _clip(grads: list[torch.Tensor], outs: list[torch.Tensor] | None, max_norm: float, norm_type: float | None,
          total: torch.Tensor | None) -> torch.Tensor:
    if outs is None:
        outs = grads
    else:
        refuse_derivatives("gradient clipping", outs)
    refuse_derivatives("gradient clipping", grads)
    if all(map(_CONTIGUOUS, grads)) and (outs is grads or all(map(_CONTIGUOUS, outs))):
        norm = _apply(grads, outs, max_norm, norm_type, total)
        increment_version(outs)  # autograd has to see what was written by pointer
        return norm
    # Other strides: elementwise work needs only that both sides agree on the
    # order of elements, else a contiguous copy is scaled and copied back, past
    # the library's own check of overlaps.
    src, dst, back = [], [], []
    for g, o in zip(grads, outs):
        dense, _ = _dense_storage(g), _dense_storage(o)
        if any(n > 1 and s == 0 for s, n in zip(o.stride(), o.shape)):
            raise RuntimeError("an expanded tensor cannot be clipped in place: several elements share memory")
        if g.stride() == o.stride() and dense:
            src.append(g)
            dst.append(o)
            continue
        src.append(g.contiguous())
        if o.is_contiguous():
            dst.append(o)
        else:
            dst.append(torch.empty(o.shape, dtype=o.dtype, device=o.device))
            back.append((o, dst[-1]))
    if back:
        _check_overlap(outs if total is None else [*outs, total])
    norm = _apply(src, dst, max_norm, norm_type, total)
    with torch.no_grad():
        for o, d in back:
            o.copy_(d)
    increment_version(outs)
    return norm


def clip_grads(grads: Iterable[torch.Tensor], max_norm: float, *, norm_type: float = 2.0,
               out: Iterable[torch.Tensor] | None = None) -> torch.Tensor:
    """Scale ``grads`` by min(max_norm / (total + 1e-6), 1), in place or into
    ``out`` (same shapes, bfloat16 or float32 each), and return the total
    norm of ``grads``, a 0-d fp32 tensor. In place, a tensor that appears
    twice counts and is scaled once. Nothing is recorded for autograd:
    tensors that require grad are refused outside of ``torch.no_grad()``."""
    max_norm = _max_norm(max_norm)
    _norm_kind(norm_type)
    grads = list(grads)
    if out is None:
        grads = _unique(grads)
    else:
        out = list(out)
        if len(out) != len(grads) or list(map(_SIZE, out)) != list(map(_SIZE, grads)):
            raise ValueError("out must match the gradients in number and shapes")
    if not grads:
        return torch.tensor(0.0)
    return _clip(grads, out, max_norm, norm_type, None)


def _parameter_grads(parameters) -> list[torch.Tensor]:
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else parameters
    return _unique(p.grad for p in _unique(parameters) if p.grad is not None)


def _merged(grad: torch.Tensor) -> torch.Tensor:
    """Values of a sparse gradient with each row's entries added up."""
    return rows_of(grad).values


def rows_of(grad: torch.Tensor) -> RowGrad:
    """A sparse COO gradient (sparse in its first dimension) as a RowGrad:
    entries of the same row, as accumulated passes or ``nn.Embedding(sparse=
    True)`` leave them, are added by the sorted-token kernel."""
    if grad.layout is not torch.sparse_coo or grad.sparse_dim() != 1 or grad.dense_dim() < 1:
        raise RuntimeError("sparse gradients must be COO tensors, sparse in their first dimension only")
    ids, values = grad._indices()[0], grad._values()
    if grad.is_coalesced():
        return RowGrad(grad.shape[0], ids.contiguous(), values.contiguous())
    flat = values.reshape(values.shape[0], math.prod(values.shape[1:]))
    rows = embedding_row_grad(flat, ids, grad.shape[0])
    rows.values = rows.values.view(rows.values.shape[0], *values.shape[1:])
    return rows


@torch.no_grad()
def clip_grad_norm_(parameters: torch.Tensor | Iterable[torch.Tensor], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False, foreach: bool | None = None) -> torch.Tensor:
    """``torch.nn.utils.clip_grad_norm_`` in two kernel launches: clips the
    parameters' gradients in place and returns their total norm (fp32). A
    sparse COO gradient counts with its entries of one row added up, and has
    its values scaled."""
    max_norm = _max_norm(max_norm)
    _norm_kind(norm_type)
    grads = _parameter_grads(parameters)
    if not grads:
        return torch.tensor(0.0)
    sparse = any(g.layout is not torch.strided for g in grads)
    if not sparse and not error_if_nonfinite:
        return _clip(grads, None, max_norm, norm_type, None)
    total = get_total_norm([g if g.layout is torch.strided else _merged(g) for g in grads], norm_type,
                           error_if_nonfinite)
    _clip([g if g.layout is torch.strided else g._values() for g in grads], None, max_norm, None, total)
    return total


@torch.no_grad()
def clip_grads_with_norm_(parameters: torch.Tensor | Iterable[torch.Tensor], max_norm: float,
                          total_norm: torch.Tensor, foreach: bool | None = None) -> None:
    """Scale the parameters' gradients in place by min(max_norm / (total_norm
    + 1e-6), 1), for a norm known already (one reduced over ranks, say).
    ``total_norm``: a one-element fp32 tensor on the gradients' device, in
    memory of its own."""
    max_norm = _max_norm(max_norm)
    grads = _parameter_grads(parameters)
    if not grads:
        return
    if total_norm.numel() != 1 or total_norm.dtype != torch.float32 or total_norm.device != grads[0].device:
        raise RuntimeError("total_norm must be one float32 value on the gradients' device")
    _clip([g if g.layout is torch.strided else g._values() for g in grads], None, max_norm, None, total_norm)


def _shares_memory(written: list[torch.Tensor], read: list[torch.Tensor]) -> bool:
    """Whether a written contiguous tensor overlaps another written or read one."""
    tensors = written + read
    kinds = [True] * len(written) + [False] * len(read)
    spans = sorted(span for span in zip(map(_POINTER, tensors), map(_NBYTES, tensors), kinds) if span[1])
    end = written_end = 0  # of the spans before
    for begin, size, writes in spans:
        if begin < (end if writes else written_end):
            return True
        end = max(end, begin + size)
        if writes:
            written_end = end
    return False


def _tensors_of(grad) -> tuple:
    return (grad.ids, grad.values) if isinstance(grad, RowGrad) else (grad,) if isinstance(grad, torch.Tensor) else ()


def adamw(params: list[torch.Tensor], grads: list, exp_avgs: list[torch.Tensor], exp_avg_sqs: list[torch.Tensor],
          steps: list[float], *, lr: float, beta1: float, beta2: float, eps: float, weight_decay: float) -> None:
    """One AdamW update of each parameter, in place with its fp32 moments
    (``MuonAdamW``'s AdamW group, decoupled weight decay). ``grads``: dense
    tensors, or RowGrads for parameters whose gradient is zero outside some
    rows: the same results at the cost of those rows. ``steps``: the step
    count of each, this step included. What is written may share memory with
    nothing else in the lists; empty parameters may be listed any number of
    times. With RowGrads only, a call can be captured into a graph (which
    keeps its step size); with dense gradients it raises there."""
    if not len(params) == len(grads) == len(exp_avgs) == len(exp_avg_sqs) == len(steps):
        raise ValueError("adamw lists must have one entry per parameter")
    if not params:
        return
    if min(steps) < 1:
        raise ValueError("adamw steps count from 1")
    written = [*params, *exp_avgs, *exp_avg_sqs]
    if in_dual_level() and has_tangent(chain(written, chain.from_iterable(map(_tensors_of, grads)))):
        raise RuntimeError("adamw has no forward-mode derivative")
    dense = False
    for p, g, m, v in zip(params, grads, exp_avgs, exp_avg_sqs):
        if isinstance(g, RowGrad):
            continue  # checked by the engine
        dense = True
        if not isinstance(g, torch.Tensor) or g.layout is not torch.strided or g.shape != p.shape:
            raise RuntimeError("adamw takes a dense gradient of its parameter's shape, or a RowGrad")
        if any(t.dtype != torch.float32 or t.shape != p.shape or not t.is_contiguous() for t in (m, v)):
            raise RuntimeError("AdamW moments must be contiguous float32 tensors of their parameter's shape")
    index = device_index(params[0])
    if dense or len(params) > 1:  # the tensors of one row update are checked by the library
        reads = chain.from_iterable(map(_tensors_of, grads))
        if _shares_memory(written, [t for t in reads if t.is_contiguous()]):  # others are copied
            raise ValueError("adamw parameters and moments must be distinct: no two of them, and no gradient, may "
                             "share memory")
    items = list(map(AdamItem, params, grads, exp_avgs, exp_avg_sqs, map(float, steps)))

    def call():
        if dense and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("adamw of dense gradients uploads a table, which a captured graph would read again: "
                               "it cannot be captured")
        engine_for(params[0].device, "fp16").adamw(items, lr=float(lr), beta1=float(beta1), beta2=float(beta2),
                                                   eps=float(eps), weight_decay=float(weight_decay))

    on_device(index, call)
    increment_version(written)
