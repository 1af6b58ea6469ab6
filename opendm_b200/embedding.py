"""Token embedding with scaling, and its gradient by sorted tokens.

    out[t] = round(scale * weight[ids[t]])
    dW[v]  = round(scale * sum of dOut[t] over the tokens t with ids[t] == v)

The embedding is the largest tensor of the optimizer's AdamW group, and its
gradient is zero outside the rows of the step's tokens. ``embedding`` and
``ScaledEmbedding`` give that gradient either as a dense tensor or, with
``sparse=True``, as a sparse COO tensor that
``MuonAdamW(..., sparse_grads=True)`` takes: the dense gradient is then
neither written by the backward pass nor read by the norm and AdamW.

The functions run the sm_100a kernels of ``libopendm_muon.so`` on the current
stream of the tensors' device; there is no CPU path (CPU tensors raise). Sums
are fp32, in an order fixed by the sorted tokens: two calls give the same bits.
Tensors are bfloat16 or float32, ids int64 or int32.

An id outside the vocabulary does not fault: its row of the lookup is zeros,
the gradient leaves it out, and the device's error word is set, which
``check_errors()`` (or ``MuonAdamW.check_device_errors()``, or a later
``MuonAdamW.step()`` with ``sparse_grads=True``) turns into a ``RuntimeError``.
"""

from __future__ import annotations

import threading
from ctypes import byref, c_int
from dataclasses import dataclass
from operator import attrgetter

import torch
from torch.autograd import forward_ad

from . import _native as N

_FLOAT_CODE = {torch.bfloat16: N.MUON_BF16, torch.float32: N.MUON_F32}
_REQUIRES_GRAD = attrgetter("requires_grad")
_INDEX_CODE = {torch.int32: N.MUON_I32, torch.int64: N.MUON_I64}


@dataclass
class RowGrad:
    """Gradient of a ``[num_rows, ...]`` parameter that is zero outside some rows.

    ids: [cap] int64, the rows in ascending order; values: [cap, ...] their
    gradients; count: one int64 on the device, how many of them there are
    (None: all). Entries past the count have id 0 and zero values, so that
    ``ids`` and ``values`` are a valid coordinate list without reading it.
    """

    num_rows: int
    ids: torch.Tensor
    values: torch.Tensor
    count: torch.Tensor | None = None

    def to_sparse(self) -> torch.Tensor:
        """The sparse COO tensor (not marked coalesced: entries past the count repeat id 0)."""
        return torch.sparse_coo_tensor(self.ids.unsqueeze(0), self.values, (self.num_rows, *self.values.shape[1:]))


class _ErrorWord:
    """A device's error word for out-of-range ids, with a pinned copy."""

    def __init__(self, device: torch.device):
        self.word = torch.zeros(1, dtype=torch.int32, device=device)
        self.pointer = self.word.data_ptr()
        self.host = torch.zeros(1, dtype=torch.int32).pin_memory()
        self.event = None


_WORDS: dict[int, _ErrorWord] = {}
_WORDS_LOCK = threading.Lock()

# The current stream's handle: torch.cuda.current_stream(index).cuda_stream without its
# Stream object where this torch has the call (0.1 us instead of 1.2).
raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


def device_index(t: torch.Tensor) -> int:
    index = t.get_device()
    if index < 0 or not t.is_cuda:
        raise RuntimeError("opendm_b200 runs on CUDA (sm_100) tensors only; got a tensor on " + str(t.device))
    return index


def _error_word(index: int) -> _ErrorWord:
    word = _WORDS.get(index)
    if word is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the first embedding call on a device allocates its error word: make one call "
                               "before capturing a graph")
        with _WORDS_LOCK:  # kernels keep the pointer: a device's word is made once
            word = _WORDS.get(index)
            if word is None:
                N.check(N.lib().muon_device_check(index), "muon_device_check")
                word = _ErrorWord(torch.device("cuda", index))
                torch.cuda.current_stream(index).synchronize()  # zeroed before any stream uses it
                _WORDS[index] = word
    return word


def check_errors(device: torch.device | int | None = None) -> None:
    """Synchronise the device (default: all devices used) and raise if a
    lookup or gradient met an id outside its vocabulary."""
    if device is None:
        indices = list(_WORDS)
    else:
        device = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        indices = [torch.cuda.current_device() if device.index is None else device.index]
    for index in indices:
        word = _WORDS.get(index)
        if word is None:
            continue
        with torch.cuda.device(index):
            torch.cuda.synchronize()
            word.event = None  # a copy queued before shows no more than the word itself
            code = c_int(0)
            N.check(N.lib().muon_read_error(word.pointer, byref(code), raw_stream(index)), "embedding")


def record_error_check(device: torch.device) -> None:
    """Queue a copy of the device's error word for ``poll_errors``."""
    word = _WORDS.get(device.index)
    if word is not None and word.event is None:
        word.host.copy_(word.word, non_blocking=True)
        word.event = torch.cuda.Event()
        word.event.record(torch.cuda.current_stream(device))  # of the copy, whichever device is current


def poll_errors(device: torch.device) -> None:
    """Raise if a copy queued by ``record_error_check`` has arrived with an error."""
    word = _WORDS.get(device.index)
    if word is None or word.event is None or not word.event.query():
        return
    word.event = None
    code = int(word.host.item())
    if code != 0:
        word.word.zero_()
        raise RuntimeError(f"opendm_b200 embedding reported device error 0x{code:x} (token id out of range)")


def _code(table: dict, dtype: torch.dtype, what: str) -> int:
    code = table.get(dtype)
    if code is None:
        names = " or ".join(str(d).removeprefix("torch.") for d in table)
        raise RuntimeError(f"unsupported {what} dtype {dtype}: the kernels take {names}")
    return code


def in_dual_level() -> bool:
    """Whether tensors can carry forward-mode derivatives here."""
    return forward_ad._current_level >= 0


def has_tangent(tensors) -> bool:
    """Whether one of the tensors carries a forward-mode derivative."""
    return in_dual_level() and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def refuse_derivatives(what: str, tensors) -> None:
    """Raise where autograd would have to follow a call that reads or writes its tensors by pointer."""
    if torch.is_grad_enabled() and any(map(_REQUIRES_GRAD, tensors)) or has_tangent(tensors):
        raise RuntimeError(f"{what} records no derivatives: detach its tensors, or call it under torch.no_grad()")


def on_device(index: int, call, *args):
    """Run ``call`` with the device current (the usual case costs one query)."""
    if torch.cuda.current_device() == index:
        return call(*args)
    with torch.cuda.device(index):
        return call(*args)


def _lookup(ids: torch.Tensor, weight: torch.Tensor, scale: float, out_dtype: torch.dtype) -> torch.Tensor:
    index = device_index(weight)
    if torch.cuda.current_device() != index:
        with torch.cuda.device(index):
            return _lookup(ids, weight, scale, out_dtype)
    if weight.ndim != 2:
        raise ValueError("embedding weight must be 2-D")
    if ids.get_device() != index:
        raise RuntimeError(f"ids are on {ids.device}, the weight on {weight.device}")
    w_code, o_code = _FLOAT_CODE.get(weight.dtype), _FLOAT_CODE.get(out_dtype)
    i_code = _INDEX_CODE.get(ids.dtype)
    if w_code is None or o_code is None or i_code is None:
        _code(_FLOAT_CODE, weight.dtype, "weight"), _code(_FLOAT_CODE, out_dtype, "output")
        _code(_INDEX_CODE, ids.dtype, "id")
    rows, dim = weight.shape
    if not weight.is_contiguous() and (dim > 1 and weight.stride(1) != 1 or rows > 1 and weight.stride(0) < dim):
        weight = weight.contiguous()  # columns apart, or rows that share memory
    ids = ids.contiguous()
    out = weight.new_empty((*ids.shape, dim), dtype=out_dtype)
    N.check(N.lib().muon_embedding(weight.data_ptr(), w_code, rows, dim, weight.stride(0) if rows > 1 else dim,
                                   ids.data_ptr(), i_code, ids.numel(), scale, out.data_ptr(), o_code,
                                   _error_word(index).pointer, raw_stream(index)), "muon_embedding")
    return out


def _gradient(grad: torch.Tensor, ids: torch.Tensor, num_rows: int, scale: float, padding_idx: int | None,
              dtype: torch.dtype | None, as_rows: bool):
    if has_tangent((grad,)):
        raise RuntimeError("the embedding's gradient has no forward-mode derivative")
    index = device_index(grad)
    if ids.get_device() != index:
        raise RuntimeError(f"ids are on {ids.device}, the gradient on {grad.device}")
    if grad.shape[:-1] != ids.shape or grad.ndim == 0:
        raise ValueError(f"gradient of shape {tuple(grad.shape)} does not match ids of shape {tuple(ids.shape)}")
    dtype = dtype or grad.dtype
    g_code, o_code = _code(_FLOAT_CODE, grad.dtype, "gradient"), _code(_FLOAT_CODE, dtype, "result")
    i_code = _code(_INDEX_CODE, ids.dtype, "id")
    num_rows = int(num_rows)
    pad = -1 if padding_idx is None else int(padding_idx)
    if num_rows < 0 or (padding_idx is not None and not 0 <= pad < num_rows):
        raise ValueError(f"padding_idx {padding_idx} is not one of {num_rows} rows")
    return on_device(index, _launch_gradient, index, grad.contiguous(), g_code, ids.contiguous(), i_code, num_rows,
                     pad, scale, dtype, o_code, as_rows)


def _launch_gradient(index, grad, g_code, ids, i_code, num_rows, pad, scale, dtype, o_code, as_rows):
    lib = N.lib()
    dim, tokens = grad.shape[-1], ids.numel()
    need = lib.muon_embedding_grad_workspace_bytes(tokens, num_rows, dim)
    if need < 0:
        raise RuntimeError(f"embedding gradient of {tokens} tokens, {num_rows} x {dim} is out of range")
    work = grad.new_empty(need, dtype=torch.uint8)
    if as_rows:
        cap = min(tokens, num_rows)
        out = grad.new_empty((cap, dim), dtype=dtype)
        out_ids, count = grad.new_empty(cap, dtype=torch.int64), grad.new_empty(1, dtype=torch.int64)
        count_ptr = count.data_ptr()
        ids_ptr = out_ids.data_ptr() or count_ptr  # of no ids: a null pointer would ask for the dense form
    else:
        out = grad.new_empty((num_rows, dim), dtype=dtype)
        ids_ptr = count_ptr = None
    N.check(lib.muon_embedding_grad(grad.data_ptr(), g_code, ids.data_ptr(), i_code, tokens, num_rows, dim, pad, scale,
                                    out.data_ptr(), o_code, ids_ptr, count_ptr, work.data_ptr(), need,
                                    _error_word(index).pointer, raw_stream(index)), "muon_embedding_grad")
    return RowGrad(num_rows, out_ids, out, count) if as_rows else out


def embedding_grad(grad: torch.Tensor, ids: torch.Tensor, num_rows: int, *, scale: float = 1.0,
                   padding_idx: int | None = None, dtype: torch.dtype | None = None) -> torch.Tensor:
    """Dense ``[num_rows, dim]`` gradient of an embedding weight from the
    gradient ``[*ids.shape, dim]`` of its lookup; ``dtype``: of the result
    (default: the gradient's). Tokens equal to ``padding_idx`` are left out.
    Not differentiable: a gradient that requires grad is refused."""
    refuse_derivatives("embedding_grad", (grad,))
    return _gradient(grad, ids, num_rows, float(scale), padding_idx, dtype, as_rows=False)


def embedding_row_grad(grad: torch.Tensor, ids: torch.Tensor, num_rows: int, *, scale: float = 1.0,
                       padding_idx: int | None = None, dtype: torch.dtype | None = None) -> RowGrad:
    """``embedding_grad`` as the rows of the tokens only: min(tokens,
    num_rows) entries, the distinct ids first and zeros behind them. The host
    never waits for the number of distinct ids."""
    refuse_derivatives("embedding_row_grad", (grad,))
    return _gradient(grad, ids, num_rows, float(scale), padding_idx, dtype, as_rows=True)


class _EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, ids, scale, padding_idx, sparse, out_dtype):
        ctx.save_for_backward(ids)
        ctx.save_for_forward(ids)
        ctx.args = (weight.shape[0], scale, padding_idx, sparse, weight.dtype)
        ctx.out_dtype = out_dtype
        return _lookup(ids, weight, scale, out_dtype)

    @staticmethod
    def jvp(ctx, tangent, *_):  # the lookup is linear in the weight
        ids, = ctx.saved_tensors
        _, scale, padding_idx, sparse, _ = ctx.args
        return embedding(ids, tangent, scale=scale, padding_idx=padding_idx, sparse=sparse, out_dtype=ctx.out_dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        ids, = ctx.saved_tensors
        rows, scale, padding_idx, sparse, dtype = ctx.args
        out = _gradient(grad, ids, rows, scale, padding_idx, dtype, as_rows=sparse)
        return (out.to_sparse() if sparse else out), None, None, None, None, None


def embedding(ids: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0, padding_idx: int | None = None,
              sparse: bool = False, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``round(scale * weight[ids])`` of shape ``[*ids.shape, dim]``.

    The product is fp32, rounded once to ``out_dtype`` (default: the
    weight's). Differentiable in ``weight``, once in reverse mode and in
    forward mode: the gradient is dense, or a sparse COO tensor with
    ``sparse=True``; ``padding_idx`` gets none."""
    scale = float(scale)
    out_dtype = out_dtype or weight.dtype
    if padding_idx is not None and not 0 <= int(padding_idx) < weight.shape[0]:
        raise ValueError(f"padding_idx {padding_idx} is not one of {weight.shape[0]} rows")
    if torch.is_grad_enabled() and weight.requires_grad or has_tangent((weight,)):
        return _EmbeddingFn.apply(weight, ids, scale, padding_idx, bool(sparse), out_dtype)
    return _lookup(ids, weight, scale, out_dtype)


class ScaledEmbedding(torch.nn.Embedding):
    """``torch.nn.Embedding`` (same arguments, initialisation and state dict;
    no ``max_norm`` or ``scale_grad_by_freq``) whose lookup is multiplied by
    ``scale``, on the sm_100a kernels. ``out_dtype``: of the output (default:
    the weight's, which may be fp32 under a bf16 model)."""

    def __init__(self, num_embeddings: int, embedding_dim: int, padding_idx: int | None = None, *, scale: float = 1.0,
                 sparse: bool = False, out_dtype: torch.dtype | None = None, device=None, dtype=None) -> None:
        super().__init__(num_embeddings, embedding_dim, padding_idx, sparse=sparse, device=device, dtype=dtype)
        self.scale = float(scale)
        self.out_dtype = out_dtype

    @classmethod
    def from_pretrained(cls, embeddings: torch.Tensor, freeze: bool = True, padding_idx: int | None = None, *,
                        scale: float = 1.0, sparse: bool = False, out_dtype: torch.dtype | None = None):
        """``torch.nn.Embedding.from_pretrained``: a module around ``embeddings`` itself."""
        if embeddings.ndim != 2:
            raise ValueError("embeddings must be 2-D")
        module = cls(*embeddings.shape, padding_idx, scale=scale, sparse=sparse, out_dtype=out_dtype, device="meta")
        module.weight = torch.nn.Parameter(embeddings, requires_grad=not freeze)
        return module

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        return embedding(input, self.weight, scale=self.scale, padding_idx=self.padding_idx, sparse=self.sparse,
                         out_dtype=self.out_dtype)

    def extra_repr(self) -> str:
        return super().extra_repr() + f", scale={self.scale}"
