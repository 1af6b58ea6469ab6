"""GPU tests of the embedding gradient's C entry on buffers of the caller's: everything it writes is set to 0xFF bytes
before, so that a zero that was not written shows, and the bytes around it must stay as they were.

Gradients are -1, 0 or 1: every fp32 sum below 2^24 terms is exact, and rounds once to the result's type."""

import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

GUARD = 256


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)


class Guarded:
    """``size`` bytes that start ``skew`` bytes behind a 256-byte boundary, between guards."""

    def __init__(self, size, skew=0):
        self.size, self.skew = size, skew
        self.raw = torch.full((2 * GUARD + 256 + size,), 0xFF, dtype=torch.uint8, device=_dev())
        assert self.raw.data_ptr() % 256 == 0
        self.begin = GUARD + skew
        self.pointer = self.raw.data_ptr() + self.begin

    def view(self, dtype, *shape):
        if 0 in shape:
            return torch.empty(shape, dtype=dtype, device=_dev())
        return self.raw[self.begin:self.begin + self.size].clone().view(dtype).view(shape)

    def check(self):
        assert bool((self.raw[:self.begin] == 0xFF).all()), "written in front of the buffer"
        assert bool((self.raw[self.begin + self.size:] == 0xFF).all()), "written behind the buffer"


def _call(n, rows, dim, gdt, odt, *, as_rows, skew=0, pad=-1, seed=1):
    from opendm_b200 import _native as N
    from opendm_b200.embedding import _error_word, check_errors

    dev = _dev()
    gen = torch.Generator(device=dev).manual_seed(seed)
    ids = (torch.pow(float(rows + 1), torch.rand(n, device=dev, generator=gen, dtype=torch.float64)).long() - 1)
    ids = ids.clamp_(0, rows - 1) * 7919 % rows
    grad = torch.randint(-1, 2, (n, dim), device=dev, generator=gen).to(gdt)
    code = {torch.bfloat16: N.MUON_BF16, torch.float32: N.MUON_F32}
    cap = min(n, rows)
    need = N.lib().muon_embedding_grad_workspace_bytes(n, rows, dim)
    work = Guarded(need)
    out = Guarded((cap if as_rows else rows) * dim * odt.itemsize, skew)
    out_ids, count = Guarded(8 * cap, 8 if skew else 0), Guarded(8)
    word = _error_word(0)
    N.check(N.lib().muon_embedding_grad(
        grad.data_ptr(), code[gdt], ids.data_ptr(), N.MUON_I64, n, rows, dim, pad, ctypes.c_float(1.0), out.pointer,
        code[odt], out_ids.pointer if as_rows else None, count.pointer if as_rows else None, work.pointer, need,
        word.pointer, torch.cuda.current_stream().cuda_stream), "muon_embedding_grad")
    check_errors()
    for buffer in (work, out, out_ids, count):
        buffer.check()
    use = ids != pad
    seen, back = torch.unique(ids[use], return_inverse=True)
    sums = torch.zeros(seen.numel(), dim, dtype=torch.float64, device=dev).index_add_(0, back, grad[use].double())
    if not as_rows:
        want = torch.zeros(rows, dim, dtype=odt, device=dev)
        want[seen] = sums.to(odt)
        assert torch.equal(out.view(odt, rows, dim), want)
        return
    k = seen.numel()
    assert count.view(torch.int64, 1).item() == k
    got_ids, got = out_ids.view(torch.int64, cap), out.view(odt, cap, dim)
    assert torch.equal(got_ids[:k], seen) and not got_ids[k:].any()
    assert torch.equal(got[:k], sums.to(odt)) and torch.equal(got[k:], torch.zeros_like(got[k:]))


B, F = torch.bfloat16, torch.float32

# the tokens of every sort: one block (1 or 4 keys a thread), clusters (2, 4, 8), tiles
TOKENS = [1, 300, 512, 2048, 2049, 8000, 16000, 32768, 32769]


@pytest.mark.parametrize("as_rows", [False, True])
@pytest.mark.parametrize("gdt,odt", [(B, B), (F, F), (B, F), (F, B)])
@pytest.mark.parametrize("dim,skew", [(8, 0), (33, 0), (33, 4), (36, 8), (250, 4), (520, 0), (1, 4)])
def test_every_byte_is_written_and_none_beside(dim, skew, gdt, odt, as_rows):
    for n in TOKENS:
        for rows in (7, 1000, 40000):
            _call(n, rows, dim, gdt, odt, as_rows=as_rows, skew=skew, pad=3 if n % 2 else -1)


# Zeros are written beside the sort from 1 MB of whole 16-byte words on, up to 8 MB (one block sorts) or 48 MB (a
# cluster); the sum writes the rest.
@pytest.mark.parametrize("n,megabytes", [(300, 1), (300, 8), (2049, 1), (2049, 48), (30000, 48)])
@pytest.mark.parametrize("dim,odt,skew", [(64, B, 0), (64, F, 0), (64, B, 2), (64, F, 16), (33, B, 0), (33, F, 0),
                                          (33, F, 4), (66, B, 4), (250, F, 0)])
def test_zeros_around_the_share_that_is_written_beside_the_sort(n, megabytes, dim, odt, skew):
    edge = (megabytes << 20) // (dim * odt.itemsize)
    for rows in (edge - 9, edge - 8, edge - 1, edge, edge + 1, edge + 7, edge + 33):
        _call(n, rows, dim, B, odt, as_rows=False, skew=skew, seed=rows)


def test_tables_of_few_long_rows():
    for n, rows, dim in ((100, 3, 70001), (3000, 50, 300000), (5, 40, 1 << 20)):
        for odt in (B, F):
            for as_rows in (False, True):
                _call(n, rows, dim if odt == B else dim // 2, B, odt, as_rows=as_rows, skew=4)


@pytest.mark.parametrize("as_rows", [False, True])
@pytest.mark.parametrize("rows", [900, 3_000_017])
def test_more_tokens_than_one_pass_over_the_tiles_run_starts(rows, as_rows):
    """The run starts of more than 1024 tiles of 4096 tokens are added up in two rounds."""
    _call(4_300_017, rows, 2, F, F, as_rows=as_rows, pad=5)
