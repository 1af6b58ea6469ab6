"""Host logic of the embedding, list-clipping and row-gradient AdamW entry points, with the device faked."""

import contextlib
import ctypes

import pytest
import torch

from opendm_b200 import embedding as E


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
