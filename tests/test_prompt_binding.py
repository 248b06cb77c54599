"""CPU tests of the ctypes binding of the prompt path: what it hands to the C entry points, with the library faked."""

import random
from contextlib import contextmanager
from types import SimpleNamespace

import pytest
import torch

from lightdelta_b200 import capi

H, HV, N = 1, 2, 10


class Fake:
    """The library and torch's streams: remembers on which stream memory was asked for and used."""

    def __init__(self, monkeypatch):
        self.current, self.made, self.launched = 0, [], None
        monkeypatch.setattr(capi, "lib", lambda: SimpleNamespace(ld_prefill=self.prefill, ld_prefill_workspace=lambda *a: 1000,
                                                                 ld_last_error=lambda: b""))
        monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: SimpleNamespace(cuda_stream=self.current))
        monkeypatch.setattr(torch.cuda, "ExternalStream", lambda ptr, device=None: SimpleNamespace(cuda_stream=ptr))
        monkeypatch.setattr(torch.cuda, "stream", self.stream)
        real = torch.empty

        def empty(*args, **kwargs):
            out = real(*args, **kwargs)
            self.made.append((self.current, out.data_ptr()))
            return out

        monkeypatch.setattr(torch, "empty", empty)

    @contextmanager
    def stream(self, stream):
        before, self.current = self.current, stream.cuda_stream
        yield
        self.current = before

    def prefill(self, *args):
        self.launched = dict(workspace=args[-3], size=args[-2], stream=args[-1])
        return 0


def call(**kwargs):
    bf16, i32 = torch.bfloat16, torch.int32
    capi.prefill(torch.zeros(N, (2 * H + HV) * 128, dtype=bf16), torch.zeros(N, HV, dtype=bf16), torch.zeros(N, HV, dtype=bf16),
                 torch.zeros(HV), torch.zeros(HV), torch.zeros(1, 1, dtype=i32), torch.zeros(1, dtype=i32),
                 torch.zeros(2, dtype=i32), torch.zeros(2, HV, 128, 128), torch.zeros(N, HV, 128, dtype=bf16),
                 torch.zeros(128), torch.zeros(N, HV, 128, dtype=bf16), 64, **kwargs)


@pytest.mark.parametrize("given", [None, 77, SimpleNamespace(cuda_stream=77)])
def test_prefill_takes_its_workspace_on_the_stream_that_uses_it(monkeypatch, given):
    """Memory that torch's allocator hands out belongs to a stream: there it waits for whoever had it before, and there it
    may go to the next one as soon as it is given back.  On another stream it may still be, or be again, somebody else's."""
    fake = Fake(monkeypatch)
    call(**({} if given is None else {"stream": given}))
    used = 0 if given is None else 77
    assert fake.launched["stream"] == used
    assert fake.made == [(used, fake.launched["workspace"])] and fake.launched["size"] == 1000


def test_prefill_uses_the_workspace_that_it_is_given(monkeypatch):
    mine = torch.zeros(2000, dtype=torch.uint8)
    fake = Fake(monkeypatch)
    call(workspace=mine, stream=77)
    assert fake.made == [] and fake.launched == dict(workspace=mine.data_ptr(), size=2000, stream=77)


@pytest.mark.parametrize("tokens,requests,h,hv", [(7001, 128, 16, 32), (128, 128, 16, 32), (4096, 4096, 16, 32), (300, 7, 2, 6),
                                                  (16384, 1, 16, 48), (1, 1, 1, 1)])
def test_the_workspace_is_what_the_header_says(native, tokens, requests, h, hv):
    """Room for each chunk that the requests can have: two beyond their whole ones, and never more than tokens."""
    chunks = min(tokens, tokens // 64 + 2 * requests)
    least = chunks * (32768 * h + 16640 * hv) + 4 * requests
    assert least <= native.prefill_workspace(tokens, requests, h, hv) <= least + 256 + 15 * 2 ** 20


def test_places_of_chunks_do_not_overlap():
    """The rule that gives request r of a batch its places, min(first, first // 64 + 2 r) and on, for requests of any
    lengths that begin anywhere in a chunk; none lies behind what the workspace has room for."""
    rng = random.Random(5)
    for _ in range(3000):
        lens = [rng.choice((0, 0, 1, 1, 2, 3, 63, 64, 65, 130, rng.randrange(500))) for _ in range(rng.randrange(1, 9))]
        lens += [1] * rng.randrange(4)
        total, first, end = sum(lens), 0, 0
        for r, n in enumerate(lens):
            base = min(first, first // 64 + 2 * r)
            assert base >= end
            if n:
                end = base + (rng.choice((0, 1, 62, 63)) + n + 63) // 64
            first += n
        assert end <= min(total, total // 64 + 2 * len(lens))
