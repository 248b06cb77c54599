"""GPU tests of the ctypes binding of the prompt path."""

import pytest
import torch

from lightdelta_b200 import capi
from test_prompt_path_gpu import Prompt, check_outputs, check_states

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("how", ["stream", "pointer", "current", "zero"])
def test_prefill_on_a_stream_of_its_own(how, monkeypatch):
    """A call on a stream that is not the current one, while the current one goes on allocating and writing."""
    case = Prompt([700, 64], [0, 64], seed=95)
    want, size, pool = case.expect()
    side = torch.cuda.Stream()
    given = {"stream": side, "pointer": side.cuda_stream, "current": None, "zero": 0}[how]
    made, real = [], torch.empty

    def empty(*args, **kwargs):
        out = real(*args, **kwargs)
        made.append(out.data_ptr())
        return out

    torch.cuda.synchronize()
    with monkeypatch.context() as patch:
        patch.setattr(torch, "empty", empty)
        capi.prefill(*case.args(), stream=given)
    junk = [torch.full((1 << 22,), float("nan"), device="cuda") for _ in range(8)]
    torch.cuda.synchronize()
    (address,) = made
    owners = [s["stream"] for s in torch.cuda.memory_snapshot() if s["address"] <= address < s["address"] + s["total_size"]]
    assert owners == [side.cuda_stream if how in ("stream", "pointer") else torch.cuda.default_stream().cuda_stream]
    check_outputs(case.out, want, size)
    check_states(case.state, pool)
    assert len(junk) == 8 and capi.fault_flags() == 0


@pytest.mark.parametrize("lens,contexts", [([1] * 40, [63, 64, 0, 130] * 10), ([2, 0, 1, 0, 0, 66, 1, 130, 0], [63, 0, 5, 9, 0, 62, 127, 1, 64])])
def test_prefill_stays_in_its_workspace(lens, contexts):
    """A workspace of the bytes asked for and not one more, behind it and in front of it what was there."""
    case = Prompt(lens, contexts, h=1, hv=3, seed=96)
    want, size, pool = case.expect()
    bytes_ = capi.prefill_workspace(sum(lens), len(lens), 1, 3)
    room = torch.full((bytes_ + 8192,), 0x5A, dtype=torch.uint8, device="cuda")
    start = 4096 + (-room.data_ptr()) % 128
    capi.prefill(*case.args(), workspace=room[start:start + bytes_])
    torch.cuda.synchronize()
    assert bool((room[:start] == 0x5A).all()) and bool((room[start + bytes_:] == 0x5A).all())
    check_outputs(case.out, want, size)
    check_states(case.state, pool)
    assert capi.fault_flags() == 0
