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
