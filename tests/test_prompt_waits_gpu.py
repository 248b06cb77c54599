"""GPU tests of what a launch of the prompt path leaves behind when one of its bounded waits runs out.  The test hook lets
copies announce more bytes than they bring: they land, but the wait for them runs out."""

import pytest
import torch

from lightdelta_b200 import capi
from test_prompt_path_gpu import Prompt

pytestmark = pytest.mark.gpu


def run_out(case, limit_ns):
    """Milliseconds of a call whose first waits run out."""
    capi.fault_flags()
    start, stop = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    capi.set_decode_wait_test(limit_ns, 64)
    try:
        torch.cuda.synchronize()
        start.record()
        case.run()
        stop.record()
        torch.cuda.synchronize()
    finally:
        capi.set_decode_wait_test()
    return start.elapsed_time(stop)


def test_a_wait_that_runs_out_leaves_the_zeros_of_invalid_requests_too():
    """Every multiprocessor's first item is a head of a valid prompt of three chunks, whose first copy never counts as
    landed; the heads of an invalid request come behind, and their zero outputs are stores like any other."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    case = Prompt([190, 20], [64, 64], h=1, hv=sms, seed=90)
    case.table[1, 0] = 0
    before, out = case.state.clone(), case.out.clone()
    run_out(case, 20_000_000)
    assert capi.fault_flags() == capi.LD_FAULT_WAIT_TIMEOUT
    assert torch.equal(case.state, before) and torch.equal(case.out, out)


def test_a_wait_that_runs_out_is_followed_by_one_for_what_is_in_flight():
    """Before it returns, a CTA waits once more, as long at most, for the copies that it has under way: they must not land
    in shared memory that is another CTA's by then."""
    case = Prompt([130], [64], h=1, hv=2, seed=91)
    before, out = case.state.clone(), case.out.clone()
    took = run_out(case, 20_000_000)
    assert capi.fault_flags() == capi.LD_FAULT_WAIT_TIMEOUT
    assert torch.equal(case.state, before) and torch.equal(case.out, out)
    assert 39.0 < took < 200.0
    case.check()
