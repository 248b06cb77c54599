"""GPU tests of single tokens behind prompts, as the integration notes have them: tables, conv_prefill, then decode on the
pairs of slots; and what becomes of a request without context there."""

import pytest
import torch

import prompt_oracle
from lightdelta_b200 import capi
from test_prompt_path_gpu import DIM, Prompt, ints, lib

pytestmark = pytest.mark.gpu


def test_single_tokens_take_their_windows_from_the_held_block():
    """Contexts that end inside a block and with one.  The convolution's outputs are exact to bf16's half step, 2^-8 of the
    value, and 2^-18 of the magnitudes; the new block's windows are equal to the definition's."""
    gen = torch.Generator().manual_seed(97)
    contexts, block, dim = [5, 64, 128, 1], 64, 256
    x = torch.randn(4, dim, generator=gen).bfloat16().cuda()
    weight = torch.randn(dim, 4, generator=gen).bfloat16().cuda()
    state = torch.randn(20, dim, 3, generator=gen).bfloat16().cuda()
    table = (torch.randperm(12, generator=gen) + 1).view(4, 3).int().cuda()
    cu, used, pairs = torch.empty(5, dtype=torch.int32, device="cuda"), ints([0]), torch.empty(4, 2, dtype=torch.int32, device="cuda")
    positions, slot_map = (torch.empty(4, dtype=torch.int64, device="cuda") for _ in range(2))
    lib().request_tables(ints([1] * 4), ints(contexts), ints([13, 14, 15]), table, cu, positions, slot_map, pairs, used, block)
    want, size, after = prompt_oracle.conv(x, state, weight, None, table, ints(contexts), cu, block)
    out = torch.empty_like(x)
    lib().conv_prefill(x, state, weight, None, table, ints(contexts), cu, out, block)
    torch.cuda.synchronize()
    assert int(used) == 2 and pairs[:, 0].tolist() == [int(table[0, 0]), 13, 14, int(table[3, 0])]
    off = (out.cpu().double() - want).abs() / (2.0 ** -8 * want.abs() + 2.0 ** -18 * size + 1e-30)
    assert off.max() <= 1.0
    assert torch.equal(state.cpu().double(), after)


def test_a_first_token_needs_prefill():
    """`decode` has nothing to start a request without context from: zeros, and its new slot unchanged; `prefill` runs it."""
    case = Prompt([1, 1], [0, 64], h=1, hv=2, seed=98)
    pairs = ints([[int(case.table[0, 0]), 0], [int(case.table[1, 1]), int(case.table[1, 0])]])
    before, steps, out = case.state.clone(), case.state.clone(), torch.full_like(case.out, 7.0)
    lib().decode(case.qkv, case.a, case.b, case.a_log, case.dt_bias, pairs, case.cu, ints([2, 2]), steps, case.gate,
                 case.weight, out, 1e-6)
    case.check()
    assert bool((out[0] == 0).all()) and torch.equal(steps[pairs[0, 0]], before[pairs[0, 0]])
    got, want = steps[pairs[1, 0]].cpu(), case.state[pairs[1, 0]].cpu()
    # Two fp32 recurrences, one step: sums of 128 in either, 2 * 2^-17 of the largest value.
    assert (got - want).abs().max() <= 2.0 ** -16 * want.abs().max()
    assert capi.fault_flags() == 0 and out.shape[-1] == DIM


@pytest.mark.parametrize("lens,contexts,pad", [([0, 0], [0, 64], 5), ([0], [0], 1), ([0, 3, 0, 0], [7, 64, 0, 64], 2)])
def test_a_batch_padded_with_empty_requests(lens, contexts, pad):
    """Rows of a captured batch that hold no request now: nothing is written for them, whatever their contexts say."""
    case = Prompt(lens, contexts, h=1, hv=2, pad=pad, seed=99)
    case.check()
