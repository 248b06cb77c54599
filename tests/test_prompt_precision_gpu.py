"""GPU tests of what the prompt path's arithmetic keeps, against the 64-bit definitions.

Tolerances.
  * Share of outputs that are not the nearest bf16 to the exact value.  Every product's operands have 22 bits or more
    and sums are fp32, so a value before its rounding is off by e = 2^-18 of its row's size (128 sums of 2^-24, roots of
    independent terms, the norm's and the gate's few fp32 steps).  It rounds elsewhere when it lies within e of a border:
    for a value x of a row of unit size, 2 e / 2^-8 |x| of them at most, and the mean of 1 / |x| over a normal
    distribution, cut off where the share reaches 1, is below 8: 2^4 * 2^-18 / 2^-8 = 2^-6.
    A chunk of equal keys cancels 64 terms against one another, sqrt(64) * sqrt(2) of independent errors: 2^-4 is four
    times the above, since there e is led by operand rounding, 2^-22, alone.
  * One token that leaves the state alone: S q has operands of 22 bits and a sum of 128 products in fp32, whose
    independent roundings make sqrt(128) * 2^-24 = 2^-20.5 of |S| |q| at most: 2^-20 of it through the norm, and bf16's
    half step, 2^-8 of the value.
  * States on an fp32 pool.  In a chunk, S k is off by 2^-22 (operands) and sqrt(128) * 2^-24 = 2^-20.5 (sums) of a row's
    norm, and so is u with beta < 1; 64 independent ones times keys' elements of about 128^-1/2 add 2^-22 of the norm to
    an element, and with the norm at most 4 times the head's largest value (128^1/2 over the three standard deviations
    that the largest of 16,384 surely has), 2^-20.  Four chunks' memory (default decays): 2^-19.  States that hardly
    forget keep 16 chunks' errors and the joins': 2^-18.
"""

import pytest
import torch

import prompt_oracle
from lightdelta_b200 import capi
from test_prompt_path_gpu import DIM, Prompt, check_outputs, ints

pytestmark = pytest.mark.gpu


def check_states_closely(state, pool, bound=2.0 ** -19):
    got = state.cpu().double()
    scale = pool.abs().amax(dim=(2, 3), keepdim=True)
    half = 2.0 ** -8 if state.dtype == torch.bfloat16 else 0.0
    off = (got - pool).abs() / (half * pool.abs() + bound * scale + 1e-30)
    assert off.max() <= 1.0, f"states {off.max():.2f} times their bound off"


def rounded_elsewhere(out, want):
    live = ~want.isnan()
    return float((out.cpu()[live] != want[live].bfloat16()).double().mean())


@pytest.mark.parametrize("lens,contexts,heads,decay", [
    ([64, 200, 17], [0, 64, 100], (1, 2), 1.0),
    ([300], [64], (2, 4), 1e-3),
    ([130, 70], [30, 0], (1, 3), 10.0),
    ([2500], [70], (1, 2), 1e-2),  # in pieces
])
def test_outputs_round_as_their_exact_values(lens, contexts, heads, decay):
    case = Prompt(lens, contexts, *heads, decay=decay, seed=50 + len(lens))
    want, _, pool = case.expect()
    case.run()
    torch.cuda.synchronize()
    assert rounded_elsewhere(case.out, want) <= 2.0 ** -6
    check_states_closely(case.state, pool)


def test_outputs_of_equal_keys_round_as_their_exact_values():
    """One and the same key with steps near 1: each token's output is what is left of 64 terms that cancel."""
    case = Prompt([64, 128], [0, 64], decay=1e-3, seed=60)
    case.qkv[:, DIM:2 * DIM] = case.qkv[:1, DIM:2 * DIM]
    case.b[:] = 9.0
    want, _, _ = case.expect()
    case.run()
    torch.cuda.synchronize()
    assert rounded_elsewhere(case.out, want) <= 2.0 ** -4


@pytest.mark.parametrize("cosine", [0.1, 0.01, 0.002])
@pytest.mark.parametrize("pool", [torch.float32, torch.bfloat16])
def test_queries_nearly_orthogonal_to_what_the_state_holds(cosine, pool):
    """The norm divides by what such a query reads, so an error that is small next to |S| |q| is large there.  `decode`
    rounds relative to the output itself; so must a prompt."""
    gen = torch.Generator().manual_seed(61)
    case = Prompt([1] * 8, [64] * 8, h=1, hv=2, decay=1e-6, pool=pool, seed=61)
    f = lambda *shape: torch.randn(*shape, generator=gen, dtype=torch.float64)  # noqa: E731
    basis = torch.linalg.qr(f(DIM, DIM)).Q
    held = torch.einsum("shvi,ik->shvk", f(case.slots, 2, DIM, 32), basis[:32])
    case.state.copy_(held)
    weights = f(8, DIM)
    weights[:, :32] = 0
    weights /= weights.norm(dim=1, keepdim=True)
    weights[:, 0] = cosine
    case.qkv[:, :DIM] = (weights @ basis).bfloat16()
    case.b[:] = -30.0  # the token leaves the state alone
    qkv, state = case.qkv.cpu().double(), case.state.cpu().double()
    want, _, after = case.expect()
    case.run()
    torch.cuda.synchronize()
    q = qkv[:, :DIM]
    q = q / (q * q).sum(-1, keepdim=True).sqrt() * DIM ** -0.5
    S = state[case.table[:, 0].cpu().long()]
    o = torch.einsum("rhvk,rk->rhv", S, q)
    size = S.norm(dim=-1) * q.norm(dim=-1)[:, None, None] + 1e-12
    rstd = torch.rsqrt((o * o).mean(-1, keepdim=True) + 1e-6)
    gate = case.gate.cpu().double()
    shape = (case.weight.cpu().double() * gate * torch.sigmoid(gate)).abs()
    through = (size + size.amax(-1, keepdim=True) * (o.abs() * rstd)) * rstd * shape
    off = (case.out.cpu().double() - want).abs() / (2.0 ** -8 * want.abs() + 2.0 ** -20 * through)
    assert off.max() <= 1.0, f"outputs {off.max():.2f} times their bound off"
    check_states_closely(case.state, after)


@pytest.mark.parametrize("power", [12, 18, 22])
def test_small_channels_beside_a_large_one(power):
    """One channel of the keys is 2^power times the others and the queries leave it out, so they read the columns that
    the small ones made.  bf16's 8 bits of those are kept (q, k as one fp16 each, 2^-24 the smallest step, the row's
    largest at 2^13 or more), P's entries, 2^-power, are good to 2^-25 of a range of 2^11, 2^(power - 36) = 2^-14 at 22,
    and the sums of 127 terms to 2^-17: 2^-13 of sum |q| |k| |u| over the small channels, and bf16's half step."""
    case = Prompt([5, 3], [0, 0], h=1, hv=2, decay=1e-3, seed=62)
    case.qkv[:, DIM] = 2.0 ** power * torch.sign(case.qkv[:, DIM].float()).bfloat16()
    case.qkv[:, 0] = 0
    case.b[:] = case.b * 0.3 - 1  # steps of about a quarter, so that tokens do not cancel one another
    want, _, _ = case.expect()
    case.run()
    torch.cuda.synchronize()
    qkv, f64 = case.qkv.cpu().double(), lambda t: t.cpu().double()
    q, k = qkv[:, :DIM], qkv[:, DIM:2 * DIM]
    q, k = (x / ((x * x).sum(-1, keepdim=True) + 1e-6).sqrt() for x in (q, k))
    q = q * DIM ** -0.5
    gate = f64(case.gate)
    shape = (f64(case.weight) * gate * torch.sigmoid(gate)).abs()
    v = qkv[:, 2 * DIM:].view(-1, 2, DIM)
    cu = case.cu.tolist()
    for r in range(2):
        for t in range(cu[r], cu[r + 1]):
            # |u| is below twice the largest v so far of its row (steps below 1, keys of one direction).
            u = 2 * v[cu[r]:t + 1].abs().amax(0)
            size = u * (q[t].abs() * k[cu[r]:t + 1].abs()).sum()
            o = want[t] / (shape[t] + 1e-300)  # o rstd; rstd is at most 1e3
            through = (size + size.amax(-1, keepdim=True) * o.abs()) * 1e3 * shape[t]
            off = (f64(case.out[t]) - want[t]).abs() / (2.0 ** -8 * want[t].abs() + 2.0 ** -13 * through)
            assert off.max() <= 1.0, f"outputs {off.max():.2f} times their bound off"


@pytest.mark.parametrize("lens,contexts,heads,block", [
    ([64], [0], (1, 1), 64),
    ([130, 1, 64, 63, 200, 9], [64, 63, 64, 65, 57, 5], (1, 2), 64),
    ([257, 70], [128, 0], (2, 6), 128),
    ([1500], [64], (1, 2), 256),
])
def test_states_closely(lens, contexts, heads, block):
    case = Prompt(lens, contexts, *heads, block=block, seed=70 + len(lens))
    _, _, pool = case.expect()
    case.run()
    torch.cuda.synchronize()
    check_states_closely(case.state, pool)


def test_states_of_equal_keys_closely():
    """A chunk of one key with steps near 1: T's entries alternate at their largest, 1, and R's errors of 64 tokens meet
    in the one direction of the key: sqrt(64) more than the bound of independent keys, 2^-19 * 2^3."""
    case = Prompt([128], [64], decay=1e-3, seed=75)
    case.qkv[64:, DIM:2 * DIM] = case.qkv[64, DIM:2 * DIM]
    case.b[:] = 9.0
    _, _, pool = case.expect()
    case.run()
    torch.cuda.synchronize()
    check_states_closely(case.state, pool, 2.0 ** -16)


def cuts(tokens, context, requests, hv):
    """The first chunk of each piece of a request that is a call's longest by far: the rule of the header's note on
    prompts in pieces, for 148 multiprocessors."""
    slots, chunks = 148 // (requests * hv), tokens // 64
    most, whole = min(16, chunks // 5), 2 + (slots - 1) // 2
    half = slots % 2 == 0 and whole < most
    count = whole + 1 if half else min(whole, most)
    at = [2 * k - (1 if half and k >= count - 1 else 0) for k in range(count + 1)]
    own = -(-(context % 64 + tokens) // 64)
    return [own * x // at[-1] for x in at], half


@pytest.mark.parametrize("tokens,context,heads,pool,pieces,half", [
    (5300, 64, (1, 2), torch.float32, 16, False),
    (5300, 90, (1, 1), torch.bfloat16, 16, False),
    (2300, 64, (2, 18), torch.bfloat16, 6, True),
    (1700, 100, (1, 37), torch.float32, 4, True),
    (1990, 64, (1, 49), torch.float32, 3, False),
])
def test_pieces_hand_on_what_came_before_them(tokens, context, heads, pool, pieces, half):
    """Slow decays and small steps, so that the state of the first piece lasts: each piece's first state is the joined
    one, S_k M_k + B_k, and the states behind show M_k.  Without S_k M_k they would be off by many times the bound."""
    starts, has_half = cuts(tokens, context, 1, heads[1])
    assert len(starts) == pieces + 1 and has_half == half
    case = Prompt([tokens], [context], *heads, block=128, pool=pool, decay=1e-5, seed=80 + pieces)
    case.b[:] = case.b - 3
    want, size, expect = case.expect()
    state = case.state.clone()
    # What the third piece and on would be from B_1 alone: the second piece's tokens run from nothing.
    lead = context % 64
    first = starts[1] * 64 - lead
    last = min(starts[2] * 64 - lead + 128, tokens)
    rows = slice(first, last)
    forgot = prompt_oracle.prefill(case.qkv[rows], case.a[rows], case.b[rows], case.a_log, case.dt_bias, case.table,
                                   ints([context + first]), ints([0, last - first]), torch.zeros_like(state), case.gate[rows],
                                   case.weight, case.block)[2]
    slot = int(case.table[0, (context + last) // 128 - 1])  # of the last block that ends in there
    case.run()
    torch.cuda.synchronize()
    check_outputs(case.out, want, size)
    bound = 2.0 ** -18
    check_states_closely(case.state, expect, bound)
    scale = expect[slot].abs().amax(dim=(1, 2))
    missing = (forgot[slot] - expect[slot]).abs().amax(dim=(1, 2)) / scale
    assert missing.min() > 100 * (bound + (2.0 ** -8 if pool == torch.bfloat16 else 0.0) / 25), "the case shows nothing"
    assert capi.fault_flags() == 0


def test_decode_and_prefill_agree_on_orthogonal_queries():
    """The same token through `decode` and through `prefill`: both round the output once (half a step, 2^-8 of the value
    each), and `decode` its recurrence output as well, which the norm passes on: 3 * 2^-8; and fp32 sums of |S| |q|,
    about a thousand times what is read, cost either 2^-22 of it: 2^-12 of the row's largest."""
    gen = torch.Generator().manual_seed(63)
    case = Prompt([1] * 4, [64] * 4, h=1, hv=2, decay=1e-6, seed=63)
    basis = torch.linalg.qr(torch.randn(DIM, DIM, generator=gen, dtype=torch.float64)).Q
    case.state.copy_(torch.einsum("shvi,ik->shvk", torch.randn(case.slots, 2, DIM, 32, generator=gen, dtype=torch.float64),
                                  basis[:32]))
    case.qkv[:, :DIM] = (basis[40] + 0.005 * basis[0]).bfloat16()
    case.b[:] = -30.0
    steps, out = case.state.clone(), torch.empty_like(case.out)
    pairs = torch.stack((case.table[:, 1], case.table[:, 0]), 1).contiguous()
    case.run()
    torch.ops.lightdelta.decode(case.qkv, case.a, case.b, case.a_log, case.dt_bias, pairs, case.cu, ints([2] * 4), steps,
                                case.gate, case.weight, out, 1e-6)
    torch.cuda.synchronize()
    got, want = case.out.cpu().double(), out.cpu().double()
    off = (got - want).abs() / (3 * 2.0 ** -8 * want.abs() + 2.0 ** -12 * want.abs().amax(-1, keepdim=True))
    assert off.max() <= 1.0
