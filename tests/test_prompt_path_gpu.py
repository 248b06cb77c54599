"""GPU tests of the prompt path (request_tables, conv_prefill, prefill) against the 64-bit definitions.

Tolerances.
  * States.  The products on the way to the state take fp32 values as two fp16 terms (2^-22 of the row's largest) and
    sum 128 (S k) or 64 (T R, the update) of them in fp32: at most 128 * 2^-24 = 2^-17 of the sum of magnitudes each,
    and |k| = 1, beta < 1 keep those sums within a state row's norm, here at most sqrt(128) < 2^4 times its
    root mean square.  Three products per chunk, chunks decaying into each other: STATE = 2^-17 * 3 * 2 of the head's
    largest value (a row's norm against the largest value absorbs the 2^4: errors of independent terms add as a
    root), rounded up to 2^-14.  A bf16 pool adds half a step, 2^-8 of the value.
  * Outputs.  2^-9 of what the oracle reports for the two products that take single fp16 terms (derived there), then
    bf16's half step, 2^-8 of the value.
  * Convolution.  Half a step, 2^-8 of the value, and 2^-18 of the magnitudes for fp32 sums and the fast exponential.
Windows, tables and everything that must not change are compared exactly.
"""

import numpy as np
import pytest
import torch

import prompt_oracle
from helpers import bits
from lightdelta_b200 import capi
from lightdelta_b200.backend import GDNBackend
from lightdelta_b200.config import BackendConfig

pytestmark = pytest.mark.gpu
DIM = 128
STATE = 2.0 ** -14


def lib():
    from lightdelta_b200 import ops  # noqa: F401

    return torch.ops.lightdelta


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Prompt:
    """Inputs of one prefill call.  `rows`: table rows (lists of slots) or None for distinct ones."""

    def __init__(self, lens, contexts, h=1, hv=2, block=64, pool=torch.float32, seed=0, rows=None, pad=0, spare=0,
                 decay=1.0, scale=1.0, strided=True):
        gen = torch.Generator().manual_seed(seed)
        f = lambda *shape: torch.randn(*shape, generator=gen)  # noqa: E731
        n = sum(lens) + pad
        width = (2 * h + hv) * DIM
        wide = torch.empty(n, width + hv * DIM + (8 if strided else 0))
        wide[:] = f(*wide.shape)
        wide[:, :width] *= scale
        wide = wide.bfloat16().cuda()
        ab = f(n, 2 * hv + 1).bfloat16().cuda()
        self.qkv, self.gate = wide[:, :width], wide[:, width:width + hv * DIM].view(n, hv, DIM)
        self.a, self.b = ab[:, hv:2 * hv], ab[:, :hv]
        self.a_log, self.dt_bias = (f(hv) * 0.3 + np.log(decay)).cuda(), (f(hv) - 2).cuda()
        self.weight = (1 + 0.1 * f(DIM)).bfloat16().cuda()
        blocks = max([-(-(c + k) // block) for c, k in zip(contexts, lens)] + [1])
        if rows is None:
            slots = len(lens) * blocks
            rows = (torch.randperm(slots, generator=gen) + 1).view(len(lens), blocks).tolist()
        self.slots = max([max(r) for r in rows] + [1]) + 1 + spare
        self.table, self.context = ints(rows), ints(contexts)
        self.cu = ints([0] + np.cumsum(lens).tolist())
        self.state = (0.2 * scale * f(self.slots, hv, DIM, DIM)).to(pool).cuda()
        self.out = torch.full((n, hv, DIM), 7.0, dtype=torch.bfloat16, device="cuda")
        self.block, self.h, self.hv = block, h, hv

    def args(self):
        return (self.qkv, self.a, self.b, self.a_log, self.dt_bias, self.table, self.context, self.cu, self.state,
                self.gate, self.weight, self.out, self.block, 1e-6)

    def run(self):
        lib().prefill(*self.args())

    def check(self, expect=None, faults=0):
        want, size, pool = expect or self.expect()
        self.run()
        torch.cuda.synchronize()
        check_outputs(self.out, want, size)
        check_states(self.state, pool)
        assert capi.fault_flags() == faults

    def expect(self):
        return prompt_oracle.prefill(*self.args()[:-3], block_size=self.block)


def check_outputs(out, want, size):
    got = out.cpu().double()
    untouched = want.isnan()
    assert bool((got[untouched] == 7.0).all()), "rows of no request changed"
    want = torch.where(untouched, got, want)
    off = (got - want).abs() / (2.0 ** -8 * want.abs() + 2.0 ** -9 * size + 1e-30)
    assert off.max() <= 1.0, f"outputs {off.max():.2f} times their bound off"


def check_states(state, pool):
    got = state.cpu().double()
    scale = pool.abs().amax(dim=(2, 3), keepdim=True)
    half = 2.0 ** -8 if state.dtype == torch.bfloat16 else 0.0
    off = (got - pool).abs() / (half * pool.abs() + STATE * scale + 1e-30)
    assert off.max() <= 1.0, f"states {off.max():.2f} times their bound off"


@pytest.mark.parametrize("lens", [[1], [2], [63], [64], [65], [127, 1, 129], [200], [17, 0, 64, 3]])
def test_prefill_lengths(lens):
    Prompt(lens, [0] * len(lens), seed=len(lens)).check()


@pytest.mark.parametrize("heads", [(1, 1), (2, 2), (1, 3), (1, 6), (2, 10)])
def test_prefill_heads(heads):
    Prompt([70, 5], [0, 128], *heads, seed=heads[1]).check()


@pytest.mark.parametrize("pool", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("block", [64, 128])
def test_prefill_contexts_inside_and_at_block_ends(pool, block):
    """Starts and ends anywhere in a block: the source slot is the first destination where a block goes on."""
    Prompt([130, 1, 64, 63, 200, 9], [block, 63, 64, block + 1, block - 7, 5], block=block, pool=pool, seed=5).check()


def test_prefill_state_of_a_continued_block_is_read_before_it_is_written():
    case = Prompt([40, 30], [10, 64 + 20], seed=6)
    case.check()


@pytest.mark.parametrize("shape", ["odd_rows", "odd_base"])
def test_prefill_unaligned_rows(shape):
    """Rows that 16-byte copies cannot read: an odd row stride, or an odd first element."""
    case = Prompt([75, 20], [0, 30], seed=7)
    n, width = case.qkv.shape
    wide = torch.zeros(n, width + (1 if shape == "odd_rows" else 8), dtype=torch.bfloat16, device="cuda")
    view = wide[:, :width] if shape == "odd_rows" else wide[:, 1:1 + width]
    view.copy_(case.qkv)
    case.qkv = view
    gate = torch.zeros(n, case.hv * DIM + 3, dtype=torch.bfloat16, device="cuda")
    gate[:, 3:].copy_(case.gate.reshape(n, -1))
    case.gate = gate.as_strided((n, case.hv, DIM), (gate.stride(0), DIM, 1), 3)
    case.check()


def test_prefill_pool_with_gaps_and_table_with_wide_rows():
    case = Prompt([66, 80], [64, 0], seed=8)
    big = torch.full((case.slots, 3 * case.state[0].numel() // 2), 3.0, device="cuda")
    pool = big.as_strided(case.state.shape, (big.stride(0), DIM * DIM, DIM, 1))
    pool.copy_(case.state)
    case.state = pool
    table = torch.full((2, case.table.shape[1] + 5), 1 << 30, dtype=torch.int32, device="cuda")
    table[:, : case.table.shape[1]] = case.table
    case.table = table[:, : case.table.shape[1]]
    case.check()
    assert bool((big[:, case.state[0].numel():] == 3.0).all())


def test_prefill_null_destinations_and_padding():
    """Blocks without a slot are not stored, rows behind the last request stay, and slot 0 is neither read nor
    written, whatever it holds."""
    case = Prompt([150, 64], [0, 64], rows=[[0, 0, 3], [2, 0, 0]], pad=9, spare=2, seed=9)
    case.state[0] = float("nan")
    case.qkv[-9:] = float("nan")
    want, size, pool = case.expect()
    case.run()
    torch.cuda.synchronize()
    check_outputs(case.out, want, size)
    assert bool(case.state[0].isnan().all())
    check_states(case.state[1:], pool[1:])
    assert capi.fault_flags() == 0


def test_prefill_neighbours_values_do_not_spread():
    """A request whose tokens are not finite spoils itself alone, from its chunk on."""
    case = Prompt([70, 30, 64, 5], [0, 10, 0, 3], seed=10)
    want, size, pool = case.expect()
    bad = slice(70, 100)
    case.qkv[bad], case.gate[bad] = float("nan"), float("inf")
    case.run()
    torch.cuda.synchronize()
    keep = torch.ones(169, dtype=torch.bool)
    keep[bad] = False
    check_outputs(case.out[keep.cuda()], want[keep], size[keep])
    ok = [s for s in range(case.slots) if s not in case.table[1].tolist()]
    check_states(case.state[ok], pool[ok])


@pytest.mark.parametrize("decay", [1e-6, 30.0, 1e4])
def test_prefill_decays(decay):
    """From hardly any forgetting to states that are gone within a token (sums of log decays past 1e5)."""
    Prompt([140], [64], decay=decay, seed=11).check()


@pytest.mark.parametrize("scale", [1e-15, 1e12])
def test_prefill_magnitudes(scale):
    Prompt([100], [64], scale=scale, seed=12).check()


def test_prefill_zero_and_equal_keys():
    """Rows of zeros, and a chunk of one and the same key with steps near 1: the inverse's hardest case."""
    case = Prompt([128], [0], seed=13)
    case.qkv[10:14] = 0
    case.qkv[64:, DIM:2 * DIM] = case.qkv[64, DIM:2 * DIM]
    case.b[:] = 9.0
    case.check()


def test_prefill_invalid_requests():
    """A null or missing source, contexts and blocks out of range: zero outputs, no stores, and the others unharmed."""
    case = Prompt([10, 20, 30, 40, 70, 64], [64, 64, -1, 10, 0, 64], spare=1, seed=14,
                  rows=[[0, 1], [99, 2], [3, 4], [5, 6], [7, 77], [8, 9]])
    case.slots = 10
    case.state = case.state[:10].contiguous()
    case.table[3] = 5
    case.context[3] = 2 * 64 + 10
    before = case.state.clone()
    want, size, pool = case.expect()
    case.run()
    torch.cuda.synchronize()
    check_outputs(case.out, want, size)
    check_states(case.state, pool)
    for slot in (0, 1, 2, 3, 4, 5, 6):
        assert torch.equal(case.state[slot], before[slot])
    assert capi.fault_flags() == capi.LD_FAULT_DECODE_SLOT_RANGE | capi.LD_FAULT_TABLE_BLOCKS


@pytest.mark.parametrize("cu,faults", [([0, 30, 200], 2), ([-5, 30, 60], 2), ([40, 30, 60], 0), ([0, 91, 92], 2)])
def test_prefill_offsets_out_of_range_skip_the_request(cu, faults):
    """Offsets outside the tokens raise the fault, a request that ends before it begins is empty."""
    case = Prompt([30, 60], [0, 0], seed=15)
    case.cu = ints(cu)
    case.check(faults=faults)


@pytest.mark.parametrize("lens,contexts,heads,block,pool", [
    ([2500], [70], (1, 2), 64, torch.float32),
    ([6200], [0], (1, 1), 128, torch.bfloat16),
    ([7000, 100, 0, 300], [64, 3, 0, 64], (1, 2), 64, torch.float32),
    ([3100, 3100], [100, 0], (2, 12), 1024, torch.float32),
    ([2700], [1000], (1, 37), 64, torch.float32),
])
def test_prefill_long_prompts_in_pieces_at_once(lens, contexts, heads, block, pool):
    """Long prompts of few heads, which run in pieces side by side whose states are joined, beside short ones."""
    Prompt(lens, contexts, *heads, block=block, pool=pool, seed=len(lens)).check()


def test_prefill_long_prompts_that_cannot_run_or_keep_nothing():
    """Pieces of a request with a null source give zeros and raise nothing, and blocks without a slot are not stored."""
    case = Prompt([2400, 2400], [64, 0], h=1, hv=2, seed=41)
    case.table[0, 0] = 0
    case.table[1, ::2] = 0
    case.check()
    case = Prompt([2400], [64], h=1, hv=2, seed=42)
    case.table[0, 0] = case.slots
    case.check(faults=capi.LD_FAULT_DECODE_SLOT_RANGE)


def test_prefill_long_prompt_repeats_and_stops():
    """Bit for bit, and a wait that runs out in the first pass keeps the second from storing anything."""
    results = []
    for _ in range(2):
        case = Prompt([3000], [30], h=1, hv=2, seed=43)
        case.run()
        torch.cuda.synchronize()
        results.append((bits(case.out), case.state.cpu().numpy().view(np.uint32)))
    assert np.array_equal(results[0][0], results[1][0]) and np.array_equal(results[0][1], results[1][1])
    before, out = case.state.clone(), case.out.clone()
    capi.set_decode_wait_test(200_000, 64)
    try:
        case.run()
        torch.cuda.synchronize()
    finally:
        capi.set_decode_wait_test()
    assert capi.fault_flags() == capi.LD_FAULT_WAIT_TIMEOUT
    assert torch.equal(case.state, before) and torch.equal(case.out, out)


def test_prefill_requests_that_share_a_held_block():
    """One full block as the source of several requests, as prompts with a common beginning have it."""
    Prompt([70, 3, 64], [64, 64, 64], rows=[[1, 2, 3], [1, 4, 0], [1, 5, 0]], seed=44).check()


def test_prefill_long_prompt_in_a_graph():
    """The passes and joins of a split prompt captured, replayed with new inputs, bit for bit what a call gives."""
    case, new = Prompt([3000], [30], h=1, hv=2, seed=45), Prompt([3000], [30], h=1, hv=2, seed=46)
    case.run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        case.run()
    for name in ("qkv", "a", "b", "a_log", "dt_bias", "table", "gate", "weight", "state"):
        getattr(case, name).copy_(getattr(new, name))
    graph.replay()
    new.run()
    torch.cuda.synchronize()
    assert np.array_equal(bits(case.out), bits(new.out)) and torch.equal(case.state, new.state)


def test_prefill_many_requests():
    """Single tokens and empty requests by the hundred, in an order that the queue of items changes."""
    lens = [(7 * i) % 3 for i in range(300)]
    Prompt(lens, [64 * (i % 2) for i in range(300)], h=1, hv=1, seed=16).check()


def test_prefill_offsets_past_32_bits():
    """Slots more than 2^31 elements into the pool."""
    case = Prompt([70], [64], h=1, hv=1, seed=17)
    far = 2 ** 31 // (DIM * DIM) + 5
    pool = torch.empty(far + 8, 1, DIM, DIM, device="cuda")
    pool[far:] = case.state[:1]
    small = case.state.clone()
    for s in range(case.slots):
        pool[far + s] = small[s]
    want, size, expect = case.expect()
    case.state, case.table = pool, case.table + far
    case.run()
    torch.cuda.synchronize()
    check_outputs(case.out, want, size)
    check_states(pool[far:far + case.slots], expect)


def test_prefill_is_decode_token_by_token():
    """The same tokens through `decode`, whose recurrence outputs and results are both rounded to bf16: two half steps
    of 2^-8, on values whose recurrence outputs differ by the outputs' bound."""
    lens, contexts = [9, 5], [60, 0]
    case = Prompt(lens, contexts, h=2, hv=4, seed=18)
    _, size, _ = case.expect()
    steps = case.state.clone()
    steps[case.table[1, 0]] = 0  # a request without context starts from nothing
    case.run()
    out = torch.empty_like(case.out)
    for r, (n, ctx) in enumerate(zip(lens, contexts)):
        for t in range(n):
            at = int(case.cu[r]) + t
            slot = case.table[r:r + 1, (ctx + t) // 64:(ctx + t) // 64 + 1].contiguous()
            if t and (ctx + t) % 64 == 0:
                steps[slot[0, 0]] = steps[case.table[r, (ctx + t) // 64 - 1]]
            one = out[at:at + 1]
            lib().decode(case.qkv[at:at + 1], case.a[at:at + 1], case.b[at:at + 1], case.a_log, case.dt_bias, slot,
                         ints([0, 1]), ints([1]), steps, case.gate[at:at + 1], case.weight, one, 1e-6)
    used = [s for s in case.table.flatten().tolist() if s not in (0,)]
    check_states(case.state[used], steps[used].cpu().double())
    got, want = case.out.cpu().double(), out.cpu().double()
    off = (got - want).abs() / (3 * 2.0 ** -8 * want.abs() + 2.0 ** -7 * size + 1e-30)
    assert off.max() <= 1.0


@pytest.mark.parametrize("cuts", [[100], [64, 36], [1, 62, 2, 35], [37, 63]])
def test_prefill_in_pieces(cuts):
    """A prompt in one call and in pieces that start inside blocks: the same results within the states' bound."""
    whole = Prompt([100], [0], seed=19)
    expect = whole.expect()
    done = 0
    for n in cuts:
        part = slice(done, done + n)
        lib().prefill(whole.qkv[part], whole.a[part], whole.b[part], whole.a_log, whole.dt_bias, whole.table, ints([done]),
                      ints([0, n]), whole.state, whole.gate[part], whole.weight, whole.out[part], whole.block, 1e-6)
        done += n
    torch.cuda.synchronize()
    check_outputs(whole.out, expect[0], expect[1])
    check_states(whole.state, expect[2])


def test_prefill_repeats_bit_for_bit():
    """Two runs, programmatic launch on and off, the torch operator and the C entry point."""
    results = []
    for way in range(4):
        case = Prompt([130, 64, 1, 300], [0, 64, 70, 3], h=2, hv=4, seed=20)
        previous = capi.set_programmatic_launch(way != 2)
        if way == 3:
            args = case.args()
            capi.prefill(*args)
        else:
            case.run()
        capi.set_programmatic_launch(previous)
        torch.cuda.synchronize()
        results.append((bits(case.out), case.state.cpu().numpy().view(np.uint32)))
    for out, state in results[1:]:
        assert np.array_equal(out, results[0][0]) and np.array_equal(state, results[0][1])


def test_prefill_graphs_and_streams():
    """Two graphs on two layers' pools, replayed together with new inputs in place, and an eager call on another
    stream beside them; each has a workspace of its own."""
    cases = [Prompt([70, 64], [0, 64], seed=21), Prompt([70, 64], [64, 0], seed=22)]
    graphs = []
    for case in cases:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            case.run()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            case.run()
        graphs.append(graph)
    fresh = [Prompt([78, 56], [0, 64], seed=23), Prompt([100, 34], [64, 0], seed=24)]
    expect = []
    for case, new in zip(cases, fresh):
        for name in ("qkv", "a", "b", "a_log", "dt_bias", "context", "cu", "gate", "weight", "out"):
            getattr(case, name).copy_(getattr(new, name))
        case.state.copy_(new.state)
        expect.append(case.expect())
    other = Prompt([200], [0], seed=25)
    third = other.expect()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for graph, stream in zip(graphs, streams):
        with torch.cuda.stream(stream):
            graph.replay()
    with torch.cuda.stream(streams[2]):
        other.run()
    torch.cuda.synchronize()
    for case, (want, size, pool) in zip(cases + [other], expect + [third]):
        check_outputs(case.out, want, size)
        check_states(case.state, pool)


def test_prefill_wait_that_runs_out():
    """Copies that announce more bytes than they bring: the wait for them runs out, the launch stores nothing, raises
    the fault bit and returns, and the next one is right."""
    case = Prompt([130], [64], seed=26)
    before, out = case.state.clone(), case.out.clone()
    capi.fault_flags()
    capi.set_decode_wait_test(200_000, 64)
    try:
        case.run()
        torch.cuda.synchronize()
    finally:
        capi.set_decode_wait_test()
    assert capi.fault_flags() == capi.LD_FAULT_WAIT_TIMEOUT
    assert torch.equal(case.state, before) and torch.equal(case.out, out)
    case.check()


def test_prefill_refuses_other_tensors():
    case = Prompt([10], [0])
    for change in (dict(table=case.table.long()), dict(table=case.table[0]), dict(context=ints([0, 0])), dict(cu=ints([0])),
                   dict(state=case.state.half()), dict(out=case.out[:5]), dict(gate=case.gate.float()),
                   dict(qkv=case.qkv[:, :-1]), dict(a=case.a.cpu()), dict(block=63), dict(gate=case.out)):
        args = dict(qkv=case.qkv, a=case.a, b=case.b, a_log=case.a_log, dt_bias=case.dt_bias, table=case.table,
                    context=case.context, cu=case.cu, state=case.state, gate=case.gate, weight=case.weight, out=case.out,
                    block=64, eps=1e-6)
        with pytest.raises(RuntimeError):
            lib().prefill(*{**args, **change}.values())
    assert bool((case.out == 7.0).all())


# ---------------------------------------------------------------------------------------------------------------
# conv_prefill
# ---------------------------------------------------------------------------------------------------------------
class Conv:
    def __init__(self, lens, contexts, dim=256, width=4, block=64, bias=True, token_first=False, length=None, seed=0, pad=0):
        gen = torch.Generator().manual_seed(seed)
        f = lambda *shape: torch.randn(*shape, generator=gen).bfloat16().cuda()  # noqa: E731
        n = sum(lens) + pad
        self.x = f(n, dim + 8)[:, :dim]
        blocks = max([-(-(c + k) // block) for c, k in zip(contexts, lens)] + [1])
        self.table = (torch.randperm(len(lens) * blocks, generator=gen) + 1).view(len(lens), blocks).int().cuda()
        length = length or width - 1
        state = f(len(lens) * blocks + 1, length, dim) if token_first else f(len(lens) * blocks + 1, dim, length)
        self.state = state.transpose(1, 2) if token_first else state
        self.weight, self.bias = f(dim, width), f(dim) if bias else None
        self.context, self.cu = ints(contexts), ints([0] + np.cumsum(lens).tolist())
        self.out = torch.full((n, dim), 7.0, dtype=torch.bfloat16, device="cuda")
        self.block = block

    def run(self):
        lib().conv_prefill(self.x, self.state, self.weight, self.bias, self.table, self.context, self.cu, self.out, self.block)

    def check(self, faults=0):
        want, size, state = prompt_oracle.conv(self.x, self.state, self.weight, self.bias, self.table, self.context, self.cu,
                                               self.block)
        self.run()
        torch.cuda.synchronize()
        got = self.out.cpu().double()
        untouched = want.isnan()
        assert bool((got[untouched] == 7.0).all()), "rows of no request changed"
        want = torch.where(untouched, got, want)
        off = (got - want).abs() / (2.0 ** -8 * want.abs() + 2.0 ** -18 * size + 1e-30)
        assert off.max() <= 1.0, f"{off.max():.2f} times their bound off"
        assert torch.equal(self.state.cpu().double(), state), "windows"
        assert capi.fault_flags() == faults


@pytest.mark.parametrize("width", [2, 3, 4])
@pytest.mark.parametrize("token_first", [False, True])
def test_conv_prefill_widths_and_layouts(width, token_first):
    Conv([1, 2, 3, 70, 0, 64, 5], [0, 64, 3, 60, 7, 64, 1], width=width, token_first=token_first, bias=width != 3,
         length=width + 1, seed=width).check()


@pytest.mark.parametrize("dim", [4, 130, 515, 1024])
def test_conv_prefill_channel_counts(dim):
    Conv([40, 9], [0, 33], dim=dim, seed=dim).check()


@pytest.mark.parametrize("seed", range(6))
def test_conv_prefill_ragged_batches_over_tile_borders(seed):
    """Requests that begin and end everywhere in the tiles of 8 and of 32 tokens, most of them short, many going on
    inside a block (read and written slot in one)."""
    rng = np.random.default_rng(seed)
    lens = rng.integers(0, 12, 60).tolist() + [int(rng.integers(30, 200))]
    contexts = rng.integers(0, 130, len(lens)).tolist()
    rng.shuffle(lens)
    Conv(lens, contexts, dim=20, width=int(rng.integers(2, 5)), block=int(rng.choice([1, 7, 64])), seed=seed, pad=3).check()


def test_conv_prefill_long_batch():
    Conv([2500, 31, 2, 1200], [0, 64, 100, 3], dim=2560, block=512, seed=31).check()


@pytest.mark.parametrize("dim,tokens", [(2560, 4000), (8192, 3700)])
def test_conv_prefill_batches_that_take_long_tiles(dim, tokens):
    """Batches large enough for tiles of 32 and of 64 tokens, with requests that begin and end anywhere in them."""
    rng = np.random.default_rng(dim)
    lens = []
    while sum(lens) < tokens:
        lens.append(int(rng.choice([1, 2, 3, 5, 31, 32, 33, 62, 63, 64, 65, 200])))
    contexts = rng.integers(0, 100, len(lens)).tolist()
    Conv(lens, contexts, dim=dim, block=64, seed=dim).check()


def test_conv_prefill_invalid_requests():
    case = Conv([10, 20, 30, 5], [64, 64, -1, 0], seed=32)
    case.table[0, 0], case.table[1, 0], case.table[3, 0] = 0, 1000, 1001
    case.check(faults=capi.LD_FAULT_CONV_SLOT_RANGE | capi.LD_FAULT_TABLE_BLOCKS)
    case = Conv([10, 20], [0, 0], seed=33)
    case.cu = ints([0, 10, 31])
    case.check(faults=capi.LD_FAULT_DECODE_TOKENS)


def test_conv_prefill_then_conv_update_goes_on():
    """The window that a prompt leaves is what `conv_update` continues: its outputs on three more tokens are the
    prompt's own within the products and the sum that it rounds to bf16 (half a step, 2^-8, of their magnitudes each,
    times silu's slope, at most 1.1) and its result's half step."""
    case = Conv([50], [0], dim=256, block=64, seed=34)
    want, size, _ = prompt_oracle.conv(case.x, case.state, case.weight, case.bias, case.table, case.context, case.cu, 64)
    first = slice(0, 47)
    lib().conv_prefill(case.x[first], case.state, case.weight, case.bias, case.table, case.context, ints([0, 47]),
                       case.out[first], 64)
    x = case.x[47:].clone()
    for t in range(3):
        lib().conv_update(x[t:t + 1], case.state, case.weight, case.bias, case.table[:, 0].contiguous(), None, ints([0, 1]), 1)
    torch.cuda.synchronize()
    off = (x.cpu().double() - want[47:]).abs() / (2.0 ** -8 * want[47:].abs() + 2.2 * 2.0 ** -8 * size[47:])
    assert off.max() <= 1.0


def test_conv_prefill_graph_and_refusals():
    case = Conv([40, 30], [0, 64], seed=35)
    case.run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        case.run()
    new = Conv([25, 45], [0, 64], seed=36)
    for name in ("x", "state", "weight", "bias", "cu", "out"):
        getattr(case, name).copy_(getattr(new, name)[: getattr(case, name).shape[0]])
    want, size, state = prompt_oracle.conv(case.x, case.state, case.weight, case.bias, case.table, case.context, case.cu, 64)
    graph.replay()
    torch.cuda.synchronize()
    off = (case.out.cpu().double() - want).abs() / (2.0 ** -8 * want.abs() + 2.0 ** -18 * size)
    assert off.max() <= 1.0 and torch.equal(case.state.cpu().double(), state)
    with pytest.raises(RuntimeError, match="overlap"):
        x = torch.zeros(10, 256, dtype=torch.bfloat16, device="cuda")
        lib().conv_prefill(x, case.state, case.weight, None, case.table, case.context, ints([0, 5, 10]), x, 64)


# ---------------------------------------------------------------------------------------------------------------
# request_tables
# ---------------------------------------------------------------------------------------------------------------
def check_tables(query, context, block, width, n_tokens, n_free, seed=0, faults=0):
    rng = np.random.default_rng(seed)
    n = len(query)
    table = rng.integers(1, 1 << 20, (n, width))
    free = rng.integers(1, 1 << 20, n_free)
    want = prompt_oracle.tables(query, context, free.tolist(), table, n_tokens, block)
    wide = torch.full((n, width + 3), -7, dtype=torch.int32, device="cuda")
    wide[:, :width] = torch.from_numpy(table)
    got = wide[:, :width]
    cu, used, pairs = torch.empty(n + 1, dtype=torch.int32, device="cuda"), ints([0]), torch.empty(n, 2, dtype=torch.int32, device="cuda")
    positions, slot_map = (torch.empty(n_tokens, dtype=torch.int64, device="cuda") for _ in range(2))
    lib().request_tables(ints(query), ints(context), torch.from_numpy(free).int().cuda(), got, cu, positions, slot_map, pairs,
                         used, block)
    torch.cuda.synchronize()
    for x, y in zip((cu, got, positions, slot_map, pairs, used), want):
        assert np.array_equal(x.cpu().numpy().reshape(np.shape(y)), y)
    assert bool((wide[:, width:] == -7).all())
    assert capi.fault_flags() == faults


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 600, 1024, 1025, 2500])
@pytest.mark.parametrize("block", [1, 16, 48])
def test_request_tables(n, block):
    rng = np.random.default_rng(n + block)
    query, context = rng.integers(0, 40, n).tolist(), rng.integers(0, 100, n).tolist()
    need = sum(-(-(c + q) // block) - -(-c // block) for q, c in zip(query, context))
    check_tables(query, context, block, -(-140 // block), sum(query) + n % 5, need + 1, seed=n)


def test_request_tables_edges():
    blocks = capi.LD_FAULT_TABLE_BLOCKS
    check_tables([], [], 16, 4, 5, 3)
    check_tables([0, 0], [0, 5], 16, 2, 0, 0)
    check_tables([100], [0], 16, 7, 100, 7)
    check_tables([20, 30], [0, 10], 16, 4, 50, 2, faults=blocks)            # the free list runs out
    check_tables([40, 3], [30, 0], 16, 3, 43, 9, faults=blocks)              # a row is too short
    check_tables([5, -3, 4], [-2, 7, 9], 16, 3, 9, 9, faults=capi.LD_FAULT_TABLE_LENGTHS)
    check_tables([5, 6], [0, 0], 16, 3, 8, 9, faults=capi.LD_FAULT_TABLE_LENGTHS)  # more tokens than rows
    check_tables([3], [2 ** 31 - 40], 1 << 30, 2, 3, 1)                      # positions and slots past 2^31
    check_tables([10], [2 ** 31 - 5], 1 << 29, 5, 12, 3)


def test_request_tables_one_long_prompt():
    check_tables([300000, 1], [0, 300000], 16, 18752, 300001, 18752)


def test_request_tables_many_requests():
    rng = np.random.default_rng(5)
    check_tables(rng.integers(0, 4, 70000).tolist(), rng.integers(0, 64, 70000).tolist(), 16, 5, 140000 - 140000 % 7 + 70000, 80000)


# ---------------------------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("pool", [torch.float32, torch.bfloat16])
def test_prompts_then_tokens(pool):
    """The path of a server: tables from lengths, convolution, prefill, then single tokens through tables, conv_update
    and decode on the state slots that the tables give, over the end of a block; against the oracle on each request's
    whole sequence.  A bf16 pool is rounded at every token's store, half a step each, and the rounded state decays
    into the next: eight tokens' half steps of 2^-8 at most.  The tokens' convolution rounds products and results to
    bf16 where the oracle, too, is given those activations."""
    h, hv, block, lens, extra = 1, 2, 64, [60, 1, 130, 125], 8
    dim = (2 * h + hv) * DIM
    gen = torch.Generator().manual_seed(40)
    f = lambda *shape: torch.randn(*shape, generator=gen)  # noqa: E731
    total = [n + extra for n in lens]
    xs = [f(n, dim).bfloat16().cuda() for n in total]
    gates = [f(n, hv, DIM).bfloat16().cuda() for n in total]
    abs_ = [f(n, 2 * hv).bfloat16().cuda() for n in total]
    a_log, dt_bias = (f(hv) * 0.3).cuda(), (f(hv) - 2).cuda()
    weight, conv_weight = (1 + 0.1 * f(DIM)).bfloat16().cuda(), (0.5 * f(dim, 4)).bfloat16().cuda()
    n, width = len(lens), 4
    free = (torch.randperm(30, generator=gen) + 1).int().cuda()
    table = torch.zeros(n, width, dtype=torch.int32, device="cuda")
    state = torch.zeros(31, hv, DIM, DIM, dtype=pool, device="cuda")
    conv_state = torch.zeros(31, dim, 3, dtype=torch.bfloat16, device="cuda")
    backend = GDNBackend(BackendConfig(compute="cuda_fused", state_io="indexed"))
    context, query, taken = ints([0] * n), ints(lens), 0
    outs, activations = [[] for _ in lens], [[] for _ in lens]
    for step in range(1 + extra):
        count = lens if step == 0 else [1] * n
        tokens = sum(count)
        done = [0] * n if step == 0 else [k + step - 1 for k in lens]
        rows = lambda parts: torch.cat([p[d:d + c] for p, d, c in zip(parts, done, count)])  # noqa: B023, E731
        cu = torch.empty(n + 1, dtype=torch.int32, device="cuda")
        pairs, used = torch.empty(n, 2, dtype=torch.int32, device="cuda"), ints([0])
        positions, slot_map = (torch.empty(tokens, dtype=torch.int64, device="cuda") for _ in range(2))
        lib().request_tables(query, context, free[taken:], table, cu, positions, slot_map, pairs, used, block)
        x, gate, ab = rows(xs), rows(gates), rows(abs_)
        out = torch.empty(tokens, hv, DIM, dtype=torch.bfloat16, device="cuda")
        qkv = torch.empty_like(x)
        lib().conv_prefill(x, conv_state, conv_weight, None, table, context, cu, qkv, block)
        if step == 0:
            backend.prefill(qkv, ab[:, hv:], ab[:, :hv], a_log, dt_bias, table, context, cu, state, gate, weight, out, block)
        else:
            backend(qkv, ab[:, hv:], ab[:, :hv], a_log, dt_bias, pairs, cu, ints([2] * n), state, gate, weight, out)
        for r in range(n):
            part = slice(int(cu[r]), int(cu[r + 1]))
            outs[r].append(out[part])
            activations[r].append(qkv[part])
        taken += int(used)
        context, query = context + query, ints([1] * n)
    assert backend.calls == {"prefill": 1, "verify": extra}
    assert capi.fault_flags() == 0
    for r in range(n):
        mine = torch.cat(activations[r])
        want, size, expect = prompt_oracle.prefill(
            mine, abs_[r][:, hv:], abs_[r][:, :hv], a_log, dt_bias, table[r:r + 1], ints([0]), ints([0, total[r]]),
            torch.zeros(31, hv, DIM, DIM), gates[r], weight, block)
        conv_want, conv_size, windows = prompt_oracle.conv(xs[r], torch.zeros(31, dim, 3), conv_weight, None, table[r:r + 1],
                                                           ints([0]), ints([0, total[r]]), block)
        off = (mine.cpu().double() - conv_want).abs() / (2.0 ** -8 * conv_want.abs() + 2.0 ** -18 * conv_size + 1e-30)
        assert off.max() <= 1.0
        slots = table[r, : -(-total[r] // block)].tolist()
        assert torch.equal(conv_state[slots].cpu().double(), windows[slots])
        got = torch.cat(outs[r]).cpu().double()
        # decode rounds its recurrence outputs once more (half a step, on values of the outputs' size); a bf16 pool's
        # states carry up to eight half steps of 2^-8 into S q.
        loose = (2.0 ** -9 + (extra * 2.0 ** -8 if pool == torch.bfloat16 else 0.0)) * size + 2.0 ** -8 * size
        off = (got - want).abs() / (2 * 2.0 ** -8 * want.abs() + loose + 1e-30)
        assert off.max() <= 1.0
        scale = expect[slots].abs().amax(dim=(2, 3), keepdim=True)
        steps = extra * 2.0 ** -8 if pool == torch.bfloat16 else 0.0
        assert ((state[slots].cpu().double() - expect[slots]).abs() / ((STATE + steps) * scale)).max() <= 1.0
