"""CPU tests of the prompt path's boundary: host-side refusals of its C entry points, the operators' schemas and
fake kernels, and the 64-bit oracle against the decode's.  Nothing here launches a kernel: every refused call would
have to touch addresses that are not memory."""

import numpy as np
import pytest
import torch

import oracle
import prompt_oracle

FAKE = 1 << 20  # aligned, not NULL, never read
FAR = 1 << 40


def prefill_args(**changes):
    args = dict(qkv=FAKE, qkv_row=512, a=FAKE, a_row=2, b=FAKE, b_row=2, a_log=FAKE, dt_bias=FAKE, dt_dtype=0, table=FAKE,
                table_row=4, table_width=4, block=64, context=FAKE, cu=FAKE, requests=3, state=FAKE, state_dtype=0, slots=5,
                slot_stride=2 * 128 * 128, gate=FAKE, gate_row=256, weight=FAKE, w_dtype=1, out=FAR, tokens=100, h=1,
                hv=2, eps=1e-6, workspace=FAKE, size=1 << 40, stream=None)
    assert set(changes) <= set(args)
    return list({**args, **changes}.values())


@pytest.mark.parametrize("changes, message", [
    (dict(h=0), "multiple of num_k_heads"),
    (dict(h=2, hv=3), "multiple of num_k_heads"),
    (dict(eps=0.0), "epsilon"),
    (dict(block=0), "block_size"),
    (dict(block=32), "multiple of 64"),
    (dict(block=96), "multiple of 64"),
    (dict(requests=-1), "out of range"),
    (dict(tokens=-1), "out of range"),
    (dict(tokens=1 << 40), "out of range"),
    (dict(requests=1 << 31), "out of range"),
    (dict(state_dtype=2), "fp32 or bf16"),
    (dict(dt_dtype=3), "fp32 or bf16"),
    (dict(slots=0), "at least one slot"),
    (dict(slot_stride=2 * 128 * 128 - 4), "slot stride"),
    (dict(slot_stride=2 * 128 * 128 + 2), "divisible by 4"),
    (dict(state_dtype=1, slot_stride=2 * 128 * 128 + 4), "divisible"),
    (dict(table_width=0), "at least one block"),
    (dict(table_row=3), "do not overlap"),
    (dict(qkv_row=511), "smaller than the rows"),
    (dict(gate_row=255), "smaller than the rows"),
    (dict(a_row=1), "smaller than the rows"),
    (dict(qkv=None), "NULL"),
    (dict(cu=None), "NULL"),
    (dict(out=None), "NULL"),
    (dict(out=FAKE), "overlap"),
    (dict(out=FAKE + 2 * (99 * 512 + 511)), "overlap"),
    (dict(out=FAR, gate=FAR + 2 * 100 * 256 - 2), "overlap"),
    (dict(workspace=None), "workspace"),
    (dict(workspace=FAKE + 64), "128-byte aligned workspace"),
    (dict(size=1000), "workspace of"),
    (dict(state=FAKE + 4), "16-byte aligned"),
    (dict(qkv=FAKE + 1), "2-byte aligned"),
])
def test_prefill_refusals(native, changes, message):
    assert native.lib().ld_prefill(*prefill_args(**changes)) == native.LD_ERR_INVALID
    assert message in native.last_error()


def test_prefill_without_work_is_a_no_op(native):
    for changes in (dict(requests=0), dict(tokens=0), dict(requests=0, tokens=0, qkv=None, workspace=None)):
        assert native.lib().ld_prefill(*prefill_args(**changes)) == native.LD_OK


def test_prefill_workspace_size(native):
    size = native.prefill_workspace
    assert size(64, 1, 16, 32) < size(6400, 1, 16, 32) < size(6400, 100, 16, 32) < size(6400, 100, 16, 48)
    # Per chunk: q and k of a key head (32 KiB), triangular factors of a value head (16.1 KiB); requests share chunks
    # at most at two places each.  One head's long prompt runs in 16 pieces with 29 states of 64 KiB between them.
    assert size(64 * 1000, 1, 1, 1) <= 1002 * (32768 + 16640) + 29 * 65536 + 256
    assert size(64 * 1000, 1, 1, 149) <= 1002 * (32768 + 149 * 16640) + 256
    for bad in ((-1, 1, 1, 1), (1, -1, 1, 1), (1, 1, 0, 1), (1, 1, 1, 1 << 20)):
        with pytest.raises(native.LightDeltaError):
            size(*bad)


def conv_args(**changes):
    args = dict(x=FAKE, x_row=300, tokens=50, dim=256, state=FAKE, slots=4, s_slot=768, s_dim=3, s_pos=1, length=3,
                weight=FAKE, bias=None, width=4, table=FAKE, table_row=2, table_width=2, block=64, context=FAKE, cu=FAKE,
                requests=2, out=FAKE + (1 << 20), stream=None)
    assert set(changes) <= set(args)
    return list({**args, **changes}.values())


@pytest.mark.parametrize("changes, message", [
    (dict(width=1), "2 through 4"),
    (dict(width=5), "2 through 4"),
    (dict(length=2), "fewer than width - 1"),
    (dict(block=0), "block_size"),
    (dict(dim=0), "out of range"),
    (dict(tokens=1 << 33), "out of range"),
    (dict(requests=-2), "out of range"),
    (dict(table_width=0), "at least one block"),
    (dict(table_row=1), "do not overlap"),
    (dict(x_row=255), "invalid strides"),
    (dict(slots=0), "invalid strides"),
    (dict(s_dim=2), "overlap"),
    (dict(s_slot=767), "overlap"),
    (dict(x=None), "NULL"),
    (dict(table=None), "NULL"),
    (dict(out=None), "NULL"),
    (dict(out=FAKE + 1 + (1 << 20)), "2-byte aligned"),
    (dict(out=FAKE), "must not overlap"),
    (dict(out=FAKE + 2 * 300 * 49), "must not overlap"),
    (dict(out=FAKE - 2), "must not overlap"),
])
def test_conv_prefill_refusals(native, changes, message):
    assert native.lib().ld_conv_prefill(*conv_args(**changes)) == native.LD_ERR_INVALID
    assert message in native.last_error()


def test_conv_prefill_without_work_is_a_no_op(native):
    for changes in (dict(requests=0), dict(tokens=0)):
        assert native.lib().ld_conv_prefill(*conv_args(**changes)) == native.LD_OK


def tables_args(**changes):
    args = dict(query=FAKE, context=FAKE, requests=4, free=FAKE, n_free=10, table=FAKE, table_row=8, table_width=8, block=16,
                cu=FAKE, positions=FAKE, slot_map=FAKE, tokens=20, pairs=FAKE, used=FAKE, stream=None)
    assert set(changes) <= set(args)
    return list({**args, **changes}.values())


@pytest.mark.parametrize("changes, message", [
    (dict(requests=-1), "out of range"),
    (dict(tokens=-1), "out of range"),
    (dict(n_free=-1), "out of range"),
    (dict(block=0), "block_size"),
    (dict(block=(1 << 30) + 1), "block_size"),
    (dict(table_width=0), "at least one block"),
    (dict(table_row=7), "do not overlap"),
    (dict(cu=None), "NULL"),
    (dict(query=None), "NULL"),
    (dict(free=None), "NULL"),
    (dict(positions=None), "NULL"),
    (dict(used=None), "NULL"),
    (dict(query=FAKE + 2), "4-byte aligned"),
    (dict(slot_map=FAKE + 4), "8-byte aligned"),
])
def test_request_tables_refusals(native, changes, message):
    assert native.lib().ld_request_tables(*tables_args(**changes)) == native.LD_ERR_INVALID
    assert message in native.last_error()


def test_schemas(native):
    from lightdelta_b200 import ops  # noqa: F401

    assert str(torch.ops.lightdelta.prefill.default._schema) == (
        "lightdelta::prefill(Tensor qkv, Tensor a, Tensor b, Tensor a_log, Tensor dt_bias, Tensor table, Tensor context, "
        "Tensor cu, Tensor(s!) state, Tensor gate, Tensor weight, Tensor(o!) out, int block_size, float eps) -> ()")
    assert str(torch.ops.lightdelta.conv_prefill.default._schema) == (
        "lightdelta::conv_prefill(Tensor x, Tensor(c!) conv_state, Tensor conv_weight, Tensor? conv_bias, Tensor table, "
        "Tensor context, Tensor cu, Tensor(o!) out, int block_size) -> ()")
    assert str(torch.ops.lightdelta.request_tables.default._schema) == (
        "lightdelta::request_tables(Tensor query_lens, Tensor context, Tensor free_blocks, Tensor(t!) table, "
        "Tensor(c!) cu, Tensor(p!) positions, Tensor(m!) slot_map, Tensor(s!) state_slots, Tensor(u!) used, "
        "int block_size) -> ()")


def test_fake_kernels_allow_tracing(native):
    from torch._subclasses.fake_tensor import FakeTensorMode

    from lightdelta_b200 import ops  # noqa: F401

    with FakeTensorMode():
        i32, bf16 = torch.int32, torch.bfloat16
        table, context, cu = torch.zeros(2, 4, dtype=i32), torch.zeros(2, dtype=i32), torch.zeros(3, dtype=i32)
        x, out = torch.empty(10, 512, dtype=bf16), torch.empty(10, 512, dtype=bf16)
        assert torch.ops.lightdelta.conv_prefill(x, torch.empty(9, 512, 3, dtype=bf16), torch.empty(512, 4, dtype=bf16),
                                                 None, table, context, cu, out, 64) is None
        ab, gate = torch.empty(10, 2, dtype=bf16), torch.empty(10, 2, 128, dtype=bf16)
        assert torch.ops.lightdelta.prefill(out, ab, ab, torch.empty(2), torch.empty(2), table, context, cu,
                                            torch.empty(9, 2, 128, 128), gate, torch.empty(128), gate.clone(), 64,
                                            1e-6) is None
        long = torch.empty(10, dtype=torch.int64)
        assert torch.ops.lightdelta.request_tables(context, context, context, table, cu, long, long, table[:, :2], context,
                                                   64) is None


def test_oracle_of_a_prompt_is_decode_token_by_token():
    """The prompt oracle on a request continued inside a block against the decode oracle (itself pinned to the
    reference) fed the same tokens one by one.  Both recurrences keep each step within fp32 rounding: 2^-24 per
    element and operation, a hundred sums of 128 at most, so 2^-12 of the largest value is far beyond either."""
    rng = np.random.default_rng(3)
    h, hv, n, slots = 1, 2, 9, 3
    f = lambda *shape: torch.from_numpy(rng.standard_normal(shape).astype(np.float32))  # noqa: E731
    qkv, gate = f(n, (2 * h + hv) * 128).bfloat16(), f(n, hv, 128).bfloat16()
    a, b = f(n, hv).bfloat16(), f(n, hv).bfloat16()
    a_log, dt_bias, weight = f(hv) * 0.1, f(hv), f(128).bfloat16()
    state = f(slots, hv, 128, 128) * 0.1
    out, _, pool = prompt_oracle.prefill(qkv, a, b, a_log, dt_bias, torch.tensor([[2, 1]]), torch.tensor([60]),
                                         torch.tensor([0, n]), state, gate, weight, 64)
    bits = lambda t: t.view(torch.int16).numpy().view(np.uint16).copy()  # noqa: E731
    steps, got = state.numpy().copy(), np.zeros((n, hv, 128), np.uint16)
    for t in range(n):
        one = np.zeros((1, hv, 128), np.uint16)
        slot = np.array([[2 if 60 + t < 64 else 1]], np.int32)
        if 60 + t == 64:
            steps[1] = steps[2]
        oracle.decode(bits(qkv[t:t + 1]), bits(a[t:t + 1]), bits(b[t:t + 1]), a_log.numpy(), dt_bias.numpy(), slot,
                      np.array([0, 1], np.int32), np.ones(1, np.int32), steps, bits(gate[t:t + 1]), bits(weight), one,
                      num_k_heads=h)
        got[t] = one[0]
    for slot in (1, 2):
        want = pool[slot].numpy()
        assert np.abs(steps[slot] - want).max() <= 2 ** -12 * np.abs(want).max()
    # The decode rounds its recurrence outputs and its results to bf16: two half steps.
    values = oracle.bf16_to_f32(got)
    want = out.numpy()
    scale = np.abs(want) + 2 ** -6 * np.abs(want).max()
    assert (np.abs(values - want) / scale).max() <= 2 * 2 ** -8


def test_oracle_of_tables_by_hand():
    cu, table, positions, slot_map, pairs, used = prompt_oracle.tables(
        [3, 0, 5, 1], [6, 4, 0, 8], [50, 51, 52, 53], [[7, 8, 0], [9, 0, 0], [0, 0, 0], [1, 2, 3]], 11, 4)
    assert cu.tolist() == [0, 3, 3, 8, 9] and used == 4
    assert table.tolist() == [[7, 8, 50], [9, 0, 0], [51, 52, 0], [1, 2, 53]]
    assert positions.tolist() == [6, 7, 8, 0, 1, 2, 3, 4, 8, -1, -1]
    assert slot_map.tolist() == [34, 35, 200, 204, 205, 206, 207, 208, 212, -1, -1]
    assert pairs.tolist() == [[50, 8], [0, 9], [52, 0], [53, 2]]


def test_backend_prefill_needs_indexed_state():
    from lightdelta_b200.backend import GDNBackend
    from lightdelta_b200.config import BackendConfig

    backend = GDNBackend(BackendConfig(compute="cuda_fused", state_io="packed"))
    with pytest.raises(ValueError, match="indexed"):
        backend.prefill(*[None] * 13)
    assert backend.calls["prefill"] == 0
