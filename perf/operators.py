"""Cases of the prompt path's operators: what each is called with, its plain form, and its value in 64 bits.

Three operators run one after the other when a batch of prompts (or pieces of prompts) enters the server:

  tables   torch.ops.lightdelta.request_tables: from the requests' lengths, on the GPU, the token offsets, the block
           table's new entries (taken from a list of free blocks), every token's position and cache slot, and the
           state slots that a following decode reads and writes
  conv     torch.ops.lightdelta.conv_prefill: the causal depthwise convolution (and silu) over whole prompts, which
           leaves each block's convolution window in the pool
  prefill  torch.ops.lightdelta.prefill: gated delta rule attention (linear attention with a decay for each head) over
           whole prompts, with the gated norm, which leaves each block's state in the pool

Geometry: key and value heads of 128; a block of the table covers ``block`` tokens and names one slot of the state
pool, which holds the state after the block's last token (or after the prompt's last token, in its last block).
"""

import math
import random

import torch

own = False

DIM = 128
CHUNK = 64
EPS = 1e-6


# ---------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------
def _prefill(name, tokens, requests, h, hv, block, context, pool, ragged=1):
    case = {"op": "prefill", "tokens": tokens, "requests": requests, "h": h, "hv": hv, "block": block,
            "context": context, "pool": pool, "ragged": ragged}
    return {"name": name, **case} if name else case


def _conv(name, tokens, requests, h, hv, block, context, width, bias, token_first, ragged=1):
    case = {"op": "conv", "tokens": tokens, "requests": requests, "h": h, "hv": hv, "block": block,
            "context": context, "width": width, "bias": bias, "token_first": token_first, "ragged": ragged}
    return {"name": name, **case} if name else case


def _tables(name, tokens, requests, block, context, pad, ragged=1):
    case = {"op": "tables", "tokens": tokens, "requests": requests, "block": block, "context": context, "pad": pad,
            "ragged": ragged}
    return {"name": name, **case} if name else case


def listed():
    return [
        # The shortest useful prompt, alone: time to first token of an interactive request.
        _prefill("prefill 1x17", 17, 1, 16, 32, 1024, 0, "float32"),
        # One long prompt alone on the GPU: nothing but heads and state columns to spread over the SMs.
        _prefill("prefill 1x16384", 16384, 1, 16, 32, 1024, 0, "float32"),
        # A server's ordinary batch of prompts of mixed lengths.
        _prefill("prefill 24 ragged", 16000, 24, 16, 32, 1024, 0, "float32"),
        # Pieces of longer prompts on the larger geometry with a bf16 pool: each request continues from a cached block.
        _prefill("prefill 8 continued bf16", 16384, 8, 16, 48, 512, 2048, "bfloat16"),
        # Many short prompts (chat turns after a cached system prompt).
        _prefill("prefill 128 short", 7001, 128, 16, 32, 128, 256, "float32"),
        # The convolution of the same three kinds: shortest, an ordinary batch, the largest continued one.
        _conv("conv 1x17", 17, 1, 16, 32, 1024, 0, 4, False, True),
        _conv("conv 24 ragged", 16000, 24, 16, 32, 1024, 0, 4, False, True),
        _conv("conv 8 continued", 16384, 8, 16, 48, 512, 2048, 4, True, False),
        # One decode step of 8 requests, one of 256 prompts, one of 4096 requests with long caches.
        _tables("tables 8 decodes", 8, 8, 64, 1000, 0),
        _tables("tables 256 prompts", 120000, 256, 64, 0, 72),
        _tables("tables 4096 mixed", 400000, 4096, 64, 4000, 1600),
    ]


def draw(rng):
    def spread(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))

    op = rng.choice(("prefill", "prefill", "conv", "tables"))
    ragged = rng.randrange(1 << 20)
    if op == "tables":
        requests = spread(1, 4096)
        tokens = spread(requests, min(400000, requests * 2000))
        return _tables(None, tokens, requests, rng.choice((16, 64, 128, 256)), rng.choice((0, spread(1, 4000))),
                       rng.choice((0, rng.randrange(1, 512))), ragged)
    requests = spread(1, 128)
    tokens = spread(requests, 16000 if requests < 32 else 8000)
    h, hv = rng.choice(((16, 32), (16, 48), (8, 16), (4, 12), (2, 4), (4, 4)))
    block = rng.choice((128, 256, 512, 1024))
    context = rng.choice((0, 0, block, 2 * block))
    if op == "conv":
        return _conv(None, tokens, requests, h, hv, block, context, rng.choice((2, 3, 4)), rng.random() < 0.5,
                     rng.random() < 0.5, ragged)
    return _prefill(None, tokens, requests, h, hv, block, context, rng.choice(("float32", "bfloat16")), ragged)


def _lengths(case):
    """The requests' token counts: they sum to case["tokens"], each is one at least, and they differ by about a
    factor of ten from shortest to longest."""
    rng = random.Random(case["ragged"])
    n, total = case["requests"], case["tokens"]
    weight = [math.exp(rng.uniform(0.0, 2.3)) for _ in range(n)]
    scale = (total - n) / sum(weight)
    lens = [1 + int(w * scale) for w in weight]
    for i in range(total - sum(lens)):
        lens[i % n] += 1
    rng.shuffle(lens)
    return lens


def _contexts(case):
    """Tokens already held: prefill and conv continue at the end of a block (a cached prefix), some requests from
    nothing; the tables are built at any length."""
    rng = random.Random(case["ragged"] + 1)
    n, context = case["requests"], case["context"]
    if case["op"] == "tables":
        return [rng.randrange(context // 2, context + 1) if context else 0 for _ in range(n)]
    return [context if i == 0 or rng.random() < 0.75 else 0 for i in range(n)]


def _blocks(case):
    """(blocks a row of the table has, blocks that are written in all)."""
    lens, ctx, bs = _lengths(case), _contexts(case), case["block"]
    width = max(-(-(c + n) // bs) for c, n in zip(ctx, lens))
    written = sum(-(-(c + n) // bs) - c // bs for c, n in zip(ctx, lens))
    return width, written


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dev = torch.device("cuda")

    def randn(*shape, scale=1.0):
        return torch.randn(*shape, device=dev, generator=gen) * scale

    def ints(values):
        return torch.tensor(values, device=dev, dtype=torch.int32)

    lens, ctx, bs, n = _lengths(case), _contexts(case), case["block"], case["tokens"]
    requests = case["requests"]
    width, written = _blocks(case)
    s = {"op": case["op"], "block": bs, "context": ints(ctx), "tokens": n, "longest": max(lens)}
    if case["op"] == "tables":
        held = [-(-c // bs) for c in ctx]
        # Held blocks and free ones are spread over a cache of a million blocks; lengths vary with the seed by moving
        # the contexts, so that the sum of the new tokens stays the batch's.
        s["context"] = torch.clamp(s["context"] - torch.randint(0, bs, (requests,), device=dev, generator=gen), min=0)
        s["context"] = s["context"].to(torch.int32).contiguous()
        s["query_lens"] = ints(lens)
        free = torch.randperm(1 << 20, device=dev, generator=gen)[: written + sum(held) + requests + 1] + 1
        s["free"] = free.to(torch.int32)
        s["table"] = torch.randint(1, 1 << 20, (requests, width), device=dev, generator=gen, dtype=torch.int32)
        total = n + case["pad"]
        s["cu"] = torch.empty(requests + 1, device=dev, dtype=torch.int32)
        s["positions"] = torch.empty(total, device=dev, dtype=torch.int64)
        s["slot_map"] = torch.empty(total, device=dev, dtype=torch.int64)
        s["state_slots"] = torch.empty(requests, 2, device=dev, dtype=torch.int32)
        s["used"] = torch.empty(1, device=dev, dtype=torch.int32)
        return s
    offsets = [0]
    for v in lens:
        offsets.append(offsets[-1] + v)
    s["cu"] = ints(offsets)
    slots = requests * width
    s["table"] = (torch.randperm(slots, device=dev, generator=gen) + 1).to(torch.int32).view(requests, width).contiguous()
    h, hv = case["h"], case["hv"]
    dim = (2 * h + hv) * DIM
    if case["op"] == "conv":
        # The layer's projection: q, k, v beside the output gate in one row.
        proj = randn(n, dim + hv * DIM).to(torch.bfloat16)
        s["x"] = proj[:, :dim]
        w = case["width"]
        state = randn(slots + 1, w - 1, dim) if case["token_first"] else randn(slots + 1, dim, w - 1)
        state = state.to(torch.bfloat16)
        s["conv_state"] = state.transpose(1, 2) if case["token_first"] else state
        s["weight"] = randn(dim, w, scale=0.5).to(torch.bfloat16)
        s["bias"] = randn(dim, scale=0.2).to(torch.bfloat16) if case["bias"] else None
        s["out"] = torch.empty(n, dim, device=dev, dtype=torch.bfloat16)
        return s
    # q, k, v as they come out of the convolution's silu; decays and step sizes as the layer is initialised (A in
    # 1..16, a step of 0.001 to 0.1 per token), so that heads remember from a few tokens to a few thousand.
    s["qkv"] = torch.nn.functional.silu(randn(n, dim, scale=1.5)).to(torch.bfloat16)
    s["gate"] = randn(n, hv, DIM).to(torch.bfloat16)
    ab = randn(n, 2 * hv, scale=0.7).to(torch.bfloat16)
    s["a"], s["b"] = ab[:, hv:], ab[:, :hv]
    s["a_log"] = torch.log(1 + 15 * torch.rand(hv, device=dev, generator=gen))
    step = torch.exp(math.log(1e-3) + math.log(100.0) * torch.rand(hv, device=dev, generator=gen))
    s["dt_bias"] = step + torch.log(-torch.expm1(-step))
    s["weight"] = (1 + randn(DIM, scale=0.1)).to(torch.bfloat16)
    s["state"] = randn(slots + 1, hv, DIM, DIM, scale=0.05).to(getattr(torch, case["pool"]))
    s["out"] = torch.empty(n, hv, DIM, device=dev, dtype=torch.bfloat16)
    return s


# ---------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------
def run(state):
    if own:
        return _own(state)
    return {"tables": _plain_tables, "conv": _plain_conv, "prefill": _plain_prefill}[state["op"]](state)


def _own(s):
    from lightdelta_b200 import ops  # noqa: F401

    lib = torch.ops.lightdelta
    if s["op"] == "tables":
        lib.request_tables(s["query_lens"], s["context"], s["free"], s["table"], s["cu"], s["positions"],
                           s["slot_map"], s["state_slots"], s["used"], s["block"])
        return {k: s[k] for k in ("table", "cu", "positions", "slot_map", "state_slots", "used")}
    if s["op"] == "conv":
        lib.conv_prefill(s["x"], s["conv_state"], s["weight"], s["bias"], s["table"], s["context"], s["cu"], s["out"],
                         s["block"])
        return {"out": s["out"], "conv_state": s["conv_state"]}
    lib.prefill(s["qkv"], s["a"], s["b"], s["a_log"], s["dt_bias"], s["table"], s["context"], s["cu"], s["state"],
                s["gate"], s["weight"], s["out"], s["block"], EPS)
    return {"out": s["out"], "state": s["state"]}


def _ceil(x, d):
    return torch.div(x + (d - 1), d, rounding_mode="floor")


def _plain_tables(s):
    bs, table = s["block"], s["table"]
    q, ctx = s["query_lens"].long(), s["context"].long()
    dev, n, width = q.device, s["positions"].numel(), table.shape[1]
    cu = torch.cat((q.new_zeros(1), torch.cumsum(q, 0)))
    have, want = _ceil(ctx, bs), _ceil(ctx + q, bs)
    need = want - have
    first = torch.cumsum(need, 0) - need
    col = torch.arange(width, device=dev)[None, :]
    new = (col >= have[:, None]) & (col < want[:, None])
    at = torch.where(new, first[:, None] + col - have[:, None], torch.zeros_like(col))
    table.copy_(torch.where(new, s["free"][at], table))
    token = torch.arange(n, device=dev)
    row = torch.searchsorted(cu, token, right=True) - 1
    live = row < q.numel()
    row = torch.clamp(row, max=q.numel() - 1)
    pos = ctx[row] + token - cu[row]
    page = table[row, torch.clamp(torch.div(pos, bs, rounding_mode="floor"), max=width - 1)].long()
    minus = torch.full_like(pos, -1)
    last = torch.gather(table, 1, torch.clamp(want - 1, min=0)[:, None])[:, 0]
    held = torch.gather(table, 1, torch.clamp(have - 1, min=0)[:, None])[:, 0]
    zero = torch.zeros_like(last)
    pair = torch.stack((torch.where(q > 0, last, zero), torch.where(ctx > 0, held, zero)), 1)
    return {"table": table, "cu": cu.to(torch.int32), "positions": torch.where(live, pos, minus),
            "slot_map": torch.where(live, page * bs + pos % bs, minus), "state_slots": pair,
            "used": need.sum().to(torch.int32).reshape(1)}


def _block_ends(s, width):
    """For every (request, block of its row): the context-relative end of what the block holds after this call, the
    slot that takes it, and whether the block is written."""
    bs = s["block"]
    ctx, cu = s["context"].long(), s["cu"].long()
    n = cu[1:] - cu[:-1]
    col = torch.arange(width, device=ctx.device)[None, :]
    end = torch.minimum((col + 1) * bs, (ctx + n)[:, None])
    written = (n > 0)[:, None] & (col >= (ctx // bs)[:, None]) & (col * bs < (ctx + n)[:, None])
    return end - ctx[:, None], torch.where(written, s["table"].long(), torch.zeros_like(end)), written


def _plain_conv(s):
    x, state, table, cu, ctx, w = s["x"], s["conv_state"], s["table"], s["cu"].long(), s["context"].long(), s["weight"]
    taps, bs = w.shape[1], s["block"]
    n, dev = x.shape[0], x.device
    source = torch.gather(table.long(), 1, torch.clamp(_ceil(ctx, bs) - 1, min=0)[:, None])[:, 0]
    history = state[source][:, :, : taps - 1].float() * (ctx > 0)[:, None, None]
    token = torch.arange(n, device=dev)
    row = torch.searchsorted(cu, token, right=True) - 1
    local = token - cu[row]

    def tap(back):
        """The input `back` tokens before each token: an earlier row, or the request's history."""
        earlier = x[torch.clamp(token - back, min=0)].float()
        old = history[row, :, torch.clamp(taps - 1 + local - back, 0, taps - 2)]
        return torch.where((local >= back)[:, None], earlier, old)

    y = sum(tap(taps - 1 - j) * w[:, j].float() for j in range(taps))
    if s["bias"] is not None:
        y = y + s["bias"].float()
    out = (y / (1 + torch.exp(-y))).to(torch.bfloat16)
    end, slot, written = _block_ends(s, table.shape[1])
    at = end[:, :, None] - (taps - 1) + torch.arange(taps - 1, device=dev)
    inside = x[torch.clamp(cu[:-1, None, None] + at, 0, n - 1)]
    reqs = torch.arange(ctx.numel(), device=dev)[:, None, None]
    before = history.to(x.dtype)[reqs, :, torch.clamp(taps - 1 + at, 0, taps - 2)]
    window = torch.where((at >= 0)[..., None], inside, before).transpose(2, 3)
    keep = state[0, :, : taps - 1].clone()
    state[:, :, : taps - 1][slot.reshape(-1)] = torch.where(written[:, :, None, None], window, keep).flatten(0, 1)
    return {"out": out, "conv_state": state}


def _plain_prefill(s):
    """The chunked form: 64 tokens at a time at absolute positions, the tokens of a chunk coupled by the inverse of a
    unit triangular matrix, and the state carried from chunk to chunk, all requests and heads side by side."""
    pool, table, bs = s["state"], s["table"].long(), s["block"]
    cu, ctx = s["cu"].long(), s["context"].long()
    hv, n, dev = pool.shape[1], s["qkv"].shape[0], pool.device
    h = (s["qkv"].shape[1] // DIM - hv) // 2
    requests = ctx.numel()
    lead = ctx % CHUNK
    chunks = -(-(s["longest"] + CHUNK - 1) // CHUNK)
    place = torch.arange(chunks * CHUNK, device=dev)[None, :]
    local = place - lead[:, None]
    length = cu[1:] - cu[:-1]
    live = (local >= 0) & (local < length[:, None])
    token = torch.where(live, cu[:-1, None] + local, torch.zeros_like(local))

    def padded(x, heads):
        """[tokens, heads, ...] to [requests, heads, chunks, 64, ...], zero where no token is."""
        y = x[token].float() * live.view(requests, -1, *([1] * (x.dim() - 1)))
        return y.view(requests, chunks, CHUNK, heads, *x.shape[2:]).movedim(3, 1)

    parts = s["qkv"].view(n, 2 * h + hv, DIM)
    q, k, v = padded(parts[:, :h], h), padded(parts[:, h:2 * h], h), padded(parts[:, 2 * h:], hv)
    q = q / torch.sqrt((q * q).sum(-1, keepdim=True) + 1e-6) * DIM ** -0.5
    k = k / torch.sqrt((k * k).sum(-1, keepdim=True) + 1e-6)
    q, k = (x.repeat_interleave(hv // h, 1) for x in (q, k))
    x = s["a"].double() + s["dt_bias"].double()
    g = -torch.exp(s["a_log"].double()) * torch.where(x > 20, x, torch.log1p(torch.exp(torch.clamp(x, max=20))))
    mask = live.view(requests, 1, chunks, CHUNK)
    g = g[token].view(requests, chunks, CHUNK, hv).movedim(3, 1) * mask
    beta = (1 / (1 + torch.exp(-s["b"].float())))[token].view(requests, chunks, CHUNK, hv).movedim(3, 1) * mask
    total = torch.cumsum(g, -1)
    tri = torch.ones(CHUNK, CHUNK, device=dev, dtype=torch.bool).tril()
    decay = torch.where(tri, torch.exp(total[..., :, None] - total[..., None, :]), 0.0).float()
    within, out_of = torch.exp(total).float(), torch.exp(total[..., -1:] - total).float()
    low = beta[..., None] * decay * (k @ k.transpose(-1, -2)) * tri.tril(-1)
    inv = torch.eye(CHUNK, device=dev).expand_as(low).contiguous()
    for i in range(1, CHUNK):
        inv[..., i, :i] = -(low[..., i:i + 1, :i] @ inv[..., :i, :i])[..., 0, :]
    near = decay * (q @ k.transpose(-1, -2))
    source = torch.gather(table, 1, torch.clamp(_ceil(ctx, bs) - 1, min=0)[:, None])[:, 0]
    S = pool[source].float() * (ctx > 0)[:, None, None, None]
    null = pool[0].clone()
    o = torch.empty_like(v)
    for c in range(chunks):
        kc, scale = k[:, :, c], within[:, :, c, :, None]
        u = inv[:, :, c] @ (beta[:, :, c, :, None] * (v[:, :, c] - scale * (kc @ S.transpose(-1, -2))))
        o[:, :, c] = scale * (q[:, :, c] @ S.transpose(-1, -2)) + near[:, :, c] @ u
        S = within[:, :, c, -1, None, None] * S + (u * out_of[:, :, c, :, None]).transpose(-1, -2) @ kc
        stop = torch.minimum(ctx - lead + (c + 1) * CHUNK, ctx + length)
        begun = ctx - lead + c * CHUNK < ctx + length
        done = begun & ((stop % bs == 0) | (stop == ctx + length))
        slot = torch.gather(table, 1, torch.clamp(_ceil(stop, bs) - 1, min=0)[:, None])[:, 0]
        slot = torch.where(done, slot, torch.zeros_like(slot))
        pool[slot] = torch.where(done[:, None, None, None], S.to(pool.dtype), null)
    token = torch.arange(n, device=dev)
    row = torch.searchsorted(cu, token, right=True) - 1
    o = o.flatten(2, 3)[row, :, lead[row] + token - cu[row]]
    gate = s["gate"].float()
    o = o / torch.sqrt((o * o).mean(-1, keepdim=True) + EPS) * s["weight"].float() * gate / (1 + torch.exp(-gate))
    return {"out": o.to(torch.bfloat16), "state": pool}


# ---------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------
def work(case):
    n, r = case["tokens"], case["requests"]
    width, written = _blocks(case)
    if case["op"] == "tables":
        # Lengths, free blocks and the blocks of the tokens read; offsets, new entries, positions and slots written.
        return {"bytes": 8 * r + 4 * written + 4 * r * width + 4 * r + 4 * written + 16 * (n + case["pad"]) + 8 * r,
                "flops": 0}
    h, hv = case["h"], case["hv"]
    dim = (2 * h + hv) * DIM
    sources = sum(c > 0 for c in _contexts(case))
    if case["op"] == "conv":
        taps = case["width"]
        return {"bytes": 4 * n * dim + 2 * dim * (taps + case["bias"]) + 2 * dim * (taps - 1) * (sources + written),
                "flops": n * dim * (2 * taps + 4)}
    item = 4 if case["pool"] == "float32" else 2
    # Read once: q, k, v, gate, a, b; written once: the output; states read where a request continues, written per
    # block. Operations: the recurrence's decay, prediction, update and read-out of one 128 x 128 state per token.
    return {"bytes": n * (2 * dim + 4 * hv * DIM + 4 * hv) + item * hv * DIM * DIM * (sources + written),
            "flops": 7 * n * hv * DIM * DIM}


# ---------------------------------------------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "tables":
        return None
    s = prepare(case, seed)
    return (_exact_conv if case["op"] == "conv" else _exact_prefill)(case, s)


def _exact_conv(case, s):
    """Request by request: the history in front of its rows, then a correlation with the taps."""
    w = s["weight"].double()
    taps, bs = w.shape[1], case["block"]
    out = torch.empty(s["x"].shape, device=w.device, dtype=torch.float64)
    state = s["conv_state"].double()
    at = 0
    for row, ctx, n in zip(s["table"].tolist(), _contexts(case), _lengths(case)):
        line = torch.zeros(taps - 1 + n, w.shape[0], device=w.device, dtype=torch.float64)
        if ctx:
            line[: taps - 1] = s["conv_state"][row[(ctx - 1) // bs], :, : taps - 1].double().t()
        line[taps - 1:] = s["x"][at:at + n].double()
        y = torch.zeros(n, w.shape[0], device=w.device, dtype=torch.float64)
        if s["bias"] is not None:
            y += s["bias"].double()
        for j in range(taps):
            y += line[j:j + n] * w[:, j]
        out[at:at + n] = y * torch.sigmoid(y)
        stop = ctx + n
        for b in range(ctx // bs, (stop - 1) // bs + 1):
            end = min((b + 1) * bs, stop) - ctx
            state[row[b], :, : taps - 1] = line[end:end + taps - 1].t()
        at += n
    return {"out": out, "conv_state": state}


def _exact_prefill(case, s):
    """The recurrence itself, token after token, for all requests that still have one."""
    lens, ctx, bs, hv = _lengths(case), _contexts(case), case["block"], case["hv"]
    h, n, dev = case["h"], case["tokens"], s["qkv"].device
    parts = s["qkv"].double().view(n, 2 * h + hv, DIM)
    q, k, v = parts[:, :h], parts[:, h:2 * h], parts[:, 2 * h:]
    q = q * (torch.rsqrt((q * q).sum(-1, keepdim=True) + 1e-6) * DIM ** -0.5)
    k = k * torch.rsqrt((k * k).sum(-1, keepdim=True) + 1e-6)
    group = torch.arange(hv, device=dev) // (hv // h)
    keep = torch.exp(-torch.exp(s["a_log"].double())
                     * torch.nn.functional.softplus(s["a"].double() + s["dt_bias"].double(), threshold=1e6))
    beta = torch.sigmoid(s["b"].double())
    pool = s["state"].double()
    table = s["table"].tolist()
    starts = s["cu"].tolist()
    order = sorted(range(len(lens)), key=lambda i: -lens[i])
    S = torch.zeros(len(lens), hv, DIM, DIM, device=dev, dtype=torch.float64)
    for place, i in enumerate(order):
        if ctx[i]:
            S[place] = s["state"][table[i][(ctx[i] - 1) // bs]].double()
    first = torch.tensor([starts[i] for i in order], device=dev)
    o = torch.empty(n, hv, DIM, device=dev, dtype=torch.float64)
    active = len(order)
    for t in range(lens[order[0]]):
        while lens[order[active - 1]] <= t:
            active -= 1
        at = first[:active] + t
        kt, M = k[at][:, group], S[:active]
        M *= keep[at][..., None, None]
        miss = beta[at][..., None] * (v[at] - (M @ kt[..., None])[..., 0])
        M += miss[..., :, None] * kt[..., None, :]
        o[at] = (M @ q[at][:, group][..., None])[..., 0]
        for place in range(active):
            i = order[place]
            if t + 1 == lens[i] or (ctx[i] + t + 1) % bs == 0:
                pool[table[i][(ctx[i] + t) // bs]] = M[place]
    gate = s["gate"].double()
    o = o * torch.rsqrt((o * o).mean(-1, keepdim=True) + EPS) * s["weight"].double() * gate * torch.sigmoid(gate)
    return {"out": o, "state": pool}
