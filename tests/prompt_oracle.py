"""The prompt path's operators from their definitions, in 64 bits and token by token, on the CPU."""

from __future__ import annotations

import numpy as np
import torch

DIM = 128


def softplus(x):
    return torch.where(x > 30, x, torch.log1p(torch.exp(torch.clamp(x, max=30))))


def prefill(qkv, a, b, a_log, dt_bias, table, context, cu, state, gate, weight, block_size, eps=1e-6):
    """(outputs, bound, pool): the outputs [tokens, HV, 128] with NaN where no request writes, what the products that
    only reach the outputs sum up in magnitude (in units of the output), and the pool afterwards.

    The bound is meant for a factor of 2^-9.  S q takes the state S_0 that the chunk (of 64 tokens) begins with as one
    fp16 term, 2^-11 of |S_0| |q| = 2^-9 * 2^-2.  P u takes both factors so, 2 * 2^-11 = 2^-9 * 2^-1 of sum_j |P_ij| |u_j|.
    The chunk's corrections are U = T R with T's entries (at most 1) as two fp16 terms, off by 2^-25 whatever their size,
    and R's and the fp32 sums' 2^-22 of themselves: a sum over 64 tokens is off by 64 * 2^-25 = 2^-19 of the value row's
    largest R in the chunk, and as much again for the relative parts, so by 2^-18.  With |R_i| =
    |u_i + beta (e^g S_(i-1) - e^G S_0) k_i| at most 4 times the row's largest |S| in the chunk, `peak`, that is 2^-16 =
    2^-9 * 2^-7 of it; 2^-6 covers the fp32 sums of S q and P u, 2^-17 each, too.

    Requests that cannot run give zeros and write nothing, as the operator's contract says."""
    f64 = lambda t: t.detach().cpu().double()  # noqa: E731
    qkv, a, b, a_log, dt_bias, gate, weight = (f64(t) for t in (qkv, a, b, a_log, dt_bias, gate, weight))
    pool = f64(state).clone()
    slots, hv = pool.shape[:2]
    n = qkv.shape[0]
    h = (qkv.shape[1] // DIM - hv) // 2
    parts = qkv.view(n, 2 * h + hv, DIM)
    group = torch.arange(hv) // (hv // h)
    q, k, v = parts[:, :h][:, group], parts[:, h:2 * h][:, group], parts[:, 2 * h:]
    q = q * torch.rsqrt((q * q).sum(-1, keepdim=True) + 1e-6) * DIM ** -0.5
    k = k * torch.rsqrt((k * k).sum(-1, keepdim=True) + 1e-6)
    keep = torch.exp(-torch.exp(a_log) * softplus(a + dt_bias))
    beta = torch.sigmoid(b)
    out = torch.full((n, hv, DIM), float("nan"), dtype=torch.float64)
    bound = torch.zeros(n, hv, DIM, dtype=torch.float64)
    table, context, cu = table.cpu().tolist(), context.cpu().tolist(), cu.cpu().tolist()
    for r, (row, ctx) in enumerate(zip(table, context)):
        begin, end = cu[r], cu[r + 1]
        if end <= begin or begin < 0 or end > n:
            continue
        source = row[(ctx - 1) // block_size] if ctx > 0 and (ctx - 1) // block_size < len(row) else 0
        fits = ctx >= 0 and (ctx + end - begin - 1) // block_size < len(row)
        if not fits or (ctx > 0 and not 0 < source < slots):
            out[begin:end] = 0
            continue
        S = pool[source].clone() if ctx > 0 else torch.zeros(hv, DIM, DIM, dtype=torch.float64)
        norms, recurrence = [S.norm(dim=-1)], []
        for t in range(begin, end):
            if (ctx + t - begin) % 64 == 0 or t == begin:
                chunk_u, chunk_k, chunk_g = [], [], []
            chunk_g = [g * keep[t] for g in chunk_g] + [torch.ones(hv, dtype=torch.float64)]
            S *= keep[t][:, None, None]
            miss = beta[t][:, None] * (v[t] - torch.einsum("hvk,hk->hv", S, k[t]))
            S += miss[..., None] * k[t][:, None, :]
            o = torch.einsum("hvk,hk->hv", S, q[t])
            rstd = torch.rsqrt((o * o).mean(-1, keepdim=True) + eps)
            shape = weight * gate[t] * torch.sigmoid(gate[t])
            out[t] = o * rstd * shape
            norms.append(S.norm(dim=-1))
            chunk_u.append(miss.abs())
            chunk_k.append(k[t])
            pairs = torch.einsum("jhk,hk->jh", torch.stack(chunk_k), q[t]).abs() * torch.stack(chunk_g)
            recurrence.append((o, rstd, shape, torch.einsum("jh,jhv->hv", pairs, torch.stack(chunk_u))))
            position = ctx + t - begin
            if (position + 1) % block_size == 0 or t + 1 == end:
                slot = row[position // block_size]
                if 0 < slot < slots:
                    pool[slot] = S
        for t, (o, rstd, shape, sums) in zip(range(begin, end), recurrence):
            chunk = (ctx + t - begin) // 64
            first, last = max(chunk * 64 - ctx, 0), min(chunk * 64 + 64 - ctx, end - begin)
            peak = torch.stack(norms[first:last + 1]).amax(0)
            size = (2.0 ** -2 + 2.0 ** -6) * peak * q[t].norm(dim=-1, keepdim=True) + 0.5 * sums
            bound[t] = (size + size.max(-1, keepdim=True).values * (o.abs() * rstd)) * rstd * shape.abs()
    return out, bound, pool


def conv(x, conv_state, weight, bias, table, context, cu, block_size):
    """(outputs with NaN where no request writes, magnitude of their sums, conv state)."""
    xs = x.detach().cpu().double()
    w = weight.detach().cpu().double().reshape(weight.shape[0], -1)
    state = conv_state.detach().cpu().double().clone()
    n, dim = xs.shape
    taps = w.shape[1]
    out = torch.full((n, dim), float("nan"), dtype=torch.float64)
    size = torch.zeros(n, dim, dtype=torch.float64)
    add = torch.zeros(dim, dtype=torch.float64) if bias is None else bias.detach().cpu().double()
    before = state.clone()
    cu, table, context = cu.cpu().tolist(), table.cpu().tolist(), context.cpu().tolist()
    for r, (row, ctx) in enumerate(zip(table, context)):
        begin, end = cu[r], cu[r + 1]
        if end <= begin or begin < 0 or end > n:
            continue
        fits = ctx >= 0 and (ctx + end - begin - 1) // block_size < len(row)
        source = row[(ctx - 1) // block_size] if ctx > 0 and (ctx - 1) // block_size < len(row) else 0
        if not fits or (ctx > 0 and not 0 < source < state.shape[0]):
            out[begin:end] = 0
            continue
        line = torch.zeros(taps - 1 + end - begin, dim, dtype=torch.float64)
        if ctx > 0:
            line[: taps - 1] = before[source, :, : taps - 1].t()
        line[taps - 1:] = xs[begin:end]
        y = torch.stack([(line[i:i + taps] * w.t()).sum(0) for i in range(end - begin)]) + add
        out[begin:end] = y * torch.sigmoid(y)
        size[begin:end] = torch.stack([(line[i:i + taps] * w.t()).abs().sum(0) for i in range(end - begin)]) + add.abs()
        for i in range(end - begin):
            if (ctx + i + 1) % block_size == 0 or i + 1 == end - begin:
                slot = row[(ctx + i) // block_size]
                if 0 < slot < state.shape[0]:
                    state[slot, :, : taps - 1] = line[i + 1:i + taps].t()
    return out, size, state


def tables(query, context, free, table, n_tokens, block_size):
    """(cu, table, positions, slot_map, state_slots, used) as int64 arrays, request by request."""
    table = np.array(table, dtype=np.int64)
    cu, taken = [0], 0
    positions, slot_map = np.full(n_tokens, -1, np.int64), np.full(n_tokens, -1, np.int64)
    pairs = np.zeros((len(query), 2), np.int64)
    for r, (q, c) in enumerate(zip(query, context)):
        q, c = max(q, 0), max(c, 0)
        have, want = -(-c // block_size), -(-(c + q) // block_size)

        def block(i):
            return int(table[r, i]) if i < table.shape[1] else 0

        for i in range(have, want):
            if i < table.shape[1]:
                table[r, i] = free[taken] if taken < len(free) else 0
            taken += 1
        for i in range(q):
            at = cu[-1] + i
            if at < n_tokens:
                positions[at] = c + i
                page = block((c + i) // block_size)
                slot_map[at] = page * block_size + (c + i) % block_size if page > 0 else -1
        pairs[r] = (block(want - 1) if q > 0 else 0, block(have - 1) if c > 0 else 0)
        cu.append(cu[-1] + q)
    return np.array(cu), table, positions, slot_map, pairs, taken
