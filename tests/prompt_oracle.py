"""Plain 64-bit forms of the prompt operators, on the CPU, row by row and token
by token, for the tests of ``gdn_recoverssm_prefill`` / ``decode`` / ``conv`` /
``step_tables``."""

import torch


def row_plan(b, qsl, source, *, final=None, computed=None, table=None, block=None, requests=None, blocks=1):
    """(first token, tokens, C, source page or 0 for a zero state, final page,
    {position: page}) of a row, None for a row that is refused."""
    lo, n = int(qsl[b]), int(qsl[b + 1]) - int(qsl[b])
    req = int(requests[b]) if requests is not None else b
    C = 0
    if computed is not None:
        if not 0 <= req < len(computed) or int(computed[req]) < 0:
            return lo, n, None
        C = int(computed[req])
    fresh = computed is not None and C == 0
    src = int(source[b])
    fin, bounds = src, {}
    if table is not None:
        if not 0 <= req < table.shape[0]:
            return lo, n, None
        fin = int(table[req, min(max(C + n - 1, 0) // block, table.shape[1] - 1)])
        for pos in range((C // block + 1) * block, C + n, block):
            col = pos // block - 1
            page = int(table[req, col]) if col < table.shape[1] else 0
            if 0 < page < blocks and page != fin:
                bounds[pos - C] = page
    elif final is not None:
        fin = int(final[b])
    if not 0 < fin < blocks or not (fresh or 0 < src < blocks):
        return lo, n, None
    return lo, n, (0 if fresh else src, fin, bounds)


def gates(a, b, A_log, dt_bias, sb=1.0, threshold=20.0):
    x = a.double() + dt_bias.double()
    soft = torch.where(sb * x <= threshold, torch.log1p(torch.exp((sb * x).clamp(max=threshold))) / sb, x)
    return -torch.exp(A_log.double()) * soft, torch.sigmoid(b.double())


def rule(q, k, v, g, beta, pages, qsl, source, *, scale=None, l2norm=False, **rows):
    """out [T, HV, V] and the pages afterwards, both in 64 bits; the second is
    rounded to the pages' type where a page was stored. Also which tokens were
    written."""
    _, T, H, K = q.shape
    HV, V = v.shape[2:]
    q, k, v = q[0].double(), k[0].double(), v[0].double()
    g, beta = g.reshape(T, HV).double(), beta.reshape(T, HV).double()
    if l2norm:
        q, k = (x / torch.sqrt((x * x).sum(-1, keepdim=True) + 1e-6) for x in (q, k))
    q = q * (K**-0.5 if scale is None else scale)
    head = torch.arange(HV) // (HV // H)
    before, after = pages.double(), pages.double().clone()
    out = torch.zeros(T, HV, V, dtype=torch.float64)
    for b in range(len(source)):
        lo, n, plan = row_plan(b, qsl, source, blocks=pages.shape[0], **rows)
        if plan is None or n == 0:
            continue
        src, fin, bounds = plan
        S = before[src].clone() if src else torch.zeros(HV, V, K, dtype=torch.float64)
        for t in range(n):
            kt = k[lo + t][head]
            S = S * torch.exp(g[lo + t])[:, None, None]
            c = beta[lo + t][:, None] * (v[lo + t] - (S * kt[:, None, :]).sum(-1))
            S = S + c[:, :, None] * kt[:, None, :]
            out[lo + t] = (S * q[lo + t][head][:, None, :]).sum(-1)
            if t + 1 in bounds:
                after[bounds[t + 1]] = S
        after[fin] = S
    return out, after


def conv(x, weight, bias, states, qsl, source, *, silu=True, **rows):
    """out [T, D] in 64 bits and the conv states afterwards (their own bits)."""
    T, D = x.shape
    taps = weight.shape[1]
    hist = taps - 1
    out = torch.zeros(T, D, dtype=torch.float64)
    after = states.clone()
    for b in range(len(source)):
        lo, n, plan = row_plan(b, qsl, source, blocks=states.shape[0], **rows)
        if plan is None or n == 0:
            continue
        src, fin, bounds = plan
        past = states[src][:, :hist].T if src else torch.zeros(hist, D, dtype=x.dtype)
        seq = torch.cat([past, x[lo:lo + n]])
        for t in range(n):
            y = (seq[t:t + taps].double() * weight.double().T).sum(0)
            y = y if bias is None else y + bias.double()
            out[lo + t] = y * torch.sigmoid(y) if silu else y
        for length, page in bounds.items():
            after[page][:, :hist] = seq[length:length + hist].T
        after[fin][:, :hist] = seq[n:n + hist].T
    return out, after


def tables(table, free, span, computed, lens, block, num_tokens, requests=None):
    """A step's tables in plain loops."""
    table = table.clone()
    head, tail = (int(x) for x in span)
    room = min(max(tail - head, 0), len(free))
    rows = len(lens)
    res = dict(query_start_loc=[0], seq_lens=[], source_indices=[], final_indices=[], new_pages=[])
    positions, slots, asked, taken = [], [], 0, 0
    for r in range(rows):
        req = int(requests[r]) if requests is not None else r
        known = 0 <= req < table.shape[0] and req < len(computed)
        C = max(int(computed[req]), 0) if known else 0
        n = max(int(lens[r]), 0)
        have, all_ = -(-C // block), -(-(C + n) // block)
        known = known and all_ <= table.shape[1]
        need = all_ - have if known else 0
        ok = known and (need == 0 or asked + need <= room)
        if ok:
            for j in range(need):
                table[req, have + j] = free[(head + asked + j) % len(free)]
            taken += need
        asked += need
        res["query_start_loc"].append(res["query_start_loc"][-1] + n)
        res["seq_lens"].append(C + n)
        res["source_indices"].append(int(table[req, (C - 1) // block]) if known and C > 0 else 0)
        res["final_indices"].append(int(table[req, (C + n - 1) // block]) if ok and C + n > 0 else 0)
        res["new_pages"].append(need if ok else -1)
        for i in range(n):
            pos = C + i
            positions.append(pos)
            slots.append(int(table[req, pos // block]) * block + pos % block if ok else -1)
    pad = num_tokens - len(positions)
    res = {k: torch.tensor(v, dtype=torch.int32) for k, v in res.items()}
    res["positions"] = torch.tensor(positions + [-1] * pad, dtype=torch.int64)
    res["slot_mapping"] = torch.tensor(slots + [-1] * pad, dtype=torch.int64)
    res["free_span"] = torch.tensor([head + taken, tail], dtype=torch.int64)
    return table, res
