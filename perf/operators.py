"""The operators of a Gated DeltaNet layer's prompt and plain decode, measured.

A case is one call of one operator of one layer:

* op ``prefill``: a packed batch of prompts through the gated delta rule from
  each row's state page to its final page (``gdn_recoverssm_prefill``; with
  ``gated`` the gating and the q/k L2 norm inside,
  ``gdn_recoverssm_prefill_gated``; with ``block`` the states at block
  boundaries go to the pages of a block table);
* op ``decode``: one token (or a few) of every row, states updated in place
  (``gdn_recoverssm_decode`` / ``gdn_recoverssm_decode_gated``);
* op ``conv``: the causal depthwise convolution before it, with its state pages
  (``gdn_recoverssm_conv``);
* op ``tables``: the step's offsets, positions, slots, state pages and newly
  taken cache pages from the rows' lengths (``gdn_recoverssm_step_tables``).

Head geometries are the benchmark's (Hk=16, Hv=32, Dk=Dv=128), one
tensor-parallel rank of eight of it (Hk=2, Hv=4), the toy layer's and the tests'
odd ones; conv channels are q, k and v side by side.
"""

import math
import os
import sys
from types import SimpleNamespace

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gdn-recoverssm-ascend_amd")
_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_MAX_COMPUTED = 4096  # tokens a continued row has behind it, at most
_CHUNK = 64  # tokens per chunk of the plain form


def _case(name=None, **kw):
    base = dict(op="prefill", rows=1, tokens=1024, lengths="even", H=16, HV=32, K=128, V=128, act="bf16", state="f32",
                computed="none", block=0, gated=False, taps=4, bias=True)
    unknown = set(kw) - set(base)
    assert not unknown, unknown
    base.update(kw)
    return dict(base, name=name) if name else base


def listed():
    return [
        # A toy layer's three short prompts: the latency of a call.
        _case("prefill_toy", rows=3, tokens=50, lengths="skewed", H=2, HV=4, K=64, V=64),
        # One user's prompt of ordinary length: 32 heads, one sequence, so the
        # chain of its chunks is what takes the time.
        _case("prefill_prompt_2k", tokens=2048),
        # One user's long prompt: the largest case.
        _case("prefill_prompt_8k", tokens=8192),
        # A serving step's packed prompts of very different lengths, some of
        # them continued, with prefix caching: states at block boundaries.
        _case("prefill_packed_align", rows=24, tokens=7777, lengths="skewed", computed="some", block=256),
        # One tensor-parallel rank of eight continuing a long prompt, gating and
        # L2 norm fused in.
        _case("prefill_tp8_gated", tokens=4096, H=2, HV=4, computed="all", gated=True),
        # FP16 activations and pages, head dims off the 128 x 128 tile, odd
        # ragged rows, three value heads to a key head.
        _case("prefill_f16_ragged", rows=7, tokens=1301, lengths="skewed", H=4, HV=12, K=96, V=192, act="f16",
              state="f16", computed="some"),
        # A full batch without drafts: bound by reading and writing the pages.
        _case("decode_b256", op="decode", rows=256, tokens=256, computed="all"),
        # A few requests on one tensor-parallel rank, everything fused.
        _case("decode_tp8_b6_gated", op="decode", rows=6, tokens=6, H=2, HV=4, computed="all", gated=True),
        # The convolution of a packed prompt step.
        _case("conv_packed_8k", op="conv", rows=24, tokens=8191, lengths="skewed", computed="some"),
        # The convolution of a plain decode step.
        _case("conv_decode_b256", op="conv", rows=256, tokens=256, computed="all"),
        # The tables of a small decode step.
        _case("tables_decode_b6", op="tables", rows=6, tokens=6, computed="all", block=64),
        # The tables of a large mixed step: prompts among decoding rows.
        _case("tables_mixed_b512", op="tables", rows=512, tokens=16384, lengths="skewed", computed="some", block=64),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of the same ranges."""
    op = rng.choice(["prefill"] * 6 + ["decode"] * 3 + ["conv"] * 2 + ["tables"])
    H, HV = rng.choice([(2, 4), (4, 4), (4, 12), (8, 16), (16, 32), (16, 32)])
    K, V = rng.choice([(128, 128)] * 4 + [(64, 64), (96, 192), (128, 96), (64, 192), (256, 128)])
    act, state = rng.choice([("bf16", "f32")] * 5 + [("bf16", "bf16"), ("f16", "f16"), ("f32", "f32")])
    gated = op != "conv" and op != "tables" and rng.random() < 0.4
    if op == "prefill":
        rows = _log_int(rng, 1, 48)
        most = min(8192, 8192 * 32 * 128 * 128 // (HV * K * V))
        tokens = max(rows, _log_int(rng, 33, most))
        block = rng.choice([0, 0, 256, 1024])
        return _case(op=op, rows=rows, tokens=tokens, lengths=rng.choice(["even", "skewed", "skewed"]), H=H, HV=HV, K=K,
                     V=V, act=act, state=state, computed=rng.choice(["none", "some", "all"]), block=block, gated=gated)
    if op == "decode":
        rows = _log_int(rng, 1, 256)
        each = rng.choice([1, 1, 1, 2, 5])
        return _case(op=op, rows=rows, tokens=rows * each, lengths="even", H=H, HV=HV, K=K, V=V, act=act, state=state,
                     computed="all", gated=gated)
    if op == "conv":
        rows = _log_int(rng, 1, 256)
        tokens = rows if rng.random() < 0.4 else max(rows, _log_int(rng, 64, 8192))
        return _case(op=op, rows=rows, tokens=tokens, lengths="skewed" if tokens > rows else "even", H=H, HV=HV, K=K,
                     V=V, act=act, state=act, computed=rng.choice(["some", "all"]), taps=rng.choice([2, 3, 4, 4, 4]),
                     bias=rng.random() < 0.5)
    rows = _log_int(rng, 1, 1024)
    tokens = rows if rng.random() < 0.3 else max(rows, _log_int(rng, 64, 16384))
    return _case(op=op, rows=rows, tokens=tokens, lengths="skewed" if tokens > rows else "even",
                 computed=rng.choice(["some", "all"]), block=rng.choice([16, 64, 128, 144]))


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _lengths(c, gen):
    """Token counts of the rows; they add up to ``tokens``, each at least 1."""
    B, T = c["rows"], c["tokens"]
    if c["lengths"] == "even" or B == 1:
        n = torch.full((B,), T // B, dtype=torch.int64)
        n[:T - int(n.sum())] += 1
        return n
    # Lengths spread over two orders of magnitude, in a random order.
    w = torch.exp(torch.linspace(0.0, 4.0, B, dtype=torch.float64))[torch.randperm(B, generator=gen)]
    n = 1 + torch.floor(w / w.sum() * (T - B)).long()
    n[int(torch.argmax(n))] += T - int(n.sum())
    return n


def _computed(c, gen):
    """Tokens each row has behind it (0: a new request)."""
    B = c["rows"]
    C = torch.randint(1, _MAX_COMPUTED, (B,), generator=gen)
    if c["computed"] == "none":
        return torch.zeros(B, dtype=torch.int64)
    if c["computed"] == "some":
        return torch.where(torch.rand(B, generator=gen) < 0.5, torch.zeros_like(C), C)
    return C


def _plan(c, gen, dev):
    """The step as the scheduler knows it: lengths and positions on the host,
    offsets and pages on the GPU."""
    p = SimpleNamespace()
    p.n, p.C = _lengths(c, gen), _computed(c, gen)
    qsl = torch.zeros(c["rows"] + 1, dtype=torch.int64)
    qsl[1:] = torch.cumsum(p.n, 0)
    p.starts = qsl[:-1]
    p.row_of = torch.repeat_interleave(torch.arange(c["rows"]), p.n).to(dev)
    p.pos_in_row = (torch.arange(c["tokens"]) - qsl[:-1].repeat_interleave(p.n)).to(dev)
    p.qsl = qsl.to(torch.int32).to(dev)
    p.num_computed = p.C.to(torch.int32).to(dev)
    p.query_lens = p.n.to(torch.int32).to(dev)
    return p


def _state_pages(c, p, gen, dev):
    """Source and final page of every row, and the block table in align mode
    (pages for the blocks a row is in now and reaches; the rest are null)."""
    B, block = c["rows"], c["block"]
    if not block:
        pages = 2 * B + 1
        place = 1 + torch.randperm(2 * B, generator=gen)
        source = place[:B]
        # Prompts go on from one page to another; plain decode stays in place.
        final = source if c["op"] == "decode" else place[B:]
        p.table = None
    else:
        first, last = (p.C - 1).clamp(min=0) // block, (p.C + p.n - 1) // block
        # Sizes that hold whatever the positions.
        table = torch.zeros(B, (_MAX_COMPUTED + int(p.n.max())) // block + 2, dtype=torch.int64)
        room, pages = 1 + int((p.n // block + 2).sum()), 1
        for r in range(B):
            for j in range(int(first[r]), int(last[r]) + 1):
                table[r, j] = pages
                pages += 1
        pages = room
        rows = torch.arange(B)
        source, final = table[rows, first], table[rows, last]
        p.table = table.to(torch.int32).to(dev)
        p.table_host = table
    p.source_host = torch.where(p.C > 0, source, torch.zeros_like(source))
    p.final_host, p.pages = final, pages
    p.source = p.source_host.to(torch.int32).to(dev)
    p.final = final.to(torch.int32).to(dev)


def _chunks(c, p, dev):
    """The plain form's chunks: token index and mask of every chunk (a chunk
    ends at a block boundary), and for step j of the scan the chunks it takes,
    their rows and the boundary pages their states go to."""
    T = c["tokens"]
    index, steps, stores = [], [], []
    for r in range(c["rows"]):
        at, n, C, j = int(p.starts[r]), int(p.n[r]), int(p.C[r]) if c["block"] else 0, 0
        done = 0
        while done < n:
            size = min(_CHUNK - (C + done) % _CHUNK, n - done)
            index.append(torch.arange(at + done, at + done + _CHUNK).where(torch.arange(_CHUNK) < size, torch.tensor(T)))
            done += size
            if len(steps) == j:
                steps.append(([], []))
                stores.append(([], []))
            steps[j][0].append(len(index) - 1)
            steps[j][1].append(r)
            if c["block"] and (C + done) % c["block"] == 0 and done < n:
                stores[j][0].append(len(steps[j][1]) - 1)
                stores[j][1].append(int(p.table_host[r, (C + done) // c["block"] - 1]))
            j += 1
    put = lambda v: torch.tensor(v, dtype=torch.int64, device=dev)  # noqa: E731
    p.chunk_index = torch.stack(index).to(dev)
    p.chunk_steps = [(put(a), put(b)) for a, b in steps]
    p.chunk_stores = [(put(a), put(b)) if a else None for a, b in stores]


def prepare(case, seed):
    c = dict(case)
    dev = torch.device("cuda")
    gen = torch.Generator().manual_seed(int(seed))
    dgen = torch.Generator(device=dev).manual_seed(int(seed) + 1)
    s = SimpleNamespace(c=c)
    s.p = p = _plan(c, gen, dev)
    act, T, B, H, HV, K, V = _DTYPES[c["act"]], c["tokens"], c["rows"], c["H"], c["HV"], c["K"], c["V"]

    def randn(*shape):
        return torch.randn(*shape, generator=dgen, device=dev)

    def uniform(low, high, *shape):
        return low + (high - low) * torch.rand(*shape, generator=dgen, device=dev)

    if c["op"] == "tables":
        block = c["block"]
        have = (p.C + block - 1) // block
        table = torch.zeros(B, (_MAX_COMPUTED + int(p.n.max())) // block + 3, dtype=torch.int64)
        spare = int((p.n // block + 1).sum()) + 64
        place = 1 + torch.randperm(int(have.sum()) + spare, generator=gen)
        at = 0
        for r in range(B):
            table[r, :int(have[r])] = place[at:at + int(have[r])]
            at += int(have[r])
        s.block_table = table.to(torch.int32).to(dev)
        # The free pages as a ring whose first entry lies near its end.
        free = place[at:]
        head = int(torch.randint(0, 1000, (1,), generator=gen)) * free.numel() + free.numel() - 3
        s.free_pages = torch.roll(free, -3).to(torch.int32).to(dev)
        s.free_span = torch.tensor([head, head + free.numel()], dtype=torch.int64, device=dev)
        return s
    if c["op"] == "conv":
        D = 2 * H * K + HV * V
        s.x = randn(T, D).to(act)
        s.weight = (randn(D, c["taps"]) * 0.5).to(act)
        s.bias = (randn(D) * 0.1).to(act) if c["bias"] else None
        place = 1 + torch.randperm(B, generator=gen)
        p.source = p.final = place.to(torch.int32).to(dev)
        # Room for a window of four drafted tokens behind the history.
        s.conv_states = randn(B + 1, D, c["taps"] - 1 + 3).to(act)
        return s
    _state_pages(c, p, gen, dev)
    if c["op"] == "prefill":
        _chunks(c, p, dev)

    def unit(x):
        return x * torch.rsqrt((x * x).sum(-1, keepdim=True) + 1e-6)

    q, k = randn(1, T, H, K), randn(1, T, H, K)
    s.q, s.k = (q.to(act), k.to(act)) if c["gated"] else (unit(q).to(act), unit(k).to(act))
    s.v = randn(1, T, HV, V).to(act)
    # Per head decay rates over three orders of magnitude, as trained layers have them.
    s.A_log = uniform(math.log(0.01), math.log(8.0), HV)
    s.dt_bias = randn(HV)
    s.a, s.b = randn(T, HV).to(act), randn(T, HV).to(act)
    if not c["gated"]:
        s.g = -torch.exp(s.A_log) * torch.nn.functional.softplus(s.a.float() + s.dt_bias)
        s.beta = torch.sigmoid(s.b.float())
    s.pages = (randn(p.pages, HV, V, K) * 0.1).to(_DTYPES[c["state"]])
    return s


# ---------------------------------------------------------------------------
# The framework's operators
# ---------------------------------------------------------------------------


def _run_own(s):
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import gdn_recoverssm_ascend as G

    c, p = s.c, s.p
    if c["op"] == "tables":
        t = G.gdn_recoverssm_step_tables(s.block_table, s.free_pages, s.free_span, num_computed=p.num_computed,
                                         query_lens=p.query_lens, block_size=c["block"], num_tokens=c["tokens"])
        return {"block_table": s.block_table, "query_start_loc": t.query_start_loc, "positions": t.positions,
                "slot_mapping": t.slot_mapping, "seq_lens": t.seq_lens, "source": t.source_indices,
                "final": t.final_indices, "new_pages": t.new_pages, "free_span": t.free_span}
    if c["op"] == "conv":
        out = G.gdn_recoverssm_conv(s.x, s.weight, s.bias, conv_states=s.conv_states, query_start_loc=p.qsl,
                                    state_indices=p.source, num_computed=p.num_computed)
        return {"out": out, "conv_states": s.conv_states}
    rest = dict(checkpoint_state=s.pages, query_start_loc=p.qsl, state_indices=p.source, num_computed=p.num_computed)
    rest.update(dict(block_table=p.table, block_size=c["block"]) if c["block"] else dict(final_indices=p.final))
    if c["gated"]:
        call = G.gdn_recoverssm_prefill_gated if c["op"] == "prefill" else G.gdn_recoverssm_decode_gated
        out = call(s.a, s.b, s.q, s.k, s.v, A_log=s.A_log, dt_bias=s.dt_bias, **rest)
    else:
        call = G.gdn_recoverssm_prefill if c["op"] == "prefill" else G.gdn_recoverssm_decode
        out = call(s.g, s.beta, s.q, s.k, s.v, **rest)
    return {"out": out, "pages": s.pages}


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------


def _plain_inputs(s):
    """q (scaled), k, v, g and beta in 32 bits, q and k once per value head."""
    c = s.c
    T, H, HV, K, V = c["tokens"], c["H"], c["HV"], c["K"], c["V"]
    q, k, v = s.q.view(T, H, K).float(), s.k.view(T, H, K).float(), s.v.view(T, HV, V).float()
    if c["gated"]:
        q, k = (x * torch.rsqrt((x * x).sum(-1, keepdim=True) + 1e-6) for x in (q, k))
        x = s.a.float() + s.dt_bias
        g = -torch.exp(s.A_log) * torch.where(x <= 20.0, torch.log1p(torch.exp(x.clamp(max=20.0))), x)
        beta = 1.0 / (1.0 + torch.exp(-s.b.float()))
    else:
        g, beta = s.g, s.beta
    group = HV // H
    return (q * K ** -0.5).repeat_interleave(group, 1), k.repeat_interleave(group, 1), v, g, beta


def _plain_start(s):
    p = s.p
    fresh = (p.num_computed == 0).view(-1, 1, 1, 1)
    return torch.where(fresh, torch.zeros((), device=s.pages.device), s.pages[p.source.long()].float())


def _plain_tokens(s):
    """A few tokens of every row, one after the other."""
    c, p = s.c, s.p
    q, k, v, g, beta = _plain_inputs(s)
    S, decay = _plain_start(s), torch.exp(g)[..., None, None]
    out = torch.empty_like(v)
    for t in range(c["tokens"] // c["rows"]):
        tok = p.qsl[:-1].long() + t
        S = S * decay[tok]
        corr = (v[tok] - torch.matmul(S, k[tok].unsqueeze(-1)).squeeze(-1)) * beta[tok].unsqueeze(-1)
        S = S + corr.unsqueeze(-1) * k[tok].unsqueeze(-2)
        out[tok] = torch.matmul(S, q[tok].unsqueeze(-1)).squeeze(-1)
    s.pages[p.final.long()] = S.to(s.pages.dtype)
    return {"out": out.to(s.v.dtype).unsqueeze(0), "pages": s.pages}


def _plain_chunked(s):
    """Whole rows, a chunk of tokens at a time: within a chunk the corrections
    solve a unit lower triangular system, from chunk to chunk goes the state."""
    c, p = s.c, s.p
    at = p.chunk_index
    q, k, v, g, beta = _plain_inputs(s)

    def chunked(x):  # [T, HV, ...] -> [chunks, HV, 64, ...], zeros past a chunk's end
        x = torch.cat([x, torch.zeros_like(x[:1])])
        return x[at].transpose(1, 2).contiguous()

    q, k, v, g, beta = chunked(q), chunked(k), chunked(v), chunked(g), chunked(beta)
    G = torch.cumsum(g, -1)
    low = torch.ones(_CHUNK, _CHUNK, dtype=torch.bool, device=at.device).tril()
    decay = torch.where(low, torch.exp((G.unsqueeze(-1) - G.unsqueeze(-2)).clamp(max=0.0)), torch.zeros_like(G[..., :1, None]))
    kt = k.transpose(-1, -2)
    L = beta.unsqueeze(-1) * decay * torch.matmul(k, kt)
    inverse = torch.eye(_CHUNK, device=at.device).expand_as(L).contiguous()
    for i in range(1, _CHUNK):
        inverse[..., i, :i] = -torch.matmul(L[..., i:i + 1, :i], inverse[..., :i, :i]).squeeze(-2)
    inverse = inverse * beta.unsqueeze(-2)
    P = decay * torch.matmul(q, kt)
    k_in, q_in = k * torch.exp(G).unsqueeze(-1), q * torch.exp(G).unsqueeze(-1)
    k_out = k * torch.exp(G[..., -1:] - G).unsqueeze(-1)
    end = torch.exp(G[..., -1])[..., None, None]
    S = _plain_start(s)
    out = torch.empty(c["tokens"] + 1, c["HV"], c["V"], device=at.device)
    for (chunks, rows), store in zip(p.chunk_steps, p.chunk_stores):
        S0 = S[rows]
        S0t = S0.transpose(-1, -2)
        corr = torch.matmul(inverse[chunks], v[chunks] - torch.matmul(k_in[chunks], S0t))
        o = torch.matmul(q_in[chunks], S0t) + torch.matmul(P[chunks], corr)
        out[at[chunks]] = o.transpose(1, 2)
        S1 = end[chunks] * S0 + torch.matmul(corr.transpose(-1, -2), k_out[chunks])
        S[rows] = S1
        if store is not None:
            s.pages[store[1]] = S1[store[0]].to(s.pages.dtype)
    s.pages[p.final.long()] = S.to(s.pages.dtype)
    return {"out": out[:-1].to(s.v.dtype).unsqueeze(0), "pages": s.pages}


def _plain_conv(s):
    c, p = s.c, s.p
    history = c["taps"] - 1
    x, w = s.x.float(), s.weight.float()
    state = s.conv_states[p.source.long()][..., :history].float().transpose(1, 2)  # [rows, history, channels]
    state = torch.where((p.num_computed == 0).view(-1, 1, 1), torch.zeros((), device=x.device), state)
    token = torch.arange(c["tokens"], device=x.device)
    out = torch.zeros_like(x) if s.bias is None else s.bias.float().expand_as(x)
    for j in range(c["taps"]):
        back = history - j
        here = (p.pos_in_row >= back).unsqueeze(-1)
        before = state[p.row_of, (history + p.pos_in_row - back).clamp(0, history - 1)]
        out = out + torch.where(here, x[(token - back).clamp(min=0)], before) * w[:, j]
    out = out / (1.0 + torch.exp(-out))
    # The last inputs of every row, history first.
    ago = torch.arange(-history, 0, device=x.device)
    pos = p.query_lens.long().unsqueeze(-1) + ago
    last = p.qsl[1:].long().unsqueeze(-1) + ago
    new = torch.where((pos >= 0).unsqueeze(-1), x[last.clamp(min=0)],
                      torch.gather(state, 1, (history + pos).clamp(0, history - 1).unsqueeze(-1).expand_as(state)))
    s.conv_states[p.final.long(), :, :history] = new.transpose(1, 2).to(s.conv_states.dtype)
    return {"out": out.to(s.x.dtype), "conv_states": s.conv_states}


def _plain_tables(s):
    c, p = s.c, s.p
    block, dev = c["block"], s.block_table.device
    C, n = p.num_computed.long(), p.query_lens.long()
    seq = C + n
    have, need = (C + block - 1) // block, (seq + block - 1) // block
    new = need - have
    ends = torch.cumsum(new, 0)
    head = s.free_span[0]
    fits = (ends <= s.free_span[1] - head) | (new == 0)
    new = torch.where(fits, new, torch.full_like(new, -1))
    qsl = torch.zeros(c["rows"] + 1, dtype=torch.int64, device=dev)
    qsl[1:] = torch.cumsum(n, 0)
    taken = new.clamp(min=0)
    # The new pages' columns, at most as many as tokens: token t opens one if
    # its position starts a block.
    token = torch.arange(c["tokens"], device=dev)
    row = torch.searchsorted(qsl[1:], token, right=True).clamp(max=c["rows"] - 1)
    pos = C[row] + token - qsl[row]
    col = pos // block
    opened = (col >= have[row]) & fits[row]
    page = s.free_pages[((head + (ends - taken)[row] + col - have[row]) % s.free_pages.numel())].long()
    page = torch.where(opened, page, s.block_table[row, col].long())
    starts = opened & (pos % block == 0)
    flat = torch.where(starts, row * s.block_table.shape[1] + col, torch.full_like(row, s.block_table.numel()))
    room = torch.cat([s.block_table.flatten(), s.block_table.new_zeros(1)])
    room[flat] = page.to(torch.int32)
    s.block_table.copy_(room[:-1].view_as(s.block_table))
    slots = torch.where(fits[row], page * block + pos % block, torch.full_like(page, -1))
    rows = torch.arange(c["rows"], device=dev)
    table = s.block_table
    source = torch.where(C > 0, table[rows, (C - 1).clamp(min=0) // block], table.new_zeros(()))
    final = torch.where(fits, table[rows, (seq - 1).clamp(min=0) // block], table.new_zeros(()))
    span = torch.stack([head + taken.sum(), s.free_span[1]])
    return {"block_table": table, "query_start_loc": qsl.to(torch.int32), "positions": pos, "slot_mapping": slots,
            "seq_lens": seq.to(torch.int32), "source": source, "final": final, "new_pages": new.to(torch.int32),
            "free_span": span}


def run(state):
    if own:
        return _run_own(state)
    c = state.c
    if c["op"] == "tables":
        return _plain_tables(state)
    if c["op"] == "conv":
        return _plain_conv(state)
    return _plain_chunked(state) if c["op"] == "prefill" else _plain_tokens(state)


# ---------------------------------------------------------------------------
# What a pass cannot do without, and what it should give
# ---------------------------------------------------------------------------


def work(case):
    c = dict(case)
    T, B, H, HV, K, V = c["tokens"], c["rows"], c["H"], c["HV"], c["K"], c["V"]
    act, state = (4 if c[x] == "f32" else 2 for x in ("act", "state"))
    gen = torch.Generator().manual_seed(0)
    n, C = _lengths(c, gen), _computed(c, gen)
    if c["op"] == "tables":
        block = c["block"]
        new = int(((C + n + block - 1) // block - (C + block - 1) // block).sum())
        # Lengths and pages in; positions, slots, offsets and per-row words out.
        return {"bytes": 4 * (2 * B + 2 * new + B) + 16 * T + 4 * (6 * B + 1) + 32, "flops": 0}
    continued = int((C > 0).sum())
    if c["op"] == "conv":
        D = 2 * H * K + HV * V
        pages = (continued + B) * (c["taps"] - 1) * D
        return {"bytes": act * (2 * T * D + (c["taps"] + bool(c["bias"])) * D + pages),
                "flops": T * D * (2 * c["taps"] + 5)}
    gates = 2 * T * HV * (act if c["gated"] else 4)
    stored = B
    if c["block"]:
        stored += int(((C + n - 1) // c["block"] - C // c["block"]).sum())
    moved = act * (2 * T * H * K + 2 * T * HV * V) + gates + state * (continued + stored) * HV * V * K
    return {"bytes": moved, "flops": 6 * T * HV * K * V}


def exact(case, seed):
    """The definition in 64 bits, token by token over all rows at once."""
    s = prepare(case, seed)
    c, p = s.c, s.p
    if c["op"] == "tables":
        return None
    if c["op"] == "conv":
        history, rows = c["taps"] - 1, []
        new = s.conv_states.double()
        for r in range(c["rows"]):
            at, n, page = int(p.starts[r]), int(p.n[r]), int(p.source[r])
            past = s.conv_states[page, :, :history].double().T * (1.0 if int(p.C[r]) else 0.0)
            seq = torch.cat([past, s.x[at:at + n].double()])
            y = (seq.unfold(0, c["taps"], 1) * s.weight.double()).sum(-1)
            rows.append(y if s.bias is None else y + s.bias.double())
            new[page, :, :history] = seq[-history:].T
        y = torch.cat(rows)
        return {"out": y * torch.sigmoid(y), "conv_states": new}
    T, H, HV, K, V = c["tokens"], c["H"], c["HV"], c["K"], c["V"]
    q, k, v = s.q[0].double(), s.k[0].double(), s.v[0].double()
    if c["gated"]:
        q, k = (x / torch.sqrt((x ** 2).sum(-1, keepdim=True) + 1e-6) for x in (q, k))
        x = s.a.double() + s.dt_bias.double()
        g = -s.A_log.double().exp() * torch.where(x > 20.0, x, torch.log(1.0 + x.exp()))
        beta = torch.sigmoid(s.b.double())
    else:
        g, beta = s.g.double(), s.beta.double()
    head = torch.arange(HV, device=q.device) // (HV // H)
    pages = s.pages.double()
    S = pages[p.source_host.to(q.device)]
    S[(p.C == 0).to(q.device)] = 0.0
    out = torch.zeros(T, HV, V, dtype=torch.float64, device=q.device)
    ends = p.n.tolist()
    order = sorted(range(c["rows"]), key=lambda r: -ends[r])  # longest first: live rows are a prefix
    S = S[torch.tensor(order, device=q.device)]
    starts = p.starts[order].to(q.device)
    block = c["block"]
    live = len(order)
    for t in range(max(ends)):
        while ends[order[live - 1]] <= t:
            live -= 1
        tok = starts[:live] + t
        St, kt = S[:live], k[tok][:, head]
        St *= g[tok].exp()[..., None, None]
        corr = beta[tok].unsqueeze(-1) * (v[tok] - (St @ kt.unsqueeze(-1)).squeeze(-1))
        St += corr.unsqueeze(-1) * kt.unsqueeze(-2)
        out[tok] = (St @ q[tok][:, head].unsqueeze(-1)).squeeze(-1) / math.sqrt(K)
        for i, r in enumerate(order[:live]):
            if t + 1 == ends[r]:
                pages[int(p.final_host[r])] = S[i]
            elif block and (int(p.C[r]) + t + 1) % block == 0:
                pages[int(p.table_host[r, (int(p.C[r]) + t + 1) // block - 1])] = S[i]
    return {"out": out.unsqueeze(0), "pages": pages}
