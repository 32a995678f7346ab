"""One Gated DeltaNet layer serving a few requests: prompts in chunks, plain
decode, and speculative steps, over one pool of state pages.

Every step goes the same way: ``gdn_recoverssm_step_tables`` makes the step's
offsets and pages from its lengths, ``gdn_recoverssm_conv`` mixes the projected
tokens, and ``gdn_recoverssm_prefill_gated`` or ``gdn_recoverssm_decode_gated``
take the gated delta rule from each request's page to its next. A speculative
step verifies its drafts with ``gdn_recoverssm_verify_gated``, commits what was
accepted, and hands pages that it took for rejected tokens back. No step waits
for the GPU.

    PYTHONPATH=gdn-recoverssm-ascend_amd python examples/gdn_serving.py
"""

from __future__ import annotations

import torch

import gdn_recoverssm_ascend as G


class GDNLayer:
    """The layer's weights, its pool of pages, and the requests' tables.

    The pool keeps one spare page per request at its end, for convolution states
    of tokens that may still be rejected."""

    def __init__(self, *, heads, value_heads, key_dim, value_dim, taps=4, pages=64, block_size=16, requests=8,
                 columns=32, window=4, dtype=torch.bfloat16, device="cuda", seed=0):
        gen = torch.Generator().manual_seed(seed)
        randn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
        self.shape, self.window, self.block_size = (heads, value_heads, key_dim, value_dim), window, block_size
        self.channels = 2 * heads * key_dim + value_heads * value_dim
        self.conv_weight = (randn(self.channels, taps) * taps**-0.5).to(device, dtype)
        self.A_log, self.dt_bias = randn(value_heads).to(device), randn(value_heads).to(device)
        self.states = torch.zeros(pages, value_heads, value_dim, key_dim, device=device)
        self.conv_states = torch.zeros(pages + requests, self.channels, taps - 1, dtype=dtype, device=device)
        self.spare = torch.arange(pages, pages + requests, dtype=torch.int32, device=device)
        self.table = torch.zeros(requests, columns, dtype=torch.int32, device=device)
        self.free = torch.arange(1, pages + 1, dtype=torch.int32, device=device)  # the last place stays empty
        self.span = torch.tensor([0, pages - 1], dtype=torch.int64, device=device)
        self.computed = torch.zeros(requests, dtype=torch.int64, device=device)
        # Keys as the rule sees them, normalised: more bits than the projections'.
        self.records = G.ReplayRecordBuffers.allocate(requests, value_heads, heads, window, value_dim, key_dim,
                                                      device=device, key_dtype=torch.float32)
        # The commit folds states; the convolution's go on from the accepted
        # tokens themselves, so the windows it would compact are not kept.
        unused = torch.zeros(pages, 1, window, dtype=dtype, device=device)
        self.commit = G.GDNRecoverSSMCommitContext.from_tensors([unused], [self.states], [self.records],
                                                                spec_query_len=window, max_num_reqs=requests)

    def _tables(self, requests, lens, tokens):
        t = G.gdn_recoverssm_step_tables(self.table, self.free, self.span, num_computed=self.computed,
                                         query_lens=lens, block_size=self.block_size, num_tokens=tokens,
                                         request_indices=requests)
        self.span = t.free_span
        return t

    def _rows(self, t, requests):
        return dict(query_start_loc=t.query_start_loc, state_indices=t.source_indices, num_computed=self.computed,
                    block_table=self.table, block_size=self.block_size, request_indices=requests)

    def _split(self, mixed):
        heads, value_heads, key_dim, value_dim = self.shape
        q, k, v = mixed.unsqueeze(0).split((heads * key_dim, heads * key_dim, value_heads * value_dim), dim=-1)
        return q.unflatten(-1, (heads, key_dim)), k.unflatten(-1, (heads, key_dim)), v.unflatten(-1, (value_heads, value_dim))

    def step(self, requests, lens, x, a, b, *, prompt):
        """``lens`` new tokens of each request, packed in ``x`` [T, channels] and
        the gates' projections ``a``, ``b`` [T, value heads]. Returns the layer's
        output before its norm and gate, [T, value heads, value dim]."""
        t = self._tables(requests, lens, x.shape[0])
        rows = self._rows(t, requests)
        mixed = G.gdn_recoverssm_conv(x, self.conv_weight, conv_states=self.conv_states, **rows)
        rule = G.gdn_recoverssm_prefill_gated if prompt else G.gdn_recoverssm_decode_gated
        out = rule(a, b, *self._split(mixed), A_log=self.A_log, dt_bias=self.dt_bias, checkpoint_state=self.states, **rows)
        self.computed.index_add_(0, requests, lens.to(torch.int64))
        return out[0]

    def speculate(self, requests, x, a, b, accept):
        """``window`` drafts of each request; ``accept`` takes their outputs
        [requests, window, value heads, value dim] and returns how many of each
        request's hold (int32). Returns the outputs."""
        n, Q = requests.shape[0], self.window
        lens = torch.full((n,), Q, dtype=torch.int32, device=x.device)
        t = self._tables(requests, lens, n * Q)
        mixed = G.gdn_recoverssm_conv(x, self.conv_weight, conv_states=self.conv_states,
                                      query_start_loc=t.query_start_loc, state_indices=t.source_indices,
                                      final_indices=self.spare[:n])
        out = G.gdn_recoverssm_verify_gated(a, b, *self._split(mixed), A_log=self.A_log, dt_bias=self.dt_bias,
                                            checkpoint_state=self.states, replay_cache=self.records,
                                            query_start_loc=t.query_start_loc, state_indices=t.source_indices,
                                            spec_query_len=Q)
        out = out[0].unflatten(0, (n, Q))
        held = accept(out)
        accepted = torch.zeros_like(self.computed, dtype=torch.int32).index_copy_(0, requests, held)  # by request
        self.commit.commit(accepted, t.source_indices, t.query_start_loc, request_indices=requests,
                           block_table=self.table, num_computed_tokens=self.computed,
                           mamba_block_size=self.block_size, commit_conv=False)
        # The convolution's states after the accepted tokens: every request's row
        # is cut behind them, and the rest is a row of the null page.
        start = t.query_start_loc[:-1]
        qsl = torch.cat([torch.stack([start, start + held], 1).flatten(), t.query_start_loc[-1:]])
        source = torch.stack([t.source_indices, torch.zeros_like(t.source_indices)], 1).flatten()
        outside = torch.full_like(requests, -1)
        G.gdn_recoverssm_conv(x, self.conv_weight, conv_states=self.conv_states, query_start_loc=qsl,
                              state_indices=source, num_computed=self.computed, block_table=self.table,
                              block_size=self.block_size,
                              request_indices=torch.stack([requests, outside], 1).flatten())
        self._hand_back(requests, held)
        return out

    def _hand_back(self, requests, held):
        """Pages taken for rejected tokens: at most one a request, in the column
        behind its last block."""
        taken = -(-(self.computed[requests] + self.window) // self.block_size)
        self.computed.index_add_(0, requests, held.to(torch.int64))
        column = -(-self.computed[requests] // self.block_size)
        last = column.clamp(max=self.table.shape[1] - 1)
        entry = self.table[requests, last]
        extra = torch.where(column < taken, entry, torch.zeros_like(entry))
        self.table[requests, last] = entry - extra
        self.span = G.gdn_recoverssm_release_pages(
            extra.unsqueeze(1), self.free, self.span, requests=torch.arange(len(requests), device=requests.device),
            seq_lens=torch.ones_like(requests), block_size=self.block_size)

    def end(self, requests):
        """The requests' pages go back to the pool."""
        self.span = G.gdn_recoverssm_release_pages(self.table, self.free, self.span, requests=requests,
                                                   seq_lens=self.computed[requests], block_size=self.block_size)
        self.computed[requests] = 0

    def free_count(self):
        return int(self.span[1] - self.span[0])


def main():
    layer = GDNLayer(heads=2, value_heads=4, key_dim=128, value_dim=128, pages=128, requests=4, block_size=64)
    device, dtype = "cuda", torch.bfloat16
    gen = torch.Generator(device=device).manual_seed(1)

    def tokens(n):
        return [torch.randn(n, width, generator=gen, device=device).to(dtype) for width in (layer.channels, 4, 4)]

    requests = torch.tensor([2, 0, 1], device=device)
    prompts = torch.tensor([700, 33, 250], dtype=torch.int32, device=device)
    out = layer.step(requests, prompts, *tokens(983), prompt=True)
    print("prompt: ", tuple(out.shape), "free pages", layer.free_count())
    out = layer.step(requests, torch.ones_like(prompts), *tokens(3), prompt=False)
    print("decode: ", tuple(out.shape), "free pages", layer.free_count())
    held = torch.tensor([1, 4, 2], dtype=torch.int32, device=device)
    out = layer.speculate(requests, *tokens(12), accept=lambda drafts: held)
    print("drafts: ", tuple(out.shape), "accepted", held.tolist(), "tokens", layer.computed[requests].tolist())
    layer.end(requests)
    print("ended:   free pages", layer.free_count())


if __name__ == "__main__":
    main()
