"""Pages far into a large pool, and rows far into a long batch: offsets past 32
bits give the bits that small ones give."""

import pytest
import torch

import gdn_recoverssm_ascend as G

pytestmark = pytest.mark.gpu


def inputs(T, H, HV, K, V, dev, seed=0):
    gen = torch.Generator().manual_seed(seed)
    q, k = (torch.nn.functional.normalize(torch.randn(1, T, H, K, generator=gen), dim=-1) for _ in range(2))
    v = torch.randn(1, T, HV, V, generator=gen)
    g, beta = -torch.rand(T, HV, generator=gen), torch.rand(T, HV, generator=gen)
    return [x.to(dev) for x in (g, beta)] + [x.to(dev, torch.bfloat16) for x in (q, k, v)]


@pytest.mark.parametrize("form,tokens,rows", [("prefill", 100, 1), ("prefill", 70, 6), ("decode", 1, 1), ("decode", 1, 40)])
def test_pages_past_32_bits(form, tokens, rows, gpu_device):
    """A pool of 4200 pages of 2 MB: 2.2 billion elements."""
    H, HV, K, V, pages = 2, 32, 128, 128, 4200
    args = inputs(tokens * rows, H, HV, K, V, gpu_device)
    start = torch.randn(rows, HV, V, K, device=gpu_device) * 0.1
    qsl = torch.arange(0, tokens * rows + 1, tokens, device=gpu_device)
    run = getattr(G, "gdn_recoverssm_" + form)
    small = torch.cat([torch.zeros_like(start[:1]), start, torch.zeros_like(start)])
    low = torch.arange(1, rows + 1, device=gpu_device)
    out = run(*args, checkpoint_state=small, query_start_loc=qsl, state_indices=low, final_indices=low + rows)
    pool = torch.empty(pages, HV, V, K, device=gpu_device)
    high = pages - 2 * rows - 1 + low
    pool[high] = start
    far = run(*args, checkpoint_state=pool, query_start_loc=qsl, state_indices=high, final_indices=high + rows)
    assert torch.equal(out, far) and torch.equal(pool[high + rows], small[low + rows])
    assert torch.equal(pool[high], start)


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 16384)])
def test_tokens_past_32_bits(dtype, D, gpu_device):
    """The last of 150 thousand tokens: the convolution's offsets, and the rule's
    with heads side by side, pass 2^31 elements."""
    T, n = 150_000, 90
    x = torch.empty(T, D, dtype=dtype, device=gpu_device)
    gen = torch.Generator().manual_seed(1)
    x[T - n:] = torch.randn(n, D, generator=gen).to(gpu_device, dtype)
    weight = torch.randn(D, 4, generator=gen).to(gpu_device, dtype)
    states = torch.zeros(4, D, 3, dtype=dtype, device=gpu_device)
    page = torch.tensor([0, 1], device=gpu_device)
    out = G.gdn_recoverssm_conv(x, weight, conv_states=states, query_start_loc=torch.tensor([0, T - n, T], device=gpu_device),
                                state_indices=page)
    near = torch.zeros_like(states)
    want = G.gdn_recoverssm_conv(x[T - n:], weight, conv_states=near,
                                 query_start_loc=torch.tensor([0, n], device=gpu_device), state_indices=page[1:])
    assert torch.equal(out[T - n:], want) and torch.equal(states, near)
    assert not out[:n].any() and not out[T - n - 1].any()  # the null page's row
    HV, V, K = 128, 128, 64
    v = out.view(1, T, HV, V)
    g, beta, q, k, _ = inputs(n, 1, HV, K, 8, gpu_device)
    far = [torch.zeros(1, T, 1, K, dtype=dtype, device=gpu_device) for _ in range(2)]
    gates = [torch.zeros(T, HV, device=gpu_device) for _ in range(2)]
    for to, part in zip((*gates, far[0][0], far[1][0]), (g, beta, q[0], k[0])):
        to[T - n:] = part
    state = torch.zeros(2, HV, V, K, device=gpu_device)
    mine = G.gdn_recoverssm_prefill(*gates, *far, v, checkpoint_state=state, state_indices=page,
                                    query_start_loc=torch.tensor([0, T - n, T], device=gpu_device))
    other = torch.zeros_like(state)
    want = G.gdn_recoverssm_prefill(g, beta, q, k, v[:, T - n:], checkpoint_state=other, state_indices=page[1:],
                                    query_start_loc=torch.tensor([0, n], device=gpu_device))
    assert torch.equal(state, other) or torch.allclose(state, other, rtol=0, atol=1e-5 * float(other.abs().max()))
    err = float((mine[0, T - n:].float() - want[0].float()).norm() / want.float().norm())
    assert err <= 2.0**-7  # two roundings to BF16: the two launches' tiles differ
