"""The serving example on the GPU: requests that come and go, prompts in chunks,
decode and speculative steps, against each request's whole sequence computed at
once in 64 bits.

Bars: FP32 inputs, the rule's 1e-5 and the convolution's 1e-6 on each of q, k and
v, which the L2 norm and the state can double: 3e-5 norm-wise, and for the states
max-abs over max-abs."""

import os
import sys

import pytest
import torch

import gdn_oracle as O
import prompt_oracle as P

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

pytestmark = pytest.mark.gpu
BAR = 3e-5


def whole(layer, x, a, b):
    """Outputs of a request's tokens and its state after them, in 64 bits."""
    heads, value_heads, K, V = layer.shape
    n = x.shape[0]
    qsl, page = torch.tensor([0, n]), torch.tensor([1])
    new = dict(computed=torch.tensor([0]))
    mixed, _ = P.conv(x, layer.conv_weight.cpu(), None, torch.zeros(2, layer.channels, 3), qsl, page, **new)
    q, k, v = mixed.unsqueeze(0).split((heads * K, heads * K, value_heads * V), dim=-1)
    g, beta = P.gates(a, b, layer.A_log.cpu(), layer.dt_bias.cpu())
    out, pages = P.rule(q.unflatten(-1, (heads, K)), k.unflatten(-1, (heads, K)), v.unflatten(-1, (value_heads, V)),
                        g, beta, torch.zeros(2, value_heads, V, K), qsl, page, l2norm=True, **new)
    return out, pages[1]


@pytest.mark.parametrize("block", [8, 16, 64])
def test_requests_over_many_steps(block, gpu_device):
    from gdn_serving import GDNLayer

    dev = gpu_device
    pages = 2 + 4 * -(-260 // block)
    layer = GDNLayer(heads=2, value_heads=4, key_dim=64, value_dim=32, pages=pages, block_size=block, requests=4,
                     columns=-(-260 // block), dtype=torch.float32, device=dev)
    gen = torch.Generator().manual_seed(block)
    inputs = [[torch.randn(260, w, generator=gen) for w in (layer.channels, 4, 4)] for _ in range(5)]
    at, got = [0] * 5, [[] for _ in range(5)]

    def packed(who, lens):
        return [torch.cat([inputs[r][i][at[r]:at[r] + n] for r, n in zip(who, lens)]).to(dev) for i in range(3)]

    def step(who, lens, prompt, places):
        out = layer.step(torch.tensor(places, device=dev), torch.tensor(lens, dtype=torch.int32, device=dev),
                         *packed(who, lens), prompt=prompt).cpu()
        for r, part in zip(who, out.split(lens)):
            got[r].append(part)
            at[r] += len(part)

    def speculate(who, held, places):
        out = layer.speculate(torch.tensor(places, device=dev), *packed(who, [4] * len(who)),
                              accept=lambda drafts: torch.tensor(held, dtype=torch.int32, device=dev)).cpu()
        for r, part, n in zip(who, out, held):
            got[r].append(part[:n])
            at[r] += n

    def check(r, place):
        n = at[r]
        out, state = whole(layer, *(t[:n] for t in inputs[r]))
        mine = torch.cat(got[r]).double()
        assert float((mine - out).norm() / out.norm()) <= BAR
        page = int(layer.table[place, (n - 1) // block])
        assert O.max_abs_rel(layer.states[page].cpu().double(), state) <= BAR

    step([0, 1, 2], [100, 1, 37], True, [2, 0, 3])
    step([0, 3], [30, 150], True, [2, 1])
    for _ in range(3):
        step([0, 1, 2, 3], [1, 1, 1, 1], False, [2, 0, 3, 1])
    for i in range(9):
        speculate([2, 0, 3], [(1, 4, 2), (3, 1, 4), (4, 4, 1)][i % 3], [3, 2, 1])
    for r, place in ((0, 2), (1, 0), (2, 3), (3, 1)):
        check(r, place)
    layer.end(torch.tensor([2, 1], device=dev))
    held = [-(-at[1] // block), -(-at[2] // block)]
    assert layer.free_count() == pages - 1 - sum(held)  # nothing has been lost
    step([4, 2], [200, 20], True, [2, 3])  # another request in a place that was left
    speculate([2, 4], [4, 4], [3, 2])
    check(4, 2)
    check(2, 3)
    layer.end(torch.tensor([0, 2, 3], device=dev))
    assert layer.free_count() == pages - 1
    order = layer.free[(torch.arange(pages - 1) + int(layer.span[0])) % len(layer.free)].tolist()
    assert sorted(order) == list(range(1, pages))


def test_main_runs(gpu_device, capsys):
    import gdn_serving

    gdn_serving.main()
    assert "free pages 127" in capsys.readouterr().out
