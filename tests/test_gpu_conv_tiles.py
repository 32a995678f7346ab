"""The convolution's tiles, each reached by the number of tokens, rows and
channels; rows that cross tiles, in place, with other threads at work on the same
row. Bars as for the other tests of it: states bit for bit, outputs norm-wise
2^-8 BF16, 2^-11 F16, 1e-6 FP32."""

import pytest
import torch

from test_gpu_conv_rows import check, problem

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("lengths,D", [([1] * 300, 260), ([2, 3, 1, 2] * 150, 259), ([5, 4, 7] * 100, 130),
                                       ([600, 17, 3, 0, 1500, 1, 2], 8192 + 3)], ids=["single", "short", "mixed", "long"])
def test_in_place_over_tiles(lengths, D, dtype, gpu_device):
    """Tokens of one row in several tiles: none reads the page after it has been
    written."""
    p = problem(lengths, D, 4, dtype, window=6, seed=len(lengths))
    check(p, gpu_device)


@pytest.mark.parametrize("taps", [2, 3, 5])
def test_taps_over_tiles(taps, gpu_device):
    p = problem([3, 1, 4, 2, 9] * 40, 65, taps, "bf16", seed=taps)
    check(p, gpu_device)


@pytest.mark.parametrize("lengths,D", [([2, 5, 3, 40, 1] * 6, 70), ([700, 900, 450], 8192)], ids=["short", "long"])
def test_refused_rows_over_tiles(lengths, D, gpu_device):
    p = problem(lengths, D, 4, "bf16", seed=9)
    p["source"][1] = 0
    p["final"][0] = -3
    check(p, gpu_device, rows=dict(final=p["final"]))


def test_block_table_over_tiles(gpu_device):
    """Boundary pages of a long row, the first of them within the history."""
    D, block = 8192, 64
    p = problem([1500, 700], D, 4, "bf16", seed=3)
    C = torch.tensor([62, 0])
    table = torch.arange(1, 2 * 40 + 1).view(2, 40)
    p["states"] = torch.randn(90, D, 3, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    p["source"] = table[:, 0].int()
    check(p, gpu_device, rows=dict(computed=C, table=table, block=block))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_silu_of_any_size(dtype, gpu_device):
    """Sums from -200 to 200: what SiLU leaves of a large negative one, and large
    ones as they are."""
    p = problem([400], 64, 4, dtype, seed=5, bias=False)
    p["x"] = (torch.linspace(-50, 50, 400)[:, None] * torch.ones(64)).to(p["x"].dtype)
    p["weight"] = torch.ones_like(p["weight"])
    p["states"].zero_()
    check(p, gpu_device)
