"""The chunked rule over many rows: workgroups take them by length, 64 at a time,
and every row is taken once. And FP32 operands straight from memory for launches of
many column tiles. Bars as for the other prompt tests."""

import pytest
import torch

from test_gpu_prompt import check, problem

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [2, 63, 64, 65, 150])
@pytest.mark.parametrize("HV", [1, 12], ids=["few", "many"])
def test_rows_by_length(rows, HV, gpu_device):
    gen = torch.Generator().manual_seed(rows)
    lengths = [int(x) for x in torch.tensor([0, 1, 1, 3, 9, 64, 65, 100])[torch.randint(0, 8, (rows,), generator=gen)]]
    lengths[-1] = 131  # the longest last
    p = problem(lengths, 1, HV, 64, 20, seed=rows)
    check("prefill", p, gpu_device, rows=dict(final=p["final"]))


def test_rows_of_one_length(gpu_device):
    p = problem([65] * 70, 1, 8, 64, 32, seed=3)
    check("prefill", p, gpu_device, rows=dict(final=p["final"]))


@pytest.mark.parametrize("K", [128, 256])
def test_fp32_operands_of_many_tiles(K, gpu_device):
    HV = 800  # a tile each, two rows
    p = problem([66, 70], 2, HV, K, 10, "f32", seed=K)
    check("prefill", p, gpu_device, rows=dict(final=p["final"]))


@pytest.mark.parametrize("HV", [1, 1100], ids=["split", "eight"])
def test_single_small_values_at_a_chunks_end(HV, gpu_device):
    """Chunks that end in one, two or three tokens whose values are next to nothing."""
    p = problem([57, 66, 3, 1], 1, HV, 64, 16, "f32", seed=7)
    at = 0
    for n in (57, 66, 3, 1):
        at += n
        p["v"][0, at - 1] *= 1e-7
    check("prefill", p, gpu_device, rows=dict(final=p["final"]))
