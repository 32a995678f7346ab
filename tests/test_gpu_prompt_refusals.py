"""What the prompt operators refuse, with tensors on the GPU: a call that breaks a
rule does not pass for one that keeps them all, and nothing is launched."""

import pytest
import torch

import gdn_recoverssm_ascend as G
from gdn_recoverssm_ascend import kernels
from test_prompt_host import CONV_REFUSALS, POOL_REFUSALS, RULE_REFUSALS, TABLE_REFUSALS, call, conv_call, table_call, z

pytestmark = pytest.mark.gpu
I = torch.int32


def on(device, change):
    """The tensors of a call on the GPU, of the strides they have."""
    return {n: torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=device).zero_()
            if torch.is_tensor(t) and t.device.type == "cpu" else t for n, t in change.items()}


def cases(refusals):
    return [pytest.param(m, c, id=f"{i}-{m}") for i, (m, c) in enumerate(refusals) if "HIP device" not in m]


@pytest.fixture(autouse=True)
def nothing_launched():
    before = dict(kernels._COUNTS)
    yield
    assert dict(kernels._COUNTS) == before


def rule_tensors(T=6, H=2, HV=4, K=16, V=8):
    bf = torch.bfloat16
    return dict(g=z(1, T, HV), beta=z(1, T, HV), q=z(1, T, H, K, dtype=bf), k=z(1, T, H, K, dtype=bf),
                v=z(1, T, HV, V, dtype=bf), checkpoint_state=z(3, HV, V, K), query_start_loc=z(3, dtype=I),
                state_indices=z(2, dtype=I))


@pytest.mark.parametrize("fn", ["prefill", "decode"])
@pytest.mark.parametrize("message,change", cases(RULE_REFUSALS))
def test_rule_arguments(fn, message, change, gpu_device):
    with pytest.raises(ValueError, match=f"GDN RecoverSSM: .*{message}"):
        call(fn, **on(gpu_device, {**rule_tensors(), **change}))


ROW_REFUSALS = [
    ("one entry more than state_indices", dict(query_start_loc=z(4, dtype=I))),
    ("one entry more than state_indices", dict(state_indices=z(2, 1, dtype=I))),
    ("final_indices must have one entry", dict(final_indices=z(3, dtype=I))),
    ("num_computed must be one-dimensional", dict(num_computed=z(2, 2, dtype=I))),
    ("request_indices must have one entry", dict(request_indices=z(1, dtype=I))),
    ("num_computed needs one entry per row", dict(num_computed=z(1, dtype=I))),
    ("takes the place of final_indices", dict(block_table=z(2, 2, dtype=I), block_size=16)),
    ("takes the place of final_indices", dict(block_table=z(2, 2, dtype=I), num_computed=z(2, dtype=I))),
    ("takes the place of final_indices", dict(block_table=z(2, 2, dtype=I), num_computed=z(2, dtype=I), block_size=0)),
    ("takes the place of final_indices", dict(block_table=z(2, 2, dtype=I), num_computed=z(2, dtype=I), block_size=16,
                                              final_indices=z(2, dtype=I))),
    ("block_size comes with a block table", dict(block_size=16)),
    ("must be two-dimensional", dict(block_table=z(2, dtype=I), num_computed=z(2, dtype=I), block_size=16)),
    ("must be two-dimensional", dict(block_table=z(2, 0, dtype=I), num_computed=z(2, dtype=I), block_size=16)),
    ("must be int32 or int64", dict(query_start_loc=z(3))), ("must be int32 or int64", dict(state_indices=z(2))),
    ("must be int32 or int64", dict(final_indices=z(2, dtype=torch.int16))),
    ("must be int32 or int64", dict(num_computed=z(2))), ("must be int32 or int64", dict(request_indices=z(2))),
    ("same device", dict(final_indices=z(2, dtype=I, device="meta"))),
    ("same device", dict(num_computed=z(2, dtype=I, device="meta"))),
    ("same device", dict(request_indices=z(2, dtype=I, device="meta"))),
    ("same device", dict(state_indices=z(2, dtype=I, device="meta"))),
]


@pytest.mark.parametrize("fn", ["prefill", "decode", "conv"])
@pytest.mark.parametrize("message,change", cases(ROW_REFUSALS))
def test_row_arguments(fn, message, change, gpu_device):
    with pytest.raises(ValueError, match=f"GDN RecoverSSM: .*{message}"):
        if fn == "conv":
            base = dict(x=z(6, 8), weight=z(8, 4), bias=z(8), conv_states=z(3, 8, 3), query_start_loc=z(3, dtype=I),
                        state_indices=z(2, dtype=I))
            conv_call(**on(gpu_device, {**base, **change}))
        else:
            call(fn, **on(gpu_device, {**rule_tensors(), **change}))


@pytest.mark.parametrize("message,change", cases(CONV_REFUSALS))
def test_convolution_arguments(message, change, gpu_device):
    base = dict(x=z(6, 8), weight=z(8, 4), bias=z(8), conv_states=z(3, 8, 3), query_start_loc=z(3, dtype=I),
                state_indices=z(2, dtype=I))
    with pytest.raises(ValueError, match=f"GDN RecoverSSM: .*{message}"):
        conv_call(**on(gpu_device, {**base, **change}))


def test_convolution_in_place_is_refused(gpu_device):
    x = torch.zeros(6, 8, device=gpu_device)
    base = on(gpu_device, dict(weight=z(8, 4), bias=z(8), conv_states=z(3, 8, 3), query_start_loc=z(3, dtype=I),
                               state_indices=z(2, dtype=I)))
    with pytest.raises(ValueError, match="may not share memory"):
        conv_call(x=x, out=x, **base)


def pool():
    return dict(block_table=z(4, 8, dtype=I), free_pages=z(16, dtype=I), free_span=z(2, dtype=torch.int64))


@pytest.mark.parametrize("message,change", cases(TABLE_REFUSALS) + cases([r for r in POOL_REFUSALS if not
                         {"seq_lens", "requests"} & set(r[1])]))
def test_table_arguments(message, change, gpu_device):
    base = dict(**pool(), num_computed=z(4, dtype=I), query_lens=z(4, dtype=I))
    with pytest.raises(ValueError, match=f"GDN RecoverSSM: .*{message}"):
        table_call(**on(gpu_device, {**base, **change}))


def test_table_outputs(gpu_device):
    base = on(gpu_device, dict(**pool(), num_computed=z(4, dtype=I), query_lens=z(4, dtype=I)))
    good = G.StepTables.allocate(4, 8, gpu_device)
    for out, message in ((G.StepTables.allocate(3, 8, gpu_device), "out.query_start_loc"),
                         (G.StepTables.allocate(4, 7, gpu_device), "out.positions"),
                         (G.StepTables.allocate(4, 8, "cpu"), "out.query_start_loc")):
        with pytest.raises(ValueError, match=message):
            table_call(**base, out=out)
    with pytest.raises(ValueError, match="out.free_span must not be free_span"):
        table_call(**{**base, "free_span": good.free_span}, out=good)


@pytest.mark.parametrize("message,change", cases(POOL_REFUSALS))
def test_release_arguments(message, change, gpu_device):
    a = on(gpu_device, {**pool(), "requests": z(2, dtype=I), "seq_lens": z(2, dtype=I), "block_size": 16, **change})
    with pytest.raises(ValueError, match=f"GDN RecoverSSM: .*{message}"):
        G.gdn_recoverssm_release_pages(a.pop("block_table"), a.pop("free_pages"), a.pop("free_span"), **a)


def test_gates_with_strided_heads(gpu_device):
    base = on(gpu_device, rule_tensors())
    with pytest.raises(ValueError, match="heads must be contiguous"):
        call("decode", **{**base, "g": torch.zeros(6, 8, device=gpu_device)[:, ::2]})
