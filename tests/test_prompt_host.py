"""Host side of the prompt operators, on the CPU (nothing is launched): the C
structures' layouts, what the C entry points refuse before any launch, the
argument checks of the Python functions, and their kernels' registers."""

import ctypes
import os
import re
import subprocess

import pytest
import torch

import gdn_recoverssm_ascend as G
from gdn_recoverssm_ascend import _native as N
from gdn_recoverssm_ascend._build import INCLUDE_DIR, LIB_PATH
from gdn_recoverssm_ascend.step_tables import MAX_TABLE_ROWS
from test_kernel_registers import _spills

STRUCTS = {"gdn_row_pages": N.RowPages, "gdn_rule_launch": N.RuleLaunch, "gdn_conv_rows": N.ConvRows,
           "gdn_step_tables": N.StepTablesLaunch}


def test_struct_layouts_match_the_c_compiler(tmp_path):
    lines = [f'printf("{s} %zu\\n", sizeof({s}));' for s in STRUCTS]
    lines += [f'printf("{s}.{f} %zu\\n", offsetof({s}, {f}));' for s, cls in STRUCTS.items() for f, *_ in cls._fields_]
    src = tmp_path / "probe.c"
    src.write_text("#include <stddef.h>\n#include <stdio.h>\n#include \"gdn_recoverssm_hip.h\"\n"
                   "int main(void) {\n" + "\n".join(lines) + "\nreturn 0;\n}\n")
    subprocess.run(["gcc", "-I", INCLUDE_DIR, str(src), "-o", str(tmp_path / "probe")], check=True)
    out = subprocess.run([str(tmp_path / "probe")], capture_output=True, text=True, check=True).stdout
    got = {k: int(v) for k, v in (line.split() for line in out.splitlines())}
    for s, cls in STRUCTS.items():
        assert got[s] == ctypes.sizeof(cls)
        for f, *_ in cls._fields_:
            assert got[f"{s}.{f}"] == getattr(cls, f).offset, f"{s}.{f}"
    text = open(os.path.join(INCLUDE_DIR, "gdn_recoverssm_hip.h")).read()
    assert f"#define GDN_TABLES_MAX_ROWS {MAX_TABLE_ROWS}" in text


# --- the C entry points ---------------------------------------------------------

def fake():
    return 0x1000  # never read: every call here is refused, or has nothing to do


def pages(**change):
    p = dict(query_start_loc=fake(), state_indices=fake(), rows=2, tokens=10, blocks=4, qsl_stride=1, si_stride=1,
             qsl_dtype=N.DT_I32, si_dtype=N.DT_I32)
    p.update(change)
    return N.RowPages(**p)


def rule(pages_=None, **change):
    l = dict(pages=pages_ or pages(), q=fake(), k=fake(), v=fake(), g=fake(), beta=fake(), out=fake(), state=fake(),
             heads=2, value_heads=4, key_dim=64, value_dim=32, q_stride=128, k_stride=128, v_stride=128, g_stride=4,
             beta_stride=4, out_stride=128, state_block_stride=8192, state_head_stride=2048, state_v_stride=64,
             act_dtype=N.DT_BF16, g_dtype=N.DT_F32, beta_dtype=N.DT_F32, out_dtype=N.DT_BF16, state_dtype=N.DT_F32,
             scale=1.0)
    l.update(change)
    return N.RuleLaunch(**l)


def conv(pages_=None, **change):
    l = dict(pages=pages_ or pages(), x=fake(), weight=fake(), out=fake(), conv_states=fake(), dim=8, taps=4, window=6,
             x_stride=8, out_stride=8, state_block_stride=48, state_dim_stride=6, state_token_stride=1,
             dtype=N.DT_BF16, silu=1)
    l.update(change)
    return N.ConvRows(**l)


BAD_PAGES = [dict(rows=-1), dict(tokens=-1), dict(blocks=0), dict(tokens=1 << 30), dict(rows=1 << 25),
             dict(qsl_dtype=N.DT_F32), dict(si_dtype=9), dict(final_indices=0x1000, final_dtype=N.DT_BF16),
             dict(num_computed=0x1000, computed_dtype=N.DT_F32), dict(request_indices=0x1000, map_dtype=-1),
             dict(num_computed=0x1000, computed_dtype=N.DT_I32, computed_len=-1),
             dict(block_table=0x1000, table_dtype=N.DT_I32, block_size=16, table_width=2),
             dict(block_table=0x1000, table_dtype=N.DT_I32, num_computed=0x1000, computed_dtype=N.DT_I32, table_width=2),
             dict(block_table=0x1000, table_dtype=N.DT_I32, num_computed=0x1000, computed_dtype=N.DT_I32, block_size=16),
             dict(block_table=0x1000, table_dtype=N.DT_I32, num_computed=0x1000, computed_dtype=N.DT_I32, block_size=16,
                  table_width=2, final_indices=0x1000, final_dtype=N.DT_I32),
             dict(query_start_loc=None), dict(state_indices=None)]
BAD_RULES = [dict(heads=0), dict(heads=3), dict(value_heads=65536), dict(value_dim=0), dict(value_dim=1 << 21),
             dict(key_dim=0), dict(key_dim=257), dict(key_dim=66), dict(state_v_stride=32), dict(state_v_stride=66),
             dict(state_head_stride=2050), dict(state_block_stride=1), dict(state=0x1004), dict(act_dtype=N.DT_I32),
             dict(state_dtype=N.DT_I64), dict(g_dtype=N.DT_F16), dict(beta_dtype=N.DT_F16), dict(out_dtype=N.DT_F16),
             dict(q=None), dict(k=None), dict(v=None), dict(g=None), dict(beta=None), dict(out=None), dict(state=None),
             dict(state_v_stride=1 << 26)]


def refused(status):
    assert status in (N.GDN_ERR_INVALID, N.GDN_ERR_UNSUPPORTED)
    assert N.load().gdn_recoverssm_last_error()


@pytest.mark.parametrize("change", BAD_PAGES, ids=str)
def test_bad_rows_are_refused(change):
    lib, p = N.load(), pages(**change)
    refused(lib.gdn_recoverssm_decode(rule(p), None))
    refused(lib.gdn_recoverssm_prefill(rule(p), 0x1000, 1 << 40, None))
    assert lib.gdn_recoverssm_prefill_workspace(rule(p)) < 0
    refused(lib.gdn_recoverssm_conv(conv(p), None))


@pytest.mark.parametrize("change", BAD_RULES, ids=str)
def test_bad_rules_are_refused(change):
    lib = N.load()
    refused(lib.gdn_recoverssm_decode(rule(**change), None))
    refused(lib.gdn_recoverssm_prefill(rule(**change), 0x1000, 1 << 40, None))
    assert lib.gdn_recoverssm_prefill_workspace(rule(**change)) < 0


def test_bad_gating_is_refused():
    lib = N.load()
    for ext, more in ((N.GatingExt(N.DT_I32, N.DT_F32, 1.0, 20.0), {}), (N.GatingExt(N.DT_F32, N.DT_I64, 1.0, 20.0), {}),
                      (N.GatingExt(N.DT_F32, N.DT_F32, 0.0, 20.0), {}), (N.GatingExt(N.DT_F32, N.DT_F32, 1.0, 20.0), dict(dt_bias=None)),
                      (N.GatingExt(N.DT_F32, N.DT_F32, float("nan"), 20.0), {})):
        l = rule(gating=ctypes.pointer(ext), **{"a_log": 0x1000, "dt_bias": 0x1000, **more})
        refused(lib.gdn_recoverssm_decode(l, None))
        refused(lib.gdn_recoverssm_prefill(l, 0x1000, 1 << 40, None))


@pytest.mark.parametrize("change", [dict(v_stride=16), dict(out_stride=-128), dict(v_stride=1 << 23), dict(out_stride=1 << 40)],
                         ids=str)
def test_prefill_refuses_token_strides_it_cannot_reach(change):
    refused(N.load().gdn_recoverssm_prefill(rule(**change), 0x1000, 1 << 40, None))


def test_prefill_workspace_is_checked():
    lib = N.load()
    need = lib.gdn_recoverssm_prefill_workspace(rule())
    # 10 tokens and 2 rows: two chunks. A key head has 12 KB per 32 columns, a
    # value head 14 + 6 KB per plane of a BF16 output.
    assert need == 2 * (2 * 12 * 2 + 4 * (14 + 6)) * 1024
    assert lib.gdn_recoverssm_prefill_workspace(rule(out_dtype=N.DT_F32)) == 2 * (2 * 12 * 2 + 4 * (14 + 12)) * 1024
    assert lib.gdn_recoverssm_prefill_workspace(rule(act_dtype=N.DT_F32, out_dtype=N.DT_F32)) == \
        2 * (2 * 12 * 2 * 2 + 4 * (14 + 12)) * 1024
    for ws, size in ((None, need), (0x1000, need - 1), (0x1008, need)):
        refused(lib.gdn_recoverssm_prefill(rule(), ws, size, None))
    assert lib.gdn_recoverssm_prefill_workspace(rule(pages(rows=0))) == 0
    assert lib.gdn_recoverssm_prefill_workspace(None) < 0


@pytest.mark.parametrize("change", [dict(dim=0), dict(dim=1 << 25), dict(taps=1), dict(taps=6), dict(window=2),
                                    dict(dtype=N.DT_I32), dict(x=None), dict(weight=None), dict(out=None),
                                    dict(conv_states=None)], ids=str)
def test_bad_convolutions_are_refused(change):
    refused(N.load().gdn_recoverssm_conv(conv(**change), None))


def tables(**change):
    l = dict(num_computed=0x1000, query_lens=0x1000, block_table=0x1000, free_pages=0x1000, free_span=0x1000,
             free_span_out=0x2000, query_start_loc=0x1000, seq_lens=0x1000, source_indices=0x1000,
             final_indices=0x1000, new_pages=0x1000, positions=0x1000, slot_mapping=0x1000, rows=4, num_tokens=8,
             computed_len=4, computed_stride=1, lens_stride=1, table_rows=4, table_width=8, table_row_stride=8,
             free_len=16, block_size=16, computed_dtype=N.DT_I32, lens_dtype=N.DT_I32)
    l.update(change)
    return N.StepTablesLaunch(**l)


@pytest.mark.parametrize("change", [dict(rows=-1), dict(rows=4097), dict(num_tokens=-1), dict(num_tokens=1 << 30),
                                    dict(table_width=0), dict(table_rows=-1), dict(free_len=0), dict(block_size=0),
                                    dict(computed_len=-1), dict(computed_dtype=N.DT_F32), dict(lens_dtype=7),
                                    dict(request_indices=0x1000, map_dtype=N.DT_BF16), dict(free_pages=None),
                                    dict(free_span=None), dict(free_span_out=None), dict(query_start_loc=None),
                                    dict(positions=None), dict(slot_mapping=None), dict(num_computed=None),
                                    dict(query_lens=None), dict(block_table=None), dict(new_pages=None),
                                    dict(free_span_out=0x1000)], ids=str)
def test_bad_tables_are_refused(change):
    refused(N.load().gdn_recoverssm_step_tables(tables(**change), None))


def test_bad_releases_are_refused():
    good = dict(requests=0x1000, requests_dtype=N.DT_I32, num=2, lens=0x1000, lens_dtype=N.DT_I32, lens_stride=1,
                table=0x1000, rows=4, width=8, stride=8, block=16, free=0x1000, free_len=16, span=0x1000, out=0x2000)
    for change in (dict(num=-1), dict(rows=-1), dict(width=0), dict(block=0), dict(free_len=0), dict(free=None),
                   dict(span=None), dict(out=None), dict(out=0x1000), dict(requests=None), dict(lens=None),
                   dict(table=None), dict(requests_dtype=N.DT_F32), dict(lens_dtype=N.DT_F16)):
        refused(N.load().gdn_recoverssm_release_pages(*{**good, **change}.values(), None))


def test_nothing_to_do_needs_no_device():
    lib = N.load()
    for p in (pages(rows=0), pages(tokens=0)):
        assert lib.gdn_recoverssm_decode(rule(p), None) == N.GDN_OK
        assert lib.gdn_recoverssm_prefill(rule(p), None, 0, None) == N.GDN_OK
        assert lib.gdn_recoverssm_conv(conv(p), None) == N.GDN_OK
    refused(lib.gdn_recoverssm_decode(None, None))
    refused(lib.gdn_recoverssm_prefill(None, None, 0, None))
    refused(lib.gdn_recoverssm_conv(None, None))
    refused(lib.gdn_recoverssm_step_tables(None, None))


# --- the Python functions -------------------------------------------------------

I = torch.int32


def call(fn, **change):
    T, H, HV, K, V = 6, 2, 4, 16, 8
    bf = torch.bfloat16
    a = dict(g=torch.zeros(1, T, HV), beta=torch.zeros(1, T, HV), q=torch.zeros(1, T, H, K, dtype=bf),
             k=torch.zeros(1, T, H, K, dtype=bf), v=torch.zeros(1, T, HV, V, dtype=bf),
             checkpoint_state=torch.zeros(3, HV, V, K), query_start_loc=torch.zeros(3, dtype=I),
             state_indices=torch.zeros(2, dtype=I))
    a.update(change)
    gated = "A_log" in a
    first = [a.pop(n) for n in ("g", "beta", "q", "k", "v")]
    return getattr(G, "gdn_recoverssm_" + fn + ("_gated" if gated else ""))(*first, **a)


z = torch.zeros
RULE_REFUSALS = [
    ("q must have shape", dict(q=z(6, 2, 16))), ("q must have shape", dict(q=z(2, 6, 2, 16))),
    ("q and k shapes differ", dict(k=z(1, 6, 2, 8))), ("v must have shape", dict(v=z(1, 5, 4, 8))),
    ("positive multiple", dict(v=z(1, 6, 3, 8))), ("positive multiple", dict(v=z(1, 6, 1, 8))),
    ("heads must be contiguous", dict(v=z(1, 6, 4, 16)[..., ::2])),
    ("heads must be contiguous", dict(q=z(1, 6, 4, 16, dtype=torch.bfloat16)[:, :, ::2])),
    ("share one activation dtype", dict(k=z(1, 6, 2, 16))),
    ("share one activation dtype", {n: z(1, 6, h, d, dtype=torch.float64) for n, h, d in (("q", 2, 16), ("k", 2, 16), ("v", 4, 8))}),
    ("gate or beta shape", dict(g=z(1, 5, 4))), ("gate or beta shape", dict(beta=z(6, 2))),
    ("gate and beta must be FP32", dict(g=z(1, 6, 4, dtype=torch.float16))),
    ("four-dimensional", dict(checkpoint_state=z(4, 8, 16))),
    ("checkpoint shape", dict(checkpoint_state=z(3, 4, 8, 8))), ("checkpoint shape", dict(checkpoint_state=z(0, 4, 8, 16))),
    ("checkpoint dtype", dict(checkpoint_state=z(3, 4, 8, 16, dtype=torch.float64))),
    ("16-byte aligned", dict(checkpoint_state=z(3, 4, 8, 17)[..., :16])),
    ("16-byte aligned", dict(checkpoint_state=z(3, 4, 16, 8).transpose(2, 3))),
    ("output shape", dict(out=z(1, 6, 4, 9))), ("output shape", dict(out=z(1, 6, 4, 16)[..., ::2])),
    ("out must be FP32", dict(out=z(1, 6, 4, 8, dtype=torch.float16))),
    ("one contiguous entry per value head", dict(A_log=z(3), dt_bias=z(4))),
    ("one contiguous entry per value head", dict(A_log=z(4), dt_bias=z(8)[::2])),
    ("softplus beta", dict(A_log=z(4), dt_bias=z(4), softplus_beta=0.0)),
    ("same device", dict(k=z(1, 6, 2, 16, dtype=torch.bfloat16, device="meta"))),
    ("run on a HIP device", {}),
]


@pytest.mark.parametrize("fn", ["prefill", "decode"])
@pytest.mark.parametrize("message,change", RULE_REFUSALS, ids=[f"{i}-{m}" for i, (m, _) in enumerate(RULE_REFUSALS)])
def test_rule_arguments(fn, message, change):
    with pytest.raises(ValueError, match=f"GDN RecoverSSM: .*{message}"):
        call(fn, **change)


def conv_call(**change):
    a = dict(x=z(6, 8), weight=z(8, 4), bias=z(8), conv_states=z(3, 8, 3), query_start_loc=z(3, dtype=I),
             state_indices=z(2, dtype=I))
    a.update(change)
    return G.gdn_recoverssm_conv(a.pop("x"), a.pop("weight"), a.pop("bias"), **a)


CONV_REFUSALS = [
    ("x must have shape", dict(x=z(6))), ("share one dtype", dict(weight=z(8, 4, dtype=torch.bfloat16))),
    ("share one dtype", dict(bias=z(8, dtype=torch.float16))), ("share one dtype", dict(conv_states=z(3, 8, 3).half())),
    ("2 to 5 taps", dict(weight=z(8, 6))), ("2 to 5 taps", dict(weight=z(8, 1))), ("2 to 5 taps", dict(weight=z(4, 8).t())),
    ("bias must be contiguous", dict(bias=z(9))), ("conv states must", dict(conv_states=z(3, 8, 2))),
    ("conv states must", dict(conv_states=z(3, 7, 3))), ("conv states must", dict(conv_states=z(0, 8, 3))),
    ("channels must be contiguous", dict(x=z(8, 6).t())), ("output shape", dict(out=z(6, 9))),
    ("activation must be", dict(activation="gelu")), ("same device", dict(bias=z(8, device="meta"))),
    ("runs on a HIP device", {}),
]


@pytest.mark.parametrize("message,change", CONV_REFUSALS, ids=[f"{i}-{m}" for i, (m, _) in enumerate(CONV_REFUSALS)])
def test_convolution_arguments(message, change):
    with pytest.raises(ValueError, match=f"GDN RecoverSSM: .*{message}"):
        conv_call(**change)


def table_call(**change):
    a = dict(block_table=z(4, 8, dtype=I), free_pages=z(16, dtype=I), free_span=z(2, dtype=torch.int64),
             num_computed=z(4, dtype=I), query_lens=z(4, dtype=I), block_size=16, num_tokens=8)
    a.update(change)
    return G.gdn_recoverssm_step_tables(a.pop("block_table"), a.pop("free_pages"), a.pop("free_span"), **a)


TABLE_REFUSALS = [
    ("one-dimensional", dict(num_computed=z(4, 1, dtype=I))), ("one entry per row", dict(request_indices=z(3, dtype=I))),
    ("one entry per row when", dict(num_computed=z(3, dtype=I))), ("int32 or int64", dict(query_lens=z(4))),
    ("at most 4096 rows", dict(query_lens=z(4097, dtype=I), num_computed=z(4097, dtype=I))),
    ("num_tokens must be", dict(num_tokens=-1)), ("run on a HIP device", {}),
]


@pytest.mark.parametrize("message,change", TABLE_REFUSALS, ids=[f"{i}-{m}" for i, (m, _) in enumerate(TABLE_REFUSALS)])
def test_table_arguments(message, change):
    with pytest.raises(ValueError, match=f"GDN RecoverSSM: .*{message}"):
        table_call(**change)


POOL_REFUSALS = [
    ("block table must be int32", dict(block_table=z(4, 8, dtype=torch.int64))),
    ("block table must be int32", dict(block_table=z(8, 4, dtype=I).t())),
    ("contiguous int32 ring", dict(free_pages=z(16, dtype=torch.int64))),
    ("contiguous int32 ring", dict(free_pages=z(0, dtype=I))), ("contiguous int64 pair", dict(free_span=z(2, dtype=I))),
    ("block_size must be positive", dict(block_size=0)), ("same device", dict(free_pages=z(16, dtype=I, device="meta"))),
    ("one entry per ended request", dict(seq_lens=z(3, dtype=I))), ("int32 or int64", dict(requests=z(2))),
    ("requests must be contiguous", dict(requests=z(4, dtype=I)[::2])), ("run on a HIP device", {}),
]


@pytest.mark.parametrize("message,change", POOL_REFUSALS, ids=[f"{i}-{m}" for i, (m, _) in enumerate(POOL_REFUSALS)])
def test_release_arguments(message, change):
    a = dict(block_table=z(4, 8, dtype=I), free_pages=z(16, dtype=I), free_span=z(2, dtype=torch.int64),
             requests=z(2, dtype=I), seq_lens=z(2, dtype=I), block_size=16)
    a.update(change)
    with pytest.raises(ValueError, match=f"GDN RecoverSSM: .*{message}"):
        G.gdn_recoverssm_release_pages(a.pop("block_table"), a.pop("free_pages"), a.pop("free_span"), **a)


@pytest.mark.skipif(not os.path.exists(LIB_PATH), reason="the library is built by __graft_entry__.build()")
def test_kernels_spill_no_vector_register(tmp_path):
    """The prefill's scans are not among them: what they keep over the walk of a
    chunk may go to memory outside their loops."""
    spills = {k: n for k, n in _spills(tmp_path).items()
              if re.search("decode_kernel|conv_kernel|step_tables_kernel|release_pages_kernel", k)}
    assert len(spills) > 60
    assert not {k: n for k, n in spills.items() if n}
