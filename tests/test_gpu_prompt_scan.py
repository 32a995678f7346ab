"""The chunked rule's scans, each reached by the number of column tiles (rows x
value heads x ceil(V / 16)): up to 512 a tile has a workgroup to itself, then
four waves and, past 1024, eight share one; FP32 operands of K >= 128 go
straight from memory past 1024. And chunks that the rule stretches, whose values
are followed out of F16's range and back.

Bars as for the other prompt tests (outputs norm-wise 2^-8 BF16, 2^-11 F16, 1e-5
FP32; pages 1e-5). Where a chunk may stretch values, an operand's error of 2^-22
grows with the factor between what cancels and what is left; FP32 outputs and
pages there get 1e-4, for factors of up to 2^8. Columns are compared each by its
own norm where their sizes differ."""

import pytest
import torch

import gdn_oracle as O
import prompt_oracle as P
from test_gpu_prompt import OUT_TOL, check, problem, run

pytestmark = pytest.mark.gpu

TILES = {"split": 300, "four": 700, "eight": 1100}


def value_heads(form, H, rows, V):
    """Value heads, a multiple of H, that take a launch of these rows to the form."""
    per = rows * ((V + 15) // 16)
    HV = -(-TILES[form] // per)
    return -(-HV // H) * H


TYPES = [("bf16", "f32"), ("f16", "f16"), ("f32", "f32")]


@pytest.mark.parametrize("types", TYPES, ids="-".join)
@pytest.mark.parametrize("dims", [(2, 64, 128), (1, 128, 72), (1, 40, 200), (3, 104, 9)], ids=lambda d: "x".join(map(str, d)))
@pytest.mark.parametrize("form", ["four", "eight"])
def test_heads_dims_and_types(form, dims, types, gpu_device):
    H, K, V = dims
    p = problem([70, 1, 64, 0, 130], H, value_heads(form, H, 5, V), K, V, *types, seed=sum(dims))
    check("prefill", p, gpu_device, rows=dict(final=p["final"]))


@pytest.mark.parametrize("K", [128, 256])
@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_operands_past_the_shared_memory(act, K, gpu_device):
    p = problem([66, 129], 2, value_heads("eight", 2, 2, 100), K, 100, act, seed=K)
    check("prefill", p, gpu_device, rows=dict(final=p["final"]))


@pytest.mark.parametrize("form", ["four", "eight"])
def test_gated_with_l2norm_and_fp32_out(form, gpu_device):
    lengths = [100, 65, 3]
    HV = value_heads(form, 4, 3, 64)
    p = problem(lengths, 4, HV, 64, 64, gated=True, unit=False, seed=1)
    p["k"] *= 40.0
    p["k"][0, 5] = 0.0
    out = torch.empty(1, sum(lengths), HV, 64, dtype=torch.float32, device=gpu_device)
    check("prefill", p, gpu_device, rows=dict(final=p["final"]), l2norm=True, out=out)


@pytest.mark.parametrize("block", [1, 40, 64, 100, 192])
@pytest.mark.parametrize("form", ["four", "eight"])
def test_block_table(form, block, gpu_device):
    lengths = [1, 65, 130, 0, 97]
    HV, V, K = value_heads(form, 1, 5, 24), 24, 64
    C = torch.tensor([0, 63, 31, 7, 2 * block], dtype=torch.int32)
    p = problem(lengths, 1, HV, K, V, seed=block)
    table = torch.zeros(5, max((int(c) + n + block) // block for c, n in zip(C, lengths)), dtype=torch.int32)
    pages = 1
    for r, (c, n) in enumerate(zip(C.tolist(), lengths)):
        for col in range(max(c - 1, 0) // block, (c + max(n, 1) - 1) // block + 1):
            # Few pages for one-token blocks: boundaries in between go nowhere.
            if block > 1 or col % 20 == 0 or c + n - 1 == col or c - 1 == col:
                table[r, col] = pages
                pages += 1
        p["source"][r] = table[r, max(c - 1, 0) // block] if c else 0
    p["pages"] = torch.randn(pages + 1, HV, V, K, generator=torch.Generator().manual_seed(block)) * 0.1
    check("prefill", p, gpu_device, rows=dict(computed=C, table=table, block=block))


@pytest.mark.parametrize("form", ["four", "eight"])
def test_refused_rows_in_place_pages_and_strides(form, gpu_device):
    lengths, V = [20, 70, 9, 66], 33
    HV = value_heads(form, 2, 4, V)
    p = problem(lengths, 2, HV, 64, V, seed=10)
    p["source"][0] = 0
    p["source"][2] = p["pages"].shape[0]

    def move(name, t):
        t = t.to(gpu_device)
        if name in ("q", "k", "v"):
            room = torch.zeros(1, t.shape[1], t.shape[2] * t.shape[3] + 3, dtype=t.dtype, device=gpu_device)
            part = room[..., 1:-2].unflatten(2, t.shape[2:])
            part.copy_(t)
            return part
        return t

    room = torch.full((1, sum(lengths), HV * V + 7), 7.0, dtype=torch.bfloat16, device=gpu_device)
    check("prefill", p, gpu_device, move=move, out=room[..., :HV * V].unflatten(2, (HV, V)))
    assert (room[..., HV * V:] == 7.0).all()


@pytest.mark.parametrize("form", ["four", "eight"])
def test_other_rows_nan_stays_there(form, gpu_device):
    p = problem([70, 65, 70], 1, value_heads(form, 1, 3, 32), 64, 32, seed=16)
    clean, pages = run("prefill", p, gpu_device, rows=dict(final=p["final"]))
    for n in ("q", "k", "v"):
        p[n][0, 70:135] = float("nan")
    p["pages"][int(p["source"][1])] = float("nan")
    out, got = run("prefill", p, gpu_device, rows=dict(final=p["final"]))
    keep = torch.cat([torch.arange(70), torch.arange(135, 205)])
    assert torch.equal(out[0, keep], clean[0, keep])
    for r in (0, 2):
        assert torch.equal(got[int(p["final"][r])], pages[int(p["final"][r])])


@pytest.mark.parametrize("form", ["four", "eight"])
def test_same_bits_every_time(form, gpu_device):
    p = problem([130, 64, 33, 1], 2, value_heads(form, 2, 4, 128), 128, 128, seed=20)
    out, pages = run("prefill", p, gpu_device, rows=dict(final=p["final"]))
    again, same = run("prefill", p, gpu_device, rows=dict(final=p["final"]))
    assert torch.equal(out, again) and torch.equal(pages, same)


def by_column(p, dev, tol, **rows):
    """Each value column of a row against the column's own norm."""
    want, pages = P.rule(p["q"], p["k"], p["v"], p["g"], p["beta"], p["pages"], p["qsl"], p["source"], **rows)
    out, got = run("prefill", p, dev, rows=rows)
    off = (out.cpu()[0].double() - want).norm(dim=0) / want.norm(dim=0)
    assert float(off.max()) <= tol, f"out: {float(off.max()):.3g}"
    for b in range(len(p["source"])):
        page = int(rows["final"][b])
        off = (got[page].cpu().double() - pages[page]).norm(dim=-1) / pages[page].norm(dim=-1)
        assert float(off.max()) <= 1e-4, f"pages: {float(off.max()):.3g}"


FORMS = ["split", "four", "eight"]


@pytest.mark.parametrize("act", ["bf16", "f32"])
@pytest.mark.parametrize("form", FORMS)
def test_columns_of_any_size(form, act, gpu_device):
    """Columns of v and of the state from 1e-30 to 1e30, and zero states."""
    V = 20
    p = problem([140, 3], 1, value_heads(form, 1, 2, V), 64, V, act, seed=30)
    size = 10.0 ** torch.linspace(-30, 30, V)
    p["v"] = (p["v"].float() * size).to(p["v"].dtype)
    p["pages"] = p["pages"] * size[:, None]
    p["pages"][int(p["source"][1])] = 0.0
    by_column(p, gpu_device, OUT_TOL[p["v"].dtype], final=p["final"])


@pytest.mark.parametrize("form", FORMS)
def test_values_that_jump_and_fade(form, gpu_device):
    """From one chunk to the next v grows a million times, and a state that
    came in large fades away under steep decays."""
    V = 20
    p = problem([200, 200], 1, value_heads(form, 1, 2, V), 64, V, "f32", seed=31)
    p["v"][0, 70:140] *= 1e6
    p["v"][0, 140:] *= 1e-6
    p["pages"] *= 1e12
    p["g"][:] = -0.5
    by_column(p, gpu_device, 1e-4, final=p["final"])


@pytest.mark.parametrize("act", ["bf16", "f32"])
@pytest.mark.parametrize("form", FORMS)
def test_steps_that_stretch(form, act, gpu_device):
    """beta past 2, keys longer than 2, decays that grow: chunks whose values
    are checked one by one."""
    V, K = 20, 64
    p = problem([130, 70], 1, value_heads(form, 1, 2, V), K, V, act, seed=32)
    p["beta"][:64] *= 3.0
    p["k"][0, 64:128] *= 4.0
    p["beta"][64:128] *= 0.15
    p["g"][130:] = 0.05
    by_column(p, gpu_device, max(OUT_TOL[p["v"].dtype], 1e-4), final=p["final"])


@pytest.mark.parametrize("form", FORMS)
def test_checked_chunks_out_of_range(form, gpu_device):
    """Short keys with a large beta make corrections far larger than v: the
    column leaves F16's range inside a chunk and is brought back."""
    V = 20
    p = problem([100, 64], 1, value_heads(form, 1, 2, V), 64, V, "f32", seed=33)
    p["k"][0, :64] *= 2.0**-12
    p["beta"][:64] *= 2.0**22
    p["k"][0, 100:] *= 2.0**9
    p["beta"][100:] *= 2.0**-18
    by_column(p, gpu_device, 1e-4, final=p["final"])


@pytest.mark.parametrize("form", FORMS)
def test_negative_beta(form, gpu_device):
    p = problem([100], 1, value_heads(form, 1, 1, 16), 64, 16, "f32", seed=34)
    p["beta"] -= 0.7
    by_column(p, gpu_device, 1e-4, final=p["final"])


def test_forms_agree(gpu_device):
    """One row alone (split) and among many (eight waves): the same FP32 state
    up to rounding."""
    H, HV, K, V = 2, 16, 128, 128
    p = problem([130] * 9, H, HV, K, V, seed=35)
    assert 8 * HV <= 512 < 1024 < 9 * 8 * HV
    _, pages = run("prefill", p, gpu_device, rows=dict(final=p["final"]))
    one = dict(p, **{n: p[n][:, :130] for n in ("q", "k", "v")}, g=p["g"][:130], beta=p["beta"][:130],
               source=p["source"][:1], qsl=p["qsl"][:2])
    _, alone = run("prefill", one, gpu_device, rows=dict(final=p["final"][:1]))
    page = int(p["final"][0])
    assert O.max_abs_rel(alone[page].cpu(), pages[page].cpu()) <= 1e-5


DECODE = [(1, 2, 128, 128), (40, 4, 128, 128), (3, 2, 64, 20), (300, 4, 64, 32), (20, 32, 256, 72)]


@pytest.mark.parametrize("dims", DECODE, ids=lambda d: "x".join(map(str, d)))
@pytest.mark.parametrize("types", [("bf16", "f32"), ("f16", "bf16"), ("f32", "f32")], ids="-".join)
def test_decode_of_few_and_many_rows(dims, types, gpu_device):
    rows, HV, K, V = dims
    lengths = [1 + (b % 7 == 3) + 2 * (b % 11 == 5) - (b % 13 == 9) for b in range(rows)]
    p = problem(lengths, 2, HV, K, V, *types, seed=rows)
    check("decode", p, gpu_device, rows=dict(final=p["final"]))
