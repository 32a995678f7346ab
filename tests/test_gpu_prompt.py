"""The prompt operators on the GPU against their definitions in 64 bits
(``prompt_oracle``): the gated delta rule over whole rows, chunked
(``gdn_recoverssm_prefill``) and recurrent (``gdn_recoverssm_decode``).

Bars, derived from the arithmetic (FP32 sums; one rounding where a tensor of
fewer bits is written): outputs norm-wise 2^-8 BF16 / 2^-11 F16 (half a unit in
the last place is 2^-9 / 2^-12 of a value) and 1e-5 FP32; pages max-abs over
max-abs 1e-5 FP32, 2^-8 BF16, 2^-11 F16. Pages that no row ends in keep their
bits; refused rows give exact zeros.
"""

import pytest
import torch

import gdn_oracle as O
import gdn_recoverssm_ascend as G
import prompt_oracle as P

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
OUT_TOL = {torch.float32: 1e-5, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
PAGE_TOL = {torch.float32: 1e-5, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
FORMS = ("prefill", "decode")


def problem(lengths, H, HV, K, V, act="bf16", state="f32", seed=0, decay=1.0, gated=False, unit=True):
    gen = torch.Generator().manual_seed(seed)
    T, B = sum(lengths), len(lengths)
    randn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    l2 = lambda x: x * torch.rsqrt((x * x).sum(-1, keepdim=True) + 1e-6)  # noqa: E731
    q, k = randn(1, T, H, K), randn(1, T, H, K)
    if unit:
        q, k = l2(q), l2(k)
    p = dict(q=q.to(DT[act]), k=k.to(DT[act]), v=randn(1, T, HV, V).to(DT[act]))
    if gated:
        p.update(A_log=randn(HV), dt_bias=randn(HV), g=randn(T, HV).to(DT[act]), beta=randn(T, HV).to(DT[act]))
    else:
        rate = torch.exp(torch.linspace(-4.0, 1.0, HV)) * decay
        p.update(g=-rate * torch.nn.functional.softplus(randn(T, HV)), beta=torch.sigmoid(randn(T, HV)))
    p["pages"] = (randn(2 * B + 2, HV, V, K) * 0.1).to(DT[state])
    place = 1 + torch.randperm(2 * B, generator=gen)
    p["source"], p["final"] = place[:B].int(), place[B:].int()
    p["qsl"] = torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32)
    return p


def run(form, p, dev, *, rows=None, scale=None, l2norm=False, move=None, **call):
    """The GPU's output and pages. ``rows``: final / computed / table / block /
    requests as the oracle names them; ``move`` may lay a tensor out anew."""
    names = dict(final="final_indices", computed="num_computed", table="block_table", requests="request_indices")
    rows = rows or {}
    move = move or (lambda name, t: t.to(dev))
    kw = {names[n]: move(n, t) for n, t in rows.items() if n in names and t is not None}
    if "block" in rows:
        kw["block_size"] = rows["block"]
    pages = move("pages", p["pages"])
    args = [move(n, p[n]) for n in ("g", "beta", "q", "k", "v")]
    fn = getattr(G, "gdn_recoverssm_" + form + ("_gated" if "A_log" in p else ""))
    if "A_log" in p:
        kw.update(A_log=move("A_log", p["A_log"]), dt_bias=move("dt_bias", p["dt_bias"]))
    out = fn(*args, checkpoint_state=pages, query_start_loc=move("qsl", p["qsl"]),
             state_indices=move("source", p["source"]), scale=scale, qk_already_normalized=not l2norm, **kw, **call)
    torch.cuda.synchronize()
    return out, pages


def check(form, p, dev, *, rows=None, scale=None, l2norm=False, **more):
    rows = rows or {}
    g, beta = p["g"], p["beta"]
    if "A_log" in p:
        g, beta = P.gates(g, beta, p["A_log"], p["dt_bias"])
    want, pages = P.rule(p["q"], p["k"], p["v"], g, beta, p["pages"], p["qsl"], p["source"], scale=scale,
                         l2norm=l2norm, **rows)
    out, got = run(form, p, dev, rows=rows, scale=scale, l2norm=l2norm, **more)
    compare(p, out.cpu()[0], got.cpu(), want, pages)


def compare(p, out, got, want, pages):
    norm = float(want.norm())
    err = float((out.double() - want).norm()) / norm if norm else float(out.double().abs().max()) if out.numel() else 0.0
    assert err <= OUT_TOL[out.dtype], f"out: {err:.3g}"
    zero = (want == 0).flatten(1).all(1)
    assert not out[zero].any(), "tokens of refused rows must be zero"
    touched = (pages != p["pages"].double()).flatten(1).any(1)
    assert torch.equal(got[~touched], p["pages"][~touched]), "a page that no row ends in changed"
    if touched.any():
        err = O.max_abs_rel(got[touched].double(), pages[touched])
        assert err <= PAGE_TOL[got.dtype], f"pages: {err:.3g}"


EDGES = [[1], [2], [15], [16], [17], [31], [33], [63], [64], [65], [127], [128], [129], [193, 1, 0, 64, 7]]


@pytest.mark.parametrize("lengths", EDGES, ids=lambda v: "-".join(map(str, v)))
@pytest.mark.parametrize("form", FORMS)
def test_lengths_around_the_chunk(form, lengths, gpu_device):
    p = problem(lengths, 2, 4, 128, 128, seed=sum(lengths))
    check(form, p, gpu_device, rows=dict(final=p["final"]))


DIMS = [(1, 1, 8, 1), (1, 2, 16, 3), (2, 2, 32, 17), (1, 3, 64, 64), (2, 6, 64, 192), (4, 12, 96, 192), (2, 4, 72, 33),
        (3, 3, 104, 80), (2, 4, 128, 96), (1, 4, 136, 40), (2, 2, 192, 128), (2, 4, 256, 128), (1, 8, 248, 65)]


@pytest.mark.parametrize("types", [("bf16", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f16", "f32"), ("f32", "f32"),
                                   ("f32", "bf16")], ids="-".join)
@pytest.mark.parametrize("dims", DIMS, ids=lambda d: "x".join(map(str, d)))
@pytest.mark.parametrize("form", FORMS)
def test_heads_dims_and_types(form, dims, types, gpu_device):
    p = problem([70, 5, 129], *dims, *types, seed=sum(dims))
    check(form, p, gpu_device, rows=dict(final=p["final"]))


@pytest.mark.parametrize("form", FORMS)
def test_key_dims_of_four(form, gpu_device):
    """FP32 pages take any multiple of four: heads of 16-bit activations then
    start off 16-byte boundaries."""
    for K in (4, 12, 20, 100, 132):
        p = problem([66, 3], 3, 6, K, 24, "bf16", "f32", seed=K)
        check(form, p, gpu_device, rows=dict(final=p["final"]))


@pytest.mark.parametrize("l2norm", [False, True])
@pytest.mark.parametrize("types", [("bf16", "f32"), ("f16", "bf16"), ("f32", "f32")], ids="-".join)
@pytest.mark.parametrize("form", FORMS)
def test_gated(form, types, l2norm, gpu_device):
    p = problem([100, 1, 65], 2, 4, 64, 64, *types, gated=True, unit=not l2norm, seed=5)
    check(form, p, gpu_device, rows=dict(final=p["final"]), l2norm=l2norm, scale=0.3)


@pytest.mark.parametrize("l2norm", [False, True])
@pytest.mark.parametrize("form", FORMS)
def test_l2norm_of_large_and_zero_keys(form, l2norm, gpu_device):
    p = problem([90], 1, 2, 64, 32, unit=not l2norm, seed=6)
    if l2norm:
        p["k"] *= 300.0
        p["q"] *= 0.01
    p["k"][0, 7] = 0.0
    p["q"][0, 9] = 0.0
    check(form, p, gpu_device, rows=dict(final=p["final"]), l2norm=l2norm)


@pytest.mark.parametrize("form", FORMS)
def test_out_in_fp32(form, gpu_device):
    p = problem([77, 64], 2, 4, 128, 64, seed=8)
    out = torch.empty(1, 141, 4, 64, dtype=torch.float32, device=gpu_device)
    check(form, p, gpu_device, rows=dict(final=p["final"]), out=out)


@pytest.mark.parametrize("form", FORMS)
def test_in_place_pages(form, gpu_device):
    p = problem([130, 1, 20], 2, 4, 64, 64, seed=9)
    check(form, p, gpu_device)


@pytest.mark.parametrize("form", FORMS)
def test_refused_rows_and_zero_starts(form, gpu_device):
    """Null, negative and past-the-pool pages; rows with C = 0 start from zero
    whatever their source page is (a NaN page here), C < 0 is refused."""
    p = problem([20, 70, 9, 1, 66, 3, 5], 1, 2, 64, 40, seed=10)
    p["pages"][int(p["source"][1])] = float("nan")
    p["source"][0] = 0
    p["source"][2] = p["pages"].shape[0]
    p["source"][3] = -1
    p["final"][4] = 0
    p["final"][5] = 10000
    rows = dict(final=p["final"], computed=torch.tensor([5, 0, 7, 0, 0, 2, -3], dtype=torch.int64))
    g, beta = p["g"], p["beta"]
    want, pages = P.rule(p["q"], p["k"], p["v"], g, beta, p["pages"], p["qsl"], p["source"], **rows)
    out, got = run(form, p, gpu_device, rows=rows)
    nan = int(p["source"][1])
    assert got[nan].isnan().all()
    keep = torch.arange(len(pages)) != nan
    compare(dict(p, pages=p["pages"][keep]), out.cpu()[0], got.cpu()[keep], want, pages[keep])


@pytest.mark.parametrize("block", [1, 16, 40, 48, 64, 96, 128, 200, 1024])
@pytest.mark.parametrize("form", FORMS)
def test_block_table(form, block, gpu_device):
    """Align mode: final page and every boundary's page from the table, some of
    them null, positions on, before and behind block boundaries, a table that
    ends early, a request map."""
    lengths = [1, 63, 64, 65, 130, 200, 0, 97]
    p = problem(lengths, 1, 2, 64, 48, seed=block)
    C = torch.tensor([0, 0, 64, 63, 31, 129, 7, 2 * block], dtype=torch.int32)
    gen = torch.Generator().manual_seed(block)
    requests = torch.randperm(len(lengths), generator=gen)
    computed = torch.zeros(len(lengths), dtype=torch.int32)
    computed[requests] = C
    width = max((int(c) + n + block) // block for c, n in zip(C, lengths))
    table = torch.zeros(len(lengths), width, dtype=torch.int32)
    pages = 1
    for r, (c, n) in enumerate(zip(C.tolist(), lengths)):
        for col in range(max(c - 1, 0) // block, (c + max(n, 1) - 1) // block + 1):
            table[requests[r], col] = pages
            pages += 1
            if col % 3 == 1 and col < (c + n - 1) // block and c <= col * block:
                table[requests[r], col] = (0, -1, 10**6)[r % 3]
        p["source"][r] = table[requests[r], max(c - 1, 0) // block] if c else 0
    p["pages"] = (torch.randn(pages + 1, 2, 48, 64, generator=gen) * 0.1)
    check(form, p, gpu_device, rows=dict(computed=computed, table=table, block=block, requests=requests))


@pytest.mark.parametrize("form", FORMS)
def test_table_narrower_than_the_row(form, gpu_device):
    """Columns past the table: the final page is the last column's, boundaries
    there go nowhere."""
    p = problem([200], 1, 1, 64, 16, seed=3)
    p["source"][0] = 1
    rows = dict(computed=torch.tensor([10]), table=torch.tensor([[1, 2]]), block=64)
    check(form, p, gpu_device, rows=rows)


@pytest.mark.parametrize("form", FORMS)
def test_strided_views_and_index_types(form, gpu_device):
    """q, k and v as views of one combined projection, gates as columns of a
    wider tensor, int64 and strided indices, pages and output with gaps."""
    lengths, H, HV, K, V = [65, 3, 140], 2, 4, 64, 48
    p = problem(lengths, H, HV, K, V, seed=12)
    T = sum(lengths)
    dev = gpu_device
    wide = torch.zeros(1, T, 2 * H * K + HV * V + 5, dtype=torch.bfloat16, device=dev)
    at = dict(q=(0, H, K), k=(H * K, H, K), v=(2 * H * K, HV, V))

    def move(name, t):
        if name in at:
            first, heads, dim = at[name]
            part = wide[..., first:first + heads * dim].unflatten(2, (heads, dim))
            part.copy_(t.to(dev))
            return part
        if name in ("g", "beta"):
            room = torch.zeros(T, HV + 3, dtype=t.dtype, device=dev)
            room[:, 1:1 + HV] = t.to(dev)
            return room[:, 1:1 + HV]
        if name in ("source", "final", "qsl"):
            room = torch.full((t.numel(), 3), 99, dtype=torch.int64, device=dev)
            room[:, 1] = t.to(dev)
            return room[:, 1]
        if name == "pages":
            room = torch.zeros(t.shape[0], HV + 1, V + 2, K + 4, dtype=t.dtype, device=dev)
            part = room[:, :HV, :V, :K]
            part.copy_(t.to(dev))
            return part
        return t.to(dev)

    out = torch.full((1, T, HV * V + 7), 7.0, dtype=torch.bfloat16, device=dev)
    view = out[..., :HV * V].unflatten(2, (HV, V))
    check(form, p, dev, rows=dict(final=p["final"]), move=move, out=view)
    assert (out[..., HV * V:] == 7.0).all()


@pytest.mark.parametrize("form", FORMS)
def test_odd_offsets_of_activations(form, gpu_device):
    """16-bit activations that start at an odd element."""
    p = problem([70, 40], 2, 4, 64, 32, seed=13)

    def move(name, t):
        if name in ("q", "k", "v"):
            room = torch.zeros(t.numel() + 1, dtype=t.dtype, device=gpu_device)
            room[1:] = t.flatten().to(gpu_device)
            return room[1:].view(t.shape)
        return t.to(gpu_device)

    check(form, p, gpu_device, rows=dict(final=p["final"]), move=move)


@pytest.mark.parametrize("form", FORMS)
def test_decays_from_none_to_all(form, gpu_device):
    """g = 0, g of minus infinity (the state is dropped) and steep decays next
    to slow ones: differences of cumulative decays keep their precision."""
    p = problem([150, 64], 1, 4, 64, 32, seed=14)
    p["g"][:, 0] = 0.0
    p["g"][10, 1] = -float("inf")
    p["g"][70:73, 1] = -float("inf")
    p["g"][5:60, 2] = -90.0
    p["g"][60:, 2] = -1e-4
    p["g"][:, 3] = -1e-3
    p["g"][::9, 3] = -30.0
    check(form, p, gpu_device, rows=dict(final=p["final"]))


@pytest.mark.parametrize("form", FORMS)
def test_repeated_keys_with_full_beta(form, gpu_device):
    """One key over and over with beta = 1 and no decay: the triangular system
    is all ones, and every token replaces what the one before it wrote."""
    p = problem([130], 1, 1, 64, 32, act="f32", seed=15)
    p["k"][:] = p["k"][:, :1]
    p["g"][:] = 0.0
    p["beta"][:] = 1.0
    check(form, p, gpu_device, rows=dict(final=p["final"]))


@pytest.mark.parametrize("form", FORMS)
def test_other_rows_nan_stays_there(form, gpu_device):
    """A row of NaN inputs, and a NaN source page, leave the rows beside them alone."""
    p = problem([70, 65, 70], 1, 2, 64, 32, seed=16)
    clean, pages = run(form, p, gpu_device, rows=dict(final=p["final"]))
    for n in ("q", "k", "v"):
        p[n][0, 70:135] = float("nan")
    p["pages"][int(p["source"][1])] = float("nan")
    out, got = run(form, p, gpu_device, rows=dict(final=p["final"]))
    keep = torch.cat([torch.arange(70), torch.arange(135, 205)])
    assert torch.equal(out[0, keep], clean[0, keep])
    for r in (0, 2):
        assert torch.equal(got[int(p["final"][r])], pages[int(p["final"][r])])


@pytest.mark.parametrize("form", FORMS)
def test_causal_within_a_row(form, gpu_device):
    """Later tokens' values leave earlier outputs alone, bit for bit."""
    p = problem([140], 1, 2, 64, 32, seed=17)
    one, _ = run(form, p, gpu_device, rows=dict(final=p["final"]))
    for n in ("q", "k", "v"):
        p[n][0, 100:] *= 3.0
    two, _ = run(form, p, gpu_device, rows=dict(final=p["final"]))
    assert torch.equal(one[0, :100], two[0, :100])


def test_prefill_and_decode_agree_with_split_rows(gpu_device):
    """A prompt in one call, and in pieces through both forms, ends in the same
    state up to FP32 rounding."""
    p = problem([300], 2, 4, 128, 128, seed=18)
    _, whole = run("prefill", p, gpu_device, rows=dict(final=p["final"]))
    pages = p["pages"].to(gpu_device)
    src, fin = p["source"].to(gpu_device), p["final"].to(gpu_device)
    at = 0
    for n, form in ((100, "prefill"), (1, "decode"), (130, "prefill"), (5, "decode"), (64, "prefill")):
        part = {x: p[x][:, at:at + n].to(gpu_device) for x in ("q", "k", "v")}
        getattr(G, "gdn_recoverssm_" + form)(
            p["g"][at:at + n].to(gpu_device), p["beta"][at:at + n].to(gpu_device), **part, checkpoint_state=pages,
            query_start_loc=torch.tensor([0, n], device=gpu_device), state_indices=src, final_indices=fin)
        src, at = fin, at + n
    page = int(p["final"][0])
    assert O.max_abs_rel(pages[page].cpu(), whole[page].cpu()) <= 1e-5


@pytest.mark.parametrize("form", FORMS)
def test_long_row(form, gpu_device):
    """A few thousand tokens of slow decay: the error does not pile up."""
    p = problem([2500], 1, 2, 128, 64, decay=0.01, seed=19)
    check(form, p, gpu_device, rows=dict(final=p["final"]))


@pytest.mark.parametrize("form", FORMS)
def test_same_bits_every_time_and_in_any_batch(form, gpu_device):
    """Results are bit-identical from run to run, and a row's do not depend on
    the rows beside it."""
    p = problem([130, 64, 33, 1], 2, 4, 128, 128, seed=20)
    rows = dict(final=p["final"])
    out, pages = run(form, p, gpu_device, rows=rows)
    again, same = run(form, p, gpu_device, rows=rows)
    assert torch.equal(out, again) and torch.equal(pages, same)
    one = dict(p, **{n: p[n][:, 194:227] for n in ("q", "k", "v")}, g=p["g"][194:227], beta=p["beta"][194:227],
               source=p["source"][2:3], qsl=torch.tensor([0, 33]))
    alone, pages1 = run(form, one, gpu_device, rows=dict(final=p["final"][2:3]))
    assert torch.equal(alone[0], out[0, 194:227])
    assert torch.equal(pages1[int(p["final"][2])], pages[int(p["final"][2])])


@pytest.mark.parametrize("form", FORMS)
def test_on_another_stream_and_in_a_graph(form, gpu_device):
    dev = gpu_device
    p = problem([100, 7], 2, 4, 64, 64, seed=21)
    want, want_pages = run(form, p, dev, rows=dict(final=p["final"]))
    t = {n: p[n].to(dev) for n in ("g", "beta", "q", "k", "v", "qsl", "source", "final")}
    pages = p["pages"].to(dev)
    fn = getattr(G, "gdn_recoverssm_" + form)

    def call():
        return fn(t["g"], t["beta"], t["q"], t["k"], t["v"], checkpoint_state=pages, query_start_loc=t["qsl"],
                  state_indices=t["source"], final_indices=t["final"])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = call()
    side.synchronize()
    assert torch.equal(out, want) and torch.equal(pages, want_pages)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for _ in range(3):
        pages.copy_(p["pages"])
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(pages, want_pages)


@pytest.mark.parametrize("form", FORMS)
def test_empty_batches(form, gpu_device):
    p = problem([4], 1, 1, 64, 16, seed=22)
    empty = dict(p, **{n: p[n][:, :0] for n in ("q", "k", "v")}, g=p["g"][:0], beta=p["beta"][:0])
    out, pages = run(form, dict(empty, qsl=torch.tensor([0, 0])), gpu_device)
    assert out.shape == (1, 0, 1, 16) and torch.equal(pages.cpu(), p["pages"])
    out, pages = run(form, dict(empty, qsl=torch.tensor([0]), source=torch.zeros(0, dtype=torch.int32)), gpu_device)
    assert out.numel() == 0 and torch.equal(pages.cpu(), p["pages"])


@pytest.mark.parametrize("form", FORMS)
def test_offsets_outside_the_batch_touch_nothing_else(form, gpu_device):
    """Offsets past the tokens are cut to them: the row that has tokens is
    right, nothing outside the output is written."""
    p = problem([70], 1, 1, 64, 16, seed=23)
    p["qsl"] = torch.tensor([0, 70, 900, 950], dtype=torch.int32)
    p["source"] = torch.tensor([1, 2, 3], dtype=torch.int32)
    p["pages"] = torch.randn(5, 1, 16, 64, generator=torch.Generator().manual_seed(1)) * 0.1
    out, pages = run(form, p, gpu_device)
    p["qsl"] = torch.tensor([0, 70], dtype=torch.int32)
    p["source"] = p["source"][:1]
    want, want_pages = P.rule(p["q"], p["k"], p["v"], p["g"], p["beta"], p["pages"], p["qsl"], p["source"])
    compare(p, out.cpu()[0], pages.cpu(), want, want_pages)


def _random(seed):
    gen = torch.Generator().manual_seed(seed)
    pick = lambda *v: v[int(torch.randint(0, len(v), (1,), generator=gen))]  # noqa: E731
    H = pick(1, 2, 3)
    state = pick("f32", "f32", "bf16", "f16")
    K = pick(8, 24, 40, 64, 88, 128, 160, 256)
    lengths = [pick(0, 1, 2, 5, 30, 64, 65, 100, 180) for _ in range(pick(1, 2, 4, 6))]
    lengths[0] = max(lengths[0], 1)
    return dict(lengths=lengths, H=H, HV=H * pick(1, 2, 3), K=K, V=pick(1, 9, 16, 50, 64, 128), act=pick("bf16", "f16", "f32"),
                state=state, seed=seed, gated=pick(False, True)), pick(False, True), pick(0, 32, 64, 100)


@pytest.mark.parametrize("seed", range(24))
@pytest.mark.parametrize("form", FORMS)
def test_random_problems(form, seed, gpu_device):
    kw, l2norm, block = _random(seed)
    p = problem(**kw, unit=not l2norm)
    rows = dict(final=p["final"])
    if block:
        gen = torch.Generator().manual_seed(seed)
        C = torch.randint(0, 300, (len(kw["lengths"]),), generator=gen) * (torch.rand(len(kw["lengths"]), generator=gen) < 0.7)
        table = torch.zeros(len(C), 600 // block + 2, dtype=torch.int64)
        pages = 1
        for r, n in enumerate(kw["lengths"]):
            for col in range(max(int(C[r]) - 1, 0) // block, (int(C[r]) + max(n, 1) - 1) // block + 1):
                table[r, col] = pages
                pages += 1
            p["source"][r] = table[r, max(int(C[r]) - 1, 0) // block]
        p["pages"] = (torch.randn(pages, kw["HV"], kw["V"], kw["K"], generator=gen) * 0.1).to(DT[kw["state"]])
        rows = dict(computed=C, table=table, block=block)
    check(form, p, gpu_device, rows=rows, l2norm=l2norm)
