"""A step's tables and the return of pages, on the GPU, against plain loops:
whole numbers, equal."""

import pytest
import torch

import gdn_recoverssm_ascend as G
import prompt_oracle as P

pytestmark = pytest.mark.gpu


def pool(C, lens, block, width, seed=0, spare=None, requests=None, table_rows=None):
    """A table that holds the pages of C tokens a request and a ring of free pages."""
    gen = torch.Generator().manual_seed(seed)
    have = [-(-max(int(c), 0) // block) for c in C]
    place = (1 + torch.randperm(sum(have) + 5000, generator=gen)).tolist()
    table = torch.zeros(table_rows or len(C), width, dtype=torch.int32)
    for r, n in enumerate(have):
        for j in range(min(n, width)):
            table[r, j] = place.pop()
    ring = torch.tensor(place[:spare or 4000], dtype=torch.int32)
    return table, ring


def check(table, ring, span, C, lens, block, num_tokens, dev, requests=None, dtype=torch.int32, out=None):
    want_table, want = P.tables(table, ring, span, C, lens, block, num_tokens, requests)
    span = torch.tensor(span, dtype=torch.int64, device=dev)
    t = table.to(dev)
    got = G.gdn_recoverssm_step_tables(
        t, ring.to(dev), span, num_computed=torch.as_tensor(C).to(dev, dtype),
        query_lens=torch.as_tensor(lens).to(dev, dtype), block_size=block, num_tokens=num_tokens,
        request_indices=None if requests is None else torch.as_tensor(requests).to(dev), out=out)
    torch.cuda.synchronize()
    for name, value in want.items():
        assert torch.equal(getattr(got, name).cpu(), value), name
    assert torch.equal(t.cpu(), want_table)
    return got, t


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("block", [1, 3, 16, 64, 1000])
def test_mixed_lengths(block, dtype, gpu_device):
    C = [0, 0, 1, 63, 64, 65, 128, 200, 5, 0]
    lens = [1, 130, 1, 1, 1, 70, 0, 300, 64, 0]
    table, ring = pool(C, lens, block, 600 // block + 2, seed=block)
    check(table, ring, (7, 7 + 4000), C, lens, block, sum(lens) + 9, gpu_device, dtype=dtype)


@pytest.mark.parametrize("rows", [1, 2, 63, 64, 65, 255, 256, 257, 1000, 4096])
def test_row_counts(rows, gpu_device):
    gen = torch.Generator().manual_seed(rows)
    C = torch.randint(0, 400, (rows,), generator=gen).tolist()
    lens = torch.randint(0, 4, (rows,), generator=gen).tolist()
    lens[rows // 2] = 300
    table, ring = pool(C, lens, 32, 700 // 32 + 2, seed=rows)
    check(table, ring, (0, 4000), C, lens, 32, sum(lens), gpu_device)


def test_ring_wraps(gpu_device):
    C, lens = [0, 10, 20], [100, 50, 7]
    table, ring = pool(C, lens, 8, 30, spare=40)
    check(table, ring, (10**12 + 33, 10**12 + 33 + 40), C, lens, 8, 157, gpu_device)


@pytest.mark.parametrize("free", [0, 1, 5, 12, 13, 18, 19])
def test_pages_run_out(free, gpu_device):
    """Rows are served in order until their pages no longer fit; rows that need
    none are served all the same."""
    C, lens = [0, 3, 16, 8, 0, 9], [40, 1, 40, 3, 20, 50]
    table, ring = pool(C, lens, 8, 30, spare=64)
    check(table, ring, (100, 100 + free), C, lens, 8, sum(lens) + 3, gpu_device)


def test_request_map_and_refusals(gpu_device):
    """Requests outside the table, more columns than it has, negative lengths."""
    C = [0, 5, -4, 100, 31, 7]
    lens = [9, 6, 5, 3, -2, 300, 4]
    requests = [3, 0, 2, 9, 1, 5, -1]
    table, ring = pool(C, lens, 16, 9, table_rows=6)
    check(table, ring, (0, 500), C, lens, 16, 400, gpu_device, requests=requests)


def test_no_rows_and_reused_buffers(gpu_device):
    table, ring = pool([0], [0], 16, 4)
    got, _ = check(table, ring, (3, 10), [], [], 16, 5, gpu_device)
    C, lens = [4, 0], [2, 30]
    table, ring = pool(C, lens, 16, 4)
    out = G.StepTables.allocate(2, 40, gpu_device)
    got, _ = check(table, ring, (3, 100), C, lens, 16, 40, gpu_device, out=out)
    assert got is out


def test_steps_and_release(gpu_device):
    """Steps that go on from each other's tables and span, a request that ends
    and gives its pages back, and one that takes them; no page is ever held
    twice or lost."""
    dev, block, pages = gpu_device, 4, 24
    table = torch.zeros(4, 12, dtype=torch.int32, device=dev)
    ring = torch.arange(1, pages + 1, dtype=torch.int32, device=dev)
    span = torch.tensor([0, pages], dtype=torch.int64, device=dev)
    C = torch.zeros(4, dtype=torch.int32, device=dev)

    def whole(span):
        head, tail = span.tolist()
        free = [int(ring[i % pages]) for i in range(head, tail)]
        held = [int(x) for x in table.flatten() if x]
        assert sorted(free + held) == list(range(1, pages + 1))

    for lens in ([5, 9, 1, 0], [4, 1, 1, 7], [1, 1, 12, 1]):
        n = torch.tensor(lens, dtype=torch.int32, device=dev)
        t = G.gdn_recoverssm_step_tables(table, ring, span, num_computed=C, query_lens=n, block_size=block,
                                         num_tokens=sum(lens))
        assert (t.new_pages >= 0).all()
        assert t.final_indices.tolist() == [int(table[r, (int(s) - 1) // block]) for r, s in enumerate(t.seq_lens)]
        C, span = t.seq_lens.clone(), t.free_span
        whole(span)
    span = G.gdn_recoverssm_release_pages(table, ring, span, requests=torch.tensor([1, 3], device=dev),
                                          seq_lens=C[[1, 3]], block_size=block)
    whole(span)
    assert not table[[1, 3]].any()
    C[[1, 3]] = 0
    lens = torch.tensor([0, 40, 0, 0], dtype=torch.int32, device=dev)
    t = G.gdn_recoverssm_step_tables(table, ring, span, num_computed=C, query_lens=lens, block_size=block, num_tokens=40)
    assert t.new_pages.tolist() == [0, 10, 0, 0]
    whole(t.free_span)


def test_release_many_columns(gpu_device):
    """Rows longer than a workgroup, holes in the table, requests outside it."""
    dev = gpu_device
    gen = torch.Generator().manual_seed(3)
    table = torch.randint(0, 3, (3, 700), generator=gen, dtype=torch.int32) * torch.arange(1, 2101, dtype=torch.int32).view(3, 700)
    ring = torch.zeros(5000, dtype=torch.int32)
    want = [int(x) for r, n in ((2, 699), (0, 300)) for x in table[r, :n] if x]
    t, ring = table.to(dev), ring.to(dev)
    span = torch.tensor([4990, 4995], device=dev)
    got = G.gdn_recoverssm_release_pages(t, ring, span, requests=torch.tensor([2, 7, 0, -1], device=dev),
                                         seq_lens=torch.tensor([699, 5, 300, 4], device=dev), block_size=1)
    assert got.tolist() == [4990, 4995 + len(want)]
    assert [int(ring[i % 5000]) for i in range(4995, 4995 + len(want))] == want
    table[2, :699] = 0
    table[0, :300] = 0
    assert torch.equal(t.cpu(), table)


def test_graph_replays(gpu_device):
    dev = gpu_device
    C, lens = [0, 70, 3], [100, 1, 64]
    table, ring = pool(C, lens, 16, 20)
    want_table, want = P.tables(table, ring, (0, 4000), C, lens, 16, 170)
    t, ring = table.to(dev), ring.to(dev)
    span = torch.tensor([0, 4000], device=dev)
    C, lens = torch.tensor(C, device=dev), torch.tensor(lens, device=dev)
    out = G.StepTables.allocate(3, 170, dev)
    graph = torch.cuda.CUDAGraph()
    call = lambda: G.gdn_recoverssm_step_tables(t, ring, span, num_computed=C, query_lens=lens, block_size=16,  # noqa: E731
                                                num_tokens=170, out=out)
    call()
    with torch.cuda.graph(graph):
        call()
    for _ in range(3):
        t.copy_(table)
        out.positions.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(t.cpu(), want_table)
        for name, value in want.items():
            assert torch.equal(getattr(out, name).cpu(), value), name
