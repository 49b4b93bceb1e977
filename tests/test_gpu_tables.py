"""build_tables (HIP) against the definition, request by request."""
import numpy as np
import pytest
import torch

from paceserve_amd.kv_transfer import append as ap
from paceserve_amd.kv_transfer.tables import BatchTables, build_tables

pytestmark = pytest.mark.gpu


def i32(x, dev):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)


def by_hand(table, lens, P, qo, nnz, num_indices):
    """(tables, requests counted)."""
    B, W = table.shape
    indices, indptr, last = np.full(num_indices, -1), np.zeros(B + 1, np.int64), np.zeros(B, np.int64)
    pos, slot = np.full(nnz, -1), np.full(nnz, -1)
    counted = 0
    for b in range(B):
        n = min(max(int(lens[b]), 0), W * P)
        pages = -(-n // P)
        indptr[b + 1] = indptr[b] + pages
        last[b] = n - max(pages - 1, 0) * P if pages else 0
        for i in range(pages):
            if indptr[b] + i < num_indices:
                indices[indptr[b] + i] = table[b, i]
        a0, a1 = (b, b + 1) if qo is None else (qo[b], qo[b + 1])
        lo = min(max(a0, 0), nnz)
        hi = min(max(a1, lo), nnz)
        for j in range(hi - lo):
            t = int(lens[b]) - (hi - lo) + j
            pos[lo + j] = max(t, -1)
            if 0 <= t < n and table[b, t // P] >= 0:
                slot[lo + j] = int(table[b, t // P]) * P + t % P
        idle = qo is None and lens[b] == 0
        counted += n != lens[b] or lo != a0 or hi != a1 or (hi - lo > lens[b] and not idle) \
            or indptr[b + 1] > num_indices
    return (indices, indptr, last, pos, slot), counted


def check(got, want):
    for name, g, w in zip(BatchTables._fields, got, want):
        assert np.array_equal(g.cpu().numpy(), w), name


@pytest.mark.parametrize("B,longest,P,most_new,pad", [
    (1, 1, 1, 1, 0), (1, 40000, 16, 30000, 3), (64, 1000, 16, 1, 0), (300, 5000, 24, 90, 17), (2500, 60, 1, 5, 0),
    (513, 700, 64, 700, 1), (7, 3, 16, 3, 9)])
def test_matches_the_definition(gpu, B, longest, P, most_new, pad):
    rng = np.random.default_rng(B + P)
    lens = rng.integers(1, longest + 1, B)
    new = rng.integers(0, np.minimum(lens, most_new) + 1)
    W = -(-longest // P) + rng.integers(0, 3)
    table = rng.permutation(B * W + 5)[:B * W].reshape(B, W)
    qo = np.concatenate([[0], np.cumsum(new)])
    nnz = int(qo[-1]) + pad
    err = torch.zeros(1, dtype=torch.int32, device=gpu)
    got = build_tables(i32(table, gpu), i32(lens, gpu), P, i32(qo, gpu), nnz, err=err)
    want, counted = by_hand(table, lens, P, qo, nnz, B * W)
    check(got, want)
    assert counted == 0 and err.item() == 0
    # the lists agree with the calls that derive the same from them
    seq = ap.get_seq_lens(got.kv_indptr, got.kv_last_page_len, P)
    assert torch.equal(seq, i32(lens, gpu))
    if nnz > pad:
        _, pos = ap.get_batch_indices_positions(i32(qo, gpu), seq, int(qo[-1]))
        assert torch.equal(pos, got.positions[:int(qo[-1])])


def test_one_token_each_and_unused_places(gpu):
    lens, table = np.array([5, 0, 16, 17, 0]), np.arange(10).reshape(5, 2)
    err = torch.zeros(1, dtype=torch.int32, device=gpu)
    got = build_tables(i32(table, gpu), i32(lens, gpu), 16, nnz=8, err=err)
    want, counted = by_hand(table, lens, 16, None, 8, 10)
    check(got, want)
    assert counted == 0 and err.item() == 0
    assert got.slot_mapping.tolist() == [4, -1, 4 * 16 + 15, 7 * 16, -1, -1, -1, -1]


def test_what_does_not_fit_is_cut_and_counted(gpu):
    P, table = 4, np.arange(18).reshape(6, 3)
    table[5, 0] = -1
    lens = np.array([13, -2, 12, 1, 3, 4])
    qo = np.array([0, 2, 3, 3, 6, 8, 12])
    for nnz, room in ((12, 18), (12, 5), (7, 18), (14, 0)):
        err = torch.zeros(1, dtype=torch.int32, device=gpu)
        got = build_tables(i32(table, gpu), i32(lens, gpu), P, i32(qo, gpu), nnz, num_indices=room, err=err)
        want, counted = by_hand(table, lens, P, qo, nnz, room)
        check(got, want)
        assert err.item() == counted > 0
    for bad in ([3, 2, 3, 3, 6, 8, 12], [-4, 2, 3, 3, 6, 8, 100], [2, 2, 3, 5, 6, 8, 9]):
        err = torch.zeros(1, dtype=torch.int32, device=gpu)
        got = build_tables(i32(table, gpu), i32(lens, gpu), P, i32(bad, gpu), 12, err=err)
        _, counted = by_hand(table, lens, P, bad, 12, 18)
        assert err.item() == counted


def test_sizes_of_nothing(gpu):
    none = torch.zeros((0, 4), dtype=torch.int32, device=gpu)
    got = build_tables(none, i32([], gpu), 16, i32([0], gpu), 3, num_indices=2)
    assert got.kv_indptr.tolist() == [0] and got.kv_indices.tolist() == [-1, -1] and got.slot_mapping.tolist() == [-1] * 3
    narrow = torch.zeros((3, 0), dtype=torch.int32, device=gpu)
    got = build_tables(narrow, i32([0, 0, 0], gpu), 16)
    assert got.kv_indptr.tolist() == [0] * 4 and got.slot_mapping.tolist() == [-1] * 3


def test_rows_of_a_larger_page_table_and_other_streams(gpu):
    wide = torch.arange(40, dtype=torch.int32, device=gpu).view(4, 10)
    lens = torch.tensor([30, 7, 1], device=gpu)                      # int64 is taken too
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = build_tables(wide[1:, 2:6], lens, 8)
    torch.cuda.current_stream().wait_stream(side)
    want, _ = by_hand(wide[1:, 2:6].cpu().numpy(), [30, 7, 1], 8, None, 3, 12)
    check(got, want)


def test_a_captured_step_follows_the_lengths(gpu):
    P, B, W = 16, 5, 6
    table = np.random.default_rng(0).permutation(B * W).reshape(B, W)
    t, lens = i32(table, gpu), i32([1] * B, gpu)
    out = build_tables(t, lens, P)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        build_tables(t, lens, P, out=out)
    rng = np.random.default_rng(1)
    for _ in range(4):
        now = rng.integers(0, W * P + 1, B)
        lens.copy_(i32(now, gpu))
        graph.replay()
        torch.cuda.synchronize()
        check(out, by_hand(table, now, P, None, B, B * W)[0])
        eager = build_tables(t, lens, P)
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_refusals(gpu):
    t, lens = torch.zeros((2, 3), dtype=torch.int32, device=gpu), i32([1, 1], gpu)
    for bad in (dict(page_table=t.cpu()), dict(page_table=t.long()), dict(page_table=t[0]), dict(page_table=t.t()),
                dict(seq_lens=lens[:1]), dict(page_size=0), dict(append_indptr=i32([0, 1, 2], gpu)),
                dict(append_indptr=i32([0, 2], gpu), nnz=2), dict(nnz=1), dict(num_indices=-1),
                dict(out=build_tables(t[:1], lens[:1], 4))):
        args = dict(page_table=t, seq_lens=lens, page_size=4)
        args.update(bad)
        with pytest.raises(ValueError):
            build_tables(**args)
