"""Pages copied between places of a cache (attn/cache.py copy_pages, umb_pages_copy) against plain indexing."""
import pytest
import torch

from umbrella_amd import _lib
from umbrella_amd.attn.cache import copy_pages

EINVAL, AT = -22, 1 << 20


def store(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    n = torch.tensor([], dtype=dtype).element_size()
    return torch.randint(0, 256, (*shape[:-1], shape[-1] * n), generator=g, dtype=torch.uint8)


def rows_of(pools):
    """the descriptors of byte stores [pages, groups, rows, row] with their tokens a row"""
    return torch.tensor([[t.data_ptr(), t[0].numel(), t.shape[1], t.shape[2], t.shape[3], per] for t, per in pools], dtype=torch.int64).reshape(-1, 6)


def plain(t, per, moves):
    t = t.clone()
    for src, dst, tokens in moves:
        if 0 <= src < t.shape[0] and 0 <= dst < t.shape[0] and src != dst and tokens > 0:
            n = t.shape[2] if per == 0 else min(t.shape[2], -(-tokens // per))
            t[dst, :, :n] = t[src, :, :n]
    return t


def check(shapes, moves, table=None, where=None, n_pages=None):
    """shapes: [(pages, groups, rows, row, dtype, per)]"""
    hosts = [(store(s[:4], s[4], i), s[5]) for i, s in enumerate(shapes)]
    devs = [(t.cuda(), per) for t, per in hosts]
    mv = torch.tensor(moves, dtype=torch.int32).reshape(-1, 3).cuda()
    tab = None if table is None else table.cuda()
    copy_pages(rows_of(devs), mv, n_pages or hosts[0][0].shape[0], table=tab, where=None if where is None else where.cuda())
    for (h, per), (d, _) in zip(hosts, devs):
        assert torch.equal(d.cpu(), plain(h, per, moves))
    return None if tab is None else tab.cpu()


MOVES = [(0, 5, 1), (0, 6, 7), (3, 1, 16), (2, 9, 3), (4, 8, 1000), (3, 7, 15)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.uint8])
@pytest.mark.parametrize("groups,rows,row", [(1, 16, 8), (2, 16, 24), (3, 16, 25), (8, 16, 128), (1, 16, 576), (2, 16, 1), (5, 7, 33)])
def test_rows_of_every_size(dtype, groups, rows, row):
    check([(10, groups, rows, row, dtype, 1), (10, groups, -(-rows // 3), row, torch.float32, 3), (10, 1, 1, 4 * row + 4, torch.float32, 0)], MOVES)


@pytest.mark.gpu
@pytest.mark.parametrize("pools", [1, 47, 48, 49, 100])
def test_many_pools(pools):
    check([(10, 2, 16, 40, torch.bfloat16, 1 + i % 3) for i in range(pools)], MOVES)


@pytest.mark.gpu
def test_pages_of_many_pieces():
    check([(6, 8, 64, 256, torch.float32, 1), (6, 1, 1, 300001, torch.uint8, 0)], [(0, 3, 64), (1, 4, 63), (5, 2, 1)])


@pytest.mark.gpu
@pytest.mark.parametrize("groups,rows,row,per", [(1 << 23, 2, 1, 1), (1 << 21, 3, 2, 1), (3000001, 3, 1, 1), ((1 << 22) - 1, 2, 1, 1), (70001, 50, 4, 7)])
def test_pages_of_very_many_groups(groups, rows, row, per):
    """a row a group: more groups than a fraction of 24 bits tells apart"""
    check([(4, groups, rows, row, torch.uint8, per)], [(0, 2, 1), (3, 1, rows * per - 1)])


@pytest.mark.gpu
def test_many_moves():
    """more than a grid's rows"""
    n = 70000
    moves = [(i, n + i, 1 + i % 2) for i in range(n)]
    check([(2 * n, 1, 2, 8, torch.uint8, 1)], moves)


@pytest.mark.gpu
def test_moves_that_do_nothing():
    """pages that are not there, a page to itself, no tokens; no moves at all"""
    check([(10, 2, 16, 24, torch.bfloat16, 1)], [(-1, 3, 16), (3, -1, 16), (10, 2, 16), (2, 10, 16), (4, 4, 16), (5, 6, 0), (5, 7, -3), (1 << 30, 1, 16), (8, 9, 2)])
    check([(10, 2, 16, 24, torch.bfloat16, 1)], [])
    # a cache whose pages beyond n_pages are another's
    check([(8, 2, 16, 24, torch.bfloat16, 1)], [(0, 5, 16)], n_pages=8)


@pytest.mark.gpu
@pytest.mark.parametrize("moves", [[], MOVES])
def test_the_table_beside_them(moves):
    where = torch.randperm(10, generator=torch.Generator().manual_seed(1)).to(torch.int32)
    table = torch.randint(-2, 13, (37, 1001), generator=torch.Generator().manual_seed(2), dtype=torch.int32)
    got = check([(10, 2, 16, 24, torch.bfloat16, 1)], moves, table, where)
    at = (table >= 0) & (table < 10)
    assert torch.equal(got, torch.where(at, where[table.clamp(0, 9).long()], table))
    copy = table.cuda()
    copy_pages(torch.zeros(0, 6, dtype=torch.int64), torch.zeros(0, 3, dtype=torch.int32, device="cuda:0"), 10, table=copy, where=where.cuda())
    assert torch.equal(copy.cpu(), got)


@pytest.mark.gpu
def test_a_table_shorter_than_the_moves():
    where = torch.randperm(400, generator=torch.Generator().manual_seed(1)).to(torch.int32)
    table = torch.tensor([3, 399, -1, 0, 17], dtype=torch.int32)
    got = check([(400, 1, 4, 8, torch.uint8, 1)], [(i, 200 + i, 4) for i in range(200)], table, where)
    assert got.tolist() == [int(where[p]) if p >= 0 else -1 for p in table.tolist()]


@pytest.mark.gpu
def test_a_store_beyond_32_bits():
    """6 GiB: pages behind 2^32 bytes"""
    pages, page = 6144, 1 << 20
    t = torch.zeros(pages, 1, 1024, 1024, dtype=torch.uint8, device="cuda:0")
    g = torch.Generator().manual_seed(1)
    first, last = (torch.randint(0, 256, (1, 1024, 1024), generator=g, dtype=torch.uint8) for _ in range(2))
    t[1], t[pages - 1] = first.cuda(), last.cuda()
    copy_pages(rows_of([(t, 1)]), torch.tensor([[1, pages - 2, 1024], [pages - 1, 0, 1000]], dtype=torch.int32).cuda(), pages)
    assert torch.equal(t[pages - 2].cpu(), first) and torch.equal(t[0, :, :1000].cpu(), last[:, :1000]) and not t[0, :, 1000:].any() and not t[2:pages - 2].any()
    assert t[0].numel() == page


@pytest.mark.gpu
def test_captured_and_replayed():
    host = store((10, 2, 16, 24), torch.bfloat16, 3)
    dev, moves = host.cuda(), torch.zeros(2, 3, dtype=torch.int32, device="cuda:0")
    pools = rows_of([(dev, 1)])
    copy_pages(pools, moves, 10)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with _lib.capturing(graph):
        copy_pages(pools, moves, 10)
    for mv in ([(0, 5, 4), (1, 6, 16)], [(5, 2, 16), (6, 3, 9)], [(2, 9, 1), (2, 8, 16)]):
        moves.copy_(torch.tensor(mv, dtype=torch.int32))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        host = plain(host, 1, mv)
        assert torch.equal(dev.cpu(), host)


def test_refusals_of_the_wrapper():
    pools, moves = torch.zeros(1, 6, dtype=torch.int64), torch.zeros(1, 3, dtype=torch.int32)
    for a, b in ((pools, moves), (pools.int(), moves), (pools[:, :5], moves), (pools[0], moves)):
        with pytest.raises(ValueError):
            copy_pages(a, b, 4)


def test_refusals_of_the_entry_point():
    lib, pool = _lib.load_seq(), [AT, 4096, 2, 16, 64, 1]

    def call(pool=pool, n_pools=1, moves=AT, n_moves=1, n_pages=8, table=None, n_table=0, where=None):
        t = torch.tensor([pool], dtype=torch.int64)
        return lib.umb_pages_copy(t.data_ptr() if n_pools else None, n_pools, moves, n_moves, n_pages, table, n_table, where, None)
    bad = [dict(n_pools=-1), dict(moves=None), dict(n_moves=-1), dict(n_pages=0), dict(n_table=4), dict(n_table=4, table=AT), dict(n_table=-1, table=AT, where=AT)]
    for i, v in ((0, 0), (1, 2047), (1, 0), (2, 0), (2, 5), (3, 0), (3, 1 << 40), (4, 0), (4, 1 << 60), (5, -1)):
        bad.append(dict(pool=pool[:i] + [v] + pool[i + 1:]))
    for kw in bad:
        assert call(**kw) == EINVAL, kw
    assert call(n_pools=0, n_moves=0) == 0 and call(n_moves=0) == 0           # nothing to do: nothing is launched
