"""Pages copied between sequences, accepted drafts moved to the front: what moves is equal bit for bit, the rest untouched."""
import pytest
import torch

import paged_ref as ref
from util import note

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 7, 64, 200])
@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
def test_copy_pages(pkg, dev, n, wide):
    note(f"copy {n} pages of pools of all kinds")
    gen = torch.Generator().manual_seed(n)
    P = 2 * n + 5
    r = lambda *s: torch.randn(P, *s, generator=gen)
    pools = [r(4, 64, 64).bfloat16(), r(5, 64, 128).half(), r(2, 128), r(5), (r(3) * 100).to(torch.uint8),
             (r(7, 3) * 1000).to(torch.int16), r(4097).double(), (r() * 10).to(torch.int8)]
    pools = [p.to(dev) for p in pools]
    order = torch.randperm(P, generator=gen)
    src, dst = order[:n].to(dev, wide), order[n:2 * n].to(dev, wide)
    src[n // 2] = src[0]  # a page may be copied more than once
    want = [p.clone() for p in pools]
    for p in want:
        p[dst.long()] = p[src.long()]
    pkg.copy_pages(pools, src, dst)
    assert all(torch.equal(a, b) for a, b in zip(pools, want))
    # indices out of range and pages onto themselves change nothing
    bad = torch.tensor([-1, P, 0, 3, 2 ** 31 - 1], device=dev).to(wide)
    pkg.copy_pages(pools, bad, torch.tensor([0, 1, P + 7, 3, 2], device=dev).to(wide))
    assert all(torch.equal(a, b) for a, b in zip(pools, want))
    pkg.copy_pages(pools, src[:0], dst[:0])
    pkg.copy_pages(pools[:1], [0, 1], [2, 3])
    assert torch.equal(pools[0][2:4], want[0][:2])


def test_more_than_the_last_cache_holds(pkg, dev):
    note("a move of 330 MB, read and written")
    gen = torch.Generator(device=dev).manual_seed(3)
    P, n = 2603, 1300
    pools = [torch.randint(0, 256, (P, 127008), device=dev, dtype=torch.uint8, generator=gen),
             torch.randn(P, 33, device=dev, generator=gen)]
    order = torch.randperm(P, device=dev, generator=gen)
    src, dst = order[:n], order[n:2 * n]
    want = [p.clone() for p in pools]
    for p in want:
        p[dst] = p[src]
    for _ in range(2):  # (nothing that is written is read: once more changes nothing)
        pkg.copy_pages(pools, src, dst)
        assert all(torch.equal(a, b) for a, b in zip(pools, want))


def test_copy_views(pkg, dev):
    note("a pool that begins between two multiples of 16 bytes")
    whole = torch.randn(1 + 10 * 33, device=dev).bfloat16()
    pool = whole[1:].view(10, 33)
    want = pool.clone()
    want[4] = want[7]
    pkg.copy_pages([pool], [7], [4])
    assert torch.equal(pool, want)


def _path(parents, length, gen):
    """The way from the root to a token of the tree, cut at `length`."""
    t = int(torch.randint(0, len(parents), (1,), generator=gen))
    way = []
    while t >= 0:
        way.append(t)
        t = parents[t]
    return way[::-1][:length]


@pytest.mark.parametrize("H,D", [(1, 64), (8, 128), (3, 64), (4, 256)])
@pytest.mark.parametrize("T,n", [(1, 1), (9, 4), (64, 16), (200, 256)])
def test_accept(pkg, dev, H, D, T, n):
    note(f"accept {n} of {T}, {H} heads of {D}")
    B, pages = 6, 6
    gen = torch.Generator().manual_seed(T)
    k, v, table = ref.cache(gen, B, pages, H, D, dev)
    base = [0, 3, 63, 64, 120, pages * 64 - T]
    wide = 0.05 if T == 200 else 1.0
    ways = [_path(ref.tree(gen, T, wide), n, gen) for _ in range(B)]
    path = torch.full((B, n), -1, dtype=torch.int32)
    for b, w in enumerate(ways):
        path[b, : len(w)] = torch.tensor(w)
    path[1] = -1  # nothing accepted
    want_k, want_v = k.clone(), v.clone()
    for b in range(B):
        for i, x in enumerate(ways[b] if b != 1 else []):
            to, fr = base[b] + i, base[b] + x
            for pool, old in ((want_k, k), (want_v, v)):
                pool[table[b, to // 64].long(), :, to % 64] = old[table[b, fr // 64].long(), :, fr % 64]
    pkg.paged_accept(k, v, table, torch.tensor(base, dtype=torch.int32, device=dev), path.to(dev))
    assert torch.equal(k, want_k) and torch.equal(v, want_v)


def test_accept_odd_paths(pkg, dev):
    note("paths that stop growing, leave the table or cross pages that are not mapped; an int base")
    gen = torch.Generator().manual_seed(2)
    k, v, table = ref.cache(gen, 5, 3, 2, 64, dev)
    table[3, 1] = -1
    path = torch.tensor([[1, 3, 3, 7], [2, 1, 5, 6], [0, 2, 300, 400], [0, 1, 30, 70], [5, 2 ** 31 - 1, 6, 7]], dtype=torch.int32)
    moves = [{0: 1, 1: 3}, {0: 2}, {1: 2}, {3: 70}, {0: 5}]
    base = 60
    want_k, want_v = k.clone(), v.clone()
    for b, m in enumerate(moves):
        for to, fr in m.items():
            a, c = base + to, base + fr
            for pool, old in ((want_k, k), (want_v, v)):
                pool[table[b, a // 64].long(), :, a % 64] = old[table[b, c // 64].long(), :, c % 64]
    pkg.paged_accept(k, v, table, base, path.to(dev))
    assert torch.equal(k, want_k) and torch.equal(v, want_v)
    pkg.paged_accept(k, v, table, base, path[:, :0].to(dev))
    neg = torch.full((5,), -3, dtype=torch.int32, device=dev)
    pkg.paged_accept(k, v, table, neg, path.to(dev))
    assert torch.equal(k, want_k) and torch.equal(v, want_v)


def test_moves_replay(pkg, dev):
    note("copies and acceptance captured")
    gen = torch.Generator().manual_seed(4)
    k, v, table = ref.cache(gen, 1, 4, 2, 64, dev)
    path = torch.tensor([[1, 4, 5]], dtype=torch.int32, device=dev)
    base = torch.tensor([10], dtype=torch.int32, device=dev)
    src, dst = table[0, 1:2].clone(), table[0, 3:4].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pkg.paged_accept(k, v, table, base, path)
        pkg.copy_pages([k, v], src, dst)
    for i in range(3):
        base.add_(40)
        k1, v1 = k.clone(), v.clone()
        graph.replay()
        pkg.paged_accept(k1, v1, table, base, path)
        pkg.copy_pages([k1, v1], src, dst)
        torch.cuda.synchronize()
        assert torch.equal(k, k1) and torch.equal(v, v1)
