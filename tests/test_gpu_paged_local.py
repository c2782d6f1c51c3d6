"""Local branch straight on the pages, for single tokens, chains and trees of drafted tokens, against the 64-bit form."""
import math

import pytest
import torch

import paged_ref as ref
from util import note

pytestmark = pytest.mark.gpu


def _run(pkg, dev, B, T, max_pages, heads, lengths, window, parents=None, seed=0, mask_lmk=True, expand=True, scale=None):
    HQ, H, D = heads
    gen = torch.Generator().manual_seed(seed)
    k, v, table = ref.cache(gen, B, max_pages, H, D, dev)
    q = torch.randn(B, T, HQ, D, generator=gen).bfloat16().to(dev)
    ln = lengths if isinstance(lengths, int) else torch.tensor(lengths, dtype=torch.int32, device=dev)
    got = pkg.paged_flex_attn(q, k, v, table, ln, window, parents=None if parents is None else parents.to(dev),
                              mask_lmk=mask_lmk, expand_to_chunk=expand, sm_scale=scale)
    torch.cuda.synchronize()
    ref.check_attention(got, ref.attend(q, k, v, table, ln, window, parents, mask_lmk, expand, scale))


HEADS = [(4, 4, 64), (16, 2, 64), (32, 8, 128), (5, 1, 128), (16, 1, 128), (6, 2, 64)]


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("T,lengths,window", [
    (1, [1, 64, 65, 577, 640], 64), (1, [63, 128, 129, 500, 640], 512), (1, [1, 2, 3, 639, 640], 1 << 30),
    (2, [2, 64, 66, 639, 640], 1), (7, [7, 64, 70, 130, 640], 100), (40, [40, 64, 104, 600, 640], 200),
    (130, [130, 200, 320, 511, 640], 512)])
def test_chain(pkg, dev, heads, T, lengths, window):
    note(f"chain T{T} window {window} heads {heads}")
    _run(pkg, dev, 5, T, 10, heads, lengths, window, seed=T + window % 1000)


@pytest.mark.parametrize("mask_lmk,expand", [(False, True), (True, False), (False, False)])
@pytest.mark.parametrize("T", [1, 5, 70])
def test_mask_options(pkg, dev, mask_lmk, expand, T):
    note(f"chain T{T} mask_lmk {mask_lmk} expand {expand}")
    for window in (1, 63, 64, 65, 300):
        _run(pkg, dev, 3, T, 8, (8, 2, 64), [T, 256, 509], window, seed=window, mask_lmk=mask_lmk, expand=expand, scale=0.3)


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("T,wide", [(1, 1.0), (2, 1.0), (13, 0.3), (33, 1.0), (64, 0.5), (100, 0.05), (256, 0.1)])
@pytest.mark.parametrize("window", [1, 64, 512])
def test_tree(pkg, dev, heads, T, wide, window):
    note(f"tree of {T} window {window} heads {heads}")
    gen = torch.Generator().manual_seed(T)
    lengths = [T, T + 1, max(T, 128), T + 191, 640]
    parents = torch.tensor([ref.tree(gen, T, wide) for _ in lengths], dtype=torch.int32)
    _run(pkg, dev, 5, T, 10, heads, lengths, window, parents, seed=T)


def test_chain_as_a_tree(pkg, dev):
    note("a chain given as a tree, shared by the batch")
    for T in (1, 16, 65, 200):
        parents = torch.arange(-1, T - 1, dtype=torch.int32)
        for window in (8, 64, 512):
            for mask_lmk in (True, False):
                _run(pkg, dev, 3, T, 8, (8, 2, 128), [T, 300, 509], window, parents, seed=T, mask_lmk=mask_lmk,
                     expand=window != 8)


def test_padding_and_wrong_parents(pkg, dev):
    """A token whose parent is no earlier token, and what follows it, sees nothing; the others are as they are without it."""
    note("padded trees")
    parents = torch.tensor([[-1, 0, 0, 1, 3, -2, -2, -2], [-1, 0, 2, 9, 3, 1, 4, 2 ** 31 - 1], [-5, 0, 1, -1, 3, 3, 6, 5],
                            [-1, 0, 1, 2, 3, 4, 5, 6]], dtype=torch.int32)
    _run(pkg, dev, 4, 8, 6, (8, 2, 64), [8, 200, 300, 384], 100, parents)
    _run(pkg, dev, 4, 8, 6, (32, 2, 128), [8, 200, 300, 384], 100, parents)


def test_sequences_that_take_no_part(pkg, dev):
    note("lengths below T, zero, negative, past the table")
    for T, parents in ((3, None), (3, torch.tensor([-1, 0, 0], dtype=torch.int32)), (90, None)):
        _run(pkg, dev, 6, T, 4, (8, 2, 64), [0, 2, -7, T, 256, 200], 64, parents)
    # a length that the table does not reach: what lies past it is not mapped
    _run(pkg, dev, 2, 3, 4, (8, 2, 64), [258, 300], 128)


@pytest.mark.parametrize("T,tree", [(1, False), (20, False), (24, True), (90, True), (90, False)])
def test_unmapped_pages(pkg, dev, T, tree):
    note(f"pages that are not mapped, T{T}")
    B, n, HQ, H, D = 3, 8, 8, 2, 128
    gen = torch.Generator().manual_seed(5)
    k, v, table = ref.cache(gen, B, n, H, D, dev)
    table[0, 5] = -1
    table[1, 6:] = 10 ** 6
    table[2] = -1
    q = torch.randn(B, T, HQ, D, generator=gen).bfloat16().to(dev)
    parents = torch.tensor(ref.tree(gen, T), dtype=torch.int32) if tree else None
    got = pkg.paged_flex_attn(q, k, v, table, 490, 300, parents=None if parents is None else parents.to(dev))
    ref.check_attention(got, ref.attend(q, k, v, table, 490, 300, parents))
    assert (got[0][2] == 0).all()


@pytest.mark.parametrize("heads", [(8, 2, 64), (8, 2, 128)])
@pytest.mark.parametrize("T,tree", [(1, False), (6, False), (20, True), (90, True), (90, False)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_is_not_seen_does_not_matter(pkg, dev, heads, T, tree, bad):
    """No number in stale slots, before the window, at landmarks and in other branches' drafts reaches a row."""
    note(f"{bad} in masked places, T{T} heads {heads}")
    HQ, H, D = heads
    B, n, window = 2, 8, 100
    gen = torch.Generator().manual_seed(6)
    k, v, table = ref.cache(gen, B, n, H, D, dev)
    q = torch.randn(B, T, HQ, D, generator=gen).bfloat16().to(dev)
    parents = torch.tensor(ref.tree(gen, T), dtype=torch.int32) if tree else None
    lengths = torch.tensor([T + 70, 437], dtype=torch.int32, device=dev)
    for b in range(B):
        see = ref.visible(T, int(lengths[b]), window, None if parents is None else parents.tolist(), True, True, n * 64)
        hide = ~see.any(0)
        if tree:  # the last token's own slot: nobody else sees it, and its row is not looked at
            hide[int(lengths[b]) - 1] = True
        for s in hide.nonzero().flatten().tolist():
            k[table[b, s // 64].long(), :, s % 64] = bad
            v[table[b, s // 64].long(), :, s % 64] = bad
    o, lse = pkg.paged_flex_attn(q, k, v, table, lengths, window, parents=None if parents is None else parents.to(dev))
    want = ref.attend(q, k, v, table, lengths, window, parents)
    keep = T - 1 if tree else T
    ref.check_attention((o[:, :keep], lse[:, :keep]), tuple(x[:, :keep] for x in want))
    if tree:
        assert not torch.isfinite(o[:, -1]).any()


def test_numbers_that_are_none_show(pkg, dev):
    note("NaN in seen places")
    gen = torch.Generator().manual_seed(7)
    for T in (1, 3, 90):
        k, v, table = ref.cache(gen, 1, 4, 2, 64, dev)
        q = torch.randn(1, T, 8, 64, generator=gen).bfloat16().to(dev)
        v2 = v.clone()
        v2[table[0, 3].long(), 1, 5, 9] = float("nan")
        o, _ = pkg.paged_flex_attn(q, k, v2, table, 250, 128, mask_lmk=False)
        see = ref.visible(T, 250, 128, None, False, True, 256)[:, 3 * 64 + 5]
        assert o[0, see, 4:, 9].isnan().all() and not o[0, :, :4].isnan().any() and not o[..., 10:].isnan().any()
        q2 = q.clone()
        q2[0, T - 1, 3, 0] = float("nan")
        o, lse = pkg.paged_flex_attn(q2, k, v, table, 250, 128)
        o0, lse0 = pkg.paged_flex_attn(q, k, v, table, 250, 128)
        assert o[0, T - 1, 3].isnan().all() and lse[0, T - 1, 3].isnan()
        o[0, T - 1, 3], lse[0, T - 1, 3] = o0[0, T - 1, 3], lse0[0, T - 1, 3]
        assert torch.equal(o, o0) and torch.equal(lse, lse0)


@pytest.mark.parametrize("T,heads,pages", [(1, (16, 2, 64), 300), (1, (32, 8, 128), 129), (3, (8, 2, 128), 200),
                                           (20, (8, 2, 128), 150), (70, (4, 1, 128), 140), (64, (16, 2, 64), 130)])
@pytest.mark.parametrize("tree", [False, True])
def test_long_context_split(pkg, dev, T, heads, pages, tree):
    note(f"a long context over several workgroups, T{T} heads {heads}")
    gen = torch.Generator().manual_seed(8)
    parents = torch.tensor([ref.tree(gen, T) for _ in range(2)], dtype=torch.int32) if tree else None
    _run(pkg, dev, 2, T, pages, heads, [pages * 64 - 37, T + 3], 1 << 20, parents, mask_lmk=tree)


def test_matches_the_contiguous_local_branch(pkg, dev):
    note("paged against flex_attn_tl")
    gen = torch.Generator().manual_seed(9)
    for T, n in ((1, 600), (64, 600), (300, 640)):
        k, v, table = ref.cache(gen, 2, 10, 2, 128, dev)
        q = torch.randn(2, T, 8, 128, generator=gen).bfloat16().to(dev)
        flat = lambda x: x[table.long()].permute(0, 1, 3, 2, 4).reshape(2, 640, 2, 128)[:, :n].contiguous()
        o0, lse0 = pkg.flex_attn_tl(q, flat(k), flat(v), 100, 64, training=False)
        o1, lse1 = pkg.paged_flex_attn(q, k, v, table, n, 100)
        # both round alike (o <= 4: two steps of the probabilities' and the outputs' rounding)
        assert (o0.float() - o1.float()).abs().max() <= 4 * 2 * 2 ** -7 and (lse0 - lse1).abs().max() <= 1e-4


def test_offsets_past_32_bits(pkg, dev):
    """Pages past 2^31 elements (and bytes) of a pool."""
    note("a pool of more than 4 GiB")
    H, D, pages = 8, 128, 36000  # 64 Ki elements a page
    gen = torch.Generator().manual_seed(10)
    k = torch.zeros(pages, H, 64, D, dtype=torch.bfloat16, device=dev)
    v = torch.zeros_like(k)
    used = [35999, 5, 34000, 33333]
    for p in used:
        k[p] = torch.randn(H, 64, D, generator=gen).bfloat16()
        v[p] = torch.randn(H, 64, D, generator=gen).bfloat16()
    table = torch.tensor([used], dtype=torch.int32, device=dev)
    small_k, small_v, small_t = k[used], v[used], torch.arange(4, dtype=torch.int32, device=dev).view(1, 4)
    for T in (1, 12, 80):
        q = torch.randn(1, T, 16, D, generator=gen).bfloat16().to(dev)
        a = pkg.paged_flex_attn(q, k, v, table, 251, 512)
        b = pkg.paged_flex_attn(q, small_k, small_v, small_t, 251, 512)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and a[0].abs().max() > 0


def test_strided_queries_and_streams(pkg, dev):
    note("views of a fused projection, a stream of its own, replays of a graph")
    gen = torch.Generator().manual_seed(11)
    B, T, HQ, H, D = 3, 5, 8, 2, 128
    k, v, table = ref.cache(gen, B, 40, H, D, dev)
    qkv = torch.randn(B, T, HQ + 2 * H, D, generator=gen).bfloat16().to(dev)
    q = qkv[:, :, :HQ]
    lengths = torch.tensor([2500, 5, 1111], dtype=torch.int32, device=dev)
    parents = torch.tensor(ref.tree(gen, T), dtype=torch.int32, device=dev)
    call = lambda x: pkg.paged_flex_attn(x, k, v, table, lengths, 4096, parents=parents)
    o0, lse0 = call(q.contiguous())
    for x in (q, q.transpose(0, 1).contiguous().transpose(0, 1), q.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2)):
        o, lse = call(x)
        assert torch.equal(o, o0) and torch.equal(lse, lse0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o, lse = call(q)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(o, o0) and torch.equal(lse, lse0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lse = call(q)
    for i in range(3):  # other lengths, parents and queries of the same shapes, between eager calls
        lengths.copy_(torch.tensor([2500 - 700 * i, 5 + i, 1111 + i], dtype=torch.int32))
        qkv.mul_(-1)
        graph.replay()
        o1, lse1 = call(q)
        torch.cuda.synchronize()
        assert torch.equal(o, o1) and torch.equal(lse, lse1)


def test_empty_calls(pkg, dev):
    k, v, table = ref.cache(torch.Generator().manual_seed(1), 2, 2, 2, 64, dev)
    o, lse = pkg.paged_flex_attn(torch.zeros(2, 0, 4, 64, dtype=torch.bfloat16, device=dev), k, v, table, 10, 64)
    assert o.shape == (2, 0, 4, 64) and lse.shape == (2, 0, 4)


def test_inference_only(pkg, dev):
    k, v, table = ref.cache(torch.Generator().manual_seed(1), 1, 2, 2, 64, dev)
    q = torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16, device=dev, requires_grad=True)
    o, lse = pkg.paged_flex_attn(q, k, v, table, 10, 64)
    with pytest.raises(RuntimeError, match="inference operator"):
        o.float().sum().backward()
