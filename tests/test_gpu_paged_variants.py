"""The attention on the pages at sizes that each of its kernels, block heights and share counts serve: few and many rows,
shares of one page and of more than 64, up to 64 shares a range.  Against the 64-bit form."""
import pytest
import torch

import paged_ref as ref
from util import note

pytestmark = pytest.mark.gpu

# query heads, KV heads, sequences, new tokens, window, longest context
CASES = [(32, 8, 2, 64, 512, 1024), (32, 8, 8, 33, 1 << 20, 900), (32, 8, 8, 64, 512, 1024), (32, 8, 5, 100, 1 << 20, 900),
         (32, 8, 5, 200, 1 << 20, 900), (32, 8, 8, 256, 512, 900), (16, 1, 16, 33, 1 << 20, 900), (16, 1, 8, 256, 300, 900),
         (4, 4, 5, 200, 1 << 20, 900), (6, 2, 5, 100, 1 << 20, 4500), (32, 8, 3, 33, 1 << 20, 4500), (5, 1, 16, 33, 1 << 20, 4500),
         (32, 8, 1, 33, 1 << 20, 18000), (32, 8, 2, 33, 1 << 20, 9000), (4, 4, 1, 33, 1 << 20, 18000), (6, 2, 2, 33, 1 << 20, 18000),
         (5, 1, 2, 33, 1 << 20, 18000), (4, 4, 16, 33, 1 << 20, 18000), (32, 8, 16, 7, 1 << 20, 4500), (32, 8, 8, 7, 1 << 20, 18000),
         (4, 4, 16, 1, 1 << 20, 18000), (5, 1, 1, 1, 1 << 20, 18000), (32, 8, 16, 40, 1 << 20, 9000), (32, 8, 16, 4, 1 << 20, 9000),
         (32, 8, 1, 256, 512, 1024), (6, 2, 3, 7, 1 << 20, 18000), (4, 4, 5, 20, 1 << 20, 18000), (6, 2, 3, 33, 1 << 20, 18000),
         (32, 8, 1, 100, 1 << 20, 4500), (32, 8, 2, 33, 1 << 20, 18000)]


def _inputs(dev, D, HQ, H, B, T, ctx, tree, seed):
    gen = torch.Generator().manual_seed(seed)
    n = -(-ctx // 64)
    k, v, table = ref.cache(gen, B, n, H, D, dev)
    q = torch.randn(B, T, HQ, D, generator=gen).bfloat16().to(dev)
    # one full, one that starts here, one that ends on a page's edge, one that takes no part, the rest anywhere
    lengths = ([ctx, T, max(T, ctx // 2 // 64 * 64), T - 1] + torch.randint(T, ctx + 1, (B,), generator=gen).tolist())[:B]
    parents = torch.tensor([ref.tree(gen, T, 0.3) for _ in range(B)], dtype=torch.int32) if tree else None
    return q, k, v, table, torch.tensor(lengths, dtype=torch.int32, device=dev), parents


def _call(pkg, q, k, v, table, lengths, window, parents, **kw):
    return pkg.paged_flex_attn(q, k, v, table, lengths, window, parents=None if parents is None else parents.to(q.device), **kw)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_sizes(pkg, dev, case, tree, D):
    HQ, H, B, T, window, ctx = case
    note(f"paged attention {case} D{D} tree {tree}")
    q, k, v, table, lengths, parents = _inputs(dev, D, HQ, H, B, T, ctx, tree, seed=T + ctx)
    got = _call(pkg, q, k, v, table, lengths, window, parents)
    again = _call(pkg, q, k, v, table, lengths, window, parents)
    assert all(torch.equal(x, y) for x, y in zip(got, again))  # (no order of sums depends on what ends first)
    for b in range(B):
        want = ref.attend_dense(q[b:b + 1], k, v, table[b:b + 1], lengths[b:b + 1], window, None if parents is None else parents[b:b + 1])
        ref.check_attention(tuple(x[b:b + 1] for x in got), want)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("case", [(8, 2, 2, 1000, 200, 2100), (6, 1, 1, 3001, 1 << 20, 3001), (32, 8, 3, 513, 512, 4500),
                                  (4, 4, 2, 700, 1 << 20, 9000)], ids=str)
def test_slices_of_a_prompt(pkg, dev, case, D):
    HQ, H, B, T, window, ctx = case
    note(f"paged attention of many tokens {case} D{D}")
    q, k, v, table, lengths, _ = _inputs(dev, D, HQ, H, B, T, ctx, False, seed=T)
    got = _call(pkg, q, k, v, table, lengths, window, None)
    for b in range(B):
        want = ref.attend_dense(q[b:b + 1], k, v, table[b:b + 1], lengths[b:b + 1], window)
        ref.check_attention(tuple(x[b:b + 1] for x in got), want)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("case", [(32, 8, 8, 64, 130, 1024), (32, 8, 5, 200, 1 << 20, 900), (16, 1, 16, 33, 1 << 20, 900),
                                  (4, 4, 1, 33, 1 << 20, 18000), (32, 8, 2, 33, 1 << 20, 9000), (4, 4, 16, 33, 1 << 20, 4500)], ids=str)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_stale_numbers(pkg, dev, case, tree, D, bad):
    """Numbers in slots that no row sees do not reach one, and what one row alone sees stays with it."""
    HQ, H, B, T, window, ctx = case
    note(f"stale {bad}, paged attention {case} D{D} tree {tree}")
    q, k, v, table, lengths, parents = _inputs(dev, D, HQ, H, B, T, ctx, tree, seed=T)
    spoilt, wants = 0, []
    for b in range(B):
        wants.append(ref.attend_dense(q[b:b + 1], k, v, table[b:b + 1], lengths[b:b + 1], window, None if parents is None else parents[b:b + 1]))
    for b in range(B):
        see = ref.visible(T, int(lengths[b]), window, None if parents is None else parents[b].tolist(), True, True, table.shape[1] * 64)
        hide = ~see.any(0)
        if tree and int(lengths[b]) >= T:  # the last token's own slot, which only its row sees
            hide[int(lengths[b]) - 1] = True
        at = hide.nonzero().flatten().to(dev)
        k[table[b, at // 64].long(), :, at % 64] = bad
        v[table[b, at // 64].long(), :, at % 64] = bad
        spoilt += at.numel()
    assert spoilt > B
    o, lse = _call(pkg, q, k, v, table, lengths, window, parents)
    keep = T - 1 if tree else T
    for b, want in enumerate(wants):
        ref.check_attention((o[b:b + 1, :keep], lse[b:b + 1, :keep]), tuple(x[:, :keep] for x in want))


def test_a_sequence_apart(pkg, dev):
    """Lengths from none to all of the table in one batch, whose shares the sequences divide by their lengths."""
    note("very uneven lengths")
    for HQ, H, B, T, D, lens in ((32, 8, 3, 33, 128, [9000, 33, 40]), (16, 2, 64, 1, 64, [9000] + [0, 1, 64, 65, 130, 500, 7] * 9),
                                 (8, 2, 65, 2, 64, [9000] + [2, 64, 3, 900] * 16), (4, 1, 2, 1, 128, [0, 0]),
                                 (32, 4, 5, 64, 128, [70, 9000, 64, 8999, 4000]), (4, 1, 40, 3, 128, [9000] * 2 + [3] * 38)):
        gen = torch.Generator().manual_seed(B)
        k, v, table = ref.cache(gen, B, 141, H, D, dev)
        q = torch.randn(B, T, HQ, D, generator=gen).bfloat16().to(dev)
        lengths = torch.tensor(lens, dtype=torch.int32, device=dev)
        got = _call(pkg, q, k, v, table, lengths, 1 << 20, None)
        ref.check_attention(got, ref.attend_dense(q, k, v, table, lengths, 1 << 20))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("case", [(32, 8, 8, 64, 512, 1024), (4, 4, 1, 33, 1 << 20, 18000), (32, 8, 3, 40, 1 << 20, 4500)], ids=str)
def test_scores_far_from_the_first_page(pkg, dev, case, D):
    """Rows whose largest score lies far above and far below what their first keys give, by more than 32 bits' range of exp."""
    HQ, H, B, T, window, ctx = case
    note(f"steep scores, paged attention {case} D{D}")
    # scores before scaling reach 12 * 200, where half a step of fp32 is 2^-13; 128 sums of such, scaled by 128^-0.5, are off by at
    # most 1.4e-3, and the scaled score by 2^-23 * 300 more: lse by 2e-3, a probability (its score and lse) by 4e-3 of itself
    for seed, steep in ((1, 200.0), (2, -200.0), (3, 0.0)):
        q, k, v, table, lengths, _ = _inputs(dev, D, HQ, H, B, T, ctx, False, seed)
        ramp = torch.linspace(-1, 1, table.shape[1], device=dev)
        if steep == 0.0:  # one far key, anywhere
            ramp = torch.zeros_like(ramp)
            ramp[table.shape[1] // 3] = 1.0
            steep = 200.0
        for b in range(B):
            k[table[b].long(), :, :, 0] = (ramp * steep)[:, None, None].bfloat16()
        q[..., 0] = 8 + q[..., 0].abs().clamp(max=4)
        got = _call(pkg, q, k, v, table, lengths, window, None)
        ref.check_attention(got, ref.attend_dense(q, k, v, table, lengths, window), lse_tol=2e-3, slack=4e-3)


def test_captured_and_replayed(pkg, dev):
    """Two captured calls whose shares meet in workspaces, and eager ones between the replays."""
    note("captured paged attention")
    a = _inputs(dev, 128, 32, 8, 2, 1, 9000, False, 1)
    b = _inputs(dev, 64, 16, 2, 3, 33, 4500, True, 2)
    first = [_call(pkg, *a[:5], 1 << 20, a[5]), _call(pkg, *b[:5], 1 << 20, b[5])]
    parents = b[5].to(dev)
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x, par in ((a, None), (b, parents)):
            pkg.paged_flex_attn(*x[:5], 1 << 20, parents=par)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                outs.append(pkg.paged_flex_attn(*x[:5], 1 << 20, parents=par))
            graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(4):
        for g in graphs:
            g.replay()
        eager = [_call(pkg, *a[:5], 1 << 20, a[5]), _call(pkg, *b[:5], 1 << 20, b[5])]
        torch.cuda.synchronize()
        for want, got, more in zip(first, outs, eager):
            for w, x, y in zip(want, got, more):
                assert torch.equal(w, x) and torch.equal(w, y)
                x.zero_()
        torch.cuda.synchronize()


@pytest.mark.parametrize("HQ,H,D", [(8, 2, 128), (16, 2, 64), (4, 1, 128)])
@pytest.mark.parametrize("T,tree", [(1, False), (6, True), (70, True)])
def test_stale_numbers_in_some_features(pkg, dev, HQ, H, D, T, tree):
    """A NaN in one feature of a hidden value: what computes the other features of the row does not see it."""
    note(f"stale numbers in some features, T{T} heads {HQ}/{H} x {D}")
    for feature, ctx, window in ((0, 700, 200), (D - 1, 700, 1 << 20), (D // 2, 5000, 1 << 20)):
        q, k, v, table, lengths, parents = _inputs(dev, D, HQ, H, 2, T, ctx, tree, seed=T + feature)
        lengths[1] = ctx - 70
        want = ref.attend_dense(q, k, v, table, lengths, window, parents)
        for b in range(2):
            see = ref.visible(T, int(lengths[b]), window, None if parents is None else parents[b].tolist(), True, True, table.shape[1] * 64)
            at = (~see.any(0)).nonzero().flatten().to(dev)
            v[table[b, at // 64].long(), :, at % 64, feature] = float("nan")
        got = _call(pkg, q, k, v, table, lengths, window, parents)
        ref.check_attention(got, want)
        again = _call(pkg, q, k, v, table, lengths, window, parents)
        assert all(torch.equal(x, y) for x, y in zip(got, again))


def test_a_captured_step_over_growing_sequences(pkg, dev):
    """Append and attend of a ragged batch in a graph whose lengths grow on the GPU, replay by replay, against eager calls."""
    note("a captured step, lengths growing")
    for HQ, H, D, lens, window in ((16, 2, 64, [40, 700, 63, 3000], 1 << 20), (8, 2, 128, [5, 9000, 127, 6000], 1 << 20),
                                   (32, 8, 128, [511, 512, 64, 1], 100)):
        B, n = len(lens), 145
        gen = torch.Generator().manual_seed(D)
        k, v, table = ref.cache(gen, B, n, H, D, dev)
        inv, scale = pkg.rotary_frequencies(D, device=dev)
        new = [torch.randn(B, 1, h, D, generator=gen).bfloat16().to(dev) for h in (HQ, H, H)]

        def step(kp, vp, lengths):
            lengths.add_(1)
            q = pkg.paged_append(new[1], new[2], kp, vp, table, lengths, q=new[0], inv_freq=inv, scale=scale)
            return pkg.paged_flex_attn(q, kp, vp, table, lengths, window)

        mine, lengths = (k.clone(), v.clone()), torch.tensor(lens, dtype=torch.int32, device=dev)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(k.clone(), v.clone(), lengths.clone())
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                out = step(*mine, lengths)
        torch.cuda.synchronize()
        at = torch.tensor(lens, dtype=torch.int32, device=dev)
        assert torch.equal(at, lengths)  # (captured, not run)
        for _ in range(70):  # (past a page's end for every sequence)
            g.replay()
            want = step(k, v, at)
            assert all(torch.equal(x, y) for x, y in zip(out, want))
        torch.cuda.synchronize()
        assert torch.equal(at, lengths) and torch.equal(mine[0], k) and torch.equal(mine[1], v)
        ref.check_attention(want, ref.attend_dense(pkg.rotary_embedding(new[0], None, (at - 1).view(B, 1), inv, scale=scale)[0], k, v, table, at, window))
