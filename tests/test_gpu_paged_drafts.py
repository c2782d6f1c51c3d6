"""Drafted tokens on the paged cache layer, used as a server does: rotate and append, local branch, remote branch, merge,
accept; and forks, roll-backs, released and compacted pages.  The yardstick is the layer fed token by token."""
import pytest
import torch

import paged_ref as ref
from util import assert_close_bf16, note

pytestmark = pytest.mark.gpu


def _layer(pkg, dev, B, H, HQ, D, pages=64, max_pages=12, order=None, **kw):
    return pkg.HiLSPagedLayer(num_pages=pages, batch=B, max_pages_per_seq=max_pages, num_kv_heads=H, head_dim=D, device=dev,
                              page_order=order, **kw)


def _state(c):
    k, v = c.gather_contiguous()
    n = c.pooled_chunks
    return [k, v, c.lmk_hm[:, :, :n].clone(), c.lmk_pages[c.page_table[:, :n].long()]]


def _same(a, b):
    assert a.seq_len == b.seq_len and a.pooled_chunks == b.pooled_chunks
    for x, y in zip(_state(a), _state(b)):
        assert torch.equal(x, y)


def _books(c):
    """The host's list of pages, the table and the free list agree."""
    need = (c.seq_len + c.drafted + 63) // 64
    users = [0] * c.num_pages
    for b, pages in enumerate(c._pages):
        assert len(pages) == need and c.page_table[b, :need].tolist() == pages and (c.page_table[b, need:] == -1).all()
        for p in pages:
            users[p] += 1
    assert users == c._users and sorted(c.free_pages) == [p for p in range(c.num_pages) if not users[p]]


def _step(c, q, topk, window):
    o, lse = c.local_attend(q, window)
    r, w, idx = c.hils_attend(q, lse, topk, window)
    return torch.addcmul(r, o, w[..., -1:]), idx


@pytest.mark.parametrize("HQ,H,D,window,topk", [(8, 2, 128, 64, 4), (16, 2, 64, 100, 3), (4, 4, 64, 130, 8), (6, 2, 64, 512, 4)])
@pytest.mark.parametrize("kind", ["tree", "trees", "chain"])
def test_drafts_match_token_by_token(pkg, dev, HQ, H, D, window, topk, kind):
    """Trees verified at lengths around chunk borders: every accepted token's output and the cache it leaves are those of a
    layer that was given the accepted tokens one at a time."""
    note(f"verification, {kind}, heads {HQ}/{H} x {D}, window {window}")
    B, T, L0 = 2, 13, 300
    gen = torch.Generator().manual_seed(window)
    order = torch.randperm(64, generator=gen).tolist()
    a, b = _layer(pkg, dev, B, H, HQ, D, order=order), _layer(pkg, dev, B, H, HQ, D)
    inv, scale = pkg.rotary_frequencies(D, scaling="yarn", factor=2, original_length=256, device=dev)
    turn = {"inv_freq": inv, "scale": scale}
    r = lambda t, h: torch.randn(B, t, h, D, generator=gen).bfloat16().to(dev)
    k, v = r(L0, H), r(L0, H)
    for c in (a, b):
        c.update(k, v, **turn)
    for step in range(7):
        q, k, v = r(T, HQ), r(T, H), r(T, H)
        rows = None if kind == "chain" else [ref.tree(gen, T, 0.4) for _ in range(B if kind == "trees" else 1)]
        qa = a.draft(k, v, parents=rows if kind != "tree" else rows[0], q=q, **turn)
        _books(a)
        o, idx = _step(a, qa, topk, window)
        up = [list(range(-1, T - 1))] if rows is None else rows
        ways = []
        for i in range(B):  # a way from the root to a leaf
            way = [T - 1]
            while up[i % len(up)][way[-1]] >= 0:
                way.append(up[i % len(up)][way[-1]])
            ways.append(way[::-1])
        n = min(len(w) for w in ways) if step != 3 else 0
        a.accept([w[:n] for w in ways] if kind == "trees" else ways[0][:n])
        ways = [(ways[i] if kind == "trees" else ways[0])[:n] for i in range(B)]
        _books(a)
        for i in range(n):
            pick = torch.tensor([w[i] for w in ways], device=dev)
            one = lambda x: x[torch.arange(B, device=dev), pick].unsqueeze(1)
            qb = b.update(one(k), one(v), q=one(q), **turn)
            o1, idx1 = _step(b, qb, topk, window)
            assert torch.equal(one(idx), idx1)
            assert_close_bf16(one(o), o1.float(), f"token {i} of {n} at {b.seq_len - 1}")
        _same(a, b)
        if a.seq_len % 64 > 40 or step == 5:  # closer to a border, or past it
            more = 64 - a.seq_len % 64 - 5 if a.seq_len % 64 < 55 else 3
            k, v = r(more, H), r(more, H)
            for c in (a, b):
                c.update(k, v, **turn)
    a.free()
    _books(a)
    assert len(a.free_pages) == 64


def test_draft_with_prior_and_pages_of_keys(pkg, dev):
    """Attention-pooled chunk keys and their bias, keys read by page."""
    note("drafts with a prior bias")
    B, H, HQ, D = 2, 2, 8, 64
    gen = torch.Generator().manual_seed(1)
    r = lambda t, h: torch.randn(B, t, h, D, generator=gen).bfloat16().to(dev)
    a, b = (_layer(pkg, dev, B, H, HQ, D, num_q_heads=HQ, chunk_pooling=False) for _ in range(2))
    k, v, mu = r(250, H), r(250, H), r(3, HQ)
    for c in (a, b):
        c.update(k, v, mu_q=mu)
    q, k, v, mu = r(9, HQ), r(9, H), r(9, H), r(1, HQ)
    a.draft(k, v, parents=[-1, 0, 0, 1, 3, 4, 5, 6, 2])
    o, lse = a.local_attend(q, 64)
    x, w, idx = a.hils_attend(q, lse, 2, 64)
    y, w1, idx1 = a.hils_attend(q, lse, 2, 64, dense_keys=False)
    assert torch.equal(idx, idx1) and torch.equal(w, w1) and torch.equal(x, y)
    way = [0, 1, 3, 4, 5, 6]
    a.accept(way, mu_q=mu)
    for i, t in enumerate(way):
        b.update(k[:, t:t + 1], v[:, t:t + 1], mu_q=mu if i == 5 else None)
        o1, lse1 = b.local_attend(q[:, t:t + 1], 64)
        if i < 5:  # (the last one fills the chunk: its own keys are pooled by then)
            x1, _, idx1 = b.hils_attend(q[:, t:t + 1], lse1, 2, 64)
            assert torch.equal(idx[:, t:t + 1], idx1)
            assert_close_bf16(x[:, t:t + 1], x1.float(), f"token {i}")
    _same(a, b)
    assert a.pooled_chunks == 4 and torch.equal(a.prior_hm, b.prior_hm)


@pytest.mark.parametrize("L0", [64, 100, 191])
def test_fork(pkg, dev, L0):
    """Forked sequences share pages and go their own ways: each is what a cache of its own would be."""
    note(f"forks at {L0} tokens")
    B, H, HQ, D = 4, 2, 8, 64
    gen = torch.Generator().manual_seed(L0)
    r = lambda t, h: torch.randn(B, t, h, D, generator=gen).bfloat16().to(dev)
    a, b = (_layer(pkg, dev, B, H, HQ, D, num_q_heads=HQ) for _ in range(2))
    log_k, log_v = r(L0, H), r(L0, H)
    mu = r(L0 // 64, HQ)
    a.update(log_k, log_v, mu_q=mu)
    used = 64 - len(a.free_pages)
    for source in ([1, 1, 1, 0], [0, 1, 2, 3], [3, 2, 1, 0], [2, 2, 2, 2]):
        a.fork(source)
        _books(a)
        assert 64 - len(a.free_pages) <= used
        log_k, log_v, mu = log_k[source], log_v[source], mu[source]
        for t in (1, 7, 64):
            k, v = r(t, H), r(t, H)
            done = a.pooled_chunks
            log_k, log_v = torch.cat([log_k, k], 1), torch.cat([log_v, v], 1)
            new = r(log_k.shape[1] // 64 - done, HQ)
            mu = torch.cat([mu, new], 1)
            a.update(k, v, mu_q=new if new.shape[1] else None)
            _books(a)
        used = 64 - len(a.free_pages)
        q = r(1, HQ)
        b.free()
        b.update(log_k, log_v, mu_q=mu)
        _same(a, b)
        n = a.pooled_chunks
        assert torch.equal(a.prior_hm[:, :, :n], b.prior_hm[:, :, :n])
        for x, y in zip(_step(a, q, 4, 64), _step(b, q, 4, 64)):
            assert torch.equal(x, y)
        # back into a shared part, and on from there
        cut = log_k.shape[1] - 70
        a.truncate(cut)
        _books(a)
        log_k, log_v, mu = log_k[:, :cut], log_v[:, :cut], mu[:, : cut // 64]
    a.free()
    _books(a)


def test_drafts_after_a_fork_and_compaction(pkg, dev):
    note("drafts on shared pages, compaction")
    B, H, HQ, D = 3, 2, 8, 128
    gen = torch.Generator().manual_seed(9)
    r = lambda t, h: torch.randn(B, t, h, D, generator=gen).bfloat16().to(dev)
    a = _layer(pkg, dev, B, H, HQ, D, order=torch.randperm(64, generator=gen).tolist())
    b = _layer(pkg, dev, B, H, HQ, D)
    k, v = r(333, H), r(333, H)
    a.update(k, v)
    a.fork([0, 0, 2])
    a.truncate(290)
    dk, dv, q = r(40, H), r(40, H), r(40, HQ)
    a.draft(dk, dv, parents=list(range(-1, 39)))
    a.accept(range(40))
    b.update(k[[0, 0, 2], :290], v[[0, 0, 2], :290])
    b.update(dk, dv)
    _same(a, b)
    before = _step(a, q, 4, 64)
    n = a.compact()
    _books(a)
    assert n == 64 - len(a.free_pages) and int(a.page_table.max()) == n - 1 and a.compact() == n
    _same(a, b)
    for x, y in zip(before, _step(a, q, 4, 64)):
        assert torch.equal(x, y)
    a.update(dk, dv), b.update(dk, dv)
    _same(a, b)


def test_layer_refusals(pkg, dev):
    note("what the layer refuses")
    B, H, D = 2, 2, 64
    a = _layer(pkg, dev, B, H, 4, D, pages=9, max_pages=4)
    z = lambda t, h=H: torch.zeros(B, t, h, D, dtype=torch.bfloat16, device=dev)
    a.update(z(100), z(100))
    with pytest.raises(ValueError, match="earlier"):
        a.draft(z(2), z(2), parents=[0, -1])
    with pytest.raises(AssertionError, match="parents"):
        a.draft(z(2), z(2), parents=[-1, 0, 1])
    with pytest.raises(AssertionError, match="needs a token"):
        a.draft(z(0), z(0))
    with pytest.raises(AssertionError, match="no tokens"):
        a.accept([0])
    with pytest.raises(ValueError, match="sequences"):
        a.fork([0, 2])
    with pytest.raises(AssertionError, match="of 100"):
        a.truncate(101)
    with pytest.raises(AssertionError, match="too short"):
        a.update(z(157), z(157))
    a.draft(z(3), z(3), parents=[-1, 0, 0])
    for call in (lambda: a.update(z(1), z(1)), lambda: a.draft(z(1), z(1)), lambda: a.fork([0, 0])):
        with pytest.raises(AssertionError, match="on trial"):
            call()
    with pytest.raises(ValueError, match="no way"):
        a.accept([0, 1, 2])
    with pytest.raises(ValueError, match="no way"):
        a.accept([3])
    with pytest.raises(AssertionError, match="got 2"):
        a.local_attend(z(2, 4), 64)
    a.accept([0, 2])
    assert a.seq_len == 102
    a.fork([1, 1])
    b = _layer(pkg, dev, B, H, 4, D, pages=3, max_pages=4)
    b.update(z(50), z(50))
    b.fork([0, 0])
    b.free_pages.clear()
    with pytest.raises(AssertionError, match="out of pages"):
        b.update(z(1), z(1))
    c = _layer(pkg, dev, B, H, 4, D, pages=40)
    c.update(z(100), z(100))
    c.draft(z(70), z(70))
    with pytest.raises(ValueError, match="too deep"):
        c.hils_attend(z(70, 4), torch.zeros(B, 70, 4, device=dev), 1, 16)


def test_a_refused_call_changes_nothing(pkg, dev):
    """A call that is refused after pages were mapped for it, or for its prior queries, leaves the sequences as they were."""
    note("refused appends and acceptances")
    B, H, HQ, D = 2, 2, 4, 64
    gen = torch.Generator().manual_seed(4)
    r = lambda t, h=H: torch.randn(B, t, h, D, generator=gen).bfloat16().to(dev)
    a = _layer(pkg, dev, B, H, HQ, D, num_q_heads=HQ)
    b = _layer(pkg, dev, B, H, HQ, D, num_q_heads=HQ)
    k, v, mu = r(100), r(100), torch.randn(B, 1, HQ, D, generator=gen).bfloat16().to(dev)
    for c in (a, b):
        c.update(k, v, mu_q=mu)
        c.fork([0, 0])
    k, v, mu = r(70), r(70), torch.randn(B, 1, HQ, D, generator=gen).bfloat16().to(dev)
    for call, kind in ((lambda: a.update(k, v, mu_q=mu, q=r(70, HQ)), AssertionError),      # q without frequencies
                       (lambda: a.update(k.float(), v.float(), mu_q=mu), TypeError),
                       (lambda: a.update(k, v), AssertionError),                            # no prior queries for a chunk
                       (lambda: a.update(k, v, mu_q=mu[:, :, :2]), AssertionError),
                       (lambda: a.draft(k, v, q=r(70, HQ)), AssertionError),
                       (lambda: a.draft(k, v[:, :3]), AssertionError)):
        with pytest.raises(kind):
            call()
        _books(a)
        assert a.seq_len == 100 and a.drafted == 0 and a.pooled_chunks == 1
    for c in (a, b):
        c.draft(k, v)
    with pytest.raises(AssertionError, match="mu_q"):
        a.accept(list(range(40)))
    assert a.drafted == 70 and a.seq_len == 100
    for c in (a, b):
        c.accept(list(range(40)), mu_q=mu)
        _books(c)
    _same(a, b)
    assert torch.equal(a.prior_hm, b.prior_hm) and a.pooled_chunks == 2


def test_pages_that_want_gradients(pkg, dev):
    note("no backward through the attention on pages")
    gen = torch.Generator().manual_seed(1)
    k, v, table = ref.cache(gen, 1, 2, 1, 64, dev)
    q = torch.randn(1, 1, 2, 64, generator=gen).bfloat16().to(dev)
    o, lse = pkg.paged_flex_attn(q, k.requires_grad_(), v, table, 100, 64)
    with pytest.raises(RuntimeError, match="not supported"):
        (o.float().sum() + lse.sum()).backward()
