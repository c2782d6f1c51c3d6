"""What the operators on a paged cache promise for calls that never reach a kernel, without a GPU: refusals of the C ABI, of
the layer and of autograd's modes."""
import ctypes
import warnings

import pytest
import torch
from torch.autograd import forward_ad

A = 1 << 20  # an address that is never read: every call is refused before a launch


def at(byte):
    return ctypes.c_void_p(A + byte)


def test_attention_refuses_buffers_between_its_loads(pkg):
    """Pages are read, shares and outputs written, in pieces of 16 and 8 bytes."""
    from hils_attention_amd.ops import _cabi
    lib = _cabi.load()
    need = lib.hils_paged_attn_workspace(1, 1, 4, 2, 64, 1 << 20, 4096)
    assert need > 0

    def call(k=0, v=0, o=0, lse=0, ws=0):
        rc = lib.hils_paged_attn(at(0), at(k), at(v), at(0), None, None, at(o), at(lse), at(ws), need, 512, 256, 64, 1, 1, 4, 2, 64,
                                 4096, 9, 1 << 18, 0, 1 << 20, 1, 1, 0.1, None)
        return rc, lib.hils_last_error().decode()

    for kw in ({"k": 2}, {"k": 8}, {"v": 2}, {"v": 4}, {"ws": 4}, {"ws": 8}, {"o": 2}, {"o": 4}, {"lse": 2}):
        rc, text = call(**kw)
        assert rc == 1 and "must lie at" in text, (kw, rc, text)


def _books(c):
    return c.seq_len, c.drafted, c.page_table.clone().tolist(), list(c.free_pages), [list(p) for p in c._pages], list(c._users)


def test_draft_refuses_a_tree_that_the_attention_does_not_take(pkg):
    c = pkg.HiLSPagedLayer(num_pages=24, batch=2, max_pages_per_seq=12, num_kv_heads=1, head_dim=16, device="cpu")
    z = lambda t: torch.ones(2, t, 1, 16, dtype=torch.bfloat16)
    c.update(z(10), z(10))
    was = _books(c)
    with pytest.raises(AssertionError, match="at most 256"):
        c.draft(z(257), z(257), parents=list(range(-1, 256)))
    assert _books(c) == was
    c.draft(z(256), z(256), parents=list(range(-1, 255)))
    c.truncate(10)
    c.draft(z(300), z(300))  # (a chain may be longer)
    c.truncate(10)
    assert _books(c)[0] == 10 and len(c.free_pages) == 22


@pytest.mark.parametrize("order", [[7, 1, 4, 9, 3, 8], [5, 3, 1, 0, 2, 4, 9, 8, 7, 6]])
def test_compact_keeps_to_the_pages_of_the_layer(pkg, monkeypatch, order):
    """A layer that has only some of the pools' pages moves nothing onto the others and hands none of them out."""
    import hils_attention_amd.utils.hils_cache_utils as utils

    def copy(pools, src, dst):
        for pool in pools:
            pool[dst] = pool[src].clone()

    monkeypatch.setattr(utils, "copy_pages", copy)
    c = pkg.HiLSPagedLayer(num_pages=10, batch=2, max_pages_per_seq=3, num_kv_heads=1, head_dim=16, device="cpu", page_order=order)
    others = [p for p in range(10) if p not in order]
    c.k_pages[others] = c.v_pages[others] = 7.0
    gen = torch.Generator().manual_seed(1)
    z = lambda t: torch.randn(2, t, 1, 16, generator=gen).bfloat16()
    c.update(z(50), z(50))
    c.draft(z(100), z(100))
    c.truncate(50)
    k, v = c.gather_contiguous()
    assert c.compact() == 2
    assert c._pages == [[p] for p in c.page_table[:, 0].tolist()] and sorted(sum(c._pages, [])) == sorted(order)[:2]
    assert sorted(c.free_pages) == sorted(order)[2:] and c.free_pages[-1] == min(c.free_pages)
    assert all(torch.equal(x, y) for x, y in zip(c.gather_contiguous(), (k, v)))
    assert (c.k_pages[others] == 7).all() and (c.v_pages[others] == 7).all()
    c.free()
    assert c.compact() == 0 and sorted(c.free_pages) == sorted(order)


def test_copied_pairs_that_are_left_out_are_in_no_ones_way(pkg):
    """Of pairs given as numbers only those that move a page have to be apart."""
    pool = torch.zeros(5, 8)
    for src, dst in (([0, 1, 2], [-1, -1, 3]), ([5, 6, 2], [3, 3, 3]), ([0, -1, 9], [1, 0, 0]), ([2, 2, 0], [2, 2, 2]),
                     ([0, 7], [2, 2])):
        with pytest.raises(RuntimeError, match="no CPU path"):  # (what pairs that are taken end in here)
            pkg.copy_pages([pool], src, dst)
    for src, dst in (([0, 1], [4, 4]), ([0, 4], [4, 3])):
        with pytest.raises(ValueError, match="another pair"):
            pkg.copy_pages([pool], src, dst)


def _put(to, x):
    """A write behind torch's back, as the native operators write."""
    x = x.detach().contiguous()
    ctypes.memmove(to.data_ptr(), x.data_ptr(), x.numel() * x.element_size())


class _StandIn:
    """The native operators in place of which something simple is computed on the same arguments."""

    def paged_append(self, k, v, k_pages, v_pages, table, seq_len, q, inv_freq, positions, interleaved, scale):
        _put(k_pages, k)
        _put(v_pages, v)
        if q is None:
            return None
        out = torch.empty_like(q)
        _put(out, q.detach() * scale)
        return out

    def paged_flex_attn(self, q, k_pages, *_):
        out = torch.empty_like(q)
        _put(out, q.detach() + k_pages.detach().flatten()[:1])
        return out, out.float().sum(-1)

    def paged_accept(self, k_pages, v_pages, table, base, path):
        _put(k_pages, k_pages.detach() * 3)

    def copy_pages(self, pools, src, dst):
        for pool in pools:
            _put(pool, pool.detach() + 1)


def _calls(pkg):
    """(name, call on (k, q, k_pages, v_pages), arguments it writes)"""
    table = torch.zeros(1, 2, dtype=torch.int32)
    one = torch.ones(1, dtype=torch.int32)
    return [("paged_append", lambda k, q, kp, vp: pkg.paged_append(k, k, kp, vp, table, 10, q=q, inv_freq=torch.ones(32), scale=2.0), (2, 3)),
            ("paged_append", lambda k, q, kp, vp: pkg.paged_append(k, k, kp, vp, table, 10), (2, 3)),
            ("paged_flex_attn", lambda k, q, kp, vp: pkg.paged_flex_attn(q, kp, vp, table, 10, 64)[0], ()),
            ("copy_pages", lambda k, q, kp, vp: pkg.copy_pages([kp, vp], one, one), (2, 3)),
            ("paged_accept", lambda k, q, kp, vp: pkg.paged_accept(kp, vp, table, 3, torch.zeros(1, 2, dtype=torch.int32)), (2, 3))]


def _tensors(seed):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(*s, generator=gen).bfloat16() for s in ((1, 2, 2, 64), (1, 2, 4, 64), (4, 2, 64, 64), (4, 2, 64, 64))]


def _stand_in(monkeypatch):
    from hils_attention_amd.ops import _cabi
    monkeypatch.setattr(_cabi, "host", lambda: _StandIn())


def test_a_trace_records_the_calls(pkg, monkeypatch):
    _stand_in(monkeypatch)
    calls = [c for _, c, _ in _calls(pkg)]

    def step(k, q, kp, vp):
        q = calls[0](k, q, kp, vp)
        for call in (calls[1], calls[3], calls[4]):
            call(k, q, kp, vp)
        return calls[2](k, q, kp, vp)

    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        traced = torch.jit.trace(step, tuple(_tensors(1)), check_trace=False)
    one, two = _tensors(2), _tensors(2)
    assert torch.equal(traced(*one), step(*two)) and not torch.equal(one[2], _tensors(2)[2])
    assert all(torch.equal(x, y) for x, y in zip(one, two))


def test_tangents_and_transforms_are_refused(pkg, monkeypatch):
    _stand_in(monkeypatch)
    args = _tensors(1)
    for name, call, _ in _calls(pkg):
        given = [2, 3] if name in ("copy_pages", "paged_accept") else [1, 2, 3] if name == "paged_flex_attn" else [0, 2, 3]
        for i in given:
            was = [x.clone() for x in args]
            with forward_ad.dual_level():
                duals = list(args)
                duals[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
                with pytest.raises(NotImplementedError, match=f"{name} .* jvp"):
                    call(*duals)
            with pytest.raises(RuntimeError):
                torch.vmap(lambda x: call(*args[:i], x, *args[i + 1:]))(args[i].unsqueeze(0))
            assert all(torch.equal(x, y) for x, y in zip(args, was))
        with forward_ad.dual_level():
            call(*args)  # (no tangent: nothing is lost)


def test_pages_that_require_gradients_are_not_written(pkg):
    """(refused by the native operators, before they look where the tensors are)"""
    for name, call, written in _calls(pkg):
        for i in written:
            args = _tensors(1)
            args[i].requires_grad_()
            with pytest.raises(RuntimeError, match=f"{name} .* must not require gradients"):
                call(*args)
            with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"):
                call(*args)
            with forward_ad.dual_level(), pytest.raises(RuntimeError, match=f"{name} .* must not require gradients"):
                call(*args)
