"""Rotary positions by position and the append to a paged cache that rotates on the way, against the 64-bit form."""
import math

import pytest
import torch

import paged_ref as ref
from util import note

pytestmark = pytest.mark.gpu


def check(got, want, size):
    """One rounding to bf16, and fp32 arithmetic on cosines and sines good to a few units of 2^-24: 2^-20 of the terms."""
    bound = ref.HALF * want.abs() + 2 ** -20 * size + 1e-30
    worst = ((got.detach().double().cpu() - want.cpu()).abs() / bound.cpu()).max().item()
    assert worst <= 1, f"{worst} of the bound"


def terms(x, n, interleaved, scale):
    """|x1| + |x2| of a feature's pair times the scale."""
    a = x.detach().double().abs()
    y = a.clone()
    if interleaved:
        both = a[..., 0:2 * n:2] + a[..., 1:2 * n:2]
        y[..., 0:2 * n:2], y[..., 1:2 * n:2] = both * scale, both * scale
    else:
        both = a[..., :n] + a[..., n:2 * n]
        y[..., :n], y[..., n:2 * n] = both * scale, both * scale
    return y


@pytest.mark.parametrize("B,T,HQ,H,D,R", [(1, 1, 4, 4, 64, 64), (2, 7, 16, 2, 64, 32), (3, 65, 32, 8, 128, 128), (1, 300, 5, 1, 128, 96),
                                          (2, 33, 3, 3, 256, 16), (1, 9, 2, 1, 16, 16), (1, 2000, 40, 8, 128, 64), (2, 5, 1, 1, 1024, 1024)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("wide", [torch.float64, torch.float32])
def test_forward_and_backward(pkg, dev, B, T, HQ, H, D, R, interleaved, wide):
    note(f"rotary B{B} T{T} heads {HQ}/{H} of {D}, {R} rotated, interleaved {interleaved}")
    gen = torch.Generator().manual_seed(T)
    r = lambda h: torch.randn(B, T, h, D, generator=gen).bfloat16().to(dev)
    q, k, dq, dk = r(HQ), r(H), r(HQ), r(H)
    inv, _ = pkg.rotary_frequencies(R, device=dev)
    inv = inv.to(wide)
    pos = torch.randint(0, 100000, (B, T), generator=gen).to(dev, torch.int64 if T % 2 else torch.int32)
    q.requires_grad_(), k.requires_grad_()
    qo, ko = pkg.rotary_embedding(q, k, pos, inv, interleaved=interleaved, scale=1.25)
    gq, gk = torch.autograd.grad([qo, ko], [q, k], [dq, dk])
    for x, y, d, g in ((q, qo, dq, gq), (k, ko, dk, gk)):
        check(y, ref.rotate(x, pos, inv, interleaved, 1.25), terms(x, R // 2, interleaved, 1.25))
        check(g, ref.rotate(d, -pos, inv, interleaved, 1.25), terms(d, R // 2, interleaved, 1.25))
        # the gradient against differences: the map is linear, so <d, R(x)> = <g, x> up to the two roundings
        lhs, rhs = (d.double() * y.detach().double()).sum(), (g.double() * x.detach().double()).sum()
        room = 2 * ref.HALF * (d.double().abs() * y.detach().double().abs()).sum()
        assert (lhs - rhs).abs() <= room


def test_far_positions(pkg, dev):
    """Positions up to 2^31 - 1, where an fp32 angle has lost every digit of its turn; negative ones; an int."""
    note("far positions")
    gen = torch.Generator().manual_seed(3)
    q = torch.randn(1, 64, 2, 128, generator=gen).bfloat16().to(dev)
    inv, _ = pkg.rotary_frequencies(128, device=dev)
    pos = torch.randint(-2 ** 31 + 1, 2 ** 31 - 1, (64,), generator=gen).to(dev)
    y, none = pkg.rotary_embedding(q, None, pos, inv)
    assert none is None
    check(y, ref.rotate(q, pos, inv), terms(q, 64, False, 1.0))
    y32, _ = pkg.rotary_embedding(q, None, pos.int(), inv)
    assert torch.equal(y, y32)
    y, _ = pkg.rotary_embedding(q, None, 1000003, inv)
    check(y, ref.rotate(q, torch.arange(64, device=dev) + 1000003, inv), terms(q, 64, False, 1.0))


def test_views_missing_gradients_and_second_derivatives(pkg, dev):
    note("views of a fused projection, broadcast gradients, one output's gradient, gradients of gradients")
    gen = torch.Generator().manual_seed(4)
    B, T, HQ, H, D = 2, 19, 8, 2, 64
    qkv = torch.randn(B, T, HQ + 2 * H, D, generator=gen).bfloat16().to(dev).requires_grad_()
    inv, _ = pkg.rotary_frequencies(D, device=dev)
    pos = torch.arange(T, device=dev).flip(0)
    q, k, _ = qkv.split([HQ, H, H], 2)
    qo, ko = pkg.rotary_embedding(q, k, pos, inv)
    assert torch.equal(qo, pkg.rotary_embedding(q.contiguous(), k.contiguous(), pos, inv)[0])
    bhtd = q.detach().transpose(1, 2).contiguous().transpose(1, 2)
    odd = torch.cat([q.detach(), q.detach()], -1)[..., 1:D + 1]  # begins between two multiples of 16 bytes
    shift = pkg.rotary_embedding(odd, None, pos, inv)[0]
    assert torch.equal(pkg.rotary_embedding(bhtd, None, pos, inv)[0], qo)
    check(shift, ref.rotate(odd, pos, inv), terms(odd, D // 2, False, 1.0))
    (g,) = torch.autograd.grad(ko.sum(), qkv, retain_graph=True)  # an expanded gradient, and none for q
    assert (g[:, :, :HQ] == 0).all() and (g[:, :, HQ + H:] == 0).all()
    check(g[:, :, HQ:HQ + H], ref.rotate(torch.ones_like(k), -pos, inv), terms(torch.ones_like(k), D // 2, False, 1.0))
    # d/dx |R x|^2 / 2 = R^T R x, whose gradient along c is R^T R c
    x = q.detach().clone().requires_grad_()
    y, _ = pkg.rotary_embedding(x, None, pos, inv)
    (g,) = torch.autograd.grad((y.float() ** 2).sum() / 2, x, create_graph=True)
    c = torch.randn(x.shape, generator=gen).to(dev)
    (h,) = torch.autograd.grad((g.float() * c).sum(), x)
    assert (h.float() - c).abs().max() <= 6 * 4 * 2 ** -8 * c.abs().max()  # four roundings of bf16 on the way
    assert pkg.rotary_embedding(q[:, :0], k[:, :0], pos[:0], inv)[0].shape == (B, 0, HQ, D)


def test_backward_in_a_graph_beside_an_eager_one(pkg, dev):
    note("forward and backward captured")
    gen = torch.Generator().manual_seed(5)
    q = torch.randn(2, 100, 8, 64, generator=gen).bfloat16().to(dev)
    d = torch.randn(2, 100, 8, 64, generator=gen).bfloat16().to(dev)
    inv, scale = pkg.rotary_frequencies(64, scaling="yarn", factor=4, original_length=4096, device=dev)
    pos = torch.arange(100, device=dev, dtype=torch.int32)

    def step():
        x = q.detach().requires_grad_()
        y, _ = pkg.rotary_embedding(x, None, pos, inv, scale=scale)
        return y.detach(), torch.autograd.grad(y, x, d)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, g = step()
    for i in range(3):
        q.mul_(-1.5)
        pos.add_(1000)
        graph.replay()
        y1, g1 = step()
        torch.cuda.synchronize()
        assert torch.equal(y, y1) and torch.equal(g, g1)


@pytest.mark.parametrize("heads", [(4, 4, 64), (16, 2, 64), (32, 8, 128), (5, 1, 256)])
@pytest.mark.parametrize("T", [1, 3, 64, 200])
@pytest.mark.parametrize("turn", ["none", "keys", "both", "positions"])
def test_append(pkg, dev, heads, T, turn):
    """K and V of the new tokens to their pages, everything else of the pages as it was."""
    note(f"append T{T} heads {heads} {turn}")
    HQ, H, D = heads
    B, n = 5, 6
    gen = torch.Generator().manual_seed(T)
    kp, vp, table = ref.cache(gen, B, n, H, D, dev)
    table[3, 1] = -1
    table[3, 2] = 10 ** 7
    lengths = [T, 0, 384, max(T, 190), 401]  # one that takes no part, one past the table
    ln = torch.tensor(lengths, dtype=torch.int32, device=dev)
    qkv = torch.randn(B, T, HQ + 2 * H, D, generator=gen).bfloat16().to(dev)
    q, k, v = qkv.split([HQ, H, H], 2)
    inv, _ = pkg.rotary_frequencies(D // 2, device=dev)
    pos = torch.randint(0, 5000, (B, T), generator=gen).to(dev, torch.int32)
    k0, v0 = kp.clone(), vp.clone()
    base = ln.view(B, 1) - T
    at = pos if turn == "positions" else base + torch.arange(T, device=dev)
    kw = {} if turn == "none" else {"inv_freq": inv, "scale": 0.5, "interleaved": T == 3}
    if turn == "positions":
        kw["positions"] = pos
    qo = pkg.paged_append(k, v, kp, vp, table, ln, q=q if turn in ("both", "positions") else None, **kw)
    kr = k.double() if turn == "none" else ref.rotate(k, at, inv, T == 3, 0.5)
    if turn in ("both", "positions"):
        check(qo, ref.rotate(q, at, inv, T == 3, 0.5), terms(q, D // 4, T == 3, 0.5))
    else:
        assert qo is None
    size = terms(k, D // 4, T == 3, 0.5)
    for b in range(B):
        for t in range(T):
            slot = lengths[b] - T + t
            page = int(table[b, slot // 64]) if 0 <= slot < n * 64 else -1
            if not 0 <= page < kp.shape[0]:
                continue
            got = kp[page, :, slot % 64]
            if turn == "none":
                assert torch.equal(got, k[b, t])
            else:
                check(got, kr[b, t], size[b, t])
            assert torch.equal(vp[page, :, slot % 64], v[b, t])
            kp[page, :, slot % 64], vp[page, :, slot % 64] = k0[page, :, slot % 64], v0[page, :, slot % 64]
    assert torch.equal(kp, k0) and torch.equal(vp, v0)


def test_append_replays(pkg, dev):
    note("append captured")
    gen = torch.Generator().manual_seed(8)
    kp, vp, table = ref.cache(gen, 2, 4, 2, 64, dev)
    k, v, q = (torch.randn(2, 3, h, 64, generator=gen).bfloat16().to(dev) for h in (2, 2, 8))
    inv, _ = pkg.rotary_frequencies(64, device=dev)
    ln = torch.tensor([10, 64], dtype=torch.int32, device=dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pkg.paged_append(k, v, kp, vp, table, ln, q=q, inv_freq=inv)
    for i in range(3):
        ln.add_(30)
        k.mul_(-1)
        graph.replay()
        torch.cuda.synchronize()
        k1, v1 = kp.clone(), vp.clone()
        want = pkg.paged_append(k, v, kp, vp, table, ln, q=q, inv_freq=inv)
        assert torch.equal(out, want) and torch.equal(kp, k1) and torch.equal(vp, v1)


def test_frequencies(pkg, dev):
    note("scaled frequencies")
    base, one = pkg.rotary_frequencies(128, device=dev)
    assert one == 1.0 and base.dtype == torch.float64 and base[0] == 1 and math.isclose(base[32].item(), 0.01, rel_tol=1e-12)
    ntk, _ = pkg.rotary_frequencies(128, scaling="ntk", factor=8, device=dev)
    assert math.isclose(ntk[0].item(), 1.0) and math.isclose(ntk[-1].item(), base[-1].item() / 8, rel_tol=1e-12)
    assert torch.equal(pkg.rotary_frequencies(128, scaling="linear", factor=4, device=dev)[0], base / 4)
    for kind, high in (("yarn", 32), ("wavelength", 4)):
        inv, scale = pkg.rotary_frequencies(128, scaling=kind, factor=4, original_length=8192, device=dev)
        turns = 8192 * base / (2 * math.pi)
        assert torch.equal(inv[turns >= high], base[turns >= high])
        torch.testing.assert_close(inv[turns <= 1], base[turns <= 1] / 4, rtol=1e-14, atol=0)
        between = (turns > 1) & (turns < high)
        assert between.any() and (inv[between] < base[between]).all() and (inv[between] > base[between] / 4).all()
        assert scale == (0.1 * math.log(4) + 1 if kind == "yarn" else 1.0)
