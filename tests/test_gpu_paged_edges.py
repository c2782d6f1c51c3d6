"""Calls at the edges of what the operators on a paged cache take: sequences too short for the call, layouts of single rows,
numbers left behind by whoever had the pages before."""
import pytest
import torch

import paged_ref as ref
from util import note

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads", [(16, 2, 64), (32, 8, 128)])
@pytest.mark.parametrize("T", [2, 8, 70])
@pytest.mark.parametrize("turned", [False, True])
def test_append_leaves_short_sequences_alone(pkg, dev, heads, T, turned):
    """A sequence with fewer tokens than the call has new ones keeps every byte of its pages, all of them mapped."""
    note(f"append of {T} tokens beside shorter sequences, heads {heads}, rotated {turned}")
    HQ, H, D = heads
    lengths = [1, T - 1, T, 0, -1, T // 2, T + 1, 150]
    gen = torch.Generator().manual_seed(T)
    kp, vp, table = ref.cache(gen, len(lengths), 3, H, D, dev)
    k, v = (torch.randn(len(lengths), T, H, D, generator=gen).bfloat16().to(dev) for _ in range(2))
    inv, _ = pkg.rotary_frequencies(D, device=dev)
    ln = torch.tensor(lengths, dtype=torch.int32, device=dev)
    want_k, want_v = kp.clone(), vp.clone()
    # (the keys as the operator itself turns them: what is tested is where they go)
    at = ln.view(-1, 1) - T + torch.arange(T, device=dev)
    turned_k = pkg.rotary_embedding(k, None, at, inv)[0] if turned else k
    for b, n in enumerate(lengths):
        for t in range(T if n >= T else 0):
            slot = n - T + t
            page = table[b, slot // 64].long()
            want_k[page, :, slot % 64], want_v[page, :, slot % 64] = turned_k[b, t], v[b, t]
    pkg.paged_append(k, v, kp, vp, table, ln, inv_freq=inv if turned else None)
    assert torch.equal(kp, want_k) and torch.equal(vp, want_v)


def test_attention_refuses_pages_between_its_loads(pkg, dev):
    """(refused on the host: no kernel runs)"""
    note("pools that begin between two multiples of 16 bytes")
    whole = torch.zeros(9 * 2 * 64 * 64 + 1, device=dev).bfloat16()
    odd, even = whole[1:].view(9, 2, 64, 64), whole[:-1].view(9, 2, 64, 64)
    q, table = torch.zeros(1, 1, 4, 64, device=dev).bfloat16(), torch.zeros(1, 4, device=dev, dtype=torch.int32)
    for k, v in ((odd, even), (even, odd)):
        with pytest.raises(RuntimeError, match="multiples of 16 bytes"):
            pkg.paged_flex_attn(q, k, v, table, 100, 64)


def _single(x, strides):
    """x (1,1,1,D) with any strides of its dimensions of one."""
    whole = torch.zeros(4096, dtype=x.dtype, device=x.device)
    y = whole.as_strided(x.shape, (*strides, 1))
    return y.copy_(x)


@pytest.mark.parametrize("strides", [(65, 65, 65), (3, 129, 64), (0, 1, 2), (64, 64, 64)])
def test_strides_of_single_rows_do_not_matter(pkg, dev, strides):
    """One token of one head, cut from rows of an odd width: torch calls it contiguous whatever its strides are."""
    note(f"single rows with strides {strides}")
    gen = torch.Generator().manual_seed(3)
    kp, vp, table = ref.cache(gen, 1, 3, 1, 64, dev)
    q, k, v = (torch.randn(1, 1, 1, 64, generator=gen).bfloat16().to(dev) for _ in range(3))
    inv, _ = pkg.rotary_frequencies(64, device=dev)
    runs = []
    for cut in (lambda x: x, lambda x: _single(x, strides)):
        k1, v1 = kp.clone(), vp.clone()
        a, b = cut(q).requires_grad_(), cut(k).requires_grad_()
        turned = pkg.rotary_embedding(a, b, 70, inv)
        grads = torch.autograd.grad(turned, [a, b], [cut(v), cut(q)])
        new = pkg.paged_append(cut(k), cut(v), k1, v1, table, 100, q=cut(q), inv_freq=inv)
        out = pkg.paged_flex_attn(cut(q), k1, v1, table, 100, 512)
        runs.append([x.detach() for x in (*turned, *grads, new, *out, k1, v1)])
    assert all(torch.equal(x, y) for x, y in zip(*runs))
    ref.check_attention(out, ref.attend(q, k1, v1, table, 100, 512))


def test_autograd_notices_what_is_written(pkg, dev):
    """A backward that needs what the pages held before is refused, as after torch's own writes in place."""
    note("pages kept for a backward, then written")
    gen = torch.Generator().manual_seed(4)
    kp, vp, table = ref.cache(gen, 1, 2, 2, 64, dev)
    k = torch.randn(1, 2, 2, 64, generator=gen).bfloat16().to(dev)
    path = torch.tensor([[1]], dtype=torch.int32, device=dev)
    for call, pools in ((lambda: pkg.paged_append(k, k, kp, vp, table, 10), (kp, vp)), (lambda: pkg.paged_accept(kp, vp, table, 3, path), (kp, vp)),
                        (lambda: pkg.copy_pages([kp, vp], [0], [1]), (kp, vp))):
        for pool in pools:
            x = torch.ones_like(pool).requires_grad_()
            loss = (x * pool).sum()
            call()
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                loss.backward()
    with torch.inference_mode():
        kept = torch.zeros_like(kp), torch.zeros_like(vp)
    pkg.paged_append(k, k, *kept, table, 10)  # (tensors of inference mode have nothing that could notice)
    with torch.inference_mode():
        pkg.paged_append(k, k, *kept, table, 12)
        pkg.paged_append(k, k, kp, vp, table, 12)
    assert (kept[0] != 0).any(-1).sum() == 8


@pytest.mark.parametrize("turned", [False, True])
def test_gradients_through_the_layers_pages(pkg, dev, turned):
    """Keys and values that want gradients: the cache is that of the direct call, bit for bit, and each gets the gradient of
    the tokens that are kept, through appends, drafts, forks and compaction."""
    note(f"a paged layer with gradients, rotated {turned}")
    B, H, D, first, drafts = 2, 2, 64, 100, 4
    gen = torch.Generator().manual_seed(5)
    r = lambda t, h: torch.randn(B, t, h, D, generator=gen).bfloat16().to(dev)
    k, v, q, dk, dv, dq = r(first, H), r(first, H), r(first, 4), r(drafts, H), r(drafts, H), r(drafts, 4)
    inv, _ = pkg.rotary_frequencies(D, device=dev)
    turn = {"inv_freq": inv, "scale": 0.5} if turned else {}
    layers, outs = [], []
    leaves = [x.clone().requires_grad_() for x in (k, v, dk, dv)]
    for kk, vv, dkk, dvv in ((k, v, dk, dv), leaves):
        c = pkg.HiLSPagedLayer(num_pages=16, batch=B, max_pages_per_seq=4, num_kv_heads=H, head_dim=D, device=dev, page_order=[3, 9, 12, 5, 7, 1, 2, 15])
        out = [c.update(kk, vv, q=q if turned else None, **turn)]
        c.fork([1, 1])
        out.append(c.draft(dkk, dvv, parents=[-1, 0, 0, 2], q=dq if turned else None, **turn))
        c.accept([0, 2, 3])
        c.compact()
        layers.append(c)
        outs.append(out + list(c.gather_contiguous()) + [c.lmk_hm, c.k_pages, c.v_pages, c.lmk_pages])
    assert [c._pages for c in layers][0] == layers[1]._pages
    assert all(x is y is None or torch.equal(x, y) for x, y in zip(*outs))
    gk, gv = outs[1][2:4]
    w = [torch.randn(x.shape, generator=gen).bfloat16().to(dev) for x in (gk, gv)]
    got = torch.autograd.grad([gk, gv], leaves, w)
    # both sequences are sequence 1's first tokens and their own drafts 0, 2 and 3; a rotation's transpose turns gradients back
    want = [torch.zeros_like(x) for x in leaves]
    back = (lambda x, at: pkg.rotary_embedding(x, None, at, inv, scale=0.5)[0]) if turned else (lambda x, at: x)
    full = back(w[0], -torch.arange(first + 3, device=dev))
    at = [0, 2, 3]
    # (of tokens that both sequences have, the sum of the two gradients as one product of bf16 each: two roundings and the sum's)
    for i, (x, kept) in enumerate(((full, 0), (w[1], 1))):
        want[i + 2][:, at] = x[:, first:]
        both = x[:, :first].double().sum(0)
        err = (got[i][1].double() - both).abs()
        size = x[:, :first].double().abs().sum(0)
        if turned and i == 0:  # (rounded before and after the rotation, whose terms are up to twice as large)
            pair = size[..., : D // 2] + size[..., D // 2:]
            size = size + 2 * torch.cat([pair, pair], -1)
        assert (err <= 3 * ref.HALF * size + 1e-30).all()
        assert (got[i][0] == 0).all()
        assert torch.equal(got[i + 2], want[i + 2])


def test_update_keeps_gradients_of_the_chunk_keys(pkg, dev):
    note("chunk keys of a paged layer with gradients")
    gen = torch.Generator().manual_seed(6)
    c = pkg.HiLSPagedLayer(num_pages=8, batch=2, max_pages_per_seq=3, num_kv_heads=2, head_dim=64, device=dev)
    k = torch.randn(2, 130, 2, 64, generator=gen).bfloat16().to(dev).requires_grad_()
    c.update(k, k.detach())
    (g,) = torch.autograd.grad(c.lmk_hm.float().sum(), k)
    # the mean of 64 tokens, each weighed 1/64 (exact in bf16); the last two are in no chunk
    assert (g[:, :128] == 1 / 64).all() and (g[:, 128:] == 0).all()
    q = torch.randn(2, 1, 4, 64, generator=gen).bfloat16().to(dev)
    o, lse = c.local_attend(q, 64)
    with pytest.raises(RuntimeError, match="inference operator"):
        o.float().sum().backward()
    with torch.no_grad():
        c.update(k[:, :1], k[:, :1])
        c.fork([0, 0])
        c.update(k[:, :1], k[:, :1])
    assert c.seq_len == 132


def test_a_backward_through_an_inference_operator_is_refused(pkg, dev):
    note("inputs that want gradients")
    gen = torch.Generator().manual_seed(7)
    kp, vp, table = ref.cache(gen, 1, 2, 2, 64, dev)
    k, q = (torch.randn(1, 2, h, 64, generator=gen).bfloat16().to(dev) for h in (2, 4))
    inv, _ = pkg.rotary_frequencies(64, device=dev)
    append = lambda k, v, q: pkg.paged_append(k, v, kp, vp, table, 10, q=q, inv_freq=inv)
    want = append(k, k, q)
    for i in range(3):
        args = [k, k, q]
        args[i] = args[i].clone().requires_grad_()
        out = append(*args)
        assert torch.equal(out, want)
        with pytest.raises(RuntimeError, match="paged_append is an inference operator"):
            out.float().sum().backward()
        with torch.no_grad():
            assert not append(*args).requires_grad
    assert pkg.paged_append(k.clone().requires_grad_(), k, kp, vp, table, 10) is None
    want = pkg.paged_flex_attn(q, kp, vp, table, 10, 64)
    for i in range(3):
        args = [q, kp, vp]
        args[i] = args[i].clone().requires_grad_()
        o, lse = pkg.paged_flex_attn(*args, table, 10, 64)
        assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
        for x in (o, lse):
            with pytest.raises(RuntimeError, match="paged_flex_attn is an inference operator"):
                x.float().sum().backward()


def _shortest(call, runs=7):
    """Microseconds of the shortest of a few calls."""
    call()
    best = float("inf")
    for _ in range(runs):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        call()
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b) * 1e3)
    return best


@pytest.mark.parametrize("heads,B,T,length,window", [((32, 8, 128), 8, 1, 4090, 512), ((16, 2, 64), 4, 1, 8001, 1 << 20),
                                                     ((32, 8, 128), 4, 63, 4093, 512), ((32, 4, 128), 2, 64, 8130, 1 << 20),
                                                     ((16, 4, 64), 4, 64, 2090, 1 << 20), ((8, 2, 128), 2, 700, 2001, 512)])
def test_what_lies_behind_the_last_token_costs_nothing(pkg, dev, heads, B, T, length, window):
    """A pool whose memory held something else has numbers that are none behind its sequences' last tokens: the same result,
    bit for bit, and no row of it is worked out a second time, token by token (12 to 160 times the call)."""
    note(f"NaN behind the last token, heads {heads}, {B} x {T} tokens of {length}")
    HQ, H, D = heads
    gen = torch.Generator().manual_seed(T)
    k, v, table = ref.cache(gen, B, -(-length // 64) + 1, H, D, dev)
    q = torch.randn(B, T, HQ, D, generator=gen).bfloat16().to(dev)
    parents = torch.tensor(ref.tree(gen, T), dtype=torch.int32, device=dev) if 1 < T <= 256 else None
    call = lambda: pkg.paged_flex_attn(q, k, v, table, length, window, parents=parents)
    want, clean = call(), _shortest(call)
    last, at = table[:, length // 64].long(), length % 64
    k[last, :, at:] = v[last, :, at:] = float("nan")
    k[table[:, -1].long()] = v[table[:, -1].long()] = float("inf")
    got, spoilt = call(), _shortest(call)
    print(f"    {clean:.1f} us, {spoilt:.1f} with stale numbers", flush=True)
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    assert spoilt <= 2 * clean + 20


@pytest.mark.parametrize("heads,T,window", [((32, 8, 128), 63, 512), ((32, 4, 128), 64, 1 << 20), ((16, 4, 64), 64, 1 << 20),
                                            ((32, 8, 128), 1, 1 << 20)])
def test_what_lies_in_the_pools_first_page_costs_nothing(pkg, dev, heads, T, window):
    """A sequence with pages that are not mapped, and a first page of the pools that is nobody's and holds no numbers."""
    note(f"pages that are not mapped beside a stale first page, heads {heads}, {T} tokens")
    HQ, H, D = heads
    B, length = 3, 4093
    gen = torch.Generator().manual_seed(T)
    k, v, table = ref.cache(gen, B, 64, H, D, dev)
    table[table == 0] = k.shape[0] - 1 if not (table == k.shape[0] - 1).any() else -1
    table[0, 60], table[1, 58:61], table[2, :62] = -1, 10 ** 6, -1
    q = torch.randn(B, T, HQ, D, generator=gen).bfloat16().to(dev)
    parents = torch.tensor(ref.tree(gen, T), dtype=torch.int32, device=dev) if T > 1 else None
    call = lambda: pkg.paged_flex_attn(q, k, v, table, length, window, parents=parents)
    k[0] = v[0] = 0
    want, clean = call(), _shortest(call)
    k[0] = v[0] = float("nan")
    got, spoilt = call(), _shortest(call)
    print(f"    {clean:.1f} us, {spoilt:.1f} with stale numbers", flush=True)
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    assert spoilt <= 2 * clean + 20
    ref.check_attention(got, ref.attend(q, k, v, table, length, window, None if parents is None else parents.cpu()))
