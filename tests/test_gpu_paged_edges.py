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
