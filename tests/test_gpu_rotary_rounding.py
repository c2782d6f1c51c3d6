"""Rotated values are the exact ones but for their rounding: fp64 angles and rotation, rounded to fp32 and then to bf16."""
import pytest
import torch

import paged_ref as ref
from util import note

pytestmark = pytest.mark.gpu


def _check(got, want, x, n, interleaved, scale):
    """Half a step of bf16 and half a step of fp32 of the value (each of the value rounded before, 2^-16 of it more at most).
    Before: angles up to 2^17, off by 2^-53 of themselves, 2^-36, in each of four roundings (one here, and in the kernel 1/(2 pi),
    its product with the frequency and that with the position), so 2^-34 in all, and the sine, cosine and sums in fp64, far
    less: together under 2^-33 of a pair's |x1| + |x2|.  An fp32 rotation is off by 2^-24 of them, which shows wherever the two
    terms cancel to less than 2^-17 (of four million values some tens)."""
    a = x.detach().double().abs()
    pair = a.new_zeros(a.shape)
    if interleaved:
        both = a[..., 0:2 * n:2] + a[..., 1:2 * n:2]
        pair[..., 0:2 * n:2], pair[..., 1:2 * n:2] = both, both
    else:
        both = a[..., :n] + a[..., n:2 * n]
        pair[..., :n], pair[..., n:2 * n] = both, both
    bound = (ref.HALF + 2 ** -24) * (1 + 2 ** -16) * want.abs() + 2 ** -33 * scale * pair
    off = (got.detach().double() - want).abs()
    worst = (off / bound.clamp_min(1e-300)).max().item()
    cancelled = (want.abs() < 2 ** -17 * scale * pair).sum().item()
    print(f"    {worst:.4f} of the bound, {cancelled} values cancelled", flush=True)
    assert worst <= 1 and cancelled > 5


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("wide", [torch.float64, torch.float32])
def test_rounded_by_way_of_fp32(pkg, dev, interleaved, wide):
    note(f"rotary's rounding, interleaved {interleaved}, {wide}")
    gen = torch.Generator(device=dev).manual_seed(1)
    B, T, HQ, H, D, R = 1, 1000, 40, 8, 128, 96
    r = lambda h: torch.randn(B, T, h, D, device=dev, generator=gen).bfloat16()
    q, k, dq, dk = r(HQ).requires_grad_(), r(H).requires_grad_(), r(HQ), r(H)
    inv = pkg.rotary_frequencies(R, device=dev)[0].to(wide)
    pos = torch.randint(0, 1 << 17, (B, T), device=dev, generator=gen)
    qo, ko = pkg.rotary_embedding(q, k, pos, inv, interleaved=interleaved, scale=1.25)
    gq, gk = torch.autograd.grad([qo, ko], [q, k], [dq, dk])
    _check(qo, ref.rotate(q, pos, inv, interleaved, 1.25), q, R // 2, interleaved, 1.25)
    _check(gq, ref.rotate(dq, -pos, inv, interleaved, 1.25), dq, R // 2, interleaved, 1.25)
    assert torch.equal(ko, pkg.rotary_embedding(k, None, pos, inv, interleaved=interleaved, scale=1.25)[0])
    assert torch.equal(gk, pkg.rotary_embedding(dk, None, -pos, inv, interleaved=interleaved, scale=1.25)[0])
