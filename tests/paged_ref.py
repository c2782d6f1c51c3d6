"""Plain 64-bit forms of the operators on a paged cache, and random caches for their tests."""
import math

import torch

S = 64
HALF = torch.finfo(torch.bfloat16).eps / 2  # a rounding to bf16, relative


def rotate(x, positions, inv_freq, interleaved=False, scale=1.0):
    """x (B,T,H,D) -> fp64; positions (T) or (B,T)."""
    x = x.detach().double()
    B, T = x.shape[:2]
    n = inv_freq.numel()
    a = positions.double().expand(B, T).unsqueeze(-1) * inv_freq.double()
    c, s = a.cos().unsqueeze(2) * scale, a.sin().unsqueeze(2) * scale
    y = x.clone()
    if interleaved:
        x1, x2 = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        y[..., 0:2 * n:2], y[..., 1:2 * n:2] = x1 * c - x2 * s, x2 * c + x1 * s
    else:
        x1, x2 = x[..., :n], x[..., n:2 * n]
        y[..., :n], y[..., n:2 * n] = x1 * c - x2 * s, x2 * c + x1 * s
    return y


def depths(parents):
    """(T,) list of parents -> list of depths, None for a token that takes no part."""
    out = []
    for t, p in enumerate(parents):
        out.append(0 if p == -1 else out[p] + 1 if 0 <= p < t and out[p] is not None else None)
    return out


def visible(T, length, window, parents, mask_lmk, expand, n_slots):
    """(T, n_slots) truth values and the depths."""
    base = length - T
    see = torch.zeros(T, n_slots, dtype=torch.bool)
    if base < 0:
        return see
    up = list(range(-1, T - 1)) if parents is None else [int(p) for p in parents]
    dep = depths(up)
    for t in range(T):
        if dep[t] is None:
            continue
        left = base + dep[t] - window + 1
        left = left // S * S if expand else left
        mine = {}
        u = t
        while u >= 0:
            mine[base + u] = base + dep[u]
            u = up[u]
        where = torch.arange(min(base, n_slots))
        ok = where >= left
        if mask_lmk:
            ok &= where % S != S - 1
        see[t, : where.numel()] = ok
        for slot, at in mine.items():
            if slot < n_slots:
                see[t, slot] = at >= left and not (mask_lmk and at % S == S - 1)
    return see


def attend(q, k_pages, v_pages, table, lengths, window, parents=None, mask_lmk=True, expand=True, scale=None):
    """o, lse in fp64 and sum p |v| (what a rounding of the probabilities can change), on the CPU."""
    q, k_pages, v_pages, table = (x.detach().cpu() for x in (q, k_pages, v_pages, table))
    B, T, HQ, D = q.shape
    P, H = k_pages.shape[:2]
    n = table.shape[1] * S
    scale = 1 / math.sqrt(D) if scale is None else scale
    o = torch.zeros(B, T, HQ, D, dtype=torch.float64)
    lse = torch.full((B, T, HQ), -math.inf, dtype=torch.float64)
    weight = torch.zeros_like(o)
    for b in range(B):
        length = int(lengths[b]) if isinstance(lengths, torch.Tensor) else int(lengths)
        par = None if parents is None else (parents[b] if parents.dim() == 2 else parents).tolist()
        see = visible(T, length, window, par, mask_lmk, expand, n)
        page = table[b].long()
        mapped = (page >= 0) & (page < P)
        see &= mapped.repeat_interleave(S)
        some = see.any(0)
        first, last = (0, 0) if not some.any() else (int(some.nonzero()[0]) // S, int(some.nonzero()[-1]) // S + 1)
        see = see[:, first * S: last * S]
        page = page[first:last].clamp(0, P - 1)
        for h in range(H):
            k = k_pages[page, h].double().reshape(-1, D)
            v = v_pages[page, h].double().reshape(-1, D)
            for t in range(T):
                at = see[t].nonzero().flatten()
                if not at.numel():
                    continue
                g = slice(h * (HQ // H), (h + 1) * (HQ // H))
                s = q[b, t, g].double() @ k[at].T * scale
                z = torch.logsumexp(s, -1)
                p = (s - z.unsqueeze(-1)).exp()
                o[b, t, g] = p @ v[at]
                weight[b, t, g] = p @ v[at].abs()
                lse[b, t, g] = z
    return o, lse, weight


def attend_dense(q, k_pages, v_pages, table, lengths, window, parents=None, mask_lmk=True, expand=True):
    """attend() in 64-bit products over whole contexts, on the device of q: for sizes that take too long row by row."""
    B, T, HQ, D = q.shape
    H = k_pages.shape[1]
    n = table.shape[1] * S
    o = torch.zeros(B, T, HQ, D, dtype=torch.float64, device=q.device)
    lse = torch.full((B, T, HQ), -math.inf, dtype=torch.float64, device=q.device)
    weight = torch.zeros_like(o)
    for b in range(B):
        par = None if parents is None else parents[b].tolist()
        see = visible(T, int(lengths[b]), window, par, mask_lmk, expand, n).to(q.device)
        page = table[b].long()
        k, v = (torch.where(see.any(0)[:, None], x[page].double().transpose(0, 1).reshape(H, n, D), 0.0) for x in (k_pages, v_pages))
        s = (q[b].double().view(T, H, HQ // H, D).permute(1, 2, 0, 3).reshape(H, -1, D) @ k.transpose(1, 2)) / math.sqrt(D)
        s = s.view(H, HQ // H, T, n).masked_fill(~see, -math.inf)
        z = torch.logsumexp(s, -1)
        p = torch.where(see, (s - z.unsqueeze(-1)).exp(), 0.0).view(H, -1, n)
        for out, x in ((o, v), (weight, v.abs())):
            out[b] = (p @ x).view(H, HQ // H, T, D).permute(2, 0, 1, 3).reshape(T, HQ, D)
        lse[b] = z.permute(2, 0, 1).reshape(T, HQ)
    return o.cpu(), lse.cpu(), weight.cpu()


def check_attention(got, want, lse_tol=1e-4, slack=0.0):
    """o: its rounding and that of the probabilities, half a bf16 step each, and 2^-12 of the weighted values for the fp32
    scores (sums of up to 128 products of N(0,1) values: 128 * 2^-24 * sum |q k| scale <= 6e-5, twice) and exponentials.
    slack: what larger scores add to that."""
    (o, lse), (o_ref, lse_ref, weight) = got, want
    o, lse = o.detach().double().cpu(), lse.detach().double().cpu()
    assert torch.isfinite(o).all(), "not finite"
    bound = HALF * o_ref.abs() + (HALF + 2 ** -12 + slack) * weight + 1e-30
    worst = ((o - o_ref).abs() / bound).max().item()
    none = torch.isinf(lse_ref)
    assert torch.equal(torch.isinf(lse), none) and (lse[none] < 0).all() and (o[none] == 0).all()
    off = (lse - lse_ref)[~none].abs().max().item() if (~none).any() else 0.0
    print(f"    o: {worst:.3f} of its bound, lse off by {off:.2e}", flush=True)
    assert worst <= 1 and off <= lse_tol


def cache(gen, B, max_pages, H, D, dev, spare=3):
    """(k_pages, v_pages, table): random pages in random order, all mapped."""
    n = B * max_pages + spare
    k = torch.randn(n, H, S, D, generator=gen).bfloat16().to(dev)
    v = torch.randn(n, H, S, D, generator=gen).bfloat16().to(dev)
    table = torch.randperm(n, generator=gen)[: B * max_pages].view(B, max_pages).to(torch.int32).to(dev)
    return k, v, table


def tree(gen, T, wide=1.0):
    """A random tree: parents[t] in -1 .. t - 1."""
    return [int(torch.rand((), generator=gen).item() ** wide * (t + 1)) - 1 for t in range(T)]
