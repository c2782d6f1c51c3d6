"""What serving with drafted tokens on the paged cache is timed on: rotary positions, appending to pages, the local branch
on pages (single tokens, chains and trees of drafted tokens), accepting drafts, copying pages.

A cache is what ``HiLSPagedLayer`` keeps and what a serving backend that owns its pages keeps: K and V in pages of one chunk
(64 tokens), (pages, KV heads, 64, D) bf16, handed out in random order, and a page table per sequence; ragged lengths.
Head shapes are the repository's: 4/4, 16/2, 16/16, 32/4, 32/8 and 40/8 (query / KV heads) of 64 or 128; local windows of 64
or 512 tokens, or the whole context.

* ``rotary``  rotary positions of q and k given by position: forward and backward of training, or a prompt's forward.
* ``append``  the new tokens of a step or of prompts: q and k rotated, K and V written to their pages.
* ``attend``  the local branch for the last tokens of every sequence, straight on the pages.
* ``verify``  one verification of drafted tokens: append them at their depths' positions, attend with each token seeing the
              context and its own ancestors, and move the accepted ones to the front of the drafts' slots.
* ``pages``   pages of every pool copied: forks of sequences (the last, partly filled page of each), and compaction.

``own`` false: the plain form, elementary torch operations in 32 bits (64 for angles), rounded once.
"""
import math

import torch

own = False

S = 64  # tokens of a page


def _case(name, kind, batch, tokens, context, heads, window=0, tree=False, train=False, rotary=0, interleaved=False,
          stretch=1.0, copies=0):
    hq, hkv, d = heads
    case = {"kind": kind, "batch": batch, "tokens": tokens, "context": context, "q_heads": hq, "kv_heads": hkv,
            "head_dim": d, "window": window, "tree": tree, "train": train, "rotary_dim": rotary or d,
            "interleaved": interleaved, "stretch": stretch, "copies": copies}
    return {"name": name, **case} if name else case


def listed():
    return [
        # the benchmark's training layer: q and k of eight packed sequences, forward and backward
        _case("rotary_train_b8_8k", "rotary", 8, 8192, 8192, (16, 16, 64), train=True),
        # the benchmark's 32K prompt, interleaved pairs in half of the features, frequencies stretched for long contexts
        _case("rotary_prompt_32k", "rotary", 1, 32768, 32768, (32, 8, 128), rotary=64, interleaved=True, stretch=8.0),
        # one token for each of 32 sequences
        _case("append_step_b32", "append", 32, 1, 16384, (32, 8, 128), stretch=4.0),
        # four prompts of an odd length into empty caches
        _case("append_prompt_4x8k", "append", 4, 8191, 8191, (32, 4, 128)),
        # one user's chat with a small model: latency alone
        _case("attend_b1_4k", "attend", 1, 1, 4097, (16, 2, 64), 512),
        # a busy server's step, the layer's window
        _case("attend_b32_16k", "attend", 32, 1, 16384, (32, 8, 128), 512),
        # the same in a layer that sees everything
        _case("attend_b16_32k_full", "attend", 16, 1, 32768, (32, 8, 128), 32768),
        # a few drafts for one user
        _case("verify_b1_4k", "verify", 1, 26, 4096, (16, 2, 64), 512, tree=True),
        # trees for eight users
        _case("verify_b8_8k", "verify", 8, 63, 8192, (32, 8, 128), 512, tree=True, stretch=4.0),
        # large trees in a layer that sees everything
        _case("verify_b4_16k_full", "verify", 4, 64, 16384, (32, 4, 128), 16384, tree=True),
        # 32 forks: the last page of each
        _case("fork_b32", "pages", 32, 1, 4096, (32, 8, 128), copies=32),
        # half of a pool moved together
        _case("compact_2k_pages", "pages", 32, 1, 8192, (32, 8, 128), copies=2048),
    ]


_HEADS = [(4, 4, 64), (16, 2, 64), (16, 16, 64), (32, 4, 64), (32, 4, 128), (32, 8, 128), (40, 8, 128)]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["rotary", "append", "attend", "attend", "verify", "verify", "pages"])
    heads = rng.choice(_HEADS)
    hq, hkv, d = heads
    stretch = rng.choice([1.0, 4.0, 8.0])
    interleaved = rng.random() < 0.4
    rotary = rng.choice([d, d, d // 2])
    window = rng.choice([64, 512, 512, 1 << 20])
    if kind == "rotary":
        tokens = _log_int(rng, 1, 32768)
        batch = _log_int(rng, 1, max(1, min(32, 8192 * 8 * 16 * 64 // (tokens * hq * d))))
        return _case(None, kind, batch, tokens, tokens, heads, train=rng.random() < 0.5, rotary=rotary,
                     interleaved=interleaved, stretch=stretch)
    if kind == "append":
        tokens = _log_int(rng, 1, 8191)
        batch = _log_int(rng, 1, max(1, min(32, 4 * 8191 * 32 * 128 // (tokens * hq * d))))
        return _case(None, kind, batch, tokens, max(tokens, _log_int(rng, 64, 8192)), heads, rotary=rotary,
                     interleaved=interleaved, stretch=stretch)
    if kind == "pages":
        copies = _log_int(rng, 1, 2048)
        return _case(None, kind, _log_int(rng, 1, 32), 1, _log_int(rng, 64, 8192), heads, copies=copies)
    context = _log_int(rng, 256, 32768 if kind == "attend" else 16384)
    tokens = 1 if kind == "attend" and rng.random() < 0.6 else _log_int(rng, 1, min(128, context))
    # no more keys and values, and no more scores, than the listed cases have
    seen = min(window + tokens, context)
    batch = _log_int(rng, 1, max(1, min(32, 16 * 32768 * 8 * 128 // (context * hkv * d),
                                        4 * 64 * 32 * 16384 // (tokens * hq * seen))))
    return _case(None, kind, batch, tokens, context, heads, min(window, context), tree=kind == "verify" and rng.random() < 0.8,
                 rotary=rotary, interleaved=interleaved, stretch=stretch)


# ---- inputs ------------------------------------------------------------------------------------

def _randn(shape, gen, chunk=1 << 28):
    out = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
    flat = out.view(-1)
    for a in range(0, flat.numel(), chunk):
        flat[a:a + chunk].normal_(generator=gen)
    return out


def _frequencies(dim, stretch):
    """Angle per position of each pair, 64 bits: base 10000, long wavelengths divided by ``stretch`` with a ramp between the
    pairs that turn 32 times and once over 4096 positions; and the factor on the rotated features that goes with it."""
    inv = 10000.0 ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)
    turns = 4096 * inv / (2 * math.pi)
    keep = ((turns - 1) / (32 - 1)).clamp(0, 1)
    return inv * keep + inv / stretch * (1 - keep), 0.1 * math.log(stretch) + 1.0


def prepare(case, seed):
    c = dict(case)
    b, t, hq, hkv, d = c["batch"], c["tokens"], c["q_heads"], c["kv_heads"], c["head_dim"]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    st = {"case": c}
    st["inv_freq"], st["scale"] = _frequencies(c["rotary_dim"], c["stretch"])
    if c["kind"] == "pages":
        n = c["copies"]
        pages = 2 * n + 3
        st["pools"] = [_randn((pages, hkv, S, d), gen), _randn((pages, hkv, S, d), gen), _randn((pages, hkv, d), gen),
                       torch.randn(pages, hq, device="cuda", generator=gen)]  # K, V, chunk keys, prior bias
        order = torch.randperm(pages, device="cuda", generator=gen)
        st["src"], st["dst"] = order[:n].to(torch.int32), order[n:2 * n].to(torch.int32)
        return st
    st["q"] = _randn((b, t, hq, d), gen)
    if c["kind"] == "rotary":
        st["k"] = _randn((b, t, hkv, d), gen)
        # sequences packed one after the other: positions start again at a random place of each row
        cut = torch.randint(0, t + 1, (b, 1), device="cuda", generator=gen)
        at = torch.arange(t, device="cuda").view(1, t)
        st["positions"] = torch.where(at >= cut, at - cut, at).to(torch.int32)
        if c["train"]:
            st["d_q"], st["d_k"] = _randn((b, t, hq, d), gen), _randn((b, t, hkv, d), gen)
            st["q"].requires_grad_()
            st["k"].requires_grad_()
        return st
    # a cache: ragged lengths (the new tokens included), pages in random order
    least = max(t, c["context"] // 2) if c["kind"] != "append" or t == 1 else c["context"]
    st["lengths"] = torch.randint(least, c["context"] + 1, (b,), device="cuda", generator=gen, dtype=torch.int32)
    n = -(-c["context"] // S)
    st["table"] = torch.randperm(b * n + 5, device="cuda", generator=gen)[: b * n].view(b, n).to(torch.int32)
    st["k_pages"], st["v_pages"] = _randn((b * n + 5, hkv, S, d), gen), _randn((b * n + 5, hkv, S, d), gen)
    base = st["lengths"].view(b, 1) - t
    if c["kind"] == "attend":
        return st
    st["k"], st["v"] = _randn((b, t, hkv, d), gen), _randn((b, t, hkv, d), gen)
    st["positions"] = base + torch.arange(t, device="cuda", dtype=torch.int32)
    if c["kind"] == "verify":
        st["base"] = base.view(b).contiguous()
        st["parents"] = None
        seen = torch.ones(b, t, t, device="cuda").tril()
        if c["tree"]:
            place = torch.rand(b, t, device="cuda", generator=gen) * torch.arange(1, t + 1, device="cuda")
            st["parents"] = place.to(torch.int32).clamp_max(torch.arange(t, device="cuda", dtype=torch.int32)) - 1
            seen = _ancestors(st["parents"])
        st["positions"] = base + seen.sum(-1).to(torch.int32) - 1
        # the accepted tokens: the way to one of the drafts, cut at 16
        leaf = torch.randint(0, t, (b,), device="cuda", generator=gen)
        on = seen[torch.arange(b, device="cuda"), leaf] > 0
        way = torch.where(on, torch.arange(t, device="cuda"), t).sort(-1).values[:, :16]
        st["path"] = torch.where(way < t, way, -1).to(torch.int32).contiguous()
    return st


# ---- the plain form ----------------------------------------------------------------------------

def _ancestors(parents):
    """(B, T, T): 1 where the second token is the first or an ancestor of it.  With A the matrix of parents, the sum of all
    powers of A, which is the inverse of 1 - A (whole numbers throughout)."""
    b, t = parents.shape
    links = torch.zeros(b, t, t + 1, device=parents.device)
    links.scatter_(2, parents.long().unsqueeze(-1) + 1, 1.0)
    one = torch.eye(t, device=parents.device).expand(b, t, t)
    return torch.linalg.solve_triangular(one - links[:, :, 1:], one, upper=False)


def _rotate(x, positions, inv_freq, scale, interleaved):
    r = 2 * inv_freq.numel()
    angle = positions.to(torch.float64).unsqueeze(-1) * inv_freq
    cos, sin = (angle.cos() * scale).float().unsqueeze(2), (angle.sin() * scale).float().unsqueeze(2)
    head, rest = x[..., :r].float(), x[..., r:].float()
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        out = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = head[..., : r // 2], head[..., r // 2:]
        out = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([out, rest], -1).to(x.dtype)


def _slots(st, first, count):
    """(page, place in it) of `count` tokens from `first` (B, 1) on."""
    slot = first.long() + torch.arange(count, device=first.device)
    return st["table"].long().gather(1, slot // S), slot % S


def _plain_append(st, c):
    q = _rotate(st["q"], st["positions"], st["inv_freq"], st["scale"], c["interleaved"])
    k = _rotate(st["k"], st["positions"], st["inv_freq"], st["scale"], c["interleaved"])
    page, at = _slots(st, st["lengths"].view(-1, 1) - c["tokens"], c["tokens"])
    st["k_pages"][page, :, at] = k
    st["v_pages"][page, :, at] = st["v"]
    return q


def _plain_attend(st, c, q, parents):
    b, t, hq, d = q.shape
    h, w = c["kv_heads"], c["window"]
    base = st["lengths"].long().view(b, 1) - t
    first = torch.div(base - w + 1, S, rounding_mode="floor").clamp_min(0)  # page where the first token's window begins
    n = min(st["table"].shape[1], (w + t + 2 * S - 2) // S)
    number = first + torch.arange(n, device=q.device)
    page = st["table"].long().gather(1, number.clamp_max(st["table"].shape[1] - 1))
    k = st["k_pages"][page].float().transpose(1, 2).reshape(b, h, n * S, d)
    v = st["v_pages"][page].float().transpose(1, 2).reshape(b, h, n * S, d)
    slot = (number.unsqueeze(-1) * S + torch.arange(S, device=q.device)).view(b, 1, n * S)
    if parents is None:
        seen = torch.ones(t, t, device=q.device).tril().expand(b, t, t)
    else:
        seen = _ancestors(parents)
    where = base + seen.sum(-1).long() - 1                                  # position of every new token
    left = torch.div(where - w + 1, S, rounding_mode="floor").unsqueeze(-1) * S
    draft = (slot - base.unsqueeze(-1)).clamp(0, t - 1)                     # new token that lies in a slot
    is_new = (slot >= base.unsqueeze(-1)) & (slot < base.unsqueeze(-1) + t)
    at = torch.where(is_new, where.unsqueeze(1).gather(2, draft), slot)     # position of a slot's token
    mine = seen.gather(2, draft.expand(b, t, n * S)) > 0
    visible = (at >= left) & ((at + 1) % S != 0) & ((slot < base.unsqueeze(-1)) | (is_new & mine))
    qq = q.float().view(b, t, h, hq // h, d).permute(0, 2, 1, 3, 4).reshape(b, h, t * (hq // h), d)
    s = torch.matmul(qq, k.transpose(-1, -2)).view(b, h, t, hq // h, n * S) / math.sqrt(d)
    s = torch.where(visible.view(b, 1, t, 1, n * S), s, -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m > -math.inf, m, 0.0)
    e = (s - m).exp()
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e.view(b, h, -1, n * S), v).view(b, h, t, hq // h, d) / torch.where(total > 0, total, 1.0)
    lse = (total.log() + m).squeeze(-1)
    return (o.permute(0, 2, 1, 3, 4).reshape(b, t, hq, d).to(q.dtype), lse.permute(0, 2, 1, 3).reshape(b, t, hq))


def _plain_accept(st, c):
    path = st["path"].long()
    b, n = path.shape
    base = st["base"].long().view(b, 1)
    to_page, to_at = _slots(st, base, n)
    slot = base + path.clamp_min(0)
    page, at = st["table"].long().gather(1, slot // S), slot % S
    taken = (path >= 0).view(b, n, 1, 1)
    k, v = st["k_pages"], st["v_pages"]
    k[to_page, :, to_at] = torch.where(taken, k[page, :, at], k[to_page, :, to_at])
    v[to_page, :, to_at] = torch.where(taken, v[page, :, at], v[to_page, :, to_at])


def _plain(st, c):
    kind = c["kind"]
    if kind == "rotary":
        rot = lambda x: _rotate(x, st["positions"], st["inv_freq"], st["scale"], c["interleaved"])
        q, k = rot(st["q"]), rot(st["k"])
        if not c["train"]:
            return {"q": q, "k": k}
        d_q, d_k = torch.autograd.grad([q, k], [st["q"], st["k"]], [st["d_q"], st["d_k"]])
        return {"q": q.detach(), "k": k.detach(), "d_q": d_q, "d_k": d_k}
    if kind == "append":
        return {"q": _plain_append(st, c), "k_pages": st["k_pages"], "v_pages": st["v_pages"]}
    if kind == "attend":
        o, lse = _plain_attend(st, c, st["q"], None)
        return {"o": o, "lse": lse}
    if kind == "verify":
        o, lse = _plain_attend(st, c, _plain_append(st, c), st["parents"])
        _plain_accept(st, c)
        return {"o": o, "lse": lse, "k_pages": st["k_pages"], "v_pages": st["v_pages"]}
    src, dst = st["src"].long(), st["dst"].long()
    keys, values, chunk_keys, bias = st["pools"]
    keys[dst] = keys[src]
    values[dst] = values[src]
    chunk_keys[dst] = chunk_keys[src]
    bias[dst] = bias[src]
    return {"pools": st["pools"]}


# ---- one pass ----------------------------------------------------------------------------------

_package = None


def _pkg():
    global _package
    if _package is None:
        import __graft_entry__
        _package = __graft_entry__.load_package()
    return _package


def _own(st, c):
    pkg, kind = _pkg(), c["kind"]
    turn = {"interleaved": c["interleaved"], "scale": st["scale"]}
    if kind == "rotary":
        q, k = pkg.rotary_embedding(st["q"], st["k"], st["positions"], st["inv_freq"], **turn)
        if not c["train"]:
            return {"q": q, "k": k}
        d_q, d_k = torch.autograd.grad([q, k], [st["q"], st["k"]], [st["d_q"], st["d_k"]])
        return {"q": q.detach(), "k": k.detach(), "d_q": d_q, "d_k": d_k}
    if kind == "pages":
        pkg.copy_pages(st["pools"], st["src"], st["dst"])
        return {"pools": st["pools"]}
    cache = (st["k_pages"], st["v_pages"], st["table"])
    q, parents = st["q"], None
    if kind in ("append", "verify"):
        q = pkg.paged_append(st["k"], st["v"], *cache, st["lengths"], q=q, inv_freq=st["inv_freq"],
                             positions=st["positions"], **turn)
        if kind == "append":
            return {"q": q, "k_pages": st["k_pages"], "v_pages": st["v_pages"]}
        parents = st["parents"]
    o, lse = pkg.paged_flex_attn(q, *cache, st["lengths"], c["window"], parents=parents)
    if kind == "attend":
        return {"o": o, "lse": lse}
    pkg.paged_accept(*cache, st["base"], st["path"])
    return {"o": o, "lse": lse, "k_pages": st["k_pages"], "v_pages": st["v_pages"]}


def run(state):
    return _own(state, state["case"]) if own else _plain(state, state["case"])


# ---- work --------------------------------------------------------------------------------------

def work(case):
    c = case
    b, t, hq, hkv, d = c["batch"], c["tokens"], c["q_heads"], c["kv_heads"], c["head_dim"]
    q_bytes, kv_bytes = 2 * b * t * hq * d, 2 * b * t * hkv * d  # of q, and of k or v
    turned = b * t * (hq + hkv) * c["rotary_dim"]                # features that are rotated
    if c["kind"] == "rotary":
        times = 2 if c["train"] else 1
        return {"bytes": times * 2 * (q_bytes + kv_bytes) + 4 * b * t, "flops": times * 3 * turned}
    if c["kind"] == "pages":
        return {"bytes": 2 * c["copies"] * (2 * 2 * hkv * S * d + 2 * hkv * d + 4 * hq), "flops": 0}
    append = {"bytes": 2 * q_bytes + 4 * kv_bytes + 4 * b * t, "flops": 3 * turned}
    if c["kind"] == "append":
        return append
    # lengths are spread evenly over the upper half of the context; a window begins at its chunk's first token
    length = (max(t, c["context"] // 2) + c["context"]) / 2
    context = min(length - t, c["window"] - 1 + (S - 1) / 2)
    ancestors = max(1.0, math.log(t + 1)) if c["tree"] else (t + 1) / 2  # a random tree's depth, a chain's mean
    attend = {"bytes": 2 * q_bytes + 4 * b * t * hq + 4 * b * hkv * d * (context + t),
              "flops": 4 * d * hq * b * t * (context + ancestors)}
    if c["kind"] == "attend":
        return attend
    moved = 2 * 4 * b * hkv * d * min(16, ancestors)  # K and V of the accepted tokens, read and written
    return {"bytes": append["bytes"] + attend["bytes"] + moved, "flops": append["flops"] + attend["flops"]}


# ---- in 64 bits, from the definitions ------------------------------------------------------------

def _exact_rotation(x, positions, st, c):
    """Pairs as complex numbers times scale * exp(i angle)."""
    r = c["rotary_dim"]
    x = x.detach().double()
    pairs = x[..., :r].unflatten(-1, (r // 2, 2)) if c["interleaved"] else x[..., :r].unflatten(-1, (2, r // 2)).transpose(-1, -2)
    angle = torch.outer(positions.reshape(-1).double(), st["inv_freq"]).view(*positions.shape, 1, r // 2)
    z = torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.full_like(angle, st["scale"]), angle)
    y = torch.view_as_real(z)
    y = y.flatten(-2) if c["interleaved"] else y.transpose(-1, -2).flatten(-2)
    return torch.cat([y, x[..., r:]], -1)


def _exact_cache(st, c):
    """Keys and values of every sequence in token order after the append, bf16 as the cache holds them, and the pages."""
    pages = {"k": st["k_pages"].clone(), "v": st["v_pages"].clone()}
    if "k" in st:
        new = {"k": _exact_rotation(st["k"], st["positions"], st, c).to(torch.bfloat16), "v": st["v"]}
        for i in range(c["batch"]):
            n = int(st["lengths"][i])
            slot = torch.arange(n - c["tokens"], n, device="cuda")
            page = st["table"][i].long()[slot // S]
            for x in ("k", "v"):
                pages[x][page, :, slot % S] = new[x][i]
    return pages


def exact(case, seed):
    c = dict(case)
    st = prepare(case, seed)
    kind, t, h, d = c["kind"], c["tokens"], c["kv_heads"], c["head_dim"]
    if kind == "pages":
        pools = []
        for pool in st["pools"]:
            order = torch.arange(pool.shape[0], device="cuda")
            order[st["dst"].long()] = st["src"].long()
            pools.append(pool.index_select(0, order).double())
        return {"pools": pools}
    if kind == "rotary":
        out = {x: _exact_rotation(st[x], st["positions"], st, c) for x in ("q", "k")}
        if c["train"]:  # the transposed map: the rotation the other way round
            out |= {"d_" + x: _exact_rotation(st["d_" + x], -st["positions"], st, c) for x in ("q", "k")}
        return out
    pages = _exact_cache(st, c)
    if kind == "append":
        # (pages in 64 bits are those of the state with the new tokens' exact values, before their rounding)
        q = _exact_rotation(st["q"], st["positions"], st, c)
        k = _exact_rotation(st["k"], st["positions"], st, c)
        wide = {x: st[x + "_pages"].double() for x in ("k", "v")}
        for i in range(c["batch"]):
            n = int(st["lengths"][i])
            slot = torch.arange(n - t, n, device="cuda")
            page = st["table"][i].long()[slot // S]
            wide["k"][page, :, slot % S] = k[i]
            wide["v"][page, :, slot % S] = st["v"][i].double()
        return {"q": q, "k_pages": wide["k"], "v_pages": wide["v"]}
    # the query that the attention is given is the rounded one
    q = st["q"] if kind == "attend" else _exact_rotation(st["q"], st["positions"], st, c).to(torch.bfloat16)
    o, z = torch.empty(q.shape, dtype=torch.float64, device="cuda"), torch.empty(q.shape[:3], dtype=torch.float64, device="cuda")
    for i in range(c["batch"]):
        n = int(st["lengths"][i])
        base = n - t
        up = list(range(-1, t - 1)) if st.get("parents") is None else st["parents"][i].tolist()
        ways = []
        for x in range(t):
            ways.append((ways[up[x]] if up[x] >= 0 else []) + [x])
        start = max(0, (base - c["window"] + 1) // S * S)
        at = torch.cat([torch.arange(start, base), torch.tensor([base + len(w) - 1 for w in ways])])
        sees = torch.zeros(t, base - start + t, dtype=torch.bool)
        for x, w in enumerate(ways):
            here = base + len(w) - 1
            sees[x, : base - start] = True
            sees[x, torch.tensor(w) + base - start] = True
            sees[x] &= (at >= (here - c["window"] + 1) // S * S) & (at % S != S - 1)
        sees = sees.cuda()
        page = st["table"][i].long()[start // S: -(-n // S)]
        k, v = (pages[x][page].double().permute(1, 0, 2, 3).reshape(h, -1, d)[:, start % S: start % S + n - start] for x in ("k", "v"))
        for g in range(h):
            mine = slice(g * (c["q_heads"] // h), (g + 1) * (c["q_heads"] // h))
            s = (q[i, :, mine].double().reshape(-1, d) @ k[g].T).view(t, -1, n - start) / math.sqrt(d)
            s = s.masked_fill(~sees.unsqueeze(1), -math.inf)
            z[i, :, mine] = torch.logsumexp(s, -1)
            p = (s - z[i, :, mine].unsqueeze(-1).clamp_min(-1e300)).exp()
            o[i, :, mine] = (p.view(-1, n - start) @ v[g]).view(t, -1, d)
    if kind == "attend":
        return {"o": o, "lse": z}
    for i in range(c["batch"]):
        way = [x for x in st["path"][i].tolist() if x >= 0]
        table = st["table"][i].long()
        new = torch.arange(len(way), device="cuda") + int(st["base"][i])
        old = torch.tensor(way, device="cuda") + int(st["base"][i])
        for x in ("k", "v"):
            pages[x][table[new // S], :, new % S] = pages[x][table[old // S], :, old % S].clone()
    return {"o": o, "lse": z, "k_pages": pages["k"].double(), "v_pages": pages["v"].double()}
