"""New and drafted tokens on a paged cache (page = chunk = 64 tokens): append, local branch, acceptance, page copies.

The layouts are those of ``HiLSPagedLayer`` and ``paged_hils_attend``: k_pages, v_pages (num_pages, H, 64, D) bf16,
page_table (B, max_pages) int32 (entries outside the pool: not mapped).  Lengths are an int for all sequences or an int32
tensor (B,) on the GPU; a sequence shorter than the T tokens of a call takes no part in it.  Everything runs on the current
stream and synchronises nothing; inference only: a backward through an output, tangents and pages that require gradients
where they are written are refused.
"""
import torch

from . import _cabi
from ._native_op import InferenceOp


class _PagedAppend(InferenceOp):
    label, written = "paged_append", slice(2, 4)

    @staticmethod
    def native(*args):
        return _cabi.host().paged_append(*args)

    @staticmethod
    def forward(ctx, *args):
        return _PagedAppend.native(*args)

    @staticmethod
    def backward(ctx, *grads):
        _PagedAppend.refuse()


class _PagedFlexAttn(InferenceOp):
    label = "paged_flex_attn"

    @staticmethod
    def native(*args):
        return _cabi.host().paged_flex_attn(*args)

    @staticmethod
    def forward(ctx, *args):
        return _PagedFlexAttn.native(*args)

    @staticmethod
    def backward(ctx, *grads):
        _PagedFlexAttn.refuse()


class _PagedAccept(InferenceOp):
    label, written = "paged_accept", slice(0, 2)

    @staticmethod
    def native(*args):
        return _cabi.host().paged_accept(*args)

    @staticmethod
    def forward(ctx, *args):
        return _PagedAccept.native(*args)


class _CopyPages(InferenceOp):
    label, written = "copy_pages", slice(2, None)

    @staticmethod
    def native(src, dst, *pools):
        return _cabi.host().copy_pages(pools, src, dst)

    @staticmethod
    def forward(ctx, *args):
        return _CopyPages.native(*args)


def paged_append(k, v, k_pages, v_pages, page_table, seq_len, q=None, inv_freq=None, positions=None, interleaved=False,
                 scale=1.0):
    """Write keys and values (B,T,H,D) of the last T of ``seq_len`` tokens into their pages, in one launch; tokens whose
    page is not mapped, and sequences shorter than T, are left out.  With ``inv_freq`` the keys, and q (B,T,H_q,D) if given,
    are rotated on the way as by ``rotary_embedding``, at ``positions`` (B,T) or, without them, at the tokens' slots.
    Returns the rotated q or None."""
    return _PagedAppend.apply(k, v, k_pages, v_pages, page_table, seq_len, q, inv_freq, positions, bool(interleaved), float(scale))


def paged_flex_attn(q, k_pages, v_pages, page_table, seq_len, window_size, parents=None, mask_lmk=True,
                    expand_to_chunk=True, sm_scale=None):
    """Local branch of the last T tokens straight on the pages: ``flex_attn_tl(..., training=False)`` on the cache that the
    pages hold (chunks of 64), and its form for trees of drafted tokens.

    q (B,T,H_q,D) bf16, any strides; ``seq_len`` tokens with the T new ones, which are in the pages already.  ``parents``
    int32 (T,) or (B,T): token t follows the new token parents[t] < t, or the last committed one (-1); it sits at position
    seq_len - T + depth and sees the committed tokens of its window, itself and its ancestors.  Tokens with any other parent,
    and those that follow them, see nothing (padding).  Without ``parents`` the tokens are a chain.  T <= 256 for a tree.
    Returns o (B,T,H_q,D) bf16 and lse (B,T,H_q) fp32, natural log; rows that see nothing: 0 and -inf.  The same call gives
    the same bits; a sequence's last bits may depend on how many others, and how long ones, are in the batch."""
    return _PagedFlexAttn.apply(q, k_pages, v_pages, page_table, seq_len, int(window_size), parents, bool(mask_lmk),
                                bool(expand_to_chunk), sm_scale)


def paged_accept(k_pages, v_pages, page_table, base_len, path):
    """Move accepted drafts to the front: keys and values at slots ``base_len + path[b][i]`` go to ``base_len + i``.
    ``path`` int32 (B,n) on the GPU, growing strictly; the first entry that does not (-1, say) ends it.  The pages from slot
    ``base_len`` on must be the sequence's own."""
    _PagedAccept.apply(k_pages, v_pages, page_table, base_len, path)


def copy_pages(pools, src, dst):
    """``pool[dst[i]] = pool[src[i]]`` for every i and every pool, in one launch.  ``pools``: up to eight contiguous tensors
    with the same number of pages (first dimension), any types.  ``src``, ``dst``: int32 or int64 vectors on the GPU, or
    sequences of ints.  Pairs with an index out of range are left out.  A page that is written must be in no other pair:
    checked for sequences, the caller's duty for tensors on the GPU (pieces of the pages that meet there are mixed)."""
    pools = list(pools)
    if not isinstance(src, torch.Tensor) or not isinstance(dst, torch.Tensor):
        src, dst = [int(x) for x in src], [int(x) for x in dst]
        if len(src) != len(dst):
            raise ValueError(f"copy_pages: {len(src)} sources and {len(dst)} destinations")
        n = pools[0].shape[0] if pools and pools[0].dim() else 0
        pairs = [(a, b) for a, b in zip(src, dst) if a != b and 0 <= a < n and 0 <= b < n]  # (the others are left out)
        written = [b for _, b in pairs]
        if len(set(written)) < len(written) or set(written) & {a for a, _ in pairs}:
            raise ValueError("copy_pages: a page that is written is in another pair too")
        dev = pools[0].device if pools else None
        src, dst = (torch.tensor(x, dtype=torch.int64, device=dev) for x in (src, dst))
    _CopyPages.apply(src, dst, *pools)
