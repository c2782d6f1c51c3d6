"""The paged layer's lists of pages where a call is refused, on the CPU."""
import pytest
import torch

from util import note


def test_refused_update_gives_its_pages_back(pkg):
    note("a refused update on the CPU")
    c = pkg.HiLSPagedLayer(num_pages=6, batch=2, max_pages_per_seq=3, num_kv_heads=1, head_dim=16, device="cpu")
    z = lambda t: torch.ones(2, t, 1, 16, dtype=torch.bfloat16)
    c.update(z(10), z(10))
    for n in (3, 60, 100):
        with pytest.raises(AssertionError, match="rotation"):
            c.update(z(n), z(n), q=z(n)) if n < 54 else c.draft(z(n), z(n), q=z(n))
        assert c.seq_len == 10 and [len(p) for p in c._pages] == [1, 1] and len(c.free_pages) == 4
        assert (c.page_table[:, 1:] == -1).all() and sorted(c.free_pages + c._pages[0] + c._pages[1]) == list(range(6))
    c.update(z(50), z(50))
    c.draft(z(60), z(60))
    assert c.seq_len == 60 and [len(p) for p in c._pages] == [2, 2] and len(c.free_pages) == 2
    k, _ = c.gather_contiguous()
    assert k.shape == (2, 60, 1, 16) and (k == 1).all()
