"""What the operators on a paged cache and the rotary positions refuse: through the C ABI and from Python without a GPU
(no kernel is launched), and with tensors on a GPU."""
import ctypes

import pytest
import torch

from util import note

B = ctypes.c_void_p(1 << 20)  # never read: every call is refused before a launch


def _lib(pkg):
    from hils_attention_amd.ops import _cabi
    return _cabi.load()


def _refused(lib, rc, text):
    assert rc == 1 and text in lib.hils_last_error().decode(), lib.hils_last_error()


def test_attention_arguments(pkg):
    lib = _lib(pkg)

    def call(q=B, parents=None, lengths=None, ws=None, wsb=0, st=(512, 256, 64), nb=1, T=4, HQ=4, H=2, D=64, mp=4, n=9, sl=200,
             window=64, scale=0.1, table=B):
        return lib.hils_paged_attn(q, B, B, table, lengths, parents, B, B, ws, wsb, *st, nb, T, HQ, H, D, mp, n, sl, 0, window, 1, 1,
                                   scale, None)

    for kw, text in [({"q": None}, "null pointer"), ({"table": None}, "null pointer"), ({"T": 0}, "positive"), ({"n": 0}, "positive"),
                     ({"HQ": 5}, "multiple of H"), ({"D": 96}, "64 or 128"), ({"window": 0}, "window"), ({"scale": 0.0}, "sm_scale"),
                     ({"scale": -1.0}, "sm_scale"), ({"scale": float("inf")}, "sm_scale"), ({"scale": float("nan")}, "sm_scale"),
                     ({"parents": B, "T": 257, "sl": 256, "mp": 5}, "at most 256"), ({"sl": 3}, "seq_len"), ({"sl": 257}, "seq_len"),
                     ({"st": (512, 256, 60)}, "16 bytes"), ({"q": ctypes.c_void_p((1 << 20) + 8)}, "16 bytes"),
                     ({"mp": 1 << 25}, "too wide"), ({"nb": 70000}, "grid"),
                     ({"T": 1, "window": 1 << 20, "mp": 4096, "sl": 1 << 18}, "workspace too short")]:
        _refused(lib, call(**kw), text)
    need = lib.hils_paged_attn_workspace(1, 1, 4, 2, 64, 1 << 20, 4096)
    assert need > 0
    _refused(lib, call(T=1, window=1 << 20, mp=4096, sl=1 << 18, ws=B, wsb=need - 1), "workspace too short")
    assert lib.hils_paged_attn_workspace(32, 1, 32, 8, 128, 64, 4096) == 0
    assert lib.hils_paged_attn_workspace(0, 1, 32, 8, 128, 64, 4096) == 0


def test_rotary_arguments(pkg):
    lib = _lib(pkg)

    def call(q=B, k=B, inv=B, st=(512, 256, 64), nb=1, T=4, HQ=4, H=2, D=64, R=64):
        return lib.hils_rotary(q, k, B, B, None, inv, *st, *st, nb, T, HQ, H, D, R, 0, 0, 0, 0, 1, 1.0, 1.0, None)

    for kw, text in [({"q": None}, "null"), ({"k": None}, "null"), ({"inv": None}, "null"), ({"T": 0}, "positive"), ({"D": 72}, "multiple of 16"),
                     ({"D": 2048}, "1024"), ({"R": 24}, "rotary_dim"), ({"R": 0}, "rotary_dim"), ({"R": 80}, "rotary_dim"),
                     ({"st": (512, 256, 4)}, "16 bytes"), ({"HQ": 1 << 20}, "heads")]:
        _refused(lib, call(**kw), text)


def test_append_arguments(pkg):
    lib = _lib(pkg)

    def call(q=B, k=B, v=B, inv=B, st=(512, 256, 64), nb=1, T=4, HQ=4, H=2, D=64, R=64, mp=4, n=9, sl=100, table=B):
        return lib.hils_paged_append(q, k, v, B, B, B, table, None, None, inv, *st, *st, *st, nb, T, HQ, H, D, R, 0, 0, 1, mp, n, sl, 1.0, None)

    for kw, text in [({"k": None}, "null"), ({"v": None}, "null"), ({"q": None}, "null"), ({"inv": None}, "null"), ({"table": None}, "null"),
                     ({"H": 0}, "positive"), ({"R": 0}, "inv_freq"), ({"R": 65}, "rotary_dim"), ({"sl": 3}, "seq_len"), ({"sl": 257}, "seq_len"),
                     ({"D": 24}, "multiple of 16"), ({"st": (512, 250, 64)}, "16 bytes"), ({"mp": 1 << 25, "sl": 4}, "too wide")]:
        _refused(lib, call(**kw), text)


def test_move_arguments(pkg):
    lib = _lib(pkg)
    acc = lambda path=B, nb=1, n=4, D=64, base=0, mp=4: lib.hils_paged_accept(B, B, B, None, path, nb, n, 2, D, mp, 9, base, None)
    for kw, text in [({"path": None}, "null"), ({"n": 0}, "256"), ({"n": 257}, "256"), ({"D": 12}, "multiple of 8"), ({"base": -1}, "base"),
                     ({"nb": 70000}, "sequences"), ({"nb": 0}, "positive"), ({"mp": 1 << 25}, "too wide")]:
        _refused(lib, acc(**kw), text)
    pools, sizes = (ctypes.c_void_p * 9)(*[1 << 20] * 9), (ctypes.c_size_t * 9)(*[128] * 9)
    cp = lambda p=pools, s=sizes, np=2, n=3, pages=9, src=B: lib.hils_copy_pages(p, s, src, B, np, n, pages, 0, None)
    for kw, text in [({"p": None}, "null"), ({"src": None}, "null"), ({"np": 0}, "pools"), ({"np": 9}, "pools"), ({"n": 0}, "positive"),
                     ({"p": (ctypes.c_void_p * 2)(1 << 20, 0)}, "null"), ({"s": (ctypes.c_size_t * 2)(0, 1)}, "page size"),
                     ({"s": (ctypes.c_size_t * 2)(1 << 39, 1 << 39), "n": 100}, "too")]:
        _refused(lib, cp(**kw), text)


def _cache(dev, D=64):
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device=dev)
    return z(9, 2, 64, D), z(9, 2, 64, D), z(2, 4, dtype=torch.int32)


def test_python_without_a_gpu(pkg):
    kp, vp, table = _cache("cpu")
    q, k = torch.zeros(2, 3, 4, 64).bfloat16(), torch.zeros(2, 3, 2, 64).bfloat16()
    inv, _ = pkg.rotary_frequencies(64, device="cpu")
    for call in (lambda: pkg.paged_flex_attn(q, kp, vp, table, 100, 64), lambda: pkg.paged_append(k, k, kp, vp, table, 100),
                 lambda: pkg.rotary_embedding(q, k, 0, inv), lambda: pkg.copy_pages([kp], [1], [2])):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
    with pytest.raises(RuntimeError, match="no CPU path"):
        pkg.paged_accept(kp, vp, table, 3, torch.zeros(2, 3, dtype=torch.int32))
    for pairs, text in ((([1, 2], [3]), "2 sources"), (([1, 2], [3, 3]), "another pair"), (([1, 2], [2, 5]), "another pair"),
                        (([1, 5], [5, 6]), "another pair")):
        with pytest.raises(ValueError, match=text):
            pkg.copy_pages([kp], *pairs)
    for kw in ({"rotary_dim": 7}, {"rotary_dim": 0}, {"rotary_dim": 64, "base": 1.0}, {"rotary_dim": 64, "factor": 0.5},
               {"rotary_dim": 64, "scaling": "other"}, {"rotary_dim": 64, "scaling": "yarn"}, {"rotary_dim": 2, "scaling": "ntk"},
               {"rotary_dim": 64, "scaling": "yarn", "original_length": 100, "low": 5, "high": 5}):
        with pytest.raises(ValueError):
            pkg.rotary_frequencies(device="cpu", **kw)


@pytest.mark.gpu
def test_python_on_a_gpu(pkg, dev):
    note("refusals of tensors on a GPU")
    kp, vp, table = _cache(dev)
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device=dev)
    q, k, inv = z(2, 3, 4, 64), z(2, 3, 2, 64), pkg.rotary_frequencies(64, device=dev)[0]
    attn = lambda **kw: pkg.paged_flex_attn(**{**dict(q=q, k_pages=kp, v_pages=vp, page_table=table, seq_len=100, window_size=64), **kw})
    i32 = lambda *s: z(*s, dtype=torch.int32)
    for kw, kind, text in [
            ({"q": q.float()}, TypeError, "bfloat16"), ({"q": q[0]}, AssertionError, "four"), ({"q": z(2, 3, 5, 64)}, AssertionError, "multiple"),
            ({"q": z(2, 3, 4, 128)}, AssertionError, "64 or 128"), ({"k_pages": kp.transpose(1, 2)}, AssertionError, "contiguous"),
            ({"v_pages": vp[:5]}, AssertionError, "contiguous"), ({"page_table": table.long()}, AssertionError, "int32"),
            ({"page_table": table[:1]}, AssertionError, "int32"), ({"page_table": table.t().contiguous().t()}, AssertionError, "contiguous"),
            ({"seq_len": 2}, AssertionError, "between 3"), ({"seq_len": 257}, AssertionError, "256"), ({"seq_len": i32(3)}, AssertionError, "lengths"),
            ({"seq_len": i32(2).long()}, AssertionError, "int32"), ({"seq_len": i32(2).cpu()}, RuntimeError, "GPU"),
            ({"window_size": 0}, AssertionError, "window"), ({"parents": i32(4)}, AssertionError, "parents"),
            ({"parents": i32(3).long()}, AssertionError, "parents"), ({"parents": i32(3).cpu()}, RuntimeError, "GPU"),
            ({"sm_scale": 0.0}, AssertionError, "sm_scale"), ({"q": z(2, 257, 4, 64), "parents": i32(257), "seq_len": i32(2)}, AssertionError, "256")]:
        with pytest.raises(kind, match=text):
            attn(**kw)
    rot = lambda **kw: pkg.rotary_embedding(**{**dict(q=q, k=k, positions=i32(3), inv_freq=inv), **kw})
    for kw, kind, text in [({"k": k[:1]}, AssertionError, "go with"), ({"positions": z(3)}, TypeError, "int32"), ({"positions": i32(4)}, AssertionError, "positions"),
                           ({"inv_freq": inv[:5]}, AssertionError, "multiple of 16"), ({"inv_freq": inv.half()}, AssertionError, "fp32"),
                           ({"inv_freq": torch.cat([inv, inv])}, AssertionError, "head dim"), ({"inv_freq": inv.clone().requires_grad_()}, RuntimeError, "gradient"),
                           ({"positions": 2 ** 31}, AssertionError, "range"), ({"q": z(2, 3, 4, 40), "k": None}, AssertionError, "multiple of 16"),
                           ({"scale": float("inf")}, AssertionError, "finite"), ({"positions": i32(3).cpu()}, RuntimeError, "tensors on")]:
        with pytest.raises(kind, match=text):
            rot(**kw)
    app = lambda **kw: pkg.paged_append(**{**dict(k=k, v=k, k_pages=kp, v_pages=vp, page_table=table, seq_len=100), **kw})
    for kw, kind, text in [({"v": k[:, :1]}, AssertionError, "must be"), ({"q": q}, AssertionError, "inv_freq is missing"), ({"positions": i32(2, 3)}, AssertionError, "missing"),
                           ({"k": z(2, 3, 4, 64), "v": z(2, 3, 4, 64)}, AssertionError, "pages of"), ({"inv_freq": inv, "positions": i32(3)}, AssertionError, "positions"),
                           ({"inv_freq": inv, "q": q[:, :2]}, AssertionError, "go with"), ({"k": k.float()}, TypeError, "bfloat16"), ({"seq_len": 2}, AssertionError, "between")]:
        with pytest.raises(kind, match=text):
            app(**kw)
    with pytest.raises(AssertionError, match="path"):
        pkg.paged_accept(kp, vp, table, 3, i32(2, 3).long())
    with pytest.raises(AssertionError, match="256"):
        pkg.paged_accept(kp, vp, table, 3, i32(2, 257))
    with pytest.raises(AssertionError, match="base_len"):
        pkg.paged_accept(kp, vp, table, -1, i32(2, 3))
    for kw, kind, text in [(dict(pools=[], src=i32(1), dst=i32(1)), AssertionError, "pools"), (dict(pools=[kp, vp[:3]], src=i32(1), dst=i32(1)), AssertionError, "pages each"),
                           (dict(pools=[kp.transpose(1, 2)], src=i32(1), dst=i32(1)), AssertionError, "contiguous"), (dict(pools=[kp], src=i32(1), dst=i32(2)), AssertionError, "one length"),
                           (dict(pools=[kp], src=z(1), dst=z(1)), TypeError, "int32"), (dict(pools=[kp] * 9, src=i32(1), dst=i32(1)), AssertionError, "pools"),
                           (dict(pools=[kp], src=i32(1).cpu(), dst=i32(1).cpu()), RuntimeError, "tensors on")]:
        with pytest.raises(kind, match=text):
            pkg.copy_pages(**kw)
