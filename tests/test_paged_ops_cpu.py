"""Refusals of the paged memory's operators on the CPU: every wrong argument is turned down before anything
reaches a kernel."""
import ctypes as C

import pytest
import torch

import sarbon_b200 as sb
from sarbon_b200 import _lib

H16 = dict(dtype=torch.float16)
I32 = dict(dtype=torch.int32)
E4M3 = torch.float8_e4m3fn


def pools(p=6, page=4, width=128, dtype=torch.float16):
    return torch.zeros(p, page, width, dtype=dtype), torch.zeros(p, page, width, dtype=dtype)


K, V = pools()
ATTEND = dict(q=torch.zeros(2, 1, 256, **H16), k_pages=K, v_pages=V, table=torch.zeros(2, 3, **I32),
              lens=torch.zeros(2, **I32), heads=4, kv_heads=2)
WRITE = dict(k=torch.zeros(2, 5, 128, **H16), v=torch.zeros(2, 5, 128, **H16), k_pages=K, v_pages=V,
             table=torch.zeros(2, 3, **I32), at=torch.zeros(2, **I32), weight=torch.zeros(2, 2, 12),
             born=torch.zeros(2, 2, 12, **I32), stamp=torch.zeros(2, 5, **I32))
EVICT = dict(k_pages=K, v_pages=V, table=torch.zeros(2, 3, **I32), lens=torch.zeros(2, **I32), weight=torch.zeros(2, 2, 12),
             keep=4, born=torch.zeros(2, 2, 12, **I32), since=torch.zeros(2, **I32))

MEMORY = [
    dict(k_pages=K.float(), v_pages=V.float()), dict(k_pages=K[0]), dict(v_pages=V[:5]), dict(v_pages=V.bfloat16()),
    dict(k_pages=torch.zeros(6, 128, 4, **H16).transpose(1, 2)), dict(table=torch.zeros(2, 3, dtype=torch.int64)),
    dict(table=torch.zeros(6, **I32)), dict(table=torch.zeros(3, 2, **I32).t()), dict(table=torch.zeros(3, 3, **I32)),
    dict(k_pages=pools(width=96)[0], v_pages=pools(width=96)[1]), dict(k_pages=pools(page=0)[0], v_pages=pools(page=0)[1]),
    dict(table=torch.zeros(2, 1, **I32).expand(2, 1 << 28)),
    dict(k_pages=torch.zeros(1, 4, 128, **H16).expand(1 << 31, 4, 128), v_pages=torch.ones(1, 4, 128, **H16).expand(1 << 31, 4, 128)),
    dict(),  # all well, but not on a GPU
]


@pytest.mark.parametrize("change", MEMORY + [
    dict(q=torch.zeros(2, 1, 256)), dict(q=torch.zeros(2, 256, **H16)), dict(q=torch.zeros(2, 1, 256, dtype=torch.bfloat16)),
    dict(q=torch.zeros(1, 1, 256, **H16)), dict(heads=3), dict(heads=8, kv_heads=3), dict(kv_heads=None), dict(heads=0),
    dict(lens=None), dict(lens=torch.zeros(2, dtype=torch.int64)), dict(lens=torch.zeros(3, **I32)),
    dict(lens=torch.zeros(4, **I32)[::2]), dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=1e39),
    dict(k_scale=float("nan")), dict(v_scale=1e39), dict(decay=-0.1), dict(decay=1.1), dict(decay=float("nan")), dict(k_scale=2.0), dict(v_scale=0.5), dict(k_scale=0.0),
    dict(weight=torch.zeros(2, 2, 11)), dict(weight=torch.zeros(2, 4, 12)), dict(weight=torch.zeros(2, 2, 12, **H16)),
    dict(weight=torch.zeros(2, 12, 2).transpose(1, 2)), dict(lse=torch.zeros(2, 4, 2)), dict(out=torch.zeros(2, 1, 128, **H16)),
    dict(out=ATTEND["q"]),
])
def test_attention_refuses(change):
    with pytest.raises(ValueError):
        sb.paged_attention(**{**ATTEND, **change})


@pytest.mark.parametrize("change", MEMORY + [
    dict(k=torch.zeros(2, 5, 128)), dict(k=torch.zeros(2, 5, 128, dtype=torch.bfloat16)), dict(v=torch.zeros(2, 4, 128, **H16)),
    dict(k=torch.zeros(2, 5, 64, **H16), v=torch.zeros(2, 5, 64, **H16)), dict(at=None), dict(at=torch.zeros(2)),
    dict(count=torch.zeros(3, **I32)), dict(count=torch.zeros(2, dtype=torch.int64)), dict(weight=torch.zeros(2, 12)),
    dict(weight=torch.zeros(2, 2, 13)), dict(born=torch.zeros(2, 2, 12)), dict(born=torch.zeros(2, 1, 12, **I32)),
    dict(stamp=None), dict(born=None), dict(stamp=torch.zeros(2, 4, **I32)), dict(stamp=torch.zeros(5, **I32)),
    dict(stamp=torch.zeros(2, 5)), dict(k_scale=2.0), dict(after=torch.zeros(3, **I32)), dict(after=WRITE["at"]),
    dict(kv_heads=4), dict(v_pages=K), dict(k=K[:2, :, :].expand(2, 4, 128), v=V[:2], stamp=torch.zeros(2, **I32)),
    dict(k_pages=torch.zeros(1, 4, 128, **H16).expand(6, 4, 128)), dict(v_pages=torch.zeros(6, 1, 128, **H16).expand(6, 4, 128)),
])
def test_write_refuses(change):
    with pytest.raises(ValueError):
        sb.paged_write(**{**WRITE, **change})


@pytest.mark.parametrize("change", MEMORY + [
    dict(weight=torch.zeros(2, 24)), dict(weight=torch.zeros(2, 2, 13)), dict(weight=torch.zeros(2, 3, 12)), dict(lens=None),
    dict(lens=torch.zeros(2)), dict(keep=-1), dict(keep=1.5), dict(keep=torch.zeros(2)), dict(keep=torch.zeros(3, **I32)),
    dict(born=None), dict(since=torch.zeros(3, **I32)), dict(born=torch.zeros(2, 2, 12)),
    dict(weight_out=torch.zeros(2, 2, 11)), dict(born=None, since=None, born_out=EVICT["born"]), dict(after=torch.zeros(1, **I32)),
    dict(weight_out=EVICT["born"].view(torch.float32)), dict(after=EVICT["since"]), dict(v_pages=K),
    dict(k_pages=torch.zeros(1, 4, 128, **H16).expand(6, 4, 128)),
])
def test_evict_refuses(change):
    with pytest.raises(ValueError):
        sb.paged_evict(**{**EVICT, **change})


def test_results_that_lie_on_others():
    """Results may be their operands themselves in eviction, but lie on nothing in part."""
    room = torch.zeros(2 * 2 * 12 + 4)
    weight, beside = room[:48].view(2, 2, 12), room[4:].view(2, 2, 12)
    with pytest.raises(ValueError, match="own memory"):
        sb.paged_evict(**{**EVICT, "weight": weight, "weight_out": beside})
    with pytest.raises(ValueError, match="CUDA"):
        sb.paged_evict(**{**EVICT, "weight": weight, "weight_out": weight, "born_out": EVICT["born"], "after": EVICT["lens"]})
    ints = torch.zeros(3, **I32)
    with pytest.raises(ValueError, match="own memory"):
        sb.paged_evict(**{**EVICT, "lens": ints[:2], "after": ints[1:]})


def test_autograd_inputs_are_refused():
    with pytest.raises(ValueError):
        sb.paged_attention(**{**ATTEND, "q": torch.zeros(2, 1, 256, **H16, requires_grad=True)})
    import torch.autograd.forward_ad as fw
    with fw.dual_level(), pytest.raises(ValueError, match="forward-mode"):
        sb.paged_attention(**{**ATTEND, "q": fw.make_dual(ATTEND["q"], torch.ones_like(ATTEND["q"]))})


def test_library_refuses():
    """The C entries turn down what the wrappers never pass, before any device call."""
    from sarbon_b200.paged_ops import _APPEND, _ATTEND, _CUT
    lib, n = _lib.lib(), C.c_longlong(0)

    def memory(kp=16, vp=32, kr=64, pt=0, p=4, page=4, table=16, tr=2, nn=2, b=1, hkv=1, dh=32):
        return kp, vp, kr, 256, kr, 256, table, tr, pt, p, page, nn, b, hkv, dh

    wrong = [dict(pt=1), dict(dh=48), dict(hkv=0), dict(b=-1), dict(page=0), dict(p=-1), dict(nn=-1), dict(page=1 << 20, nn=1 << 10),
             dict(kr=60), dict(kr=-8), dict(kp=0), dict(vp=0), dict(kp=8), dict(table=0), dict(tr=-1)]

    def attention(m=memory(), q=16, row=64, qt=0, lens=16, h=2, tq=1, scale=1.0, ks=1.0, weight=0, decay=1.0, work=0, size=0):
        return lib.sb_paged_attention(_ATTEND.pack(*m, q, 16, row, 64, row, 64, lens, 0, weight, work, size, qt, h, tq, 0, scale, ks, 1.0,
                                                   decay), None)

    def write(m=memory(), k=16, dt=0, ks=1.0, at=16, after=16, t=1, kr=32):
        return lib.sb_paged_write(_APPEND.pack(*m, k, 16, kr, 32, kr, 32, at, 0, 0, 0, 0, 0, 0, after, dt, t, ks, 1.0), None)

    def evict(m=memory(), lens=16, weight=16, since=0, born=0, born_out=0, work=16, size=1 << 20):
        return lib.sb_paged_evict(_CUT.pack(*m, lens, 0, since, weight, born, weight, born_out, 32, work, size, 2), None)

    e4m3 = memory(pt=_lib.SB_F8)
    for call in (attention, write, evict):
        for change in wrong:
            assert call(m=memory(**change)) == _lib.SB_EINVAL, (call, change)
        assert call(m=memory(b=0)) == _lib.SB_OK
    for bad in (dict(qt=1), dict(qt=2), dict(qt=3), dict(h=0), dict(m=memory(hkv=2), h=3), dict(tq=-1), dict(scale=0.0),
                dict(scale=float("nan")), dict(ks=2.0), dict(m=e4m3, ks=0.0), dict(m=e4m3, scale=1e30, ks=1e30), dict(scale=3e38),
                dict(weight=16, decay=2.0), dict(q=0), dict(q=8), dict(row=60), dict(lens=0)):
        assert attention(**bad) == _lib.SB_EINVAL, bad
    assert attention(tq=0) == _lib.SB_OK
    for bad in (dict(k=0), dict(dt=1), dict(dt=3), dict(ks=2.0), dict(m=e4m3, ks=-1.0), dict(at=0), dict(after=0), dict(t=-1),
                dict(kr=-1)):
        assert write(**bad) == _lib.SB_EINVAL, bad
    for bad in (dict(lens=0), dict(weight=0), dict(since=16), dict(born=16), dict(born_out=16), dict(m=memory(page=4096), work=0),
                dict(m=memory(page=4096), work=8)):
        assert evict(**bad) == _lib.SB_EINVAL, bad
    assert all(f(None, None) == _lib.SB_EINVAL for f in (lib.sb_paged_attention, lib.sb_paged_write, lib.sb_paged_evict))
    assert lib.sb_paged_attention_work(1, 2, 1, 48, 1, 0, 4, 2, 0, C.byref(n)) == _lib.SB_EINVAL
    assert lib.sb_paged_attention_work(1, 2, 1, 32, 1, 0, 0, 2, 0, C.byref(n)) == _lib.SB_EINVAL
    assert lib.sb_paged_attention_work(1, 2, 1, 32, 1, 1, 4, 2, 0, C.byref(n)) == _lib.SB_EINVAL
    assert lib.sb_paged_evict_work(1, 0, 4, 2, 0, C.byref(n)) == _lib.SB_EINVAL
