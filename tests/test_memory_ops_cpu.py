"""Refusals and host-side tables of the memory-reading block's operators, on the CPU: every
wrong argument is turned down before anything reaches a kernel."""
import ctypes as C

import pytest
import torch

import sarbon_b200 as sb
from sarbon_b200 import _lib, memory_ops as mo

F32 = torch.float32
H16 = dict(dtype=torch.float16)


def attend(**change):
    a = dict(q=torch.zeros(2, 5, 128, **H16), k=torch.zeros(2, 7, 64, **H16), v=torch.zeros(2, 7, 64, **H16), heads=4,
             kv_heads=2, lens=None, valid=None, scale=None, out=None, lse=None)
    a.update(change)
    return sb.cross_attention(a["q"], a["k"], a["v"], a["heads"], **{n: a[n] for n in list(a)[4:]})


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(2, 5, 128)),                                   # fp32
    dict(q=torch.zeros(10, 128, **H16)),                              # not [B, T, C]
    dict(k=torch.zeros(2, 7, 64, dtype=torch.bfloat16)),              # two types
    dict(v=torch.zeros(2, 8, 64, **H16)),                             # keys and values of two lengths
    dict(k=torch.zeros(1, 7, 64, **H16)),                             # another batch
    dict(heads=3, kv_heads=None), dict(heads=8, kv_heads=8), dict(heads=4, kv_heads=3), dict(heads=0),
    dict(k=torch.zeros(2, 64, 7, **H16).transpose(1, 2)),             # channels apart
    dict(lens=torch.zeros(2, dtype=torch.int64)), dict(lens=torch.zeros(3, dtype=torch.int32)),
    dict(valid=torch.zeros(2, 7)), dict(valid=torch.zeros(2, 6, dtype=torch.uint8)),
    dict(valid=torch.zeros(7, 2, dtype=torch.uint8).t()),
    dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan")),
    dict(out=torch.zeros(2, 5, 64, **H16)), dict(out=torch.zeros(1, 5, 128, **H16).expand(2, 5, 128)),
    dict(lse=torch.zeros(2, 4, 6)), dict(lse=torch.zeros(2, 4, 5, **H16)),
    dict(),                                                           # all well, but not on a GPU
])
def test_cross_attention_refuses(change):
    with pytest.raises(ValueError):
        attend(**change)


def test_cross_attention_backward_refuses():
    q, k, lse = torch.zeros(2, 5, 128, **H16), torch.zeros(2, 7, 128, **H16), torch.zeros(2, 4, 5)
    good = dict(dout=q, q=q, k=k, v=k, out=q, lse=lse, heads=4)
    for change in (dict(dout=q.float()), dict(dout=q[:, :4]), dict(out=q[:1]), dict(lse=lse[:, :3]), dict(dq=q[:, :4]),
                   dict(dk=torch.zeros(1, 7, 128, **H16).expand(2, 7, 128)), dict()):
        with pytest.raises(ValueError):
            sb.cross_attention_backward(**{**good, **change})


def test_results_over_inputs_are_refused():
    """Attention reads rows after others are written: a result may not lie on an operand, nor on another."""
    q, k = torch.zeros(2, 5, 128, **H16), torch.zeros(2, 5, 128, **H16)
    for x in (q, k):
        with pytest.raises(ValueError, match="own memory"):
            attend(q=q, k=k, v=k, kv_heads=4, out=x)
    lse, grad = torch.zeros(2, 4, 5), torch.zeros(2, 5, 128, **H16)
    good = dict(dout=q, q=q, k=k, v=k, out=q, lse=lse, heads=4)
    for change in (dict(dq=q), dict(dk=k), dict(dv=k), dict(dk=grad, dv=grad), dict(dq=grad, dv=grad)):
        with pytest.raises(ValueError, match="own memory"):
            sb.cross_attention_backward(**{**good, **change})


def test_rope_refuses():
    x, pos = torch.zeros(2, 6, 64), torch.zeros(6, 3, dtype=torch.int32)
    freq, axis = sb.rope_table((4, 6, 6), device="cpu")
    good = dict(x=x, pos=pos, heads=2, freq=freq, axis=axis)
    for change in (dict(x=x.double()), dict(x=x[0]), dict(heads=3), dict(heads=4), dict(pos=pos.long()),
                   dict(pos=pos[:5]), dict(pos=pos[None].expand(3, 6, 3)), dict(pos=pos.t().contiguous().t()),
                   dict(freq=freq.float()), dict(axis=axis.long()), dict(axis=axis[:5]), dict(layout="quarter"),
                   dict(out=torch.zeros(2, 6, 32)), dict()):
        with pytest.raises(ValueError):
            sb.rope_axes(**{**good, **change})


def test_gated_norm_refuses():
    x, z, w = torch.zeros(2, 6, 64), torch.zeros(2, 6, 64, **H16), torch.ones(64)
    good = dict(x=x, z=z, post=w, pre=w)
    bad = [dict(x=x[0]), dict(z=z[:, :5]), dict(x=x.double()), dict(gate=w), dict(gate=torch.ones(1, 1, 64, **H16)),
           dict(gate=torch.ones(2, 1, 64, **H16)), dict(scale=w.half()), dict(scale=w[:5]), dict(post=(w, w)),
           dict(post=w.half()), dict(pre=(None, w)), dict(kind="batch"), dict(eps=-1.0), dict(),
           dict(x=torch.zeros(1, 1, 8200), z=torch.zeros(1, 1, 8200), post=None, pre=None),
           dict(y=torch.zeros(2, 1, 64).expand(2, 6, 64)), dict(pre=None, h=z)]
    for change in bad:
        with pytest.raises(ValueError):
            sb.gated_norm(**{**good, **change})
    for change in (dict(pre=None, dh=z), dict(dy=z), dict(dh=x), dict()):
        with pytest.raises(ValueError):
            sb.gated_norm_backward(**{"dy": None, "dh": None, **good, **change})


def test_results_over_other_rows_are_refused():
    """Row by row a result may take its operand's place, with the operand's rows; with other rows, or on another
    result, one row's result would fall on another's operands."""
    base = torch.zeros(2, 6, 128)
    x, other = base[..., :64], base.view(2, 12, 64)[:, :6]
    assert x.data_ptr() == other.data_ptr()
    freq, axis = sb.rope_table((32,), device="cpu")
    pos = torch.zeros(6, 1, dtype=torch.int32)
    with pytest.raises(ValueError, match="own memory"):
        sb.rope_axes(x, pos, 1, freq, axis, out=other)
    with pytest.raises(ValueError, match="CUDA"):
        sb.rope_axes(x, pos, 1, freq, axis, out=x)
    w, z, free = torch.ones(64), torch.zeros(2, 6, 64), torch.zeros(2, 6, 64)
    for change in (dict(y=other), dict(z=x, h=other), dict(y=free, h=free)):
        with pytest.raises(ValueError, match="own memory"):
            sb.gated_norm(**{**dict(x=x, z=z, pre=w), **change})
    with pytest.raises(ValueError, match="CUDA"):
        sb.gated_norm(x, z, pre=w, y=x, h=z)
    # another type's rows begin there: its elements lie elsewhere
    half = z.view(torch.float16).view(2, 6, 128)[..., :64]
    with pytest.raises(ValueError, match="own memory"):
        sb.gated_norm(z, torch.zeros(2, 6, 64, **H16), pre=w, h=half)


def test_strides_of_views():
    wide = torch.zeros(2, 5, 192)
    assert mo._rows(wide[..., 64:128], "x", (2, 5, 64), F32)[1:] == (192, 960)
    first = torch.zeros(5, 2, 64).transpose(0, 1)  # sequence first
    assert mo._rows(first, "x", (2, 5, 64), F32, out=True)[1:] == (128, 64)
    shared = torch.zeros(1, 5, 64).expand(3, 5, 64)
    assert mo._rows(shared, "x", (3, 5, 64), F32)[1:] == (64, 0)
    one = torch.zeros(3, 9, 64)[:, 4:5]
    assert mo._rows(one, "x", (3, 1, 64), F32, out=True)[1:] == (64, 576)
    assert mo._rows(torch.zeros(3, 9, 64)[:, ::3], "x", (3, 3, 64), F32, out=True)[1:] == (192, 576)


def test_library_refuses():
    """The C entries turn down what the wrappers never pass, before any device call."""
    lib, n = _lib.lib(), C.c_longlong(0)
    one = C.c_void_p(16)

    def attention(dtype=0, b=1, h=2, hkv=1, dh=64, tq=4, tk=4, scale=1.0, row=128, q=one):
        rows = (row, 1024)
        return lib.sb_cross_attention(q, *rows, one, *rows, one, *rows, dtype, b, h, hkv, dh, tq, tk, scale, None, None, 0,
                                      one, *rows, None, None, 0, None)

    for bad in (dict(dtype=1), dict(dtype=2), dict(b=-1), dict(hkv=0), dict(h=3, hkv=2), dict(dh=48), dict(tq=-1),
                dict(scale=-1.0), dict(scale=float("nan")), dict(row=100), dict(row=-8), dict(q=None),
                dict(q=C.c_void_p(8))):
        assert attention(**bad) == _lib.SB_EINVAL, bad
    assert attention(b=0) == _lib.SB_OK and attention(tq=0) == _lib.SB_OK
    assert lib.sb_cross_attention_work(0, 0, 1, 2, 1, 48, 4, 4, C.byref(n)) == _lib.SB_EINVAL
    assert lib.sb_gated_norm_work(1, 1, 9000, C.byref(n)) == _lib.SB_EINVAL
    assert lib.sb_rope_axes(one, 64, 64, 0, 1, 1, 1, 64, one, 0, 0, 1, one, one, 33, 0, 0, one, 64, 64, None) == _lib.SB_EINVAL
    assert lib.sb_rope_axes(None, 64, 64, 0, 1, 1, 1, 64, one, 0, 0, 1, one, one, 32, 0, 0, one, 64, 64, None) == _lib.SB_EINVAL


def test_library_refuses_rows_of_one():
    """A row stride of 0 where there are several rows is turned down before anything is launched, by the
    operands that tensor maps describe: k, v and, backward, q and dout."""
    lib, one = _lib.lib(), C.c_void_p(16)
    rows = {n: (128, 1024) for n in ("dout", "q", "k", "v", "out")}

    def call(back, **change):
        r = {**rows, **change}
        names = ["dout", "q", "k", "v", "out"] if back else ["q", "k", "v"]
        a = [x for n in names for x in (one, *r[n])] + ([one] if back else [])
        a += [0, 1, 2, 1, 64, 4, 4, 1.0, None, None, 0]
        if back:
            return lib.sb_cross_attention_backward(*a, *(one, 128, 1024) * 3, None, 0, None)
        return lib.sb_cross_attention(*a, one, 128, 1024, None, None, 0, None)

    for n in ("k", "v"):
        assert call(False, **{n: (0, 1024)}) == _lib.SB_EINVAL, n
    for n in ("dout", "q", "k", "v"):
        assert call(True, **{n: (0, 1024)}) == _lib.SB_EINVAL, n


def test_autograd_inputs_are_refused():
    q = torch.zeros(1, 2, 64, **H16, requires_grad=True)
    with pytest.raises(ValueError):
        sb.cross_attention(q, q, q, 1)


def test_forward_mode_inputs_are_refused():
    """A dual tensor does not say that it requires a gradient; its tangent would be lost."""
    import torch.autograd.forward_ad as fw
    q = torch.zeros(1, 2, 64, **H16)
    x, freq, axis = torch.zeros(1, 2, 64), *sb.rope_table((32,), device="cpu")
    pos = torch.zeros(2, 1, dtype=torch.int32)
    with fw.dual_level():
        dual, dual32 = fw.make_dual(q, torch.ones_like(q)), fw.make_dual(x, torch.ones_like(x))
        lse = torch.zeros(1, 1, 2)
        for call in (lambda: sb.cross_attention(q, dual, q, 1), lambda: sb.cross_attention_backward(dual, q, q, q, q, lse, 1),
                     lambda: sb.rope_axes(dual32, pos, 1, freq, axis), lambda: sb.gated_norm(x, x, scale=dual32[0, 0]),
                     lambda: sb.gated_norm_backward(dual32, None, x, x)):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
        with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
            sb.cross_attention(dual, q, q, 1)
        with pytest.raises(ValueError, match="CUDA"):  # none among these
            sb.cross_attention(q, q, q, 1)


def test_rope_table_and_grid():
    freq, axis = sb.rope_table((2, 0, 4), theta=100.0, device="cpu")
    assert axis.tolist() == [0, 0, 2, 2, 2, 2]
    assert torch.allclose(freq, torch.tensor([1, 0.1, 1, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64))
    freq, _ = sb.rope_table((2, 2), theta=16.0, per_axis=False, device="cpu")
    assert freq.tolist() == [1.0, 0.5, 0.25, 0.125]
    pos = sb.grid_positions(2, 3, 4, device="cpu")
    assert pos.shape == (24, 3) and pos.dtype == torch.int32 and pos[13].tolist() == [1, 0, 1]
    with pytest.raises(ValueError):
        sb.rope_table((2, -1))
