"""A transformer block that reads an encoder's memory: its operators, forward and backward.

Beside the detector's own kernels (:mod:`sarbon_b200.det_ops`: attention over equal heads of 32
channels, LayerNorm, added positions) these are the pieces of a decoder or tracker block that
attends to the tokens of p8 / p16 / p32, of several frames or of images padded to a common size::

    freq, axis = rope_table((16, 24, 24))                     # time, height, width
    q = rope_axes(q, q_pos, heads, freq, axis)
    k = rope_axes(k, grid_positions(t, h, w), kv_heads, freq, axis)
    o = cross_attention(q, k, v, heads, kv_heads=kv_heads, lens=lens, lse=lse)
    x, h = gated_norm(x, proj(o), gate=gate, post=(w0, b0), pre=(w1, b1), kind="layer")

Rows are ``[B, T, channels]`` with contiguous channels; slices of wider projections, sequence-first
layouts and memories shared by all items (a batch stride of 0) are read as they are; attention copies
operands whose rows are one expanded row where its kernels cannot.  Every call
launches kernels of ``libsarbon_sparse.so`` on the current CUDA stream of its tensors' device and can
be captured in a CUDA graph after a first call outside capture.  Workspaces come from torch's
caching allocator for each call, so calls on two streams or in two graphs share none.

Gradients are calls of their own (``cross_attention_backward``, ``rope_axes(inverse=True)``,
``gated_norm_backward``) that an ``autograd.Function`` or a hand-written step makes; the forward
calls record no graph and refuse tensors that would need one, or that carry a forward-mode tangent.
"""
from __future__ import annotations

import ctypes as C
import functools

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import check, lib

DTYPES = {torch.float16: _lib.SB_F16, torch.bfloat16: _lib.SB_BF16, torch.float32: _lib.SB_F32}
_HALVES = (torch.float16, torch.bfloat16)

# library calls made through this module
CALLS = [0]

# A call's host time is what a small call costs, so the checks below format their messages only
# when they fail and read each tensor's attributes once.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)

_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _ready(*tensors):
    """All tensors on one CUDA device and none that autograd would have to follow; its index."""
    # a dual tensor does not require a gradient; looked for only inside a forward_ad.dual_level
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t, level=0).tangent is not None:
                raise ValueError("no forward-mode tangent is followed: call on primals")
    index = tensors[0].get_device()
    grad = torch.is_grad_enabled()
    for t in tensors:
        if t is not None:
            if t.get_device() != index or not t.is_cuda:
                raise ValueError("tensors of one CUDA device")
            if grad and t.requires_grad:
                raise ValueError("no autograd graph is recorded: call under torch.no_grad() or from an autograd.Function")
    return index


def _launch(name, index, *args):
    CALLS[0] += 1
    if index == _device():
        status = getattr(lib(), name)(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = getattr(lib(), name)(*args, _raw_stream(index))
    if status:
        check(status, name)


@functools.lru_cache(maxsize=4096)
def _work_bytes(name, index, *args):
    """Workspace bytes of a call with these sizes on this device."""
    n = C.c_longlong(0)
    with torch.cuda.device(index):
        check(getattr(lib(), name)(*args, C.byref(n)), name)
    return n.value


def _work(name, index, *args):
    """Workspace of a call: (tensor or None, pointer, bytes)."""
    n = _work_bytes(name, index, *args)
    if n == 0:
        return None, None, 0
    w = torch.empty(n, device=torch.device("cuda", index), dtype=torch.uint8)
    return w, w.data_ptr(), n


def _rows(t, what, shape, dtype, out=False):
    """(pointer, row stride, item stride) in elements of [B, T, C] rows."""
    if t.shape != shape or t.dtype != dtype:
        raise ValueError(f"{what}: expected {tuple(shape)} of {dtype}, got {tuple(t.shape)} of {t.dtype}")
    b, n, c = shape
    img, row, one = t.stride()
    if one != 1 and c > 1:
        raise ValueError(f"{what}: channels must be contiguous")
    # the stride of a dimension of one element is arbitrary and never used
    if n <= 1:
        row = c
    if b <= 1:
        img = n * row
    if out and (row < c or img < row * (n - 1) + c) and t.numel():
        apart = (n == 1 or row >= c) and (b == 1 or img >= c) and \
            (n == 1 or b == 1 or img >= row * (n - 1) + c or row >= img * (b - 1) + c)
        if not apart:
            raise ValueError(f"{what}: rows overlap")
    return t.data_ptr(), row, img


def _own_rows(t):
    """A copy of t, whose rows are one and the same (a row stride of 0, which no tensor map has)."""
    return t[:1].contiguous().expand(t.shape) if t.stride(0) == 0 else t.contiguous()


def _mapped(t, what, shape, dtype):
    """_rows of an operand that a tensor map describes, and what they lie in (t or a copy)."""
    rows = _rows(t, what, shape, dtype)
    if rows[1] == 0:
        t = _own_rows(t)
        rows = _rows(t, what, shape, dtype)
    return rows, t


def _apart(results, operands):
    """Results that do not begin where an operand or another result does."""
    seen = {t.data_ptr() for t in operands if t.numel()}
    for t in results:
        if t is not None and t.numel():
            if t.data_ptr() in seen:
                raise ValueError("results need their own memory")
            seen.add(t.data_ptr())


def _in_place(result, dtype, *operands):
    """A result's rows may be an operand's rows; other rows may not begin where an operand does.  Rows as
    _rows returns them, operands as (rows, type)."""
    for rows, kind in operands:
        if rows[0] == result[0] and result[0] and (rows != result or kind != dtype):
            raise ValueError("results need their own memory or an operand's very rows")


def _new(like, shape, dtype):
    """A contiguous tensor, (pointer, row stride, item stride); empty_like is the cheapest allocation."""
    t = torch.empty_like(like) if like.dtype == dtype and like.is_contiguous() and like.shape == shape else \
        torch.empty(shape, device=like.device, dtype=dtype)
    return t, (t.data_ptr(), shape[2], shape[1] * shape[2])


# ---------------------------------------------------------------- attention
def _attention_sizes(q, k, heads, kv_heads, scale):
    if q.dim() != 3 or k.dim() != 3 or q.dtype not in _HALVES:
        raise ValueError("q, k, v: [B, T, heads * dim] rows of fp16 or bf16")
    if kv_heads is None:
        kv_heads = heads
    if heads < 1 or kv_heads < 1 or heads % kv_heads:
        raise ValueError("heads: a multiple of kv_heads")
    b, tq, width = q.shape
    dim = width // heads
    if dim not in (32, 64, 128) or width != heads * dim:
        raise ValueError("heads of 32, 64 or 128 channels")
    if scale is None:
        scale = dim ** -0.5
    if not 0.0 < scale < _INF:
        raise ValueError("scale: a positive number")
    return kv_heads, b, tq, k.shape[1], dim, scale


_INF = float("inf")
_NO_MASK = (None, None, 0)


def _masks(lens, valid, b, tk):
    """Pointers of the masks: (lens, valid, valid's item stride)."""
    if lens is None and valid is None:
        return _NO_MASK
    p_lens = p_valid = None
    img = 0
    if lens is not None:
        if lens.dtype != torch.int32 or lens.shape != (b,) or (b > 1 and lens.stride(0) != 1):
            raise ValueError("lens: contiguous int32 [B]")
        p_lens = lens.data_ptr()
    if valid is not None:
        if valid.dtype not in (torch.uint8, torch.bool) or valid.shape != (b, tk) or (tk > 1 and valid.stride(1) != 1):
            raise ValueError("valid: uint8 or bool [B, Tk] with contiguous rows")
        p_valid, img = valid.data_ptr(), valid.stride(0) if b > 1 else tk
    return p_lens, p_valid, img


def _statistics(lse, b, heads, tq):
    if lse.dtype != torch.float32 or lse.shape != (b, heads, tq) or not lse.is_contiguous():
        raise ValueError("lse: contiguous fp32 [B, heads, Tq]")


def cross_attention(q, k, v, heads, kv_heads=None, lens=None, valid=None, scale=None, out=None, lse=None):
    """softmax(scale q k^T) v per head: queries [B, Tq, heads * dim] on an encoder's states k, v
    [B, Tk, kv_heads * dim] of another length; dim 32, 64 or 128, fp16 or bf16.

    Query head h reads key head ``h // (heads // kv_heads)``.  State j of item b takes part when
    ``j < lens[b]`` (int32 [B]) and ``valid[b, j]`` (uint8 or bool [B, Tk]); the others may hold
    anything.  A query without states gets zeros.  scale: 1 / sqrt(dim) unless given.  Fills out
    (allocated if None; it must not share memory with q, k or v) and, if given, lse (fp32 [B, heads,
    Tq], the log-sum-exp of the scaled scores, -inf without states), which the backward pass reads.  Few
    queries on many states (single tokens) are split over the states."""
    kv_heads, b, tq, tk, dim, scale = _attention_sizes(q, k, heads, kv_heads, scale)
    dtype, qs, ks = q.dtype, (b, tq, heads * dim), (b, tk, kv_heads * dim)
    qp, (kp, k), (vp, v) = _rows(q, "q", qs, dtype), _mapped(k, "k", ks, dtype), _mapped(v, "v", ks, dtype)
    masks = _masks(lens, valid, b, tk)
    if lse is not None:
        _statistics(lse, b, heads, tq)
    if out is not None:
        op = _rows(out, "out", qs, dtype, out=True)
        _apart((out,), (q, k, v))
    index = _ready(q, k, v, lens, valid, out, lse)
    if out is None:
        out, op = _new(q, qs, dtype)
    if b == 0 or tq == 0:
        return out
    hold, work, size = _work("sb_cross_attention_work", index, 0, valid is not None, b, heads, kv_heads, dim, tq, tk)
    _launch("sb_cross_attention", index, *qp, *kp, *vp, DTYPES[dtype], b, heads, kv_heads, dim, tq, tk, scale, *masks,
            *op, None if lse is None else lse.data_ptr(), work, size)
    return out


def cross_attention_backward(dout, q, k, v, out, lse, heads, kv_heads=None, lens=None, valid=None, scale=None,
                             dq=None, dk=None, dv=None):
    """Gradients (dq, dk, dv) of :func:`cross_attention` from dout and the forward pass's out and lse.

    The same sizes, masks and scale as forward.  dk and dv have one row for every item's state, also
    where k and v are shared by the items (sum them over the batch then); states that take no part
    get zeros.  The sums have a fixed order: the same inputs give the same bits.  dq, dk and
    dv (allocated if None) must not share memory with an operand or each other."""
    kv_heads, b, tq, tk, dim, scale = _attention_sizes(q, k, heads, kv_heads, scale)
    dtype, qs, ks = q.dtype, (b, tq, heads * dim), (b, tk, kv_heads * dim)
    (dp, dout), (qp, q), (kp, k), (vp, v) = _mapped(dout, "dout", qs, dtype), _mapped(q, "q", qs, dtype), \
        _mapped(k, "k", ks, dtype), _mapped(v, "v", ks, dtype)
    views = dp + qp + kp + vp + _rows(out, "out", qs, dtype)
    masks = _masks(lens, valid, b, tk)
    _statistics(lse, b, heads, tq)
    for what, t, shape in (("dq", dq, qs), ("dk", dk, ks), ("dv", dv, ks)):
        if t is not None:
            _rows(t, what, shape, dtype, out=True)
    if dq is not None or dk is not None or dv is not None:
        _apart((dq, dk, dv), (dout, q, k, v, out))
    index = _ready(dout, q, k, v, out, lse, lens, valid, dq, dk, dv)
    dq, dqp = _new(q, qs, dtype) if dq is None else (dq, _rows(dq, "dq", qs, dtype))
    dk, dkp = _new(k, ks, dtype) if dk is None else (dk, _rows(dk, "dk", ks, dtype))
    dv, dvp = _new(v, ks, dtype) if dv is None else (dv, _rows(dv, "dv", ks, dtype))
    if b == 0 or (tq == 0 and tk == 0):
        return dq, dk, dv
    hold, work, size = _work("sb_cross_attention_work", index, 1, valid is not None, b, heads, kv_heads, dim, tq, tk)
    _launch("sb_cross_attention_backward", index, *views, lse.data_ptr(), DTYPES[dtype], b, heads, kv_heads, dim, tq, tk,
            scale, *masks, *dqp, *dkp, *dvp, work, size)
    return dq, dk, dv


# ---------------------------------------------------------------- positions
def rope_table(sections, theta=10000.0, per_axis=True, device="cuda"):
    """(freq fp64 [R], axis int32 [R]) of :func:`rope_axes`: ``sections[a]`` pairs turn with axis a, in
    this order.  Frequencies theta ** (-i / n): i counts an axis's own n pairs (per_axis), or all R."""
    if len(sections) < 1 or any(int(n) != n or n < 0 for n in sections) or not theta > 0:
        raise ValueError("sections: numbers of pairs; theta > 0")
    total = sum(sections)
    i = [torch.arange(n, dtype=torch.float64) / max(n, 1) for n in sections]
    i = torch.cat(i) if per_axis else torch.arange(total, dtype=torch.float64) / max(total, 1)
    axis = torch.repeat_interleave(torch.arange(len(sections), dtype=torch.int32), torch.tensor(sections))
    return (float(theta) ** -i).to(device), axis.to(device)


def grid_positions(t, h, w, device="cuda"):
    """int32 [t * h * w, 3] positions (frame, row, column) of a clip's tokens in raster order."""
    axes = [torch.arange(n, dtype=torch.int32, device=device) for n in (t, h, w)]
    return torch.stack(torch.meshgrid(*axes, indexing="ij"), -1).reshape(-1, 3)


def rope_axes(x, pos, heads, freq, axis, layout="half", inverse=False, out=None):
    """Rotary positions with several axes on x [B, T, heads * dim] (fp16, bf16 or fp32).

    Pair p of every head turns by ``pos[b, t, axis[p]] * freq[p]`` (inverse: by its negative, which is
    the gradient).  pos: int32 or fp32 [B, T, A], or [T, A] for all items; freq fp64 [R], axis int32 [R]
    (:func:`rope_table`; an axis outside pos's leaves its pair).  Pairs are channels (p, p + R) of a
    head ("half") or (2p, 2p + 1) ("pairs"); channels from 2R on stay as they are.  Angles are formed in
    fp64, so positions in the millions keep their fraction of a turn.  out may be x itself (the
    very rows) and otherwise shares no memory with it."""
    dtype = x.dtype
    if x.dim() != 3 or dtype not in DTYPES:
        raise ValueError("x: [B, T, heads * dim] of fp16, bf16 or fp32")
    shape = b, t, width = x.shape
    if heads < 1 or width == 0 or width % heads:
        raise ValueError("x: a multiple of heads channels")
    dim, r = width // heads, freq.numel()
    if layout not in ("half", "pairs"):
        raise ValueError("layout: 'half' or 'pairs'")
    if freq.dtype != torch.float64 or axis.dtype != torch.int32 or freq.dim() != 1 or axis.shape != freq.shape or \
            not freq.is_contiguous() or not axis.is_contiguous():
        raise ValueError("freq: fp64 [R], axis: int32 [R]")
    if 2 * r > dim:
        raise ValueError("pairs: at most half of a head's channels")
    at, ps = pos.shape, pos.stride()
    if pos.dtype not in (torch.int32, torch.float32) or at[:-1] not in ((t,), (b, t)) or at[-1] < 1:
        raise ValueError("pos: int32 or fp32 [B, T, A] or [T, A]")
    if (at[-1] > 1 and ps[-1] != 1) or (t > 1 and ps[-2] != at[-1]):
        raise ValueError("pos: contiguous rows")
    xp = _rows(x, "x", shape, dtype)
    if out is not None:
        op = _rows(out, "out", shape, dtype, out=True)
        _in_place(op, dtype, (xp, dtype))
    index = _ready(x, pos, freq, axis, out)
    if out is None:
        out, op = _new(x, shape, dtype)
    if b == 0 or t == 0:
        return out
    _launch("sb_rope_axes", index, *xp, DTYPES[dtype], b, t, heads, dim, pos.data_ptr(), pos.dtype == torch.float32,
            ps[0] if len(at) == 3 and b > 1 else 0, at[-1], freq.data_ptr(), axis.data_ptr(), r, layout == "pairs",
            bool(inverse), *op)
    return out


# ---------------------------------------------------------------- gated residual and norms
def _norm_weights(w, what, kind):
    """A norm's weight, (weight, bias) or None -> (weight, bias)."""
    if w is None:
        return None, None
    w, b = w if isinstance(w, (tuple, list)) else (w, None)
    if w is None or (b is not None and kind != "layer"):
        raise ValueError(f"{what}: a weight, and a bias for layer norms only")
    return w, b


def _norm_inputs(x, z, gate, scale, post, pre, kind, eps):
    if x.dim() != 3 or x.dtype not in DTYPES or z.dtype not in DTYPES:
        raise ValueError("x, z: [B, T, D] of fp16, bf16 or fp32")
    if kind not in ("rms", "layer") or not eps >= 0:
        raise ValueError("kind: 'rms' or 'layer', eps >= 0")
    b, t, d = shape = x.shape
    if not 1 <= d <= 8192:
        raise ValueError("1 to 8192 channels")
    gp = (None, 0, 0)
    if gate is not None:
        n, s = gate.dim(), gate.stride()
        if gate.dtype != z.dtype or gate.shape not in ((d,), (b, d), (b, t, d)) or (d > 1 and s[-1] != 1):
            raise ValueError("gate: [D], [B, D] or [B, T, D] of z's type with contiguous channels")
        gp = (gate.data_ptr(), s[1] if n == 3 and t > 1 else 0, s[0] if n > 1 and b > 1 else 0)
    weights = _norm_weights(post, "post", kind) + _norm_weights(pre, "pre", kind)
    for t in (scale,) + weights:
        if t is not None and (t.dtype != torch.float32 or t.numel() != d or t.dim() != 1 or not t.is_contiguous()):
            raise ValueError("scale, weights and biases: contiguous fp32 [D]")
    return shape, _rows(x, "x", shape, x.dtype), _rows(z, "z", shape, z.dtype), gp, weights


def _ptr(t):
    return None if t is None else t.data_ptr()


def gated_norm(x, z, gate=None, scale=None, post=None, pre=None, kind="rms", eps=1e-6, y=None, h=None):
    """The end of a block and the start of the next: n = Npost(z), y = x + scale * gate * n, h = Npre(y).

    x (the residual) and z (the block's output): [B, T, D] rows; y has x's type and h z's.  post, pre: a
    norm's fp32 [D] weight or (weight, bias), None for no norm there (without pre, h is None).  kind:
    "rms" or "layer".  gate: z's type, [D], [B, D] (one an item) or [B, T, D].  scale: fp32 [D].  h comes
    from y before its rounding.  y may be x and h may be z (the very rows); otherwise y and h share
    no memory with an operand or each other.  Returns (y, h)."""
    shape, xp, zp, gp, weights = _norm_inputs(x, z, gate, scale, post, pre, kind, eps)
    hp = (None, 0, 0)
    if y is not None:
        yp = _rows(y, "y", shape, x.dtype, out=True)
    if h is not None:
        if pre is None:
            raise ValueError("h needs the norm pre")
        hp = _rows(h, "h", shape, z.dtype, out=True)
    if y is not None or h is not None:
        on = (xp, x.dtype), (zp, z.dtype), (gp, z.dtype)
        if y is not None:
            _in_place(yp, x.dtype, *on)
        if h is not None:
            _in_place(hp, z.dtype, *on, *(((yp, None),) if y is not None else ()))
    index = _ready(x, z, gate, scale, *weights, y, h)
    if y is None:
        y, yp = _new(x, shape, x.dtype)
    if h is None and pre is not None:
        h, hp = _new(z, shape, z.dtype)
    if shape[0] and shape[1]:
        _launch("sb_gated_norm", index, *xp, DTYPES[x.dtype], *zp, DTYPES[z.dtype], *gp, *[None if w is None else w.data_ptr() for w in (scale,) + weights],
                kind == "layer", eps, *shape, *yp, *hp)
    return y, h


def gated_norm_backward(dy, dh, x, z, gate=None, scale=None, post=None, pre=None, kind="rms", eps=1e-6):
    """Gradients of :func:`gated_norm` from dy (x's type, None: zero) and dh (z's type, None: zero).

    Returns a dict of dx (x's type), dz (z's type) and, where there is such an input, fp32 scale,
    post_w, post_b, pre_w, pre_b [D] and gate: fp32 [D] or [B, D] sums for a gate of that shape, z's
    type for one of [B, T, D]; None otherwise.  The sums over rows have a fixed order."""
    shape, xp, zp, gp, weights = _norm_inputs(x, z, gate, scale, post, pre, kind, eps)
    b, t, d = shape
    if dh is not None and pre is None:
        raise ValueError("dh needs the norm pre")
    dyp = (None, 0, 0) if dy is None else _rows(dy, "dy", shape, x.dtype)
    dhp = (None, 0, 0) if dh is None else _rows(dh, "dh", shape, z.dtype)
    index = _ready(x, z, gate, scale, *weights, dy, dh)
    g = {"dx": _new(x, shape, x.dtype)[0], "dz": _new(z, shape, z.dtype)[0]}
    make = torch.empty if b * t else torch.zeros  # no rows: every sum is zero
    for name, w in zip(("scale", "post_w", "post_b", "pre_w", "pre_b"), (scale,) + weights):
        g[name] = None if w is None else make(d, device=x.device, dtype=torch.float32)
    mode = 0 if gate is None else gate.dim()
    g["gate"] = None if gate is None else make(gate.shape, device=x.device, dtype=z.dtype if mode == 3 else torch.float32)
    if b * t == 0:
        return g
    hold, work, size = _work("sb_gated_norm_work", index, b, t, d)
    _launch("sb_gated_norm_backward", index, *dyp, *dhp, *xp, DTYPES[x.dtype], *zp, DTYPES[z.dtype], *gp, _ptr(scale),
            *map(_ptr, weights), kind == "layer", eps, b, t, d, _ptr(g["dx"]), _ptr(g["dz"]), _ptr(g["scale"]),
            _ptr(g["gate"]), mode, _ptr(g["post_w"]), _ptr(g["post_b"]), _ptr(g["pre_w"]), _ptr(g["pre_b"]), work, size)
    return g
