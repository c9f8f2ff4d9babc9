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
layouts and memories shared by all items (a batch stride of 0) are read as they are.  Every call
launches kernels of ``libsarbon_sparse.so`` on the current CUDA stream of its tensors' device and can
be captured in a CUDA graph after a first call outside capture.  Workspaces come from torch's
caching allocator for each call, so calls on two streams or in two graphs share none.

Gradients are calls of their own (``cross_attention_backward``, ``rope_axes(inverse=True)``,
``gated_norm_backward``) that an ``autograd.Function`` or a hand-written step makes; the forward
calls record no graph and refuse tensors that would need one.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._lib import check, lib

DTYPES = {torch.float16: _lib.SB_F16, torch.bfloat16: _lib.SB_BF16, torch.float32: _lib.SB_F32}

# library calls made through this module
CALLS = [0]


def _require(ok, what):
    if not ok:
        raise ValueError(what)


def _ready(*tensors):
    """All tensors on one CUDA device and none that autograd would have to follow."""
    tensors = [t for t in tensors if t is not None]
    dev = tensors[0].device
    for t in tensors:
        _require(t.is_cuda and t.device == dev, "tensors of one CUDA device")
        _require(not (t.requires_grad and torch.is_grad_enabled()),
                 "no autograd graph is recorded: call under torch.no_grad() or from an autograd.Function")
    return dev


def _launch(name, dev, *args):
    CALLS[0] += 1
    if dev.index == torch.cuda.current_device():
        status = getattr(lib(), name)(*args, torch.cuda.current_stream(dev).cuda_stream)
    else:
        with torch.cuda.device(dev):
            status = getattr(lib(), name)(*args, torch.cuda.current_stream(dev).cuda_stream)
    check(status, name)


def _work(name, dev, *args):
    """Workspace of a call: (tensor or None, pointer, bytes)."""
    n = C.c_longlong(0)
    with torch.cuda.device(dev):
        check(getattr(lib(), name)(*args, C.byref(n)), name)
    if n.value == 0:
        return None, None, 0
    w = torch.empty(n.value, device=dev, dtype=torch.uint8)
    return w, w.data_ptr(), n.value


def _rows(t, what, shape, dtype=None, out=False):
    """(pointer, row stride, item stride) in elements of [B, T, C] rows."""
    _require(t.dim() == 3 and tuple(t.shape) == tuple(shape), f"{what}: expected {tuple(shape)}, got {tuple(t.shape)}")
    _require(dtype is None or t.dtype == dtype, f"{what}: expected {dtype}, got {t.dtype}")
    b, n, c = shape
    _require(c <= 1 or t.stride(2) == 1, f"{what}: channels must be contiguous")
    # the stride of a dimension of one element is arbitrary and never used
    row = t.stride(1) if n > 1 else c
    img = t.stride(0) if b > 1 else n * row
    if out and t.numel():
        apart = (n == 1 or row >= c) and (b == 1 or img >= c) and \
            (n == 1 or b == 1 or img >= row * (n - 1) + c or row >= img * (b - 1) + c)
        _require(apart, f"{what}: rows overlap")
    return t.data_ptr(), row, img


# ---------------------------------------------------------------- attention
def _attention_sizes(q, k, v, heads, kv_heads, scale):
    _require(q.dim() == 3 and k.dim() == 3 and v.dim() == 3, "q, k, v: [B, T, heads * dim] rows")
    _require(q.dtype in (torch.float16, torch.bfloat16), "q: fp16 or bf16")
    kv_heads = heads if kv_heads is None else kv_heads
    _require(heads >= 1 and kv_heads >= 1 and heads % kv_heads == 0, "heads: a multiple of kv_heads")
    b, tq, width = q.shape
    dim = width // heads
    _require(width == heads * dim and dim in (32, 64, 128), "heads of 32, 64 or 128 channels")
    tk = k.shape[1]
    if scale is None:
        scale = dim ** -0.5
    _require(0.0 < scale < float("inf"), "scale: a positive number")
    return kv_heads, b, tq, tk, dim, float(scale)


def _masks(lens, valid, b, tk):
    """Pointers of the masks: (lens, valid, valid's item stride)."""
    p_lens = p_valid = None
    img = 0
    if lens is not None:
        _require(lens.dtype == torch.int32 and tuple(lens.shape) == (b,) and (b <= 1 or lens.stride(0) == 1),
                 "lens: contiguous int32 [B]")
        p_lens = lens.data_ptr()
    if valid is not None:
        _require(valid.dtype in (torch.uint8, torch.bool) and tuple(valid.shape) == (b, tk) and
                 (tk <= 1 or valid.stride(1) == 1), "valid: uint8 or bool [B, Tk] with contiguous rows")
        p_valid, img = valid.data_ptr(), valid.stride(0) if b > 1 else tk
    return p_lens, p_valid, img


def _statistics(lse, b, heads, tq):
    _require(lse.dtype == torch.float32 and tuple(lse.shape) == (b, heads, tq) and lse.is_contiguous(),
             "lse: contiguous fp32 [B, heads, Tq]")


def cross_attention(q, k, v, heads, kv_heads=None, lens=None, valid=None, scale=None, out=None, lse=None):
    """softmax(scale q k^T) v per head: queries [B, Tq, heads * dim] on an encoder's states k, v
    [B, Tk, kv_heads * dim] of another length; dim 32, 64 or 128, fp16 or bf16.

    Query head h reads key head ``h // (heads // kv_heads)``.  State j of item b takes part when
    ``j < lens[b]`` (int32 [B]) and ``valid[b, j]`` (uint8 or bool [B, Tk]); the others may hold
    anything.  A query without states gets zeros.  scale: 1 / sqrt(dim) unless given.  Fills out
    (allocated if None; it must not share memory with q, k or v) and, if given, lse (fp32 [B, heads,
    Tq], the log-sum-exp of the scaled scores, -inf without states), which the backward pass reads.  Few
    queries on many states (single tokens) are split over the states."""
    kv_heads, b, tq, tk, dim, scale = _attention_sizes(q, k, v, heads, kv_heads, scale)
    qp = _rows(q, "q", (b, tq, heads * dim))
    kp = _rows(k, "k", (b, tk, kv_heads * dim), q.dtype)
    vp = _rows(v, "v", (b, tk, kv_heads * dim), q.dtype)
    masks = _masks(lens, valid, b, tk)
    if lse is not None:
        _statistics(lse, b, heads, tq)
    if out is not None:
        op = _rows(out, "out", (b, tq, heads * dim), q.dtype, out=True)
    dev = _ready(q, k, v, lens, valid, out, lse)
    if out is None:
        out = torch.empty(b, tq, heads * dim, device=dev, dtype=q.dtype)
        op = (out.data_ptr(), heads * dim, tq * heads * dim)
    if out.numel() == 0:
        return out
    hold, work, size = _work("sb_cross_attention_work", dev, 0, b, heads, kv_heads, dim, tq, tk)
    _launch("sb_cross_attention", dev, *qp, *kp, *vp, DTYPES[q.dtype], b, heads, kv_heads, dim, tq, tk, scale, *masks,
            *op, None if lse is None else lse.data_ptr(), work, size)
    return out


def cross_attention_backward(dout, q, k, v, out, lse, heads, kv_heads=None, lens=None, valid=None, scale=None,
                             dq=None, dk=None, dv=None):
    """Gradients (dq, dk, dv) of :func:`cross_attention` from dout and the forward pass's out and lse.

    The same sizes, masks and scale as forward.  dk and dv have one row for every item's state, also
    where k and v are shared by the items (sum them over the batch then); states that take no part
    get zeros.  The sums have a fixed order: the same inputs give the same bits."""
    kv_heads, b, tq, tk, dim, scale = _attention_sizes(q, k, v, heads, kv_heads, scale)
    qs, ks = (b, tq, heads * dim), (b, tk, kv_heads * dim)
    views = [_rows(dout, "dout", qs, q.dtype), _rows(q, "q", qs), _rows(k, "k", ks, q.dtype),
             _rows(v, "v", ks, q.dtype), _rows(out, "out", qs, q.dtype)]
    masks = _masks(lens, valid, b, tk)
    _statistics(lse, b, heads, tq)
    for name, t, s in (("dq", dq, qs), ("dk", dk, ks), ("dv", dv, ks)):
        if t is not None:
            _rows(t, name, s, q.dtype, out=True)
    dev = _ready(dout, q, k, v, out, lse, lens, valid, dq, dk, dv)
    dq = torch.empty(qs, device=dev, dtype=q.dtype) if dq is None else dq
    dk = torch.empty(ks, device=dev, dtype=q.dtype) if dk is None else dk
    dv = torch.empty(ks, device=dev, dtype=q.dtype) if dv is None else dv
    if dq.numel() == 0 and dk.numel() == 0:
        return dq, dk, dv
    grads = [_rows(t, name, s) for name, t, s in (("dq", dq, qs), ("dk", dk, ks), ("dv", dv, ks))]
    hold, work, size = _work("sb_cross_attention_work", dev, 1, b, heads, kv_heads, dim, tq, tk)
    _launch("sb_cross_attention_backward", dev, *(x for t in views for x in t), lse.data_ptr(), DTYPES[q.dtype], b, heads,
            kv_heads, dim, tq, tk, scale, *masks, *(x for t in grads for x in t), work, size)
    return dq, dk, dv


# ---------------------------------------------------------------- positions
def rope_table(sections, theta=10000.0, per_axis=True, device="cuda"):
    """(freq fp64 [R], axis int32 [R]) of :func:`rope_axes`: ``sections[a]`` pairs turn with axis a, in
    this order.  Frequencies theta ** (-i / n): i counts an axis's own n pairs (per_axis), or all R."""
    _require(len(sections) >= 1 and all(int(n) == n and n >= 0 for n in sections) and theta > 0, "sections of pairs")
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
    fp64, so positions in the millions keep their fraction of a turn.  out may be x itself."""
    _require(x.dim() == 3 and x.dtype in DTYPES, "x: [B, T, heads * dim] of fp16, bf16 or fp32")
    b, t, width = x.shape
    _require(heads >= 1 and width % heads == 0 and width > 0, "x: a multiple of heads channels")
    dim = width // heads
    _require(layout in ("half", "pairs"), "layout: 'half' or 'pairs'")
    _require(freq.dtype == torch.float64 and axis.dtype == torch.int32 and freq.dim() == 1 and
             freq.shape == axis.shape and freq.is_contiguous() and axis.is_contiguous(), "freq fp64 [R], axis int32 [R]")
    _require(2 * freq.numel() <= dim, "pairs: at most half of a head's channels")
    _require(pos.dtype in (torch.int32, torch.float32) and pos.dim() in (2, 3) and
             tuple(pos.shape[:-1]) in ((t,), (b, t)) and pos.shape[-1] >= 1, "pos: int32 or fp32 [B, T, A] or [T, A]")
    a = pos.shape[-1]
    _require((a == 1 or pos.stride(-1) == 1) and (t <= 1 or pos.stride(-2) == a), "pos: contiguous rows")
    pos_img = pos.stride(0) if pos.dim() == 3 and b > 1 else 0
    xp = _rows(x, "x", (b, t, width))
    if out is not None:
        op = _rows(out, "out", (b, t, width), x.dtype, out=True)
    dev = _ready(x, pos, freq, axis, out)
    if out is None:
        out = torch.empty(b, t, width, device=dev, dtype=x.dtype)
        op = (out.data_ptr(), width, t * width)
    if out.numel() == 0:
        return out
    _launch("sb_rope_axes", dev, *xp, DTYPES[x.dtype], b, t, heads, dim, pos.data_ptr(), int(pos.dtype == torch.float32),
            pos_img, a, freq.data_ptr(), axis.data_ptr(), freq.numel(), int(layout == "pairs"), int(inverse), *op)
    return out


# ---------------------------------------------------------------- gated residual and norms
def _norm_weights(w, what, d, kind):
    """A norm's (weight, bias) or None -> (weight, bias) tensors or None."""
    if w is None:
        return None, None
    w, b = w if isinstance(w, (tuple, list)) else (w, None)
    for t in (w, b):
        _require(t is None or (t.dtype == torch.float32 and tuple(t.shape) == (d,) and t.is_contiguous()),
                 f"{what}: contiguous fp32 [D] weight and bias")
    _require(w is not None and (b is None or kind == "layer"), f"{what}: a weight, and a bias for layer norms only")
    return w, b


def _norm_inputs(x, z, gate, scale, post, pre, kind, eps):
    _require(x.dim() == 3 and x.dtype in DTYPES and z.dtype in DTYPES, "x, z: [B, T, D] of fp16, bf16 or fp32")
    _require(kind in ("rms", "layer") and eps >= 0, "kind: 'rms' or 'layer', eps >= 0")
    b, t, d = x.shape
    _require(1 <= d <= 8192, "1 to 8192 channels")
    gp = (None, 0, 0)
    if gate is not None:
        _require(gate.dtype == z.dtype, "gate: z's type")
        _require(tuple(gate.shape) in ((d,), (b, d), (b, t, d)), "gate: [D], [B, D] or [B, T, D]")
        _require(d == 1 or gate.stride(-1) == 1, "gate: channels must be contiguous")
        row = gate.stride(1) if gate.dim() == 3 and t > 1 else 0
        gp = (gate.data_ptr(), row, gate.stride(0) if gate.dim() > 1 and b > 1 else 0)
    _require(scale is None or (scale.dtype == torch.float32 and tuple(scale.shape) == (d,) and scale.is_contiguous()),
             "scale: contiguous fp32 [D]")
    weights = _norm_weights(post, "post", d, kind) + _norm_weights(pre, "pre", d, kind)
    return (b, t, d), _rows(x, "x", (b, t, d)), _rows(z, "z", (b, t, d)), gp, weights


def _ptr(t):
    return None if t is None else t.data_ptr()


def gated_norm(x, z, gate=None, scale=None, post=None, pre=None, kind="rms", eps=1e-6, y=None, h=None):
    """The end of a block and the start of the next: n = Npost(z), y = x + scale * gate * n, h = Npre(y).

    x (the residual) and z (the block's output): [B, T, D] rows; y has x's type and h z's.  post, pre: a
    norm's fp32 [D] weight or (weight, bias), None for no norm there (without pre, h is None).  kind:
    "rms" or "layer".  gate: z's type, [D], [B, D] (one an item) or [B, T, D].  scale: fp32 [D].  h comes
    from y before its rounding.  y may be x and h may be z.  Returns (y, h)."""
    (b, t, d), xp, zp, gp, weights = _norm_inputs(x, z, gate, scale, post, pre, kind, eps)
    _require(h is None or pre is not None, "h needs the norm pre")
    yp = _rows(y, "y", (b, t, d), x.dtype, out=True) if y is not None else None
    hp = _rows(h, "h", (b, t, d), z.dtype, out=True) if h is not None else (None, 0, 0)
    dev = _ready(x, z, gate, scale, *weights, y, h)
    if y is None:
        y = torch.empty(b, t, d, device=dev, dtype=x.dtype)
        yp = (y.data_ptr(), d, t * d)
    if h is None and pre is not None:
        h = torch.empty(b, t, d, device=dev, dtype=z.dtype)
        hp = (h.data_ptr(), d, t * d)
    if y.numel():
        _launch("sb_gated_norm", dev, *xp, DTYPES[x.dtype], *zp, DTYPES[z.dtype], *gp, _ptr(scale), *map(_ptr, weights),
                int(kind == "layer"), eps, b, t, d, *yp, *hp)
    return y, h


def gated_norm_backward(dy, dh, x, z, gate=None, scale=None, post=None, pre=None, kind="rms", eps=1e-6):
    """Gradients of :func:`gated_norm` from dy (x's type, None: zero) and dh (z's type, None: zero).

    Returns a dict of dx (x's type), dz (z's type) and, where there is such an input, fp32 scale,
    post_w, post_b, pre_w, pre_b [D] and gate: fp32 [D] or [B, D] sums for a gate of that shape, z's
    type for one of [B, T, D]; None otherwise.  The sums over rows have a fixed order."""
    (b, t, d), xp, zp, gp, weights = _norm_inputs(x, z, gate, scale, post, pre, kind, eps)
    _require(dh is None or pre is not None, "dh needs the norm pre")
    dyp = _rows(dy, "dy", (b, t, d), x.dtype) if dy is not None else (None, 0, 0)
    dhp = _rows(dh, "dh", (b, t, d), z.dtype) if dh is not None else (None, 0, 0)
    dev = _ready(x, z, gate, scale, *weights, dy, dh)
    g = {"dx": torch.empty(b, t, d, device=dev, dtype=x.dtype), "dz": torch.empty(b, t, d, device=dev, dtype=z.dtype)}
    make = torch.empty if b * t else torch.zeros  # no rows: every sum is zero
    for name, w in zip(("scale", "post_w", "post_b", "pre_w", "pre_b"), (scale,) + weights):
        g[name] = None if w is None else make(d, device=dev, dtype=torch.float32)
    mode = 0 if gate is None else gate.dim()
    g["gate"] = None if gate is None else make(gate.shape, device=dev, dtype=z.dtype if mode == 3 else torch.float32)
    if b * t == 0:
        return g
    hold, work, size = _work("sb_gated_norm_work", dev, b, t, d)
    _launch("sb_gated_norm_backward", dev, *dyp, *dhp, *xp, DTYPES[x.dtype], *zp, DTYPES[z.dtype], *gp, _ptr(scale),
            *map(_ptr, weights), int(kind == "layer"), eps, b, t, d, _ptr(g["dx"]), _ptr(g["dz"]), _ptr(g["scale"]),
            _ptr(g["gate"]), mode, _ptr(g["post_w"]), _ptr(g["post_b"]), _ptr(g["pre_w"]), _ptr(g["pre_b"]), work, size)
    return g
