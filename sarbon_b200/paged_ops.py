"""A memory that a camera stream keeps between frames: its states in pages, read, extended and cut back.

Where :func:`sarbon_b200.cross_attention` is given an encoder's whole memory with each call, a tracker
that runs for days keeps one: every frame adds its tokens, a few query tokens attend to all that is
there, and once there is more than the budget allows, the states that were looked at least go::

    n = paged_write(k, v, k_pages, v_pages, table, lens, weight=weight, born=born, stamp=frame)
    o = paged_attention(q, k_pages, v_pages, table, n, heads, kv_heads=kv_heads, weight=weight, decay=0.98)
    paged_evict(k_pages, v_pages, table, n, weight, budget, born=born, since=oldest, weight_out=weight,
                born_out=born, after=lens)

``k_pages`` and ``v_pages`` are pools ``[P, page, kv_heads * dim]`` of fp16, bf16 or e4m3 (heads of 32, 64
or 128 channels; any page size; pages and rows any multiple of 16 bytes apart, so keys and values may
lie side by side).  ``table`` (int32 [B, N]) names the pages of an item's states: state j is row
``j % page`` of page ``table[b, j // page]``.  A number outside [0, P) is no page: its states are neither
written nor read and take no part in attention (eviction does not ask for a page, see there).  Pages may be shared by items
that only read them.  Lengths (int32 [B]) outside [0, N * page] are clamped.  What a call writes shares no memory with what
it reads or else writes; rows may lie between one another, as keys and values side by side do.

``weight`` (fp32) and ``born`` (int32), ``[B, kv_heads, N * page]``, hold for each state and key head how much it was
looked at and its stamp (a frame number, say).  Eviction decides for each key head by itself, so a row's heads may
stem from different states afterwards; attention does not mind the order of states, and their positions are in
the keys (:func:`sarbon_b200.rope_axes` before they are written).

Every call launches kernels of ``libsarbon_sparse.so`` on the current CUDA stream of its tensors' device,
takes its workspace from torch's allocator and can be captured in a CUDA graph after a first call outside
capture.  No graph of gradients is recorded; tensors that would need one are refused.
"""
from __future__ import annotations

import ctypes
import math
import struct
import warnings

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import check, lib
from .memory_ops import _device, _new, _raw_stream, _ready, _rows, _statistics, _work

E4M3 = torch.float8_e4m3fn
_MOST = 3.4e38  # of fp32
_INT, _FLOAT, _HALF, _BRAIN = torch.int32, torch.float32, torch.float16, torch.bfloat16
# sb_paged_attend, sb_paged_append, sb_paged_cut, each from its sb_paged_memory on: a call's host time is what a small call
# costs, and a struct packed at once costs less of it than as many arguments
_MEMORY = "@PPqqqqPqiiiiiii4x"
_ATTEND = struct.Struct(_MEMORY + "PPqqqqPPPPqiiiiffff")
_APPEND = struct.Struct(_MEMORY + "PPqqqqPPPPPqqPiiff")
_CUT = struct.Struct(_MEMORY + "PPPPPPPPPqi4x")
PAGE_DTYPES = {torch.float16: _lib.SB_F16, torch.bfloat16: _lib.SB_BF16, E4M3: _lib.SB_F8}


# library calls made through this module
CALLS = [0]

_native = None


class _PythonSide:
    """In place of the native module: every call is left to the Python side."""
    attend = append = cut = staticmethod(lambda *arguments: None)


def _load():
    """The module that makes plainly right calls with little host time.  Measured, us a call with one token, with the checks
    below and there: attention 11.8 and 8.2 (5.0 of them the host's), writing 13.5 and 5.4, evicting 14.8 and 10.3.  Without
    it, or where it was built for another torch, all calls are made from here."""
    global _native
    so = lib()
    try:
        from . import _paged_calls
        if _paged_calls.built_for != torch.__version__:
            raise ImportError(f"built for torch {_paged_calls.built_for}")
    except ImportError as e:
        warnings.warn(f"_paged_calls is not used ({e}), small calls take longer on the host; it is built by "
                      "`python -m sarbon_b200.build_lib`", RuntimeWarning, stacklevel=3)
        _native = _PythonSide
        return _native
    _paged_calls.setup(*(ctypes.cast(f, ctypes.c_void_p).value for f in (
        so.sb_paged_attention, so.sb_paged_attention_work, so.sb_paged_write, so.sb_paged_evict, so.sb_paged_evict_work)), check)
    _native = _paged_calls
    return _native


def _call(name, index, packed):
    CALLS[0] += 1
    entry = getattr(lib(), name)
    if index == _device():
        status = entry(packed, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = entry(packed, _raw_stream(index))
    if status:
        check(status, name)


def _overlap(row, img, pages, page, width):
    """Whether rows of a pool with these strides lie on one another."""
    return (page > 1 and row < width) or (pages > 1 and img < row * (page - 1) + width and not
                                          (img >= width and (page == 1 or row >= img * (pages - 1) + width)))


def _memory(k_pages, v_pages, table, kv_heads, written=False):
    """The memory of a call: (the fields of sb_paged_memory, batch, page, entries, dim)."""
    shape, dtype = k_pages.shape, k_pages.dtype
    code = PAGE_DTYPES.get(dtype)
    if len(shape) != 3 or code is None or v_pages.shape != shape or v_pages.dtype != dtype:
        raise ValueError("k_pages, v_pages: [P, page, kv_heads * dim] pools of one shape and type, fp16, bf16 or e4m3")
    pages, page, width = shape
    dim = width // kv_heads if kv_heads >= 1 else 0
    if page < 1 or dim not in (32, 64, 128) or dim * kv_heads != width:
        raise ValueError("pools: pages of one state or more, key heads of 32, 64 or 128 channels")
    (k_img, k_row, k_one), (v_img, v_row, v_one) = k_pages.stride(), v_pages.stride()
    if k_one != 1 or v_one != 1:
        raise ValueError("pools: channels must be contiguous")
    # the stride of a dimension of one element is arbitrary and never used
    if page == 1:
        k_row = v_row = width
    if pages <= 1:
        k_img, v_img = page * k_row, page * v_row
    k, v = k_pages.data_ptr(), v_pages.data_ptr()
    if written:
        if not (k_row >= width <= v_row and k_img >= k_row * page and v_img >= v_row * page) and \
                (_overlap(k_row, k_img, *shape) or _overlap(v_row, v_img, *shape)):
            raise ValueError("pools: rows overlap")
    if table.dtype != _INT or table.dim() != 2:
        raise ValueError("table: int32 [B, N] with contiguous rows")
    (b, n), step = table.shape, table.stride()
    if step[1] != 1 and n > 1:
        raise ValueError("table: int32 [B, N] with contiguous rows")
    if n * page >= 1 << 30 or pages >= 1 << 31:
        raise ValueError("fewer than 2^30 states an item, 2^31 pages")
    return (k, v, k_row, k_img, v_row, v_img, table.data_ptr(), step[0] if b > 1 else n, code, pages, page, n, b, kv_heads, dim), \
        b, page, n, dim


def _each(t, what, b):
    """Pointer of an int32 [B]."""
    if t.dtype != _INT or t.shape != (b,) or not t.is_contiguous():
        raise ValueError(f"{what}: contiguous int32 [B]")
    return t.data_ptr()


def _account(t, what, shape, dtype):
    """Pointer of weights or stamps."""
    if t.shape != shape or t.dtype != dtype or not t.is_contiguous():
        raise ValueError(f"{what}: contiguous {dtype} {tuple(shape)}")
    return t.data_ptr()


def _one_device(floats, others):
    """memory_ops._ready for a call of many tensors, of which only `floats` could need a gradient."""
    if forward_ad._current_level >= 0:
        return _ready(*floats, *others)
    index = floats[0].get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            raise ValueError("tensors of one CUDA device")
    grad = torch.is_grad_enabled()
    for t in floats:
        if t is not None:
            if t.get_device() != index or not t.is_cuda:
                raise ValueError("tensors of one CUDA device")
            if grad and t.requires_grad:
                raise ValueError("no autograd graph is recorded: call under torch.no_grad() or from an autograd.Function")
    return index


def _scales(k_scale, v_scale, dtype):
    if not (0.0 < k_scale < _MOST and 0.0 < v_scale < _MOST):
        raise ValueError("k_scale, v_scale: positive numbers")
    if dtype != E4M3 and (k_scale != 1.0 or v_scale != 1.0):
        raise ValueError("k_scale, v_scale: of e4m3 pages only")


def _steps(t):
    """A tensor's memory: bytes of its contiguous runs, and how often each step (in bytes) goes on from the first."""
    size = run = t.element_size()
    steps = {}
    for step, n in sorted(zip(t.stride(), t.shape)):
        if n > 1 and step:
            step *= size
            if step == run and not steps:
                run *= n
            else:
                steps[step] = steps.get(step, 0) + n - 1
    return run, steps


def _meet(a, b):
    """Whether two tensors, whose first to last bytes overlap, share memory.  Rows that lie between the other's, of up to two
    different strides in all, are told apart; others only where a common divisor of their strides has room for both."""
    (run, mine), (width, its) = _steps(a), _steps(b)
    apart, steps = b.data_ptr() - a.data_ptr(), sorted(mine.keys() | its.keys())
    if not steps:
        return True
    g = math.gcd(*steps)
    if run <= apart % g <= g - width:
        return False
    if len(steps) > 2:
        return True
    # a run of b begins apart + x outer + y inner behind one of a: they meet between -width and run
    inner, outer = steps[0], steps[-1]
    y0, y1 = -mine.get(inner, 0), its.get(inner, 0)
    x0, x1 = (-mine.get(outer, 0), its.get(outer, 0)) if outer != inner else (0, 0)
    x0 = max(x0, (-width - y1 * inner - apart) // outer + 1)
    x1 = min(x1, -((apart + y0 * inner - run) // outer) - 1)
    if x1 - x0 > 64:
        return True
    for d in range(apart + x0 * outer, apart + x1 * outer + 1, outer):
        if max(y0, (-width - d) // inner + 1) <= min(y1, -((d - run) // inner) - 1):
            return True
    return False


def _own_memory(results, operands):
    """Results that share no memory with an operand or another result."""
    spans = []
    for group in results, operands:
        for t in group:
            if t is not None and t.numel():
                lo = t.data_ptr()
                last = sum((n - 1) * step for n, step in zip(t.shape, t.stride()))
                spans.append((lo, lo + (last + 1) * t.element_size(), group is results, t))
    spans.sort(key=lambda x: x[0])
    for i, (lo, hi, result, t) in enumerate(spans):
        for other in spans[i + 1:]:
            if other[0] >= hi:
                break
            if (result or other[2]) and _meet(t, other[3]):
                raise ValueError("results need their own memory")


# ---------------------------------------------------------------- attention
def paged_attention(q, k_pages, v_pages, table, lens, heads, kv_heads=None, scale=None, causal=False, k_scale=1.0,
                    v_scale=1.0, weight=None, decay=1.0, out=None, lse=None):
    """softmax(scale q k^T) v per head of a few query tokens [B, Tq, heads * dim] (fp16 or bf16) over the
    ``lens[b]`` states of each item's pages.

    Query head h reads key head ``h // (heads // kv_heads)``.  causal: the queries are the last Tq of the
    states, and query t sees those up to itself, the first ``lens[b] - Tq + 1 + t``.  A query without
    states gets zeros.  Pages have q's type, or e4m3: a code c of a key then stands for ``c * k_scale``, of a value for
    ``c * v_scale``.  scale: 1 / sqrt(dim) unless given.  Fills out (allocated if None) and, if given, lse (fp32
    [B, heads, Tq], the log-sum-exp of the scaled scores, -inf without states).

    weight (fp32 [B, kv_heads, N * page]), if given, is brought up to date: ``weight[b, h, j] = decay *
    weight[b, h, j] +`` the probabilities that the queries of key head h gave to state j, for the ``lens[b]`` states;
    sums have a fixed order.  Without queries (Tq 0) that is ``decay`` times it.  This takes a workspace of 4 bytes for each
    key head, place of the table (``N * page``, whatever the lengths) and query row, rows of a key head up to 16 counted as 1, 2,
    4, 8 or 16, more as a multiple of 16; none where a few hundred places' scores stay in shared memory.

    Made for single tokens: the states are read once for every 16 query rows of a key head (``Tq * heads // kv_heads``), and
    split over the SMs where there are few rows.  So 300 queries read them 19 times; cross_attention reads them once, but
    wants the memory in one piece and of q's type."""
    if q.is_cuda and forward_ad._current_level < 0:
        done = (_native or _load()).attend(q, k_pages, v_pages, table, lens, heads, kv_heads, scale, causal, k_scale, v_scale,
                                           weight, decay, out, lse)
        if done is not None:
            CALLS[0] += 1
            return done
    dtype, page_dtype = q.dtype, k_pages.dtype
    if q.dim() != 3 or (dtype != _BRAIN and dtype != _HALF):
        raise ValueError("q: [B, T, heads * dim] rows of fp16 or bf16")
    if kv_heads is None:
        kv_heads = heads
    if heads < 1 or kv_heads < 1 or heads % kv_heads:
        raise ValueError("heads: a multiple of kv_heads")
    memory, b, page, n, dim = _memory(k_pages, v_pages, table, kv_heads)
    if page_dtype != dtype and page_dtype != E4M3:
        raise ValueError("pages: q's type or e4m3")
    tq = q.shape[1]
    shape = (b, tq, heads * dim)
    if scale is None:
        scale = dim ** -0.5
    if not 0.0 < scale < _MOST or not 0.0 <= decay <= 1.0:
        raise ValueError("scale: a positive number; decay: from 0 to 1")
    if k_scale != 1.0 or v_scale != 1.0:
        _scales(k_scale, v_scale, page_dtype)
    if lens is None:
        raise ValueError("lens: contiguous int32 [B]")
    qp, p_lens = _rows(q, "q", shape, dtype), _each(lens, "lens", b)
    p_weight = p_lse = 0
    if weight is not None:
        p_weight = _account(weight, "weight", (b, kv_heads, n * page), _FLOAT)
    if lse is not None:
        _statistics(lse, b, heads, tq)
        p_lse = lse.data_ptr()
    if out is not None:
        op = _rows(out, "out", shape, dtype, out=True)
    _own_memory((out, lse, weight), (q, k_pages, v_pages, table, lens))
    index = _one_device((q, k_pages, v_pages, weight, out, lse), (table, lens))
    if out is None:
        out, op = _new(q, shape, dtype)
    if b == 0 or (tq == 0 and (weight is None or n == 0)):
        return out
    hold, work, size = _work("sb_paged_attention_work", index, b, heads, kv_heads, dim, tq, PAGE_DTYPES[page_dtype], page, n,
                             weight is not None)
    _call("sb_paged_attention", index, _ATTEND.pack(*memory, qp[0], op[0], qp[1], qp[2], op[1], op[2], p_lens, p_lse, p_weight,
                                                    work or 0, size, PAGE_DTYPES[dtype], heads, tq, causal, scale, k_scale,
                                                    v_scale, decay))
    return out


# ---------------------------------------------------------------- new states
def paged_write(k, v, k_pages, v_pages, table, at, count=None, k_scale=1.0, v_scale=1.0, weight=None, born=None,
                stamp=None, after=None, kv_heads=None):
    """Writes new states k, v [B, T, kv_heads * dim] (fp16 or bf16) behind the ``at[b]`` that item b has, the first
    ``count[b]`` (int32 [B]) of each or all T, and returns the new lengths (int32 [B]).

    Pages have the states' type, or e4m3: the code nearest to the fp32 quotient ``x / k_scale`` (``v_scale``), at
    most 448 of either sign.  The new states' weight becomes 0 and born their stamp (int32 [B, T], or [B] for
    all of an item's).  States behind an item's pages are dropped, rows on no page are not written, and what
    lies from ``count[b]`` on is left alone.  An item's pages that are written must be its own.  after
    is allocated if None.  kv_heads is that of weight or born where they are given;
    without them the rows are taken as heads of 32 channels."""
    if k.is_cuda and forward_ad._current_level < 0:
        done = (_native or _load()).append(k, v, k_pages, v_pages, table, at, count, k_scale, v_scale, weight, born, stamp,
                                           after, kv_heads)
        if done is not None:
            CALLS[0] += 1
            return done
    dtype, page_dtype, rows = k.dtype, k_pages.dtype, k.shape
    if len(rows) != 3 or (dtype != _BRAIN and dtype != _HALF):
        raise ValueError("k, v: [B, T, kv_heads * dim] rows of fp16 or bf16")
    if (born is None) != (stamp is None):
        raise ValueError("born and stamp: both or neither")
    if kv_heads is None:
        like = weight if weight is not None else born
        if like is not None and like.dim() != 3:
            raise ValueError("weight, born: [B, kv_heads, N * page]")
        kv_heads = rows[2] // 32 if like is None else like.shape[1]
    memory, b, page, n, dim = _memory(k_pages, v_pages, table, kv_heads, written=True)
    if page_dtype != dtype and page_dtype != E4M3:
        raise ValueError("pages: the states' type or e4m3")
    if k_scale != 1.0 or v_scale != 1.0:
        _scales(k_scale, v_scale, page_dtype)
    t = rows[1]
    shape = (b, t, kv_heads * dim)
    kp, vp = _rows(k, "k", shape, dtype), _rows(v, "v", shape, dtype)
    if at is None:
        raise ValueError("at: contiguous int32 [B]")
    p_at, p_count, p_weight, p_born, sp = _each(at, "at", b), 0, 0, 0, _NO_STAMP
    if count is not None:
        p_count = _each(count, "count", b)
    if weight is not None:
        p_weight = _account(weight, "weight", (b, kv_heads, n * page), _FLOAT)
    if born is not None:
        p_born = _account(born, "born", (b, kv_heads, n * page), _INT)
        if stamp.dtype != _INT or stamp.shape not in ((b, t), (b,)):
            raise ValueError("stamp: int32 [B, T] or [B]")
        step = stamp.stride()
        sp = stamp.data_ptr(), step[0], step[1] if len(step) == 2 else 0
    if after is not None:
        p_after = _each(after, "after", b)
    _own_memory((k_pages, v_pages, weight, born, after), (k, v, table, at, count, stamp))
    index = _one_device((k, v, k_pages, v_pages, weight), (table, at, count, born, stamp, after))
    if after is None:
        after = torch.empty_like(at)
        p_after = after.data_ptr()
    if b == 0:
        return after
    _call("sb_paged_write", index, _APPEND.pack(*memory, kp[0], vp[0], kp[1], kp[2], vp[1], vp[2], p_at, p_count, p_weight, p_born,
                                                *sp, p_after, PAGE_DTYPES[dtype], t, k_scale, v_scale))
    return after


_NO_STAMP = (0, 0, 0)


# ---------------------------------------------------------------- eviction
def paged_evict(k_pages, v_pages, table, lens, weight, keep, born=None, since=None, weight_out=None, born_out=None,
                after=None):
    """Cuts every item's ``lens[b]`` states back to ``keep`` (a number, or int32 [B]), for each key head by itself.

    Those with ``born >= since[b]`` (int32 [B]) stay before all others, then those of larger weight, of equal
    ones the first; NaN is the least.  The i-th freed place below keep takes the i-th kept state from keep
    on: keys, values, weight and stamp; nothing else moves.  Returns (after, weight, born): the new
    lengths ``min(lens, keep)``, and weights and stamps [B, kv_heads, N * page] with 0 from the new length on
    (born None without born).  after, weight_out and born_out (allocated if None) may be lens, weight and born
    themselves and otherwise share no memory with them.  An item's pages must be its own.

    Weights and stamps alone decide, also among states on no page.  So each of the ``lens[b]`` states of an item that has
    more than keep needs a page: a row is moved only where both places have one, and where one of them has none, the
    weight and stamp that move to a place are no longer those of the row that lies there."""
    if weight.is_cuda and forward_ad._current_level < 0:
        done = (_native or _load()).cut(k_pages, v_pages, table, lens, weight, keep, born, since, weight_out, born_out, after)
        if done is not None:
            CALLS[0] += 1
            return done
    places = weight.shape
    if len(places) != 3:
        raise ValueError("weight: [B, kv_heads, N * page]")
    kv_heads = places[1]
    memory, b, page, n, dim = _memory(k_pages, v_pages, table, kv_heads, written=True)
    if places != (b, kv_heads, n * page) or lens is None:
        raise ValueError("weight: [B, kv_heads, N * page]; lens: contiguous int32 [B]")
    pw, p_lens = _account(weight, "weight", places, _FLOAT), _each(lens, "lens", b)
    pb = p_since = p_keep = 0
    if born is not None:
        pb = _account(born, "born", places, _INT)
    elif since is not None or born_out is not None:
        raise ValueError("since and born_out need born")
    if since is not None:
        p_since = _each(since, "since", b)
    keep_all = 0
    if isinstance(keep, torch.Tensor):
        p_keep = _each(keep, "keep", b)
    else:
        keep_all = min(int(keep), 1 << 30) if 0 <= keep < math.inf else -1
        if keep_all < 0 or keep_all != min(keep, 1 << 30):
            raise ValueError("keep: a whole number from 0 on, or int32 [B]")
    pwo = pbo = p_after = 0
    operands = [table]
    if weight_out is not None:
        pwo = _account(weight_out, "weight_out", places, _FLOAT)
    if weight_out is None or pwo != pw:
        operands.append(weight)
    if born_out is not None:
        pbo = _account(born_out, "born_out", places, _INT)
    if born_out is None or pbo != pb:
        operands.append(born)
    if after is not None:
        p_after = _each(after, "after", b)
    here = p_after if p_after == p_lens else 0  # (lens may be since or keep too)
    operands += [t for t, p in ((lens, p_lens), (since, p_since), (keep if p_keep else None, p_keep)) if p != here]
    _own_memory((k_pages, v_pages, weight_out, born_out, after), operands)
    index = _one_device((k_pages, v_pages, weight, weight_out),
                        (table, lens, born, since, keep if p_keep else None, born_out, after))
    if after is None:
        after = torch.empty_like(lens)
        p_after = after.data_ptr()
    if weight_out is None:
        weight_out = torch.empty_like(weight)
        pwo = weight_out.data_ptr()
    if born is not None and born_out is None:
        born_out = torch.empty_like(born)
        pbo = born_out.data_ptr()
    if b == 0:
        return after, weight_out, born_out
    hold, work, size = _work("sb_paged_evict_work", index, b, kv_heads, page, n, p_after == p_lens)
    _call("sb_paged_evict", index, _CUT.pack(*memory, p_lens, p_keep, p_since, pw, pb, pwo, pbo, p_after, work or 0, size, keep_all))
    return after, weight_out, born_out
