"""The memory-reading block's operators against their formulas in 64 bits.

Bounds: a value rounded to type t is off by at most u = eps(t) / 2 of itself.  Attention rounds its
probabilities (and dS in the backward pass) once to the inputs' type before the second product, so an
output sum_j p_j v_j is off by at most u (|out| + sum_j p_j |v_j|); fp16 probabilities below 2^-14 are
rounded by at most 2^-25 absolutely.  Everything else is fp32: scores are off by at most
(dim + 2) 2^-24 sum |q||k| scale, the exponential by a few 2^-22, sums by a few 2^-22 of their
absolute terms; ``FP32`` = 2^-18 of the absolute terms covers these."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

FP32 = 2.0 ** -18


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need CUDA")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(g, *shape, dtype=torch.float32, by=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * by).to(dtype)


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def heads_of(x, heads, groups):
    """[B, T, heads * dim] -> fp64 [B, groups, heads / groups, T, dim]."""
    return x.double().unflatten(-1, (groups, heads // groups, -1)).permute(0, 2, 3, 1, 4)


def rows_of(x):
    return x.permute(0, 3, 1, 2, 4).flatten(2)


def keep_of(b, tk, lens, valid):
    keep = torch.ones(b, tk, dtype=torch.bool, device="cuda")
    if lens is not None:
        keep &= torch.arange(tk, device="cuda") < lens[:, None]
    return keep if valid is None else keep & (valid != 0)


def formula(q, k, v, heads, kv_heads, lens, valid, scale=None):
    """(out, lse, P, q, k, v) in fp64, keys that take no part left out of every sum."""
    q, k, v = heads_of(q, heads, kv_heads), heads_of(k, kv_heads, kv_heads), heads_of(v, kv_heads, kv_heads)
    keep = keep_of(q.shape[0], k.shape[3], lens, valid)
    k, v = (x.masked_fill(~keep[:, None, None, :, None], 0) for x in (k, v))
    s = q @ k.transpose(-1, -2) * (scale or q.shape[-1] ** -0.5)
    s = s.masked_fill(~keep[:, None, None, None], -math.inf)
    lse = torch.logsumexp(s, -1) if s.shape[-1] else s.new_full(s.shape[:-1], -math.inf)
    p = torch.where(lse[..., None] == -math.inf, 0.0, torch.exp(s - lse[..., None]))
    return p @ v, lse, p, q, k, v


def slack_of(q, k, scale=None):
    """Relative error of a probability from the fp32 scores."""
    s = q.abs() @ k.abs().transpose(-1, -2) * (scale or q.shape[-1] ** -0.5)
    return FP32 + 2 * (q.shape[-1] + 2) * 2.0 ** -24 * (s.amax().item() if s.numel() else 0.0)


def check_forward(out, lse, q, k, v, heads, kv_heads, lens, valid, scale=None):
    ref, ref_lse, p, qd, kd, vd = formula(q, k, v, heads, kv_heads, lens, valid, scale)
    u, e = unit(q.dtype), slack_of(qd, kd, scale)
    tol = u * ref.abs() + (u + e) * (p @ vd.abs()) + 1e-30
    if q.dtype == torch.float16:
        tol = tol + 2.0 ** -25 * (2 + vd.abs().sum(-2, keepdim=True))
    err = (out.double() - rows_of(ref)).abs()
    assert out.isfinite().all()
    assert (err <= 1.02 * rows_of(tol)).all(), (err / rows_of(tol)).max().item()
    if lse is not None:
        ref_lse = ref_lse.flatten(1, 2)
        none = ref_lse == -math.inf
        assert torch.equal(lse == -math.inf, none)
        assert ((lse.double() - ref_lse).abs()[~none] <= e * (1 + ref_lse.abs()[~none])).all()
    return ref, p


TYPES = [torch.float16, torch.bfloat16]


# one key, a full tile of 128 and its neighbours, several tiles, more query rows than a tile
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,tq,tk,heads,kv_heads,dim", [
    (2, 300, 240, 8, 8, 32), (1, 1, 1, 1, 1, 64), (2, 5, 77, 4, 2, 128), (1, 128, 128, 2, 1, 64),
    (3, 129, 127, 3, 3, 32), (2, 257, 385, 6, 2, 128), (1, 130, 129, 7, 1, 64), (4, 1, 2040, 8, 2, 128),
    (1, 1, 4097, 5, 1, 32), (2, 33, 1000, 12, 4, 64), (1, 513, 64, 2, 2, 128), (1, 3, 9001, 1, 1, 128),
    (160, 1, 8160, 4, 1, 128), (160, 1, 8160, 1, 1, 64), (80, 300, 5000, 2, 2, 32), (80, 300, 4100, 2, 2, 128),
])
def test_cross_attention(b, tq, tk, heads, kv_heads, dim, dtype):
    import sarbon_b200 as sb
    g = gen(tq * 7 + tk)
    q = rand(g, b, tq, heads * dim, dtype=dtype)
    k, v = rand(g, b, tk, kv_heads * dim, dtype=dtype), rand(g, b, tk, kv_heads * dim, dtype=dtype)
    lse = torch.empty(b, heads, tq, device="cuda")
    out = sb.cross_attention(q, k, v, heads, kv_heads=kv_heads, lse=lse)
    check_forward(out, lse, q, k, v, heads, kv_heads, None, None)
    assert torch.equal(out, sb.cross_attention(q, k, v, heads, kv_heads=kv_heads))  # with and without lse, twice


MASKS = ["lens", "valid", "both", "none_left", "ends", "holes"]


def masks_of(kind, b, tk, g):
    lens = valid = None
    if kind in ("lens", "both"):
        lens = torch.tensor([(tk * (i + 1)) // b - (i == 0) for i in range(b)], dtype=torch.int32, device="cuda")
    if kind in ("valid", "both"):
        valid = (torch.rand(b, tk, device="cuda", generator=g) < 0.6).to(torch.uint8)
    if kind == "none_left":
        lens = torch.tensor([0, tk] + [-5] * (b - 2), dtype=torch.int32, device="cuda")[:b]
        valid = torch.ones(b, tk, dtype=torch.bool, device="cuda")
        valid[min(1, b - 1)] = False
    if kind == "ends":  # outside [0, Tk]: clamped
        lens = torch.tensor([1, tk + 1000, 2 ** 31 - 1, 128][:b], dtype=torch.int32, device="cuda")
    if kind == "holes":  # whole tiles without a key between tiles with some
        valid = torch.zeros(b, tk, dtype=torch.uint8, device="cuda")
        valid[:, tk // 2] = 1
        valid[0, -1] = 255
    return lens, valid


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", MASKS)
@pytest.mark.parametrize("tq,tk,heads,kv_heads,dim", [(70, 300, 4, 2, 64), (1, 700, 4, 1, 128), (150, 129, 2, 2, 32),
                                                      (260, 520, 2, 1, 128)])
def test_cross_attention_masks(kind, tq, tk, heads, kv_heads, dim, dtype):
    """Masked places hold NaN and infinities; a row without keys gives zeros."""
    import sarbon_b200 as sb
    g = gen(tk + len(kind))
    b = 4
    q = rand(g, b, tq, heads * dim, dtype=dtype)
    kv = rand(g, b, tk, 2 * kv_heads * dim, dtype=dtype)
    lens, valid = masks_of(kind, b, tk, g)
    away = ~keep_of(b, tk, lens, valid)
    kv[away] = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(dtype).min], device="cuda", dtype=dtype).repeat(
        kv.shape[-1] // 4)
    k, v = kv[..., :kv_heads * dim], kv[..., kv_heads * dim:]
    lse = torch.empty(b, heads, tq, device="cuda")
    out = sb.cross_attention(q, k, v, heads, kv_heads=kv_heads, lens=lens, valid=valid, lse=lse)
    check_forward(out, lse, q, k, v, heads, kv_heads, lens, valid)
    if kind == "none_left":
        assert not out[0].any() and not out[1].any()


@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("tq", [1, 300])
def test_cross_attention_long_ragged(tq, dim):
    """Many key tiles a CTA of ragged, masked items: every stage of the rings is used many times."""
    import sarbon_b200 as sb
    g = gen(77)
    b, tk, heads, kv_heads = 160, 6000, 2, 1
    q = rand(g, b, tq, heads * dim, dtype=torch.bfloat16)
    kv = rand(g, b, tk, 2 * dim, dtype=torch.bfloat16)
    lens = torch.randint(0, tk + 1, (b,), device="cuda", generator=g, dtype=torch.int32)
    valid = torch.rand(b, tk, device="cuda", generator=g) < 0.8
    lse = torch.empty(b, heads, tq, device="cuda")
    for masks in ((lens, None), (None, valid), (lens, valid)):
        out = sb.cross_attention(q, kv[..., :dim], kv[..., dim:], heads, kv_heads=kv_heads, lens=masks[0], valid=masks[1],
                                 lse=lse)
        for i in range(0, b, 40):  # forty items at a time
            at = slice(i, i + 40)
            check_forward(out[at], lse[at], q[at], kv[at, :, :dim], kv[at, :, dim:], heads, kv_heads,
                          None if masks[0] is None else masks[0][at], None if masks[1] is None else masks[1][at])


def test_cross_attention_strides_and_scale():
    """Sequence-first rows, a slice of a wider projection, one memory for all items, out in place of a
    slice; what lies around out stays as it was."""
    import sarbon_b200 as sb
    g = gen(5)
    b, tq, tk, heads, dim = 3, 45, 200, 4, 64
    q = rand(g, tq, b, heads * dim, dtype=torch.bfloat16).transpose(0, 1)
    wide = rand(g, 1, tk, 3 * heads * dim, dtype=torch.bfloat16)
    k = wide[..., :heads * dim].expand(b, -1, -1)
    v = wide[..., 2 * heads * dim:].expand(b, -1, -1)
    hold = torch.full((b, tq + 2, heads * dim + 8), 7.0, device="cuda", dtype=torch.bfloat16)
    out = hold[:, 1:-1, 8:]
    assert sb.cross_attention(q, k, v, heads, scale=0.3, out=out) is out
    check_forward(out, None, q, k, v, heads, heads, None, None, scale=0.3)
    assert (hold[:, 0] == 7).all() and (hold[:, -1] == 7).all() and (hold[..., :8] == 7).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_cross_attention_large_scores(dtype):
    """Scores that grow from tile to tile and differ by hundreds: the running maximum moves often."""
    import sarbon_b200 as sb
    g = gen(6)
    b, tq, tk, heads, dim = 1, 140, 1500, 2, 64
    q = rand(g, b, tq, heads * dim, dtype=dtype)
    ramp = torch.linspace(0.1, 6.0, tk, device="cuda")[None, :, None]
    k = (rand(g, b, tk, heads * dim) * ramp).to(dtype)
    v = rand(g, b, tk, heads * dim, dtype=dtype)
    lse = torch.empty(b, heads, tq, device="cuda")
    out = sb.cross_attention(q, k, v, heads, scale=1.0, lse=lse)
    check_forward(out, lse, q, k, v, heads, heads, None, None, scale=1.0)


@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("tq", [1, 16, 40, 300])
@pytest.mark.parametrize("far", [25.0, 24.6, 30.0])
def test_cross_attention_small_probabilities(tq, dim, far):
    """One key on top of a long memory, the others 2^-far of it: their sum counts although each lies near or
    below fp16's smallest number.  P is held times 2^7, where a value below 2^-14 is rounded by at most
    2^-25, so each of them is off by at most 2^-32 of the top one (or u of itself)."""
    import sarbon_b200 as sb
    b, tk = 160, 8160
    z = dict(device="cuda", dtype=torch.float16)
    q, k, v = torch.zeros(b, tq, dim, **z), torch.zeros(b, tk, dim, **z), torch.ones(b, tk, dim, **z)
    q[..., 0] = 1
    k[:, 1:, 0] = -far  # scores in powers of two: the scale is log 2
    v[:, 0] = 0
    lse = torch.empty(b, 1, tq, device="cuda")
    out = sb.cross_attention(q, k, v, 1, scale=math.log(2.0), lse=lse)
    each = 2.0 ** k[0, 1, 0].double().item()
    total = 1 + (tk - 1) * each
    u, e = unit(torch.float16), FP32 + 2 * (dim + 2) * 2.0 ** -24 * far
    want = (tk - 1) * each / total
    tol = want * (2 * u + e) + (tk - 1) * 2.0 ** -32 + 2.0 ** -25
    assert ((out.double() - want).abs() <= 1.02 * tol).all(), (out.double().min().item(), out.double().max().item(), want)
    assert ((lse.double() - math.log(total)).abs() <= e).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tq", [1, 300])
def test_cross_attention_huge_scores(tq, dtype):
    """Scores of tens of millions, far apart and growing, with ties at the top: exact integers in fp32, and
    probabilities of 1 / ties and 0."""
    import sarbon_b200 as sb
    b, tk, dim = 160, 1400, 64
    z = dict(device="cuda", dtype=dtype)
    q, k = torch.full((b, tq, dim), 128.0, **z), torch.zeros(b, tk, dim, **z)
    v = rand(gen(8), b, tk, dim, dtype=dtype)
    k[:] = (8192.0 - 64.0 * torch.arange(13, -1, -1, device="cuda").repeat_interleave(100))[:, None].to(dtype)
    lse = torch.empty(b, 1, tq, device="cuda")
    out = sb.cross_attention(q, k, v, 1, scale=math.log(2.0), lse=lse)
    best = k[0, :, 0] == k[0, -1, 0]
    want = v[:, best].double().mean(1, keepdim=True).expand(b, tq, dim)
    tol = 2 * unit(dtype) * v[:, best].double().abs().mean(1, keepdim=True) + FP32 + 2.0 ** -25
    assert ((out.double() - want).abs() <= 1.02 * tol).all()
    score = math.log(2.0) * 64 * 128 * k[0, -1, 0].double().item()
    assert ((lse.double() - score - math.log(best.sum().item())).abs() <= 2.0 ** -22 * score).all()


def test_cross_attention_empty_sizes():
    import sarbon_b200 as sb
    z = dict(device="cuda", dtype=torch.float16)
    assert sb.cross_attention(torch.zeros(0, 3, 64, **z), torch.zeros(0, 5, 64, **z), torch.zeros(0, 5, 64, **z), 1).shape == (0, 3, 64)
    assert sb.cross_attention(torch.zeros(2, 0, 64, **z), torch.zeros(2, 5, 64, **z), torch.zeros(2, 5, 64, **z), 1).shape == (2, 0, 64)
    lse = torch.zeros(2, 2, 3, device="cuda")
    q, none = torch.ones(2, 3, 64, **z), torch.zeros(2, 0, 64, **z)
    out = sb.cross_attention(q, none, none, 2, lse=lse)
    assert not out.any() and (lse == -math.inf).all()
    dq, dk, dv = sb.cross_attention_backward(q, q, none, none, out, lse, 2)
    assert not dq.any() and dk.shape == dv.shape == (2, 0, 64)
    k = torch.ones(2, 5, 64, **z)
    empty = torch.zeros(2, 0, 64, **z)
    dq, dk, dv = sb.cross_attention_backward(empty, empty, k, k, empty, torch.zeros(2, 2, 0, device="cuda"), 2)
    assert dq.shape == (2, 0, 64) and not dk.any() and not dv.any()


def check_backward(grads, dout, q, k, v, heads, kv_heads, lens, valid, out16, scale=None, sub_ds=None, sub_p=None, one_tile=False):
    ref, lse, p, qd, kd, vd = formula(q, k, v, heads, kv_heads, lens, valid, scale)
    scale = scale or qd.shape[-1] ** -0.5
    g, o = heads_of(dout, heads, kv_heads), heads_of(out16, heads, kv_heads)
    u, e = unit(q.dtype), slack_of(qd, kd, scale)
    dp, d = g @ vd.transpose(-1, -2), (g * ref).sum(-1, keepdim=True)
    ds = p * (dp - d)
    # dS is off by its rounding, by D from the rounded out, by P and by the fp32 products
    absd = (g.abs() * ref.abs()).sum(-1, keepdim=True)
    sub = 2.0 ** -25 if q.dtype == torch.float16 else 0.0  # fp16 values below 2^-14
    from_out = 0 if one_tile else (g * (o - ref)).abs().sum(-1, keepdim=True)
    ds_tol = u * ds.abs() + p * (from_out + e * (g.abs() @ vd.abs().transpose(-1, -2) + absd)) + \
        (sub if sub_ds is None else sub_ds)
    p_tol = (u + e) * p + (sub if sub_p is None else sub_p)
    want = {"dq": (ds @ kd * scale, ds_tol @ kd.abs() * scale),
            "dk": ((ds.transpose(-1, -2) @ qd * scale).sum(2, keepdim=True),
                   (ds_tol.transpose(-1, -2) @ qd.abs() * scale).sum(2, keepdim=True)),
            "dv": ((p.transpose(-1, -2) @ g).sum(2, keepdim=True), (p_tol.transpose(-1, -2) @ g.abs()).sum(2, keepdim=True))}
    for name, got in zip(("dq", "dk", "dv"), grads):
        r, t = (rows_of(x) for x in want[name])
        t = t + u * r.abs() + sub
        err = (got.double() - r).abs()
        assert got.isfinite().all(), name
        assert (err <= 1.02 * t + 1e-30).all(), (name, (err / (t + 1e-30)).max().item())
    return {n: rows_of(w[0]) for n, w in want.items()}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,tq,tk,heads,kv_heads,dim,kind", [
    (2, 300, 240, 8, 8, 32, None), (1, 1, 1, 1, 1, 64, None), (2, 5, 77, 4, 2, 128, None), (1, 64, 128, 2, 1, 64, None),
    (3, 65, 129, 6, 2, 64, "lens"), (4, 130, 200, 4, 4, 32, "none_left"), (4, 257, 130, 4, 1, 128, "both"),
    (4, 1, 700, 4, 2, 128, "valid"), (2, 40, 385, 3, 1, 64, "holes"), (4, 33, 260, 2, 2, 128, "ends"),
    (1, 700, 3, 2, 1, 128, None),
])
def test_cross_attention_backward(b, tq, tk, heads, kv_heads, dim, kind, dtype):
    import sarbon_b200 as sb
    g = gen(tq * 3 + tk)
    q, dout = rand(g, b, tq, heads * dim, dtype=dtype), rand(g, b, tq, heads * dim, dtype=dtype)
    kv = rand(g, b, tk, 2 * kv_heads * dim, dtype=dtype)
    lens, valid = masks_of(kind, b, tk, g) if kind else (None, None)
    kv[~keep_of(b, tk, lens, valid)] = math.nan
    k, v = kv[..., :kv_heads * dim], kv[..., kv_heads * dim:]
    ref, lse, *_ = formula(q, k, v, heads, kv_heads, lens, valid)
    out, lse = rows_of(ref).to(dtype), lse.flatten(1, 2).float().contiguous()
    call = lambda: sb.cross_attention_backward(dout, q, k, v, out, lse, heads, kv_heads=kv_heads, lens=lens, valid=valid)  # noqa: E731
    grads = call()
    check_backward(grads, dout, q, k, v, heads, kv_heads, lens, valid, out)
    assert all(torch.equal(x, y) for x, y in zip(grads, call()))  # the same bits again
    away = ~keep_of(b, tk, lens, valid)
    assert not grads[1][away].any() and not grads[2][away].any()


def test_cross_attention_backward_strides():
    """Gradients written into slices of one projection's gradient; a memory shared by the items."""
    import sarbon_b200 as sb
    g = gen(9)
    b, tq, tk, heads, dim = 3, 50, 140, 2, 64
    q, dout = (rand(g, tq, b, heads * dim, dtype=torch.float16).transpose(0, 1) for _ in range(2))
    kv = rand(g, 1, tk, 2 * heads * dim, dtype=torch.float16).expand(b, -1, -1)
    k, v = kv[..., :heads * dim], kv[..., heads * dim:]
    lse = torch.empty(b, heads, tq, device="cuda")
    out = sb.cross_attention(q, k, v, heads, lse=lse)
    both = torch.full((b, tk, 2 * heads * dim + 16), 3.0, device="cuda", dtype=torch.float16)
    dk, dv = both[..., 8:8 + heads * dim], both[..., 8 + heads * dim:-8]
    grads = sb.cross_attention_backward(dout, q, k, v, out, lse, heads, dk=dk, dv=dv)
    assert grads[1] is dk and grads[2] is dv
    check_backward(grads, dout, q, k, v, heads, heads, None, None, out)
    assert (both[..., :8] == 3).all() and (both[..., -8:] == 3).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tq,tk,heads,kv_heads,dim", [(300, 2, 3, 1, 32), (7, 20, 4, 4, 64), (140, 128, 2, 1, 128), (5, 400, 2, 2, 64)])
def test_cross_attention_backward_few_keys(tq, tk, heads, kv_heads, dim, dtype):
    """Items whose keys fit one tile: D is not left with the rounding of out."""
    import sarbon_b200 as sb
    g = gen(tq + tk)
    b = 4
    q, dout = (rand(g, b, tq, heads * dim, dtype=dtype) for _ in range(2))
    k, v = (rand(g, b, tk, kv_heads * dim, dtype=dtype) for _ in range(2))
    lens = torch.tensor([min(tk, 128), 1, 0, min(tk, 19)], device="cuda", dtype=torch.int32)
    ref, lse, *_ = formula(q, k, v, heads, kv_heads, lens, None)
    out, lse = rows_of(ref).to(dtype), lse.flatten(1, 2).float().contiguous()
    grads = sb.cross_attention_backward(dout, q, k, v, out, lse, heads, kv_heads=kv_heads, lens=lens)
    check_backward(grads, dout, q, k, v, heads, kv_heads, lens, None, out, one_tile=True)


@pytest.mark.parametrize("kv_heads", [1, 4])
def test_cross_attention_backward_small_fp16(kv_heads):
    """fp16 gradients of a long memory and a small loss: P and dS lie far below fp16's normal numbers,
    and keep its precision all the same.  P is held times 2^14 and dS times a power of two that
    keeps 2 max |dout_i| max |v_j| in 2^14 .. 2^15, so a subnormal step of 2^-24 there, half of
    which a rounding may be off by, is this much smaller."""
    import sarbon_b200 as sb
    g = gen(21)
    b, tq, tk, heads, dim = 1, 40, 1500, 4, 64
    q = rand(g, b, tq, heads * dim, dtype=torch.float16)
    k, v = (rand(g, b, tk, kv_heads * dim, dtype=torch.float16) for _ in range(2))
    dout = rand(g, b, tq, heads * dim, by=2.0 ** -8).half()
    ref, lse, *_ = formula(q, k, v, heads, kv_heads, None, None)
    out, lse = rows_of(ref).half(), lse.flatten(1, 2).float().contiguous()
    grads = sb.cross_attention_backward(dout, q, k, v, out, lse, heads, kv_heads=kv_heads)
    most = (heads_of(dout, heads, kv_heads).norm(dim=-1).max() * heads_of(v, kv_heads, kv_heads).norm(dim=-1).max()).item()
    check_backward(grads, dout, q, k, v, heads, kv_heads, None, None, out, sub_ds=2.0 ** -25 * 2 * most / 2 ** 14,
                   sub_p=2.0 ** -39)


@pytest.mark.parametrize("which", ["dout", "q", "k", "v", "all"])
def test_cross_attention_rows_of_one(which):
    """Operands whose rows are one and the same (row stride 0): the gradient of a sum over the queries, one
    learned query for every place, one state for every key."""
    import sarbon_b200 as sb
    g = gen(12)
    b, tq, tk, heads, kv_heads, dim = 2, 140, 200, 4, 2, 64
    x = {n: rand(g, b, 1 if which in (n, "all") else t, h * dim, dtype=torch.bfloat16).expand(b, t, h * dim)
         for n, t, h in (("dout", tq, heads), ("q", tq, heads), ("k", tk, kv_heads), ("v", tk, kv_heads))}
    valid = torch.rand(b, tk, device="cuda", generator=g) < 0.7
    dout, qkv = x.pop("dout"), list(x.values())
    lse = torch.empty(b, heads, tq, device="cuda")
    out = sb.cross_attention(*qkv, heads, kv_heads=kv_heads, valid=valid, lse=lse)
    check_forward(out, lse, *qkv, heads, kv_heads, None, valid)
    grads = sb.cross_attention_backward(dout, *qkv, out, lse, heads, kv_heads=kv_heads, valid=valid)
    check_backward(grads, dout, *qkv, heads, kv_heads, None, valid, out)


@pytest.mark.parametrize("top", [2.0 ** 15, math.inf])
def test_cross_attention_backward_rows_of_other_sizes(top):
    """fp16: one query whose incoming gradient is 2^23 times the others', or not finite, leaves their dq
    as precise as it is without it.  A row's dS is held times 2^14 and a power of two from the
    row's own |dout_i| max |v_j|, so a step of 2^-24 there is as in the test above, row by row."""
    import sarbon_b200 as sb
    g = gen(22)
    b, tq, tk, heads, kv_heads, dim = 1, 150, 4000, 2, 1, 64
    q, k = rand(g, b, tq, heads * dim, by=2.0 ** -5).half(), rand(g, b, tk, dim, by=2.0 ** 5).half()
    v, dout = rand(g, b, tk, dim).half(), rand(g, b, tq, heads * dim, by=2.0 ** -8).half()
    dout[:, 5, 3] = top
    ref, lse, p, qd, kd, vd = formula(q, k, v, heads, kv_heads, None, None)
    out, lse = rows_of(ref).half(), lse.flatten(1, 2).float().contiguous()
    dq = sb.cross_attention_backward(dout, q, k, v, out, lse, heads, kv_heads=kv_heads)[0]
    gd, od, u, e, scale = heads_of(dout, heads, kv_heads), heads_of(out, heads, kv_heads), unit(q.dtype), slack_of(qd, kd), dim ** -0.5
    ds = p * (gd @ vd.transpose(-1, -2) - (gd * ref).sum(-1, keepdim=True))
    most = gd.norm(dim=-1, keepdim=True) * vd.norm(dim=-1).max()
    ds_tol = u * ds.abs() + 2.0 ** -25 * 2 * most / 2 ** 14 + \
        p * ((gd * (od - ref)).abs().sum(-1, keepdim=True) + e * (gd.abs() @ vd.abs().transpose(-1, -2) + (gd * ref).abs().sum(-1, keepdim=True)))
    want = rows_of(ds @ kd * scale)
    tol = rows_of(ds_tol @ kd.abs() * scale) + u * want.abs() + 2.0 ** -25
    rest = torch.arange(tq, device="cuda") != 5
    err = (dq.double() - want).abs()[:, rest]
    assert dq[:, rest].isfinite().all()
    assert (err <= 1.02 * tol[:, rest]).all(), (err / tol[:, rest]).max().item()


@pytest.mark.parametrize("kind", ["lens", "valid", "both", "queries"])
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_cross_attention_backward_long_ragged(dim, kind):
    """So many items that no range of steps is split: each CTA streams many tiles of keys (dq) or, with many
    queries, of queries (dk, dv), and every stage of its ring is used many times."""
    import sarbon_b200 as sb
    g = gen(78 + dim)
    b, tq, tk, heads, kv_heads = (160, 300, 3000, 2, 1) if kind != "queries" else (160, 1500, 200, 2, 1)
    q, dout = (rand(g, b, tq, heads * dim, dtype=torch.bfloat16) for _ in range(2))
    kv = rand(g, b, tk, 2 * dim, dtype=torch.bfloat16)
    lens = valid = None
    if kind != "valid":
        lens = torch.randint(0, tk + 1, (b,), device="cuda", generator=g, dtype=torch.int32)
    if kind != "lens":
        valid = torch.rand(b, tk, device="cuda", generator=g) < 0.8
    kv[~keep_of(b, tk, lens, valid)] = math.nan
    k, v = kv[..., :dim], kv[..., dim:]
    lse = torch.empty(b, heads, tq, device="cuda")
    out = sb.cross_attention(q, k, v, heads, kv_heads=kv_heads, lens=lens, valid=valid, lse=lse)
    grads = sb.cross_attention_backward(dout, q, k, v, out, lse, heads, kv_heads=kv_heads, lens=lens, valid=valid)
    for i in range(0, b, 20):  # twenty items at a time
        at = slice(i, i + 20)
        check_backward([x[at] for x in grads], dout[at], q[at], k[at], v[at], heads, kv_heads, None if lens is None else lens[at],
                       None if valid is None else valid[at], out[at])
    again = sb.cross_attention_backward(dout, q, k, v, out, lse, heads, kv_heads=kv_heads, lens=lens, valid=valid)
    assert all(torch.equal(x, y) for x, y in zip(grads, again))


def test_cross_attention_gradient_against_differences():
    """<gradient, direction> against the central difference of the 64-bit formula, whose own error at
    step 1e-4 is of order 1e-8; the gradients carry roundings of u to each of their many terms."""
    import sarbon_b200 as sb
    g = gen(10)
    b, tq, tk, heads, kv_heads, dim = 2, 40, 70, 4, 2, 64
    x = [rand(g, b, n, h * dim, dtype=torch.float16) for n, h in ((tq, heads), (tk, kv_heads), (tk, kv_heads))]
    dout = rand(g, b, tq, heads * dim, dtype=torch.float16)
    lens = torch.tensor([70, 33], dtype=torch.int32, device="cuda")
    lse = torch.empty(b, heads, tq, device="cuda")
    out = sb.cross_attention(*x, heads, kv_heads=kv_heads, lens=lens, lse=lse)
    grads = sb.cross_attention_backward(dout, *x, out, lse, heads, kv_heads=kv_heads, lens=lens)

    def loss(y):
        return (rows_of(formula(*y, heads, kv_heads, lens, None)[0]) * dout.double()).sum().item()

    for i in range(3):
        d = rand(g, *x[i].shape).double()
        up, down = ([y.double() + s * 1e-4 * d if j == i else y for j, y in enumerate(x)] for s in (1, -1))
        want = (loss(up) - loss(down)) / 2e-4
        got = (grads[i].double() * d).sum().item()
        # n roundings of relative size <= 4 u (P, dS, out, the result), of random sign
        tol = 4 * 4 * unit(torch.float16) * (grads[i].double() * d).square().sum().sqrt().item() + 1e-5 * abs(want)
        assert abs(got - want) <= tol, (i, got, want, tol)


# ---------------------------------------------------------------- rotary positions
def rope_formula(x, pos, heads, freq, axis, layout, inverse):
    b, t, width = x.shape
    y = x.double().view(b, t, heads, -1).clone()
    n = freq.numel()
    pos = pos.double().expand(b, t, -1)
    ok = (axis >= 0) & (axis < pos.shape[-1])
    angle = pos[..., axis.long().clamp(0, pos.shape[-1] - 1)] * freq * ok
    cos, sin = angle.cos()[:, :, None], angle.sin()[:, :, None] * (-1 if inverse else 1)
    at = (slice(0, n), slice(n, 2 * n)) if layout == "half" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    u, v = y[..., at[0]].clone(), y[..., at[1]].clone()
    y[..., at[0]], y[..., at[1]] = u * cos - v * sin, u * sin + v * cos
    size = torch.zeros_like(y)  # |u| + |v| of each channel's pair
    size[..., at[0]] = size[..., at[1]] = u.abs() + v.abs()
    return y.flatten(2), size.flatten(2)


def check_rope(out, x, *args):
    ref, size = rope_formula(x, *args)
    # sines and cosines off by about 2^-22, fp32 products and sums, one rounding to the type
    tol = unit(x.dtype) * ref.abs() + 2.0 ** -21 * size + (2.0 ** -25 if x.dtype == torch.float16 else 0)
    assert ((out.double() - ref).abs() <= 1.01 * tol).all(), ((out.double() - ref).abs() - tol).max().item()


@pytest.mark.parametrize("dtype", TYPES + [torch.float32])
@pytest.mark.parametrize("layout", ["half", "pairs"])
@pytest.mark.parametrize("b,t,heads,dim,sections,pos32", [
    (2, 300, 8, 32, (8, 8), True), (1, 1, 1, 64, (32,), False), (3, 77, 4, 128, (16, 24, 24), False),
    (2, 33, 3, 80, (4, 6, 6), False), (1, 50, 2, 20, (3, 4), True), (2, 9, 40, 64, (8, 12, 12), False),
])
def test_rope(b, t, heads, dim, sections, pos32, layout, dtype):
    import sarbon_b200 as sb
    g = gen(t + dim)
    freq, axis = sb.rope_table(sections)
    pos = torch.randint(-50, 5_000_000, (b, t, len(sections)), device="cuda", generator=g)
    pos = pos.float() + 0.25 if pos32 else pos.to(torch.int32)
    x = rand(g, b, t, heads * dim, dtype=dtype)
    for inverse in (False, True):
        out = sb.rope_axes(x, pos, heads, freq, axis, layout=layout, inverse=inverse)
        check_rope(out, x, pos, heads, freq, axis, layout, inverse)
    same = x.clone()
    assert sb.rope_axes(same, pos, heads, freq, axis, layout=layout, inverse=True, out=same) is same
    assert torch.equal(same, out)


def test_rope_views():
    """Positions shared by the items, odd offsets (no vector loads), an axis that pos lacks, a slice as
    output whose surroundings stay, no pairs at all."""
    import sarbon_b200 as sb
    g = gen(3)
    freq, axis = sb.rope_table((6, 5, 5))
    axis = axis.clone()
    axis[3], axis[4] = 7, -1
    pos = sb.grid_positions(3, 5, 7)
    wide = rand(g, 2, 105, 3 * 64 + 1, dtype=torch.bfloat16)
    x = wide[..., 1:129]
    hold = torch.full_like(wide, 9.0)
    out = sb.rope_axes(x, pos, 2, freq, axis, out=hold[..., 3:131])
    check_rope(out, x, pos[None], 2, freq, axis, "half", False)
    assert (hold[..., :3] == 9).all() and (hold[..., 131:] == 9).all()
    first = rand(g, 105, 2, 128).transpose(0, 1)
    check_rope(sb.rope_axes(first, pos, 2, freq, axis), first, pos[None], 2, freq, axis, "half", False)
    assert torch.equal(sb.rope_axes(x, pos, 2, freq[:0], axis[:0]), x)
    assert sb.rope_axes(x[:0], pos, 2, freq, axis).shape == (0, 105, 128)


@pytest.mark.parametrize("dtype", TYPES + [torch.float32])
@pytest.mark.parametrize("layout", ["half", "pairs"])
@pytest.mark.parametrize("b,t,heads,dim,sections", [(2, 20000, 3, 64, (16, 16)), (1, 30001, 8, 128, (16, 24, 8)),
                                                    (3, 16000, 5, 80, (4, 4, 8)), (1, 90000, 2, 20, (3, 4))])
def test_rope_many_tokens(b, t, heads, dim, sections, layout, dtype):
    """Enough tokens that a thread turns all of a token's heads, an odd number of them among them; also in place."""
    import sarbon_b200 as sb
    g = gen(t + heads)
    freq, axis = sb.rope_table(sections)
    pos = torch.randint(-50, 5_000_000, (b, t, len(sections)), device="cuda", generator=g, dtype=torch.int32)
    x = rand(g, b, t, heads * dim, dtype=dtype)
    out = sb.rope_axes(x, pos, heads, freq, axis, layout=layout)
    check_rope(out, x, pos, heads, freq, axis, layout, False)
    assert sb.rope_axes(x, pos, heads, freq, axis, layout=layout, out=x) is x
    assert torch.equal(x, out)


@pytest.mark.parametrize("dim", [2, 32])
def test_rope_angles(dim):
    """Sines and cosines themselves (pairs 0, 1), in fp32: one unit in the last place of the function (2^-24 below 1), half of
    one for the correction of the angle's rounding, and 2^-53 of 8e5 turns, three roundings of them."""
    import sarbon_b200 as sb
    t, n = 200_000, dim // 2
    x = torch.zeros(1, t, dim, device="cuda")
    x[..., n:] = 1
    freq = 1.0 / (1 + torch.arange(n, device="cuda", dtype=torch.float64))
    axis = torch.zeros(n, device="cuda", dtype=torch.int32)
    pos = torch.randint(-5_000_000, 5_000_000, (t, 1), device="cuda", generator=gen(4), dtype=torch.int32)
    out = sb.rope_axes(x, pos, 1, freq, axis)[0].double()
    angle = pos.double() * freq
    want = torch.cat([-angle.sin(), angle.cos()], -1)
    assert (out - want).abs().max().item() <= 1.5 * 2.0 ** -24 + 3 * 2.0 ** -53 * 5e6


# ---------------------------------------------------------------- gated residual and norms
def norm_formula(x, z, gate, scale, post, pre, kind, eps):
    def norm(v, w):
        m = v.mean(-1, keepdim=True) if kind == "layer" else 0
        r = ((v - m).square().mean(-1, keepdim=True) + eps).rsqrt()
        return (v - m) * r * w[0] + (0 if w[1] is None else w[1])

    n = norm(z, post) if post else z
    f = 1.0 if gate is None else gate[:, None] if gate.dim() == 2 else gate
    y = x + f * n * (1.0 if scale is None else scale)
    return y, norm(y, pre) if pre else None


def norm_case(g, b, t, d, xt, zt, kind, gate, scale, post, pre):
    def w(on):
        return None if not on else (1 + rand(g, d, by=0.3), rand(g, d, by=0.3) if kind == "layer" else None)

    shape = {None: None, "vector": (d,), "image": (b, d), "row": (b, t, d)}[gate]
    return dict(x=rand(g, b, t, d, dtype=xt, by=2.0), z=rand(g, b, t, d, dtype=zt),
                gate=None if shape is None else rand(g, *shape, dtype=zt), scale=rand(g, d) if scale else None,
                post=w(post), pre=w(pre), kind=kind, eps=1e-5)


def wide(s, grad=False):
    """The case's tensors in fp64."""
    f = lambda t: None if t is None else t.double().requires_grad_(grad)  # noqa: E731
    return {k: tuple(f(t) for t in v) if isinstance(v, tuple) else f(v) if torch.is_tensor(v) or v is None else v
            for k, v in s.items()}


NORMS = [
    (2, 300, 256, torch.float32, torch.float16, "layer", None, True, True, True),
    (1, 1, 8, torch.bfloat16, torch.bfloat16, "rms", "vector", False, True, True),
    (3, 17, 100, torch.float16, torch.float16, "layer", "image", True, False, True),
    (2, 40, 255, torch.float32, torch.bfloat16, "rms", "row", True, True, True),
    (2, 9, 1152, torch.bfloat16, torch.bfloat16, "layer", "image", True, True, True),
    (5, 3, 2048, torch.float32, torch.float32, "rms", "image", False, True, False),
    (1, 70, 64, torch.bfloat16, torch.float16, "layer", "row", False, True, True),
    (2, 5, 4104, torch.float32, torch.bfloat16, "layer", "vector", True, True, True),
    (1, 3, 8192, torch.bfloat16, torch.bfloat16, "rms", None, False, False, True),
    (4, 33, 768, torch.float32, torch.float16, "rms", None, True, False, False),
    (1, 1, 1, torch.float32, torch.float32, "rms", "row", True, True, True),
]


@pytest.mark.parametrize("case", NORMS, ids=lambda c: "x".join(map(str, c[:3])) + "-" + c[5])
def test_gated_norm(case):
    import sarbon_b200 as sb
    s = norm_case(gen(case[2]), *case)
    y, h = sb.gated_norm(**s)
    ry, rh = norm_formula(**wide(s))
    # fp32: products and sums of the terms of y; the norm's statistics are sums of D terms by trees
    d = wide(s)
    size = d["x"].abs() + (ry - d["x"]).abs() * 2 + 1
    assert ((y.double() - ry).abs() <= unit(y.dtype) * ry.abs() + FP32 * size + 2.0 ** -25).all()
    assert (h is None) == (s["pre"] is None)
    if h is not None:
        spread = (ry.abs().mean(-1, keepdim=True) + size) * (ry.square().mean(-1, keepdim=True) if case[5] == "rms" else
                                                             ry.var(-1, keepdim=True, unbiased=False)).add(s["eps"]).rsqrt()
        tol = unit(h.dtype) * rh.abs() + 2 * FP32 * (spread * d["pre"][0].abs() + 1) + 2.0 ** -25
        assert ((h.double() - rh).abs() <= tol).all(), ((h.double() - rh).abs() / tol).max().item()
    again = dict(s, x=s["x"].clone(), z=s["z"].clone())
    y2, h2 = sb.gated_norm(**again, y=again["x"], h=again["z"] if s["pre"] else None)  # in place
    assert torch.equal(y2, y) and (h is None or torch.equal(h2, h))


@pytest.mark.parametrize("missing", [None, "dy", "dh"])
@pytest.mark.parametrize("case", NORMS, ids=lambda c: "x".join(map(str, c[:3])) + "-" + c[5])
def test_gated_norm_backward(case, missing):
    import sarbon_b200 as sb
    g = gen(case[2] + 1)
    s = norm_case(g, *case)
    b, t, d = case[:3]
    dy = None if missing == "dy" else rand(g, b, t, d, dtype=case[3])
    dh = None if missing == "dh" or s["pre"] is None else rand(g, b, t, d, dtype=case[4])
    got = sb.gated_norm_backward(dy, dh, **s)
    w = wide(s, grad=True)
    y, h = norm_formula(**w)
    total = (y * (0 if dy is None else dy.double())).sum() + (0 if dh is None else (h * dh.double()).sum())
    total.backward()
    want = dict(dx=w["x"], dz=w["z"], gate=w["gate"], scale=w["scale"])
    for name in ("post", "pre"):
        want[name + "_w"], want[name + "_b"] = w[name] if w[name] else (None, None)
    for name, leaf in want.items():
        if leaf is None:
            assert got[name] is None
            continue
        r = torch.zeros_like(leaf) if leaf.grad is None else leaf.grad
        x = got[name].double()
        # one rounding to the type; fp32 chains of about ten operations on terms that may cancel
        # (measured by the gradient's own size), sums over rows by trees of chunks
        size = r.abs() + r.square().mean().sqrt() + (1 if name in ("dx", "dz") else math.sqrt(b * t))
        tol = unit(got[name].dtype) * r.abs() + 16 * FP32 * size + 2.0 ** -25
        assert ((x - r).abs() <= tol).all(), (name, ((x - r).abs() / tol).max().item())
    again = sb.gated_norm_backward(dy, dh, **s)
    assert all(v is None or torch.equal(v, again[k]) for k, v in got.items())


@pytest.mark.parametrize("t,d", [(70, 256), (33, 1024), (9, 4096)])
@pytest.mark.parametrize("rows", ["offset", "outlier", "flat"])
def test_gated_norm_backward_statistics(rows, t, d):
    """Layer norms of rows whose mean is hundreds of deviations, whose variance is one value's (the first:
    what the squares are taken around contains it), and whose z is one value throughout."""
    import sarbon_b200 as sb
    g = gen(d + len(rows))
    s = norm_case(g, 2, t, d, torch.float32, torch.float32, "layer", None, True, True, True)
    if rows == "offset":
        s["x"], s["z"] = s["x"] + 512, s["z"] - 256
        worse = 512.0  # roundings of values that large, measured in deviations
    elif rows == "outlier":
        s["x"][..., 0] += 4096
        s["z"][..., 0] -= 4096
        worse = d / 4.0  # E (v - c)^2 against its part (E v - c)^2
    else:
        s["z"][:] = 7.25
        worse = 1.0
    dy, dh = rand(g, 2, t, d), rand(g, 2, t, d)
    got = sb.gated_norm_backward(dy, dh, **s)
    w = wide(s, grad=True)
    y, h = norm_formula(**w)
    ((y * dy.double()).sum() + (h * dh.double()).sum()).backward()
    for name, r in (("dx", w["x"].grad), ("dz", w["z"].grad), ("post_w", w["post"][0].grad), ("pre_w", w["pre"][0].grad)):
        size = r.abs() + r.square().mean().sqrt() + (1 if name in ("dx", "dz") else math.sqrt(2 * t))
        if rows == "flat" and name == "dz":
            size = size * s["eps"] ** -0.5  # 1 / deviation is sqrt(1 / eps): every term of dz is that large
        if rows == "flat" and name == "post_w":
            assert not got[name].any()  # z - mean is exactly zero
            continue
        err = (got[name].double() - r).abs()
        assert (err <= 16 * FP32 * (1 + worse) * size).all(), (name, (err / (16 * FP32 * (1 + worse) * size)).max().item())


@pytest.mark.parametrize("d", [256, 1024, 2048, 4096, 8192])
@pytest.mark.parametrize("norm", ["post", "pre"])
def test_gated_norm_backward_deviation_of_outliers(norm, d):
    """Layer norms whose first four values are nearly all of the variance: 1 / deviation, the factor of a row's
    gradient, is as precise as a sum of D squares around a point of the row within four deviations of its
    mean: at most 17 var is summed, by chains of at most 16 + 5 + 8 additions, half of that in the root."""
    import sarbon_b200 as sb
    g = gen(d)
    b, t = 2, 20
    w, dd = 1 + rand(g, d, by=0.2), rand(g, b, t, d)
    far, near = rand(g, b, t, d), rand(g, b, t, d)
    far[..., :4] += 4096
    if norm == "post":
        got = sb.gated_norm_backward(dd, None, near, far, post=w, kind="layer", eps=1e-6)["dz"]
    else:
        got = sb.gated_norm_backward(None, dd, far, near * 2.0 ** -10, pre=w, kind="layer", eps=1e-6)["dx"]
    x = (far.double() if norm == "post" else far.double() + near.double() * 2.0 ** -10).requires_grad_(True)
    torch.nn.functional.layer_norm(x, (d,), w.double(), None, 1e-6).backward(dd.double())
    rest, want = got[..., 4:].double(), x.grad[..., 4:]
    off = ((rest * want).sum(-1) / want.square().sum(-1) - 1).abs().max().item()
    assert off <= 17 / 2 * 29 * 2.0 ** -24, off


def test_gated_norm_views_and_offset_rows():
    """Slices, an image's gate as an expanded row, rows whose mean is far from zero."""
    import sarbon_b200 as sb
    g = gen(21)
    b, t, d = 2, 30, 96
    s = norm_case(g, b, t, d, torch.float32, torch.bfloat16, "layer", None, True, True, True)
    s["x"] = (rand(g, b, t, 3 * d + 1) + 1000.0)[..., 1:d + 1]
    s["z"] = rand(g, t, b, d, dtype=torch.bfloat16).transpose(0, 1)
    s["gate"] = rand(g, b, 1, d, dtype=torch.bfloat16).expand(b, t, d)
    y, h = sb.gated_norm(**s)
    ry, rh = norm_formula(**wide(s))
    assert ((y.double() - ry).abs() <= 2.0 ** -23 * 1010).all()
    # fp32 rows around 1000 with deviations around 1: each value is known to 2^-24 * 1000
    assert ((h.double() - rh).abs() <= unit(torch.bfloat16) * rh.abs() + 8 * 2.0 ** -24 * 1000 * (1 + rh.abs())).all()
    got = sb.gated_norm_backward(y, h, **s)
    assert got["gate"].shape == (b, t, d) and got["gate"].dtype == torch.bfloat16
    none = {k: (v[:, :0] if k in ("x", "z", "gate") else v) for k, v in s.items()}
    y, h = sb.gated_norm(**none)
    assert y.shape == h.shape == (b, 0, d)
    got = sb.gated_norm_backward(y, h, **none)
    assert got["dx"].shape == (b, 0, d) and not got["post_w"].any() and not got["scale"].any()


@pytest.mark.parametrize("gate", ["image", "row"])
@pytest.mark.parametrize("d,odd", [(64, 0), (255, 0), (520, 0), (520, 1), (1152, 0), (4096, 0)])
def test_gated_norm_many_rows(d, odd, gate):
    """Many rows a team, of several items: every stage of a ring is used again, gates change on the way, and in place
    the next rows are on their way while one is written.  odd: rows that begin off 16 bytes."""
    import sarbon_b200 as sb
    g = gen(d + odd)
    b, t = (3, 9001) if d < 4096 else (5, 1803)
    s = norm_case(g, b, t, d, torch.float32, torch.bfloat16, "layer", gate, True, True, True)
    if odd:
        s["x"] = rand(g, b, t, d + 1, by=2.0)[..., 1:]
    y, h = sb.gated_norm(**s)
    again = dict(s, x=s["x"].clone(), z=s["z"].clone()) if not odd else \
        dict(s, x=torch.cat([s["x"][..., :1], s["x"]], -1)[..., 1:], z=s["z"].clone())
    y2, h2 = sb.gated_norm(**again, y=again["x"], h=again["z"])
    assert torch.equal(y2, y) and torch.equal(h2, h)
    for i in range(b):  # an item at a time
        one = wide(dict(s, x=s["x"][i:i + 1], z=s["z"][i:i + 1], gate=s["gate"][i:i + 1]))
        ry, rh = norm_formula(**one)
        size = one["x"].abs() + (ry - one["x"]).abs() * 2 + 1
        assert ((y[i:i + 1].double() - ry).abs() <= unit(y.dtype) * ry.abs() + FP32 * size + 2.0 ** -25).all()
        spread = (ry.abs().mean(-1, keepdim=True) + size) * ry.var(-1, keepdim=True, unbiased=False).add(s["eps"]).rsqrt()
        tol = unit(h.dtype) * rh.abs() + 2 * FP32 * (spread * one["pre"][0].abs() + 1) + 2.0 ** -25
        assert ((h[i:i + 1].double() - rh).abs() <= tol).all()


def grads_of(s, dy, dh):
    """The gradients in fp64, by differentiation."""
    w = wide(s, grad=True)
    y, h = norm_formula(**w)
    ((y * dy.double()).sum() + (h * dh.double()).sum()).backward()
    want = dict(dx=w["x"].grad, dz=w["z"].grad, gate=w["gate"].grad, scale=w["scale"].grad)
    for name in ("post", "pre"):
        want[name + "_w"], want[name + "_b"] = (None if v is None else v.grad for v in w[name])
    return want


@pytest.mark.parametrize("b,t,d,kind,gate,odd", [
    (3, 9001, 64, "layer", "image", 0), (3, 9001, 520, "rms", "row", 0), (3, 5001, 1152, "layer", "row", 0),
    (3, 5001, 520, "layer", "image", 1), (5, 803, 4096, "rms", "image", 0), (700, 3, 256, "layer", "image", 0),
    (300, 1, 96, "rms", "image", 0),
    (2, 70, 96, "layer", "expanded", 0), (2, 3001, 768, "layer", "expanded", 0), (2, 3001, 100, "rms", "expanded", 0),
])
def test_gated_norm_backward_many_rows(b, t, d, kind, gate, odd):
    """Rings used many times, teams whose rows are of several items, many items with a gate each, and a gate of each
    item given as rows (stride 0), whose gradient has a value a row."""
    import sarbon_b200 as sb
    g = gen(b + t + d)
    s = norm_case(g, b, t, d, torch.float32, torch.bfloat16, kind, "image" if gate == "expanded" else gate, True, True, True)
    if gate == "expanded":
        s["gate"] = s["gate"][:, None].expand(b, t, d)
    if odd:
        s["x"] = rand(g, b, t, d + 1, by=2.0)[..., 1:]
    dy, dh = rand(g, b, t, d), rand(g, b, t, d, dtype=torch.bfloat16)
    got, want = sb.gated_norm_backward(dy, dh, **s), grads_of(s, dy, dh)
    for name, r in want.items():
        if r is None:
            assert got[name] is None
            continue
        assert got[name].shape == r.shape
        x = got[name].double()
        size = r.abs() + r.square().mean().sqrt() + (1 if name in ("dx", "dz") or r.dim() == 3 else math.sqrt(b * t))
        tol = unit(got[name].dtype) * r.abs() + 16 * FP32 * size + 2.0 ** -25
        assert ((x - r).abs() <= tol).all(), (name, ((x - r).abs() / tol).max().item())


def far_apart(x):
    """x's values as the items of one buffer whose second item begins past 2^31 elements."""
    b, t, c = x.shape
    step = (2 ** 31 // max(1, b - 1) // c + 1) * c
    hold = torch.empty(step * (b - 1) + t * c, device="cuda", dtype=x.dtype)
    y = hold.as_strided((b, t, c), (step, c, 1))
    y.copy_(x)
    return y


@pytest.mark.parametrize("tq", [3, 140])
def test_items_past_32_bits(tq):
    """Items that lie more than 2^31 elements apart, in and out, give the bits of those that lie together."""
    import sarbon_b200 as sb
    g = gen(50)
    b, tk, heads, dim = 2, 300, 2, 64
    q, dout = (rand(g, b, tq, heads * dim, dtype=torch.float16) for _ in range(2))
    k, v = (rand(g, b, tk, heads * dim, dtype=torch.float16) for _ in range(2))
    valid = torch.rand(b, tk, device="cuda", generator=g) < 0.7
    lse, lse2 = torch.empty(b, heads, tq, device="cuda"), torch.empty(b, heads, tq, device="cuda")
    out = sb.cross_attention(q, k, v, heads, valid=valid, lse=lse)
    grads = sb.cross_attention_backward(dout, q, k, v, out, lse, heads, valid=valid)
    kf, of, vf = far_apart(k), far_apart(torch.zeros_like(out)), far_apart(valid[..., None])[..., 0]
    sb.cross_attention(q, kf, v, heads, valid=vf, lse=lse2, out=of)
    assert torch.equal(of, out) and torch.equal(lse2, lse)
    df = far_apart(torch.zeros_like(k))
    again = sb.cross_attention_backward(far_apart(dout), q, kf, v, of, lse, heads, valid=vf, dk=df)
    assert all(torch.equal(x, y) for x, y in zip(grads, again))
    freq, axis = sb.rope_table((16, 16))
    pos = torch.randint(0, 99, (b, tk, 2), device="cuda", generator=g, dtype=torch.int32)
    assert torch.equal(sb.rope_axes(kf, pos, heads, freq, axis, out=df), sb.rope_axes(k, pos, heads, freq, axis))
    for d in (128, 127):
        s = norm_case(g, b, tk, d, torch.float16, torch.float16, "layer", "row", True, True, True)
        far = dict(s, x=far_apart(s["x"]), gate=far_apart(s["gate"]))
        y, h = sb.gated_norm(**s)
        y2, h2 = sb.gated_norm(**far, y=far_apart(torch.zeros_like(y)))
        assert torch.equal(y2, y) and torch.equal(h2, h)
        want, got = sb.gated_norm_backward(y, h, **s), sb.gated_norm_backward(far_apart(y), h, **far)
        assert all(x is None or torch.equal(x, got[n]) for n, x in want.items())


def test_shared_queries():
    """Queries, and what comes back to them, that are one item's for all (a batch stride of 0)."""
    import sarbon_b200 as sb
    g = gen(51)
    b, tq, tk, heads, kv_heads, dim = 3, 150, 200, 4, 2, 64
    q, dout = (rand(g, 1, tq, heads * dim, dtype=torch.bfloat16).expand(b, -1, -1) for _ in range(2))
    k, v = (rand(g, b, tk, kv_heads * dim, dtype=torch.bfloat16) for _ in range(2))
    lse = torch.empty(b, heads, tq, device="cuda")
    out = sb.cross_attention(q, k, v, heads, kv_heads=kv_heads, lse=lse)
    check_forward(out, lse, q, k, v, heads, kv_heads, None, None)
    few = sb.cross_attention(q[:, :3], k, v, heads, kv_heads=kv_heads)
    check_forward(few, None, q[:, :3], k, v, heads, kv_heads, None, None)
    grads = sb.cross_attention_backward(dout, q, k, v, out, lse, heads, kv_heads=kv_heads)
    check_backward(grads, dout, q, k, v, heads, kv_heads, None, None, out)


# ---------------------------------------------------------------- together
def block(sb, g, heads, kv_heads, dim):
    """One block that reads a memory: positions, attention, gated residual and norms."""
    d = heads * dim
    freq, axis = sb.rope_table((dim // 8, dim // 8, dim // 4))
    return dict(d=d, freq=freq, axis=axis, w0=1 + rand(g, d, by=0.1), w1=1 + rand(g, d, by=0.1), heads=heads, kv=kv_heads)


def run_block(sb, p, x, q, k, v, qpos, kpos, gate, lens, lse):
    qr = sb.rope_axes(q, qpos, p["heads"], p["freq"], p["axis"])
    kr = sb.rope_axes(k, kpos, p["kv"], p["freq"], p["axis"])
    o = sb.cross_attention(qr, kr, v, p["heads"], kv_heads=p["kv"], lens=lens, lse=lse)
    y, h = sb.gated_norm(x, o, gate=gate, post=p["w0"], pre=p["w1"])
    return qr, kr, o, y, h


def back_block(sb, p, x, q, k, v, qpos, kpos, gate, lens, lse, qr, kr, o, dy, dh):
    g = sb.gated_norm_backward(dy, dh, x, o, gate=gate, post=p["w0"], pre=p["w1"])
    dqr, dkr, dv = sb.cross_attention_backward(g["dz"], qr, kr, v, o, lse, p["heads"], kv_heads=p["kv"], lens=lens)
    dq = sb.rope_axes(dqr, qpos, p["heads"], p["freq"], p["axis"], inverse=True)
    dk = sb.rope_axes(dkr, kpos, p["kv"], p["freq"], p["axis"], inverse=True)
    return g["dx"], dq, dk, dv, g["gate"], g["post_w"], g["pre_w"]


def block_inputs(g, p, b, tq, clip, dim):
    t = clip[0] * clip[1] * clip[2]
    z = dict(dtype=torch.bfloat16)
    return dict(x=rand(g, b, tq, p["d"]), q=rand(g, b, tq, p["d"], **z), k=rand(g, b, t, p["kv"] * dim, **z),
                v=rand(g, b, t, p["kv"] * dim, **z), gate=rand(g, b, p["d"], **z),
                qpos=torch.randint(0, 9, (b, tq, 3), device="cuda", generator=g, dtype=torch.int32),
                lens=torch.tensor([t, t // 2 + 1, 1][:b], dtype=torch.int32, device="cuda"),
                lse=torch.empty(b, p["heads"], tq, device="cuda"))


def test_block_forward_backward():
    """The operators one after the other against fp64 with autograd; each bf16 tensor on the way adds
    a rounding of u, and the chain multiplies them by a modest factor."""
    import sarbon_b200 as sb
    g = gen(30)
    b, tq, heads, kv_heads, dim, clip = 3, 60, 4, 2, 64, (2, 6, 10)
    p = block(sb, g, heads, kv_heads, dim)
    s = block_inputs(g, p, b, tq, clip, dim)
    kpos = sb.grid_positions(*clip)
    qr, kr, o, y, h = run_block(sb, p, kpos=kpos, **s)
    dy, dh = rand(g, *y.shape), rand(g, *h.shape, dtype=h.dtype)
    got = back_block(sb, p, kpos=kpos, **s, qr=qr, kr=kr, o=o, dy=dy, dh=dh)

    leaf = {n: s[n].double().requires_grad_(True) for n in ("x", "q", "k", "v", "gate")}
    w0, w1 = (p[n].double().requires_grad_(True) for n in ("w0", "w1"))

    def rot(x, pos, n):
        xx = x.view(b, -1, n, dim)
        a = pos.double().expand(b, -1, -1)[..., p["axis"].long()] * p["freq"]
        c, sn = a.cos()[:, :, None], a.sin()[:, :, None]
        u, v = xx[..., :dim // 2], xx[..., dim // 2:]
        return torch.cat([u * c - v * sn, u * sn + v * c], -1).flatten(2)

    ro = rows_of(formula(rot(leaf["q"], s["qpos"], heads), rot(leaf["k"], kpos, kv_heads), leaf["v"], heads, kv_heads,
                         s["lens"], None)[0])
    ry, rh = norm_formula(leaf["x"], ro, leaf["gate"], None, (w0, None), (w1, None), "rms", 1e-6)
    ((ry * dy.double()).sum() + (rh * dh.double()).sum()).backward()
    pairs = [(y, ry), (h, rh)] + list(zip(got, [t.grad for t in (*(leaf[n] for n in ("x", "q", "k", "v", "gate")), w0, w1)]))
    u = unit(torch.bfloat16)
    for i, (a, r) in enumerate(pairs):
        rel = ((a.double() - r).norm() / r.norm()).item()
        assert rel <= 6 * u, (i, rel, 6 * u)


def test_block_in_graphs_and_on_streams():
    """Two captured graphs and eager calls on a second stream, all in flight together, give the eager
    results: no workspace is shared."""
    import sarbon_b200 as sb
    b, tq, heads, kv_heads, dim, clip = 2, 3, 4, 1, 128, (4, 16, 30)
    kpos = sb.grid_positions(*clip)
    p = block(sb, gen(40), heads, kv_heads, dim)
    sets = [block_inputs(gen(41 + i), p, b, tq, clip, dim) for i in range(3)]

    def both(s):
        qr, kr, o, y, h = run_block(sb, p, kpos=kpos, **s)
        return (o, y, h) + back_block(sb, p, kpos=kpos, **s, qr=qr, kr=kr, o=o, dy=y, dh=h)

    want = [[t.clone() for t in both(s)] for s in sets]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in sets[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(both(s))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(3):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            third = both(sets[2])
    torch.cuda.synchronize()
    for w, o in zip(want, outs + [third]):
        assert all(torch.equal(x, y) for x, y in zip(w, o))
    from sarbon_b200 import det_ops
    assert det_ops.kernels_error() == 0
