"""The paged memory's operators against their formulas in 64 bits.

Bounds: a value rounded to type t is off by at most u = eps(t) / 2 of itself.  Attention multiplies its
probabilities as two 16-bit parts: what is left is u^2 of each (bf16 2^-16, fp16 2^-22), and in fp16, where
they are held times 2^7 or more, 2^-32 of the row's largest.  Everything else is fp32: scores are off by at most
(dim + 2) 2^-24 sum |q||k| scale, the exponential by a few 2^-22, sums by a few 2^-22 of their absolute terms;
``FP32`` = 2^-18 of the absolute terms covers these.  Writes and evictions move values and are exact."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

FP32 = 2.0 ** -18
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need CUDA")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(g, *shape, dtype=torch.float32, by=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * by).to(dtype)


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def same_bits(a, b):
    if a.is_floating_point():
        kind = {1: torch.uint8, 2: torch.int16, 4: torch.int32}[a.element_size()]
        a, b = a.contiguous().view(kind), b.contiguous().view(kind)
    return torch.equal(a, b)


def pages_of(g, b, n, page, width, dtype, by=1.0, spare=2):
    """Pools with what a memory holds, and a table of shuffled pages for n states an item."""
    need = max(1, -(-n // page))
    count = b * need + spare
    k, v = (rand(g, count, page, width, by=by).to(dtype) for _ in range(2))
    table = torch.randperm(count, device="cuda", generator=g)[:b * need].view(b, need).to(torch.int32)
    return k, v, table


def states(pool, table, kv_heads):
    """(fp64 [B, heads, places, dim], [B, places] of those on a page) of every item."""
    ok = (table >= 0) & (table < pool.shape[0])
    x = pool.float()[torch.where(ok, table, 0).long()].double().flatten(1, 2)
    return x.unflatten(-1, (kv_heads, -1)).transpose(1, 2), ok.repeat_interleave(pool.shape[1], 1)


def formula(q, k_pages, v_pages, table, lens, heads, kv_heads, scale=None, causal=False, k_scale=1.0, v_scale=1.0):
    """out [B, Hkv, rows, dim], lse, P, |P||V|, slack: rows are (head of the group, token)."""
    k, ok = states(k_pages, table, kv_heads)
    v, _ = states(v_pages, table, kv_heads)
    b, tq = q.shape[:2]
    n = lens.clamp(0, k.shape[2]).long()
    j = torch.arange(k.shape[2], device="cuda")
    used = ok & (j < n[:, None])
    k, v = (torch.where(used[:, None, :, None], x, 0.0) for x in (k * k_scale, v * v_scale))
    q = q.double().view(b, tq, kv_heads, heads // kv_heads, -1).permute(0, 2, 3, 1, 4).flatten(2, 3)
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    ends = n[:, None] - (torch.arange(tq - 1, -1, -1, device="cuda") if causal else torch.zeros(tq, device="cuda"))
    seen = (used[:, None] & (j < ends[..., None])).repeat(1, heads // kv_heads, 1)[:, None]
    s = (q @ k.transpose(-1, -2) * scale).masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(lse[..., None] == -math.inf, 0.0, torch.exp(s - lse[..., None]))
    # what a row does not see may be no number: its share is left out, not multiplied by 0
    finite = v.masked_fill(~v.isfinite(), 0.0)
    out = (p @ finite).masked_fill((p > 0).double() @ (~v.isfinite()).double() > 0, math.nan)
    reach = (q.abs() @ k.abs().nan_to_num(0.0).transpose(-1, -2)).masked_fill(~seen, 0.0).amax().item() * scale if k.shape[2] else 0.0
    return out, lse, p, p @ finite.abs(), finite.abs().sum(-2, keepdim=True), \
        FP32 + 2 * (q.shape[-1] + 2) * 2.0 ** -24 * reach


def rows_of(x, b, tq):
    return x.unflatten(2, (-1, tq)).permute(0, 3, 1, 2, 4).flatten(2)


def check_attention(got, lse, weight, q, k_pages, v_pages, table, lens, heads, kv_heads, before=None, decay=1.0, **how):
    out, ref_lse, p, absolute, whole, e = formula(q, k_pages, v_pages, table, lens, heads, kv_heads, **how)
    b, tq = q.shape[:2]
    half = torch.bfloat16 if k_pages.dtype == torch.bfloat16 else torch.float16
    tol = unit(q.dtype) * out.abs() + (unit(half) ** 2 + e) * absolute + 2.0 ** -32 * whole
    if q.dtype == torch.float16:
        tol = tol + 2.0 ** -25  # fp16's smallest step
    tol, out = rows_of(tol + 1e-30, b, tq), rows_of(out, b, tq)
    nan = out.isnan()
    assert torch.equal(got.isnan(), nan)
    err = (got.double() - out).abs()[~nan]
    assert (err <= 1.02 * tol[~nan]).all(), (err / tol[~nan]).max().item()
    ref_lse = ref_lse.view(b, heads, tq)
    if lse is not None:
        none = ref_lse == -math.inf
        assert torch.equal(lse == -math.inf, none)
        assert ((lse.double() - ref_lse).abs()[~none] <= e * (1 + ref_lse.abs()[~none])).all()
    if weight is not None:
        share, n = p.sum(2), lens.clamp(0, weight.shape[2])
        used = torch.arange(weight.shape[2], device="cuda") < n[:, None, None]
        ref = torch.where(used, decay * before.double() + share, before.double())
        # (a probability below fp32's normal numbers counts as 0: 2^-126 a row at most)
        tol = torch.where(used, 2.0 ** -22 * (before.double().abs() + share) + e * share + p.shape[2] * 2.0 ** -126, 0.0)
        err = (weight.double() - ref).abs()
        assert (err <= tol).all(), (err - tol).max().item()


TYPES = [(torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16), (torch.float16, E4M3), (torch.bfloat16, E4M3)]


# one state, chunks of 16 to 64 and their neighbours, pages that end inside a chunk, more query rows than 8 and 16
@pytest.mark.parametrize("qt,pt", TYPES)
@pytest.mark.parametrize("b,tq,n,heads,kv_heads,dim,page", [
    (1, 1, 1, 1, 1, 32, 1), (2, 1, 240, 8, 8, 32, 20), (3, 1, 63, 4, 2, 64, 7), (2, 1, 17, 6, 2, 128, 16), (2, 3, 300, 9, 3, 64, 1),
    (4, 1, 1030, 16, 2, 128, 64), (1, 5, 2040, 8, 1, 32, 60), (2, 17, 129, 4, 2, 128, 128), (1, 1, 9001, 5, 1, 64, 13),
    (1, 2, 42840, 8, 4, 128, 240), (64, 1, 700, 4, 4, 32, 100), (3, 1, 4097, 32, 1, 128, 48), (1, 33, 515, 2, 1, 64, 5),
    (160, 1, 1300, 4, 2, 128, 17), (2, 9, 5000, 8, 2, 64, 33), (3, 3, 9000, 3, 1, 128, 7), (1, 1, 30000, 3, 1, 32, 64),
    (300, 1, 1100, 2, 1, 128, 50), (2, 1, 384, 4, 1, 64, 8), (2, 1, 388, 4, 1, 64, 4),
])
def test_attention(b, tq, n, heads, kv_heads, dim, page, qt, pt):
    import sarbon_b200 as sb
    g = gen(n * 3 + tq)
    k, v, table = pages_of(g, b, n, page, kv_heads * dim, pt, by=1.0 if pt != E4M3 else 30.0)
    ks, vs = (2.0 ** -5, 0.03) if pt == E4M3 else (1.0, 1.0)
    q = rand(g, b, tq, heads * dim, dtype=qt)
    lens = torch.tensor([n - (i * 37) % max(1, n // 2) for i in range(b)], dtype=torch.int32, device="cuda")
    how = dict(k_scale=ks, v_scale=vs)
    before = rand(g, b, kv_heads, table.shape[1] * page).abs()
    for causal in (False, True):
        lse, weight = torch.empty(b, heads, tq, device="cuda"), before.clone()
        out = sb.paged_attention(q, k, v, table, lens, heads, kv_heads=kv_heads, causal=causal, weight=weight, decay=0.75, lse=lse, **how)
        check_attention(out, lse, weight, q, k, v, table, lens, heads, kv_heads, before=before, decay=0.75, causal=causal, **how)
        # with and without the account, twice: the same bits
        assert same_bits(out, sb.paged_attention(q, k, v, table, lens, heads, kv_heads=kv_heads, causal=causal, **how))
        again = before.clone()
        sb.paged_attention(q, k, v, table, lens, heads, kv_heads=kv_heads, causal=causal, weight=again, decay=0.75, **how)
        assert same_bits(weight, again)


@pytest.mark.parametrize("qt,pt", TYPES)
@pytest.mark.parametrize("tq,n,heads,kv_heads,dim,page", [(1, 300, 4, 2, 64, 24), (4, 700, 4, 1, 128, 60), (2, 2000, 2, 2, 32, 9)])
def test_attention_masked_places(tq, n, heads, kv_heads, dim, page, qt, pt):
    """Lengths of zero, one, below Tq and beyond the pages; missing pages; NaN wherever nothing is looked at."""
    import sarbon_b200 as sb
    g = gen(n + tq)
    b = 7
    k, v, table = pages_of(g, b, n, page, kv_heads * dim, pt)
    cap = table.shape[1] * page
    lens = ints(0, 1, 3, -5, n, cap + 1000, 2 ** 31 - 1)
    table[4, 1], table[4, 3], table[5, 0], table[6] = -1, k.shape[0], 2 ** 31 - 1, -2 ** 31
    used = torch.zeros(k.shape[:2], dtype=torch.bool, device="cuda")
    for i, m in enumerate(lens.clamp(0, cap).tolist()):
        for j in range(m):
            p = int(table[i, j // page])
            if 0 <= p < k.shape[0]:
                used[p, j % page] = True
    for x in (k, v):
        x.copy_(torch.where(used[..., None], x.float(), math.nan).to(pt))
    q = rand(g, b, tq, heads * dim, dtype=qt)
    before = rand(g, b, kv_heads, cap).abs()
    for causal in (False, True):
        lse, weight = torch.empty(b, heads, tq, device="cuda"), before.clone()
        out = sb.paged_attention(q, k, v, table, lens, heads, kv_heads=kv_heads, causal=causal, weight=weight, decay=0.5, lse=lse)
        assert out.isfinite().all() and weight.isfinite().all()
        assert not out[0].any() and not out[3].any() and not out[6].any()
        check_attention(out, lse, weight, q, k, v, table, lens, heads, kv_heads, before=before, decay=0.5, causal=causal)


@pytest.mark.parametrize("qt,pt", TYPES)
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_attention_causal_states_of_no_number(qt, pt, dim):
    """A new state that holds NaN or infinities is no matter to the queries before it."""
    import sarbon_b200 as sb
    g = gen(dim)
    b, tq, n, heads, kv_heads = 2, 6, 200, 4, 2
    k, v, table = pages_of(g, b, n, 16, kv_heads * dim, pt)
    lens = ints(n, n - 9)
    q = rand(g, b, tq, heads * dim, dtype=qt)
    for i, m in enumerate(lens.tolist()):
        at = m - 3
        v[int(table[i, at // 16]), at % 16, 5:40] = torch.tensor(math.nan if pt == E4M3 or i else math.inf).to(pt)
        k[int(table[i, (m - 2) // 16]), (m - 2) % 16, 3] = torch.tensor(math.nan).to(pt)
    lse = torch.empty(b, heads, tq, device="cuda")
    out = sb.paged_attention(q, k, v, table, lens, heads, kv_heads=kv_heads, causal=True, lse=lse)
    clean = out[:, :3]  # the first three queries see neither
    assert clean.isfinite().all()
    check_attention(clean.contiguous(), lse[..., :3].contiguous(), None, q[:, :3].contiguous(), k, v, table, lens - 3, heads, kv_heads, causal=True)
    assert not out[0, 3, 5:min(dim, 40)].isfinite().any()  # the fourth sees the channels that are none


def test_attention_peaks():
    """Scores far apart, rising and falling over the states; one state that has everything."""
    import sarbon_b200 as sb
    g = gen(5)
    for pt, qt in ((torch.bfloat16,) * 2, (torch.float16,) * 2, (E4M3, torch.bfloat16)):
        b, n, heads, dim = 2, 3000, 4, 64
        k, v, table = pages_of(g, b, n, 50, dim, pt)
        q = rand(g, b, 1, heads * dim, dtype=qt, by=4.0)
        ramp = torch.linspace(-3, 3, n, device="cuda")[:, None]
        for i, r in enumerate((ramp, -ramp)):
            k[table[i].long()] = ((k[table[i].long()].float().flatten(0, 1) * 0.1 + r) * (4.0 if pt == E4M3 else 1.0)).view(-1, 50, dim).to(pt) \
                if pt != E4M3 else k[table[i].long()]
        lse, weight = torch.empty(b, heads, 1, device="cuda"), torch.zeros(b, 1, n, device="cuda")
        out = sb.paged_attention(q, k, v, table, ints(n, n), heads, kv_heads=1, scale=1.0, lse=lse, weight=weight)
        check_attention(out, lse, weight, q, k, v, table, ints(n, n), heads, 1, before=torch.zeros_like(weight), scale=1.0)


def test_attention_bf16_queries_of_any_size_on_e4m3():
    """e4m3 pages are multiplied in fp16: bf16 queries beyond fp16's range keep their scores."""
    import sarbon_b200 as sb
    g = gen(8)
    b, n, dim = 6, 500, 64
    k, v, table = pages_of(g, b, n, 33, dim, E4M3)
    size = torch.tensor([1e-30, 1e-8, 1.0, 1e6, 1e25, 0.0], device="cuda")
    q = (rand(g, b, 1, 2 * dim) * size[:, None, None]).to(torch.bfloat16)
    lens = torch.full((b,), n, dtype=torch.int32, device="cuda")
    for i, s in enumerate(size.tolist()):
        at = slice(i, i + 1)
        scale = 0.1 / s if s else 0.1
        lse = torch.empty(1, 2, 1, device="cuda")
        out = sb.paged_attention(q[at], k, v, table[at], lens[at], 2, kv_heads=1, scale=scale, lse=lse)
        check_attention(out, lse, None, q[at], k, v, table[at], lens[at], 2, 1, scale=scale)


@pytest.mark.parametrize("size,scale", [(2.0 ** -126, 2.0 ** -40), (2.0 ** -120, 0.1), (2.0 ** -131, 2.0 ** 126), (2.0 ** 126, 2.0 ** -126), (1.0, 2.0 ** -120)])
@pytest.mark.parametrize("qt", [torch.float16, torch.bfloat16])
def test_attention_sizes_near_the_types_ends(qt, size, scale):
    """Queries and scales of any size leave states that take no part without weight, and scores of next to nothing
    share evenly."""
    import sarbon_b200 as sb
    g, b, n, heads, kv_heads = gen(21), 2, 100, 4, 2
    k, v, table = pages_of(g, b, n, 16, kv_heads * 64, E4M3)
    lens = ints(37, n)
    q = (rand(g, b, 2, heads * 64) * size).clamp(-torch.finfo(qt).max, torch.finfo(qt).max).to(qt)
    if qt == torch.float16 and size > 1:
        scale = 2.0 ** -16
    weight, lse = torch.zeros(b, kv_heads, table.shape[1] * 16, device="cuda"), torch.empty(b, heads, 2, device="cuda")
    out = sb.paged_attention(q, k, v, table, lens, heads, kv_heads, scale=scale, causal=True, weight=weight, lse=lse)
    check_attention(out, lse, weight, q, k, v, table, lens, heads, kv_heads, scale=scale, causal=True,
                    before=torch.zeros_like(weight))


def test_attention_strides_and_shared_pages():
    """Keys and values side by side, pages inside wider rows, queries of a projection, a table that is part of a larger one,
    pages that several items and several places of one item share, pages in no order in memory."""
    import sarbon_b200 as sb
    g = gen(21)
    b, n, page, heads, kv_heads, dim = 3, 330, 30, 4, 2, 64
    width = kv_heads * dim
    room = rand(g, 40, page + 2, 2 * width + 32, dtype=torch.float16)
    k, v = room[:, 1:page + 1, 16:16 + width], room[:, 1:page + 1, 16 + width:16 + 2 * width]
    tables = torch.randint(0, 40, (b, 20), dtype=torch.int32, device="cuda", generator=g)
    table = tables[:, 3:14]
    table[1] = table[0]
    table[2, 4] = table[2, 5]
    wide = rand(g, 2, b, heads * dim + 64, dtype=torch.float16).transpose(0, 1)
    q = wide[..., 32:32 + heads * dim]
    lens = ints(330, 301, 290)
    out = rand(g, b, 2, 2 * heads * dim, dtype=torch.float16)
    keep = out.clone()
    weight = rand(g, b, kv_heads, 330).abs()
    before = weight.clone()
    sb.paged_attention(q, k, v, table, lens, heads, kv_heads=kv_heads, weight=weight, out=out[..., :heads * dim])
    check_attention(out[..., :heads * dim], None, weight, q, k, v, table, lens, heads, kv_heads, before=before)
    assert same_bits(out[..., heads * dim:], keep[..., heads * dim:])
    turned = k.transpose(0, 1).contiguous().transpose(0, 1)  # the same row of all pages together
    assert same_bits(out[..., :heads * dim], sb.paged_attention(q, turned, v, table, lens, heads, kv_heads=kv_heads))


def test_attention_uneven_items():
    """CTAs share the states of items of very unequal lengths, empty ones among and behind them."""
    import sarbon_b200 as sb
    g = gen(12)
    b, n, heads, kv_heads, dim = 9, 20000, 6, 2, 64
    k, v, table = pages_of(g, b, n, 100, kv_heads * dim, torch.float16)
    q = rand(g, b, 2, heads * dim, dtype=torch.float16)
    for lens in (ints(0, 0, 20000, 1, 0, 33, 12345, 0, 0), ints(*[0] * 8, 17), ints(*[0] * 9), ints(20000, *[0] * 8), ints(*range(500, 509))):
        lse, weight = torch.empty(b, heads, 2, device="cuda"), rand(g, b, kv_heads, n).abs()
        before = weight.clone()
        out = sb.paged_attention(q, k, v, table, lens, heads, kv_heads=kv_heads, causal=True, lse=lse, weight=weight, decay=0.5)
        check_attention(out, lse, weight, q, k, v, table, lens, heads, kv_heads, before=before, decay=0.5, causal=True)


def test_nothing_there():
    import sarbon_b200 as sb
    k = torch.zeros(4, 8, 64, device="cuda", dtype=torch.float16)
    v, q = torch.ones_like(k), torch.ones(2, 1, 64, device="cuda", dtype=torch.float16)
    lse = torch.zeros(2, 1, 1, device="cuda")
    for pools, table in (((k, v), torch.zeros(2, 0, dtype=torch.int32, device="cuda")), ((k[:0], v[:0]), torch.zeros(2, 3, dtype=torch.int32, device="cuda"))):
        weight = torch.ones(2, 1, table.shape[1] * 8, device="cuda")
        out = sb.paged_attention(q, *pools, table, ints(5, 9), 1, weight=weight, decay=0.5, lse=lse)
        assert not out.any() and (lse == -math.inf).all()
        if table.shape[1]:
            assert (weight[0, 0, :5] == 0.5).all() and (weight[0, 0, 5:] == 1).all()
        after, w, born = sb.paged_evict(*pools, table, ints(5, 9), weight, 3)
        assert after.tolist() == ([3, 3] if table.shape[1] else [0, 0]) and born is None
        after = sb.paged_write(q.expand(2, 4, 64), q.expand(2, 4, 64), *pools, table, ints(0, 22), kv_heads=1)
        assert after.tolist() == ([4, 24] if table.shape[1] else [0, 0])
    table = torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    assert sb.paged_attention(q[:, :0], k, v, table, ints(1, 1), 1).shape == (2, 0, 64)
    assert sb.paged_write(q[:, :0], q[:, :0], k, v, table, ints(3, 99)).tolist() == [3, 8]
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert sb.paged_attention(q[:0], k, v, table[:0], none, 1).shape == (0, 1, 64)
    assert sb.paged_write(q[:0], q[:0], k, v, table[:0], none).shape == (0,)
    assert sb.paged_evict(k, v, table[:0], none, torch.zeros(0, 1, 8, device="cuda"), 3)[0].shape == (0,)


def test_pools_beyond_32_bit_offsets():
    """A pool of more than 2^32 elements: the last pages are written, read and moved."""
    import sarbon_b200 as sb
    g = gen(4)
    page, width = 1 << 14, 1024
    count = (1 << 32) // (page * width) + 2
    k = torch.zeros(count, page, width, device="cuda", dtype=torch.uint8).view(E4M3)
    v = torch.zeros(count, page, width, device="cuda", dtype=torch.uint8).view(E4M3)
    table = torch.tensor([[count - 1, 0, count - 2]], dtype=torch.int32, device="cuda")
    n = 2 * page + 50
    new_k, new_v = (rand(g, 1, 100, width, dtype=torch.float16) for _ in range(2))
    after = sb.paged_write(new_k, new_v, k, v, table, ints(n - 100))
    assert after.tolist() == [n]
    assert same_bits(k[count - 2, :50].view(torch.uint8), new_k[0, 50:].to(E4M3).view(torch.uint8))
    assert same_bits(v[0, page - 50:].view(torch.uint8), new_v[0, :50].to(E4M3).view(torch.uint8))
    q = rand(g, 1, 1, width, dtype=torch.float16)
    weight = torch.zeros(1, 8, 3 * page, device="cuda")
    out = sb.paged_attention(q, k, v, table, after, 8, weight=weight)
    check_attention(out, None, weight, q, k, v, table, after, 8, 8, before=torch.zeros_like(weight))
    weight[..., n - 10:n] = 9.0
    sb.paged_evict(k, v, table, after, weight, n - 10)
    low = torch.sort(weight[0, 3, :n], stable=True).indices[:10]
    assert (low < n - 10).all()
    at = low.sort().values
    rows = k.view(torch.uint8)[table[0].long()[at // page], at % page, 3 * 128:4 * 128]
    assert same_bits(rows, new_k[0, 90:, 3 * 128:4 * 128].to(E4M3).view(torch.uint8))
    del k, v
    torch.cuda.empty_cache()


def test_accounts_beyond_32_bit_offsets():
    """Weights and stamps of more than 2^31 places in all: the last item's."""
    import sarbon_b200 as sb
    g = gen(6)
    b, page, n = 5, 1 << 20, 512
    k, v = (rand(g, 2, page, 32, dtype=torch.float16) for _ in range(2))
    table = torch.full((b, n), -1, dtype=torch.int32, device="cuda")
    table[:, 0] = torch.arange(b, device="cuda") % 2
    q = rand(g, b, 1, 32, dtype=torch.float16)
    lens = ints(3, 0, 7, 1, 900)
    weight = torch.ones(b, 1, n * page, device="cuda")
    out = sb.paged_attention(q, k, v, table, lens, 1, weight=weight, decay=0.5)
    few = slice(0, 1000)
    check_attention(out, None, weight[..., few].contiguous(), q, k[:, few], v[:, few], table[:, :1], lens, 1, 1,
                    before=torch.ones(b, 1, 1000, device="cuda"), decay=0.5)
    best = torch.sort(weight[4, 0, :900], descending=True, stable=True)
    after, _, _ = sb.paged_evict(k, v, table, lens, weight, 100, weight_out=weight)
    assert after.tolist() == [3, 0, 7, 1, 100]
    assert same_bits(weight[4, 0, :100].sort(descending=True).values, best.values[:100]) and not weight[4, 0, 100:1000].any()
    assert not weight[4, 0, -1000:].any() and not weight[1].any()
    new = rand(g, b, 2, 32, dtype=torch.float16)
    weight[4, 0, 100:102] = 5.0
    assert sb.paged_write(new, new, k, v, table, after, weight=weight).tolist() == [5, 2, 9, 3, 102]
    assert not weight[4, 0, 100:102].any() and same_bits(k[0, 100:102], new[4])
    del weight
    torch.cuda.empty_cache()


# ---------------------------------------------------------------- new states
def codes(x, scale):
    # (by a tensor: torch multiplies by the reciprocal of a number, which is not the quotient)
    return (x.float() / torch.full_like(x, scale, dtype=torch.float32)).clamp(-448, 448).to(E4M3)


@pytest.mark.parametrize("qt,pt", TYPES)
@pytest.mark.parametrize("b,t,kv_heads,dim,page,ks,vs", [
    (1, 1, 1, 32, 1, 1.0, 1.0), (3, 1, 4, 128, 16, 0.5, 2.0), (2, 77, 3, 64, 7, 0.013, 3.7), (5, 130, 8, 32, 60, 2.0 ** -6, 1 / 3),
    (2, 1000, 2, 128, 64, 0.1, 0.25), (1, 9, 16, 128, 4, 1.0, 7.0),
])
def test_write(b, t, kv_heads, dim, page, ks, vs, qt, pt):
    import sarbon_b200 as sb
    g = gen(t * 11 + dim)
    width = kv_heads * dim
    if pt != E4M3:
        ks = vs = 1.0
    k, v, table = pages_of(g, b, t + 40, page, width, pt)
    cap = table.shape[1] * page
    table[0, -1] = -1
    kv = rand(g, b, t, 2 * width + 3, dtype=qt, by=3.0)
    kv[0, 0, :4] = torch.tensor([math.nan, math.inf, -math.inf, -0.0])
    at = torch.tensor([(i * 23) % 41 for i in range(b)], dtype=torch.int32, device="cuda")
    at[-1] = cap - t // 2  # runs out of pages
    count = torch.tensor([t - (i * 5) % max(1, t) for i in range(b)], dtype=torch.int32, device="cuda")
    weight, born = rand(g, b, kv_heads, cap), torch.randint(0, 99, (b, kv_heads, cap), dtype=torch.int32, device="cuda", generator=g)
    for off, n, stamp in ((0, None, torch.arange(b * t, dtype=torch.int32, device="cuda").view(b, t)), (3, count, torch.arange(b, dtype=torch.int32, device="cuda"))):
        nk, nv = kv[..., off:off + width], kv[..., width + off:2 * width + off]  # aligned to 16 bytes and not
        if off == 0 and width % 8 == 0:
            nk, nv = nk.contiguous(), nv.contiguous()
        rk, rv, rw, rb, after = k.clone(), v.clone(), weight.clone(), born.clone(), []
        for i in range(b):
            m = int(n[i]) if n is not None else t
            for x in range(m):
                pos = int(at[i]) + x
                if pos >= cap:
                    continue
                p = int(table[i, pos // page])
                if p >= 0:
                    rk[p, pos % page] = codes(nk[i, x], ks) if pt == E4M3 else nk[i, x]
                    rv[p, pos % page] = codes(nv[i, x], vs) if pt == E4M3 else nv[i, x]
                rw[i, :, pos], rb[i, :, pos] = 0, stamp[i, x] if stamp.dim() == 2 else stamp[i]
            after.append(min(cap, int(at[i]) + m))
        gk, gv, gw, gb = k.clone(), v.clone(), weight.clone(), born.clone()
        got = sb.paged_write(nk, nv, gk, gv, table, at, count=n, k_scale=ks, v_scale=vs, weight=gw, born=gb, stamp=stamp)
        assert got.tolist() == after
        # NaN is NaN, of either sign
        for a, r in ((gk, rk), (gv, rv)):
            a, r = a.float(), r.float()
            assert torch.equal(a.isnan(), r.isnan()) and torch.equal(a.nan_to_num(0.0), r.nan_to_num(0.0))
        assert same_bits(gw, rw) and same_bits(gb, rb)
        only, buf = k.clone(), torch.empty_like(at)
        assert sb.paged_write(nk, nv, only, v.clone(), table, at, count=n, k_scale=ks, v_scale=vs, after=buf, kv_heads=kv_heads) is buf
        assert same_bits(only, gk) and buf.tolist() == after


def test_write_lengths_outside():
    import sarbon_b200 as sb
    g = gen(2)
    k, v, table = pages_of(g, 4, 20, 5, 64, torch.float16)
    new, keep = rand(g, 4, 3, 64, dtype=torch.float16), k.clone()
    after = sb.paged_write(new, new, k, v, table, ints(-7, 2 ** 31 - 1, 3, 19), count=ints(2, 3, -1, 2 ** 31 - 1))
    assert after.tolist() == [2, 20, 3, 20]
    keep[table[0, 0].long(), :2] = new[0, :2]
    keep[table[3, 3].long(), 4] = new[3, 0]
    assert same_bits(k, keep)


# ---------------------------------------------------------------- eviction
def evicted(k, v, table, lens, weight, keep, born, since, kv_heads):
    """The definition, a state at a time."""
    page, cap = k.shape[1], weight.shape[2]
    k, v, w, r = (x.clone() for x in (k, v, weight, born))
    ku, vu = (x.view(torch.uint8).view(*x.shape[:2], kv_heads, -1) for x in (k, v))
    after, tab = [], table.tolist()
    for i in range(len(tab)):
        n, kp = min(max(int(lens[i]), 0), cap), min(max(int(keep[i]), 0), cap)
        for h in range(kv_heads):
            if n > kp:
                ws, bs = weight[i, h].tolist(), born[i, h].tolist()
                order = sorted(range(n), key=lambda j: (not (since is not None and bs[j] >= int(since[i])),
                                                        1 if ws[j] != ws[j] else 0, -ws[j] if ws[j] == ws[j] else 0.0, j))
                stays = set(order[:kp])
                free, moved = [j for j in range(kp) if j not in stays], sorted(j for j in stays if j >= kp)
                assert len(free) == len(moved)
                for d, s in zip(free, moved):
                    w[i, h, d], r[i, h, d] = weight[i, h, s], born[i, h, s]
                    p, c = tab[i][d // page], tab[i][s // page]
                    if 0 <= p < k.shape[0] and 0 <= c < k.shape[0]:
                        ku[p, d % page, h], vu[p, d % page, h] = ku[c, s % page, h].clone(), vu[c, s % page, h].clone()
            w[i, h, min(n, kp):], r[i, h, min(n, kp):] = 0, 0
        after.append(min(n, kp))
    return k, v, w, r, after


def check_eviction(k, v, table, lens, weight, keep, born, since, **how):
    import sarbon_b200 as sb
    kv_heads = weight.shape[1]
    keeps = [keep] * len(table) if isinstance(keep, int) else keep.tolist()
    rk, rv, rw, rb, after = evicted(k, v, table, lens, weight, keeps, born, since, kv_heads)
    gk, gv = k.clone(), v.clone()
    before = weight.clone(), born.clone(), lens.clone()
    got, w, b = sb.paged_evict(gk, gv, table, lens, weight, keep, born=born, since=since, **how)
    assert got.tolist() == after
    assert same_bits(w, rw) and same_bits(b, rb) and same_bits(gk, rk) and same_bits(gv, rv)
    assert all(same_bits(x, y) for x, y in zip((weight, born, lens), before))
    # in place
    gk, gv, w, b, n = k.clone(), v.clone(), weight.clone(), born.clone(), lens.clone()
    out = sb.paged_evict(gk, gv, table, n, w, keep, born=b, since=since, weight_out=w, born_out=b, after=n)
    assert out[0] is n and out[1] is w and out[2] is b
    assert n.tolist() == after and same_bits(w, rw) and same_bits(b, rb) and same_bits(gk, rk) and same_bits(gv, rv)
    # by weight alone, without stamps
    zero = torch.zeros_like(born)
    rk, rv, rw, _, after = evicted(k, v, table, lens, weight, keeps, zero, None, kv_heads)
    gk, gv = k.clone(), v.clone()
    got, w, none = sb.paged_evict(gk, gv, table, lens, weight, keep)
    assert none is None and got.tolist() == after and same_bits(w, rw) and same_bits(gk, rk) and same_bits(gv, rv)


@pytest.mark.parametrize("pt", [torch.float16, torch.bfloat16, E4M3])
@pytest.mark.parametrize("b,n,kv_heads,dim,page,keep", [
    (1, 2, 1, 32, 1, 1), (2, 1, 2, 64, 4, 0), (3, 241, 4, 128, 16, 240), (2, 500, 3, 64, 7, 250), (2, 1025, 1, 128, 60, 1),
    (1, 2100, 2, 32, 100, 1024), (2, 33, 2, 64, 33, 32), (1, 4000, 1, 128, 250, 3999), (2, 64, 1, 64, 3, 64), (1, 70, 1, 32, 5, 1000),
    (2, 1100, 2, 32, 60, 950), (1, 1412, 3, 32, 240, 1256), (1, 2018, 1, 128, 1, 1009), (3, 2018, 1, 32, 256, 2000),
])
def test_evict(b, n, kv_heads, dim, page, keep, pt):
    g = gen(n + keep)
    k, v, table = pages_of(g, b, n + 30, page, kv_heads * dim, pt)
    shape = (b, kv_heads, table.shape[1] * page)
    lens = torch.tensor([n - (i * 7) % max(1, n // 3) for i in range(b)], dtype=torch.int32, device="cuda")
    weight = rand(g, *shape).exp()
    born = torch.randint(-50, 50, shape, dtype=torch.int32, device="cuda", generator=g)
    for since in (-2 ** 31, 48, 20, 0, 2 ** 31 - 1):  # all, few, some, half, none protected
        check_eviction(k, v, table, lens, weight, keep, born, torch.full((b,), since, dtype=torch.int32, device="cuda"))


def test_evict_equal_and_odd_weights():
    """All weights alike, few values, zeros of both signs, infinities, NaN, negative and denormal ones."""
    g = gen(77)
    b, n, kv_heads, page = 6, 1500, 2, 25
    k, v, table = pages_of(g, b, n, page, kv_heads * 32, torch.float16)
    shape = (b, kv_heads, n)
    weight = torch.randint(0, 4, shape, device="cuda", generator=g).float()
    weight[0] = 0.0
    weight[1] = torch.where(torch.rand(kv_heads, n, device="cuda", generator=g) < 0.5, -0.0, 0.0)
    weight[2, :, ::3], weight[2, :, 1::7], weight[2, :, 5::11] = math.nan, math.inf, -math.inf
    weight[3] = -weight[3] * 2.0 ** -140
    weight[4] = 1.0 + torch.randint(0, 3, shape[1:], device="cuda", generator=g) * 2.0 ** -23
    weight[5, :, n // 2:] = 0.0
    born = torch.randint(0, 9, shape, dtype=torch.int32, device="cuda", generator=g)
    lens = torch.full((b,), n, dtype=torch.int32, device="cuda")
    for keep in (1, 700, 1499, ints(0, 10, 500, 1400, 2000, -3)):
        check_eviction(k, v, table, lens, weight, keep, born, ints(5, 9, 0, 8, 4, 7))


def test_evict_lengths_and_pages_outside():
    g = gen(3)
    k, v, table = pages_of(g, 5, 90, 10, 64, torch.bfloat16)
    weight = rand(g, 5, 1, 90)
    born = torch.zeros(5, 1, 90, dtype=torch.int32, device="cuda")
    table[1, 2], table[1, 7], table[2, 8], table[3] = -1, k.shape[0], 2 ** 31 - 1, -9
    check_eviction(k, v, table, ints(95, 90, 2 ** 31 - 1, 80, -4), weight, 40, born, None)


@pytest.mark.parametrize("n", [900, 2100, 4050, 4100, 30000, 160000])
def test_evict_partly_in_place(n):
    """One kernel, clusters and long memories; each result on its operand or apart."""
    import sarbon_b200 as sb
    g = gen(n)
    b, kv_heads, page, keep = 2, 2, 50, n * 2 // 3
    k, v, table = pages_of(g, b, n, page, kv_heads * 32, E4M3)
    weight = torch.randint(0, 500, (b, kv_heads, n), device="cuda", generator=g).float()
    born = torch.randint(0, 99, weight.shape, dtype=torch.int32, device="cuda", generator=g)
    lens, since, results = ints(n - 1, n // 2), ints(50, 3), []
    for here in range(8):
        kk, vv, w, r, m = k.clone(), v.clone(), weight.clone(), born.clone(), lens.clone()
        own = dict(weight_out=w if here & 1 else None, born_out=r if here & 2 else None, after=m if here & 4 else None)
        results.append(sb.paged_evict(kk, vv, table, m, w, keep, born=r, since=since, **own) + (kk, vv))
    assert results[0][0].tolist() == [keep, n // 2]
    for other in results[1:]:
        assert all(same_bits(x, y) for x, y in zip(results[0], other))


@pytest.mark.parametrize("cap", [18400, 18560, 48960, 147360, 147520, 245760, 245776, 300000])
def test_evict_long(cap):
    """One CTA to eight an item and head, places that just fit their shared memory, just do not, and far more, against a sort."""
    import sarbon_b200 as sb
    g = gen(cap)
    b, kv_heads, page = 2, 2, 160
    k, v, table = pages_of(g, b, cap, page, kv_heads * 32, E4M3)
    n = table.shape[1] * page
    weight = torch.randint(0, 2 ** 14, (b, kv_heads, n), device="cuda", generator=g).float()  # many ties
    born = torch.randint(0, 1000, weight.shape, dtype=torch.int32, device="cuda", generator=g)
    lens, keep, since = ints(n - 3, n - 77), cap * 5 // 8, ints(900, 300)
    order = torch.sort(weight.double() + (born >= since[:, None, None]).double() * 1e6
                       - (torch.arange(n, device="cuda") >= lens[:, None, None]).double() * 1e9, descending=True, stable=True, dim=-1).indices
    stays = torch.zeros_like(weight, dtype=torch.bool).scatter_(-1, order[..., :keep], True)
    low = torch.arange(n, device="cuda") < keep
    free, moved = (~stays & low).nonzero(as_tuple=True), (stays & ~low).nonzero(as_tuple=True)
    rw, rb = weight.masked_fill(~low, 0.0), born.masked_fill(~low, 0)
    rw[free], rb[free] = weight[moved], born[moved]
    rows = k.view(torch.uint8).view(*k.shape[:2], kv_heads, -1).clone()
    t = table.long()
    rows[t[free[0], free[2] // page], free[2] % page, free[1]] = rows[t[moved[0], moved[2] // page], moved[2] % page, moved[1]]
    after, w, r = sb.paged_evict(k, v, table, lens, weight, keep, born=born, since=since)
    assert after.tolist() == [keep, keep] and same_bits(w, rw) and same_bits(r, rb)
    assert same_bits(k.view(torch.uint8).view_as(rows), rows)


# ---------------------------------------------------------------- together
def step(sb, s, frame):
    """A frame's new states, its query tokens' attention, and the budget."""
    n = sb.paged_write(s["new_k"], s["new_v"], s["k"], s["v"], s["table"], s["lens"], k_scale=s["scale"], v_scale=s["scale"],
                       weight=s["weight"], born=s["born"], stamp=frame, after=s["n"])
    sb.paged_attention(s["q"], s["k"], s["v"], s["table"], n, 4, kv_heads=2, k_scale=s["scale"], v_scale=s["scale"], causal=True,
                       weight=s["weight"], decay=0.9, out=s["out"])
    sb.paged_evict(s["k"], s["v"], s["table"], n, s["weight"], 150, born=s["born"], since=frame, weight_out=s["weight"],
                   born_out=s["born"], after=s["lens"])


def stream(seed, pt=torch.float16, tq=2):
    g = gen(seed)
    b, dim, page, cap = 3, 64, 12, 204
    k, v, table = pages_of(g, b, cap, page, 2 * dim, pt)
    return dict(k=k, v=v, table=table, lens=ints(0, 140, 150), n=ints(0, 0, 0), new_k=rand(g, b, 40, 2 * dim, dtype=torch.float16),
                new_v=rand(g, b, 40, 2 * dim, dtype=torch.float16), q=rand(g, b, tq, 4 * dim, dtype=torch.float16), scale=0.02 if pt == E4M3 else 1.0,
                weight=rand(g, b, 2, cap).abs(), born=torch.zeros(b, 2, cap, dtype=torch.int32, device="cuda"),
                out=torch.empty(b, tq, 4 * dim, dtype=torch.float16, device="cuda"))


@pytest.mark.parametrize("pt", [torch.float16, E4M3])
def test_frames_of_a_stream(pt):
    """Write, attend and evict, frame after frame, each held to its formula on what the one before left."""
    import sarbon_b200 as sb
    s = stream(1, pt)
    g = gen(9)
    for f in range(6):
        for x in ("new_k", "new_v", "q"):
            s[x].copy_(rand(g, *s[x].shape))
        frame = ints(f, f, f)
        how = dict(k_scale=s["scale"], v_scale=s["scale"])
        n = sb.paged_write(s["new_k"], s["new_v"], s["k"], s["v"], s["table"], s["lens"], weight=s["weight"], born=s["born"], stamp=frame, **how)
        assert torch.equal(n, s["lens"] + 40)
        before = s["weight"].clone()
        out = sb.paged_attention(s["q"], s["k"], s["v"], s["table"], n, 4, kv_heads=2, causal=True, weight=s["weight"], decay=0.9, **how)
        check_attention(out, None, s["weight"], s["q"], s["k"], s["v"], s["table"], n, 4, 2, before=before, decay=0.9, causal=True, **how)
        rk, rv, rw, rb, after = evicted(s["k"], s["v"], s["table"], n, s["weight"], [150] * 3, s["born"], frame, 2)
        sb.paged_evict(s["k"], s["v"], s["table"], n, s["weight"], 150, born=s["born"], since=frame, weight_out=s["weight"],
                       born_out=s["born"], after=s["lens"])
        assert s["lens"].tolist() == after and same_bits(s["weight"], rw) and same_bits(s["born"], rb)
        assert same_bits(s["k"], rk) and same_bits(s["v"], rv)


def test_captured_steps_and_streams():
    """Two streams' steps captured as graphs and replayed at once equal the same steps one after the other."""
    import sarbon_b200 as sb
    plain = [stream(31), stream(32, E4M3)]
    frames = [ints(0, 0, 0) for _ in plain]
    for _ in range(4):
        for s, f in zip(plain, frames):
            step(sb, s, f)
            f.add_(1)
    held = [stream(31), stream(32, E4M3)]
    frames = [ints(0, 0, 0) for _ in held]
    graphs, lanes = [], [torch.cuda.Stream() for _ in held]
    torch.cuda.synchronize()
    for s, f, lane in zip(held, frames, lanes):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=lane):
            step(sb, s, f)
            f.add_(1)
        graphs.append(graph)
    for _ in range(4):
        for graph, lane in zip(graphs, lanes):
            with torch.cuda.stream(lane):
                graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(plain, held):
        assert all(same_bits(a[x], b[x]) for x in ("k", "v", "weight", "born", "lens", "out"))


def test_calls_from_either_side(monkeypatch):
    """The native side of a call and the Python side do the same; what the native side leaves alone is done all the same, and a
    status of the library's is an error on both."""
    import sarbon_b200 as sb
    from sarbon_b200 import paged_ops
    sides = [paged_ops._load()]

    class Nothing:
        attend = append = cut = staticmethod(lambda *a: None)

    sides.append(Nothing)
    for pt in (torch.float16, E4M3):
        got = []
        for side in sides:
            monkeypatch.setattr(paged_ops, "_native", side)
            s, f = stream(41, pt), ints(0, 0, 0)
            was = paged_ops.CALLS[0]
            for _ in range(3):
                step(sb, s, f)
                f.add_(1)
            assert paged_ops.CALLS[0] == was + 9
            n = sb.paged_write(s["new_k"], s["new_v"], s["k"], s["v"], s["table"], s["lens"], k_scale=s["scale"], v_scale=s["scale"])
            out = sb.paged_attention(torch.nn.Parameter(s["q"], requires_grad=False), s["k"], s["v"], s["table"], n, 4, 2)
            got.append([s[x] for x in ("k", "v", "out", "lens", "n", "weight", "born")] + [n, out] +
                       list(sb.paged_evict(s["k"], s["v"], s["table"], n, s["weight"], ints(100, 0, 150), born=s["born"], since=f)))
            assert sb.paged_evict(s["k"], s["v"], s["table"], n, s["weight"], 9)[2] is None
            with pytest.raises(ValueError):
                sb.paged_attention(s["q"], s["k"], s["v"], s["table"], n, 4, kv_heads=3)
            with pytest.raises(ValueError):
                sb.paged_attention(s["q"].clone().requires_grad_(), s["k"], s["v"], s["table"], n, 4, kv_heads=2)
            with pytest.raises(ValueError):
                sb.paged_attention(s["q"], s["k"], s["v"], s["table"], n.cpu(), 4, kv_heads=2)
            off = torch.empty(s["q"].numel() + 1, dtype=torch.float16, device="cuda")[1:].view(s["q"].shape)
            with pytest.raises(RuntimeError, match="aligned"):
                sb.paged_attention(off, s["k"], s["v"], s["table"], n, 4, kv_heads=2)
        assert all(same_bits(x, y) for x, y in zip(*got))

    class Own(torch.Tensor):
        pass

    monkeypatch.setattr(paged_ops, "_native", sides[0])
    s = stream(42)
    whole = sb.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], 4, 2)
    assert same_bits(whole, sb.paged_attention(s["q"].as_subclass(Own), s["k"], s["v"], s["table"], s["lens"], 4, 2))
    assert sb.paged_attention(s["q"][:0], s["k"], s["v"], s["table"][:0], s["lens"][:0], 4, 2).shape == (0, 2, 256)


FIRST_IN_A_CAPTURE = """
import torch
import test_gpu_paged_ops as t
import sarbon_b200 as sb

def case(n, dim, pt, heads):
    g = t.gen(n)
    k, v, table = t.pages_of(g, 2, n, 40, 2 * dim, pt)
    weight = t.rand(g, 2, 2, table.shape[1] * 40).abs()
    q, lens = t.rand(g, 2, 1, heads * dim, dtype=torch.float16), t.ints(n, n - 5)
    return lambda: (sb.paged_attention(q, k, v, table, lens, heads, 2, weight=weight.clone()),) + \\
        sb.paged_evict(k.view(k.shape), v, table, lens, weight, n // 2)[:2]

case(100, 32, torch.float16, 2)()
for n, dim, pt, heads in ((90, 64, t.E4M3, 20), (3000, 128, torch.float16, 4), (9000, 32, t.E4M3, 2), (70000, 64, torch.float16, 4)):
    run = case(n, dim, pt, heads)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = run()
    graph.replay()
    torch.cuda.synchronize()
    ref = case(n, dim, pt, heads)()
    assert all(t.same_bits(a, b) for a, b in zip(got, ref)), n
print("fine")
"""


def test_first_calls_of_a_size_inside_a_capture():
    """A process whose first call was a small one captures other types and sizes at once."""
    import pathlib
    import subprocess
    import sys
    here = pathlib.Path(__file__).resolve().parent
    r = subprocess.run([sys.executable, "-c", f"import sys; sys.path[:0] = [{str(here)!r}, {str(here.parent)!r}]\n" + FIRST_IN_A_CAPTURE],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]
