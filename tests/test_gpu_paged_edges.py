"""The paged memory's operators where values, lengths or places end.

Bounds are those of ``test_gpu_paged_ops``, whose formulas in 64 bits are used."""
import math

import pytest
import torch

from test_gpu_paged_ops import E4M3, check_attention, formula, gen, ints, pages_of, rand, rows_of, same_bits, unit

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need CUDA")


def put(pool, table, item, state, channels, value):
    """One state's channels in its page."""
    page = pool.shape[1]
    pool[int(table[item, state // page]), state % page, channels] = value


# a CTA a key head, a cluster, shared chunks; more rows than 8 and 16
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("b,tq,n,heads,kv_heads,dim,page", [
    (2, 1, 240, 8, 4, 32, 20), (2, 1, 1, 2, 1, 64, 4), (2, 3, 1500, 4, 1, 128, 50), (1, 1, 2048, 4, 4, 128, 60), (2, 2, 9001, 4, 2, 64, 13),
    (64, 1, 4100, 4, 2, 128, 64), (2, 9, 700, 4, 2, 64, 60), (2, 20, 6000, 2, 1, 32, 100),
])
def test_attention_infinite_values(b, tq, n, heads, kv_heads, dim, page, dtype):
    """A channel that holds +inf in a state with weight is +inf, with -inf too or NaN it is NaN, wherever the state lies; channels
    beside it and rows that do not see it are as without."""
    import sarbon_b200 as sb
    g = gen(n + dim)
    k, v, table = pages_of(g, b, n, page, kv_heads * dim, dtype)
    q = rand(g, b, tq, heads * dim, dtype=dtype)
    lens = torch.tensor([n - (i * 5) % max(1, n // 3) for i in range(b)], dtype=torch.int32, device="cuda")
    for i, m in enumerate(lens.tolist()):
        for x in range(12):  # +inf in states all over, -inf, both, NaN beside it
            put(v, table, i, (x * 7919 + i) % m, x, math.inf)
            put(v, table, i, (x * 6007 + i) % m, dim - 1 - x, -math.inf)
        put(v, table, i, 0, 13, math.inf)
        put(v, table, i, m - 1, 13, math.inf)
        put(v, table, i, m // 2, 14, math.inf)
        put(v, table, i, m - 1, 14, -math.inf if m > 1 else math.inf)
        put(v, table, i, m // 3, 15, math.nan)
        put(v, table, i, m - 1, 15, math.inf if m > 1 else math.nan)
    weight = rand(g, b, kv_heads, table.shape[1] * page).abs()
    for causal in (False, True):
        lse, account = torch.empty(b, heads, tq, device="cuda"), weight.clone()
        out = sb.paged_attention(q, k, v, table, lens, heads, kv_heads=kv_heads, causal=causal, weight=account, lse=lse)
        assert same_bits(out, sb.paged_attention(q, k, v, table, lens, heads, kv_heads=kv_heads, causal=causal))
        clean = v.masked_fill(~v.isfinite(), 0.0)
        ref, ref_lse, p, absolute, whole, e = formula(q, k, clean, table, lens, heads, kv_heads, causal=causal)
        takes = (p > 0).double()
        values = v[table.long()].flatten(1, 2).unflatten(-1, (kv_heads, -1)).transpose(1, 2)
        plus, minus, nan = (takes @ x.double() > 0 for x in (values == math.inf, values == -math.inf, values.isnan()))
        ref = ref.masked_fill(plus, math.inf).masked_fill(minus, -math.inf).masked_fill(nan | (plus & minus), math.nan)
        tol = unit(dtype) * ref.abs() + (unit(dtype) ** 2 + e) * absolute + 2.0 ** -32 * whole + 2.0 ** -25
        tol, ref = rows_of(tol, b, tq), rows_of(ref, b, tq)
        got, odd = out.double(), ~ref.isfinite()
        assert torch.equal(got.isnan(), ref.isnan())
        assert torch.equal((got == math.inf) | (got == -math.inf), ref.isinf()) and torch.equal(got[ref.isinf()], ref[ref.isinf()])
        assert ((got - ref).abs()[~odd] <= 1.02 * tol[~odd]).all()
        seen = ref_lse.view(b, heads, tq) > -math.inf
        assert torch.equal(lse > -math.inf, seen) and account.isfinite().all()
        again = weight.clone()  # the account and the log-sum-exp know nothing of values
        plain = torch.empty_like(lse)
        sb.paged_attention(q, k, clean, table, lens, heads, kv_heads=kv_heads, causal=causal, weight=again, lse=plain)
        assert same_bits(lse, plain) and same_bits(account, again)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("b,tq,n,heads,kv_heads,dim,page", [(2, 1, 240, 8, 4, 32, 20), (1, 1, 2048, 4, 4, 128, 60), (2, 9, 9001, 4, 2, 64, 13)])
def test_attention_values_of_the_largest_size(b, tq, n, heads, kv_heads, dim, page, dtype):
    """Sums over states stay in fp32's range: values at the type's largest, of one sign and of both, give what lies among them."""
    import sarbon_b200 as sb
    g = gen(n)
    top = torch.finfo(dtype).max
    k, v, table = pages_of(g, b, n, page, kv_heads * dim, dtype)
    v.copy_(torch.where(torch.rand(v.shape, device="cuda", generator=g) < 0.5, top, -top))
    v[..., ::3] = top
    v[..., 1::9] = -top
    q = rand(g, b, tq, heads * dim, dtype=dtype)
    lens = torch.tensor([n - 3 * i for i in range(b)], dtype=torch.int32, device="cuda")
    for causal in (False, True):
        put(v, table, 0, n - 1, 3, math.inf)  # (a causal call's odd states too)
        out = sb.paged_attention(q, k, v, table, lens, heads, kv_heads=kv_heads, causal=causal)
        ref, _, _, absolute, whole, e = formula(q, k, v, table, lens, heads, kv_heads, causal=causal)
        tol = unit(dtype) * ref.abs() + (unit(dtype) ** 2 + e) * absolute + 2.0 ** -32 * whole
        tol, ref = rows_of(tol, b, tq), rows_of(ref, b, tq)
        known = ~ref.isnan()
        assert ((out.double() - ref).abs()[known] <= 1.02 * tol[known]).all() and (out.float()[~known] == math.inf).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [200, 1900, 9000])
def test_attention_infinite_values_of_little_weight(n, dtype):
    """States whose share is far below the 16-bit types' smallest step, in the first, a middle and the last place."""
    import sarbon_b200 as sb
    g = gen(n)
    dim, page = 64, 40
    k, v, table = pages_of(g, 1, n, page, dim, dtype, by=0.1)
    q = rand(g, 1, 1, dim, dtype=dtype)
    far = (-45.0 * math.sqrt(dim) / q.float().pow(2).sum() * q.float()).to(dtype)[0, 0]  # a share of about e^-45
    for x, j in enumerate((0, n // 2, n - 1)):
        put(k, table, 0, j, slice(None), far)
        put(v, table, 0, j, x, math.inf)
        put(v, table, 0, j, 5 + x, -math.inf)
    out = sb.paged_attention(q, k, v, table, ints(n), 1)[0, 0].float()
    assert (out[:3] == math.inf).all() and (out[5:8] == -math.inf).all() and out[8:].isfinite().all() and out[3:5].isfinite().all()


def test_attention_infinite_keys_and_values():
    """A state whose score is -inf has no share: 0 times its infinite value is no number."""
    import sarbon_b200 as sb
    g = gen(3)
    k, v, table = pages_of(g, 1, 60, 20, 32, torch.float16)
    q = rand(g, 1, 1, 32, dtype=torch.float16).abs()
    put(k, table, 0, 7, 2, -math.inf)
    put(v, table, 0, 7, 4, math.inf)
    put(v, table, 0, 8, 5, math.inf)
    out = sb.paged_attention(q, k, v, table, ints(60), 1)[0, 0].float()
    assert out[4].isnan() and out[5] == math.inf and out.isfinite().sum() == 30


@pytest.mark.parametrize("page,n", [(16, 3), (100, 400)])
def test_attention_without_queries_ages_the_account(page, n):
    """No query gives a state anything: its weight is decay times what it was, of the states that are there."""
    import sarbon_b200 as sb
    g = gen(page)
    k, v, _ = pages_of(g, 1, 10, page, 128, torch.float16)
    table = torch.zeros(4, n, dtype=torch.int32, device="cuda")
    cap = n * page
    before = rand(g, 4, 2, cap)
    lens = ints(0, 5, cap - 3, cap + 9)
    ref = torch.where(torch.arange(cap, device="cuda") < lens[:, None, None], before * 0.75, before)
    q = torch.empty(4, 0, 256, dtype=torch.float16, device="cuda")
    lse = torch.empty(4, 4, 0, device="cuda")
    weight = before.clone()
    assert sb.paged_attention(q, k, v, table, lens, 4, kv_heads=2, weight=weight, decay=0.75, lse=lse).shape == q.shape
    assert same_bits(weight, ref)
    graph, weight = torch.cuda.CUDAGraph(), before.clone()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        sb.paged_attention(q, k, v, table, lens, 4, kv_heads=2, weight=weight, decay=0.5)
    graph.replay()
    graph.replay()
    assert same_bits(weight, torch.where(torch.arange(cap, device="cuda") < lens[:, None, None], before * 0.5 * 0.5, before))


def test_memories_without_places():
    """Tables without entries: nothing to write, to look at or to move, with stamps and in place too."""
    import sarbon_b200 as sb
    k = torch.ones(3, 8, 64, device="cuda", dtype=torch.float16)
    v = k.clone()
    table, new = torch.zeros(2, 0, dtype=torch.int32, device="cuda"), torch.zeros(2, 3, 64, device="cuda", dtype=torch.float16)
    weight, born = torch.zeros(2, 1, 0, device="cuda"), torch.zeros(2, 1, 0, dtype=torch.int32, device="cuda")
    lens = ints(4, 0)
    assert sb.paged_write(new, new, k, v, table, lens, weight=weight, born=born, stamp=ints(1, 2)).tolist() == [0, 0]
    assert not sb.paged_attention(new, k, v, table, lens, 1, weight=weight, decay=0.5).any()
    after, w, r = sb.paged_evict(k, v, table, lens, weight, 3, born=born, since=ints(1, 1))
    assert after.tolist() == [0, 0] and w.shape == weight.shape and r.shape == born.shape
    sb.paged_evict(k, v, table, lens, weight, 3, born=born, since=ints(1, 1), weight_out=weight, born_out=born, after=lens)
    assert lens.tolist() == [0, 0] and (k == 1).all() and (v == 1).all()


@pytest.mark.parametrize("n,keep,kv_heads,page", [(241, 240, 4, 16), (3000, 1100, 2, 7), (4090, 2000, 1, 64), (9000, 8000, 3, 60), (70000, 20000, 2, 240)])
def test_evicted_states_leave_nothing_behind(n, keep, kv_heads, page):
    """Each row carries the number of its state: afterwards a place's row, weight and stamp are one state's, no state is there
    twice, and none that went.  Entries from the last state's page on are no pages."""
    import sarbon_b200 as sb
    g = gen(n)
    b, dim = 3, 32
    lens = ints(n, n - 1, keep + 1)
    k, v, table = pages_of(g, b, n + 3 * page, page, kv_heads * dim, torch.float16)
    cap = table.shape[1] * page
    table.masked_fill_(torch.arange(table.shape[1], device="cuda") * page >= lens[:, None], -1)
    state = torch.arange(cap, device="cuda")
    number = torch.stack([state % 1024, state // 1024]).half()  # exact in fp16
    for pool, sign in ((k, 1), (v, -1)):
        rows = pool.view(-1, page, kv_heads, dim)
        for i in range(b):
            ok = table[i] >= 0
            some = number.view(2, -1, page)[:, ok].permute(1, 2, 0)
            rows[table[i][ok].long(), :, :, :2] = sign * some[:, :, None]
            rows[table[i][ok].long(), :, :, 2] = torch.arange(kv_heads, device="cuda").half()
    weight = torch.rand(b, kv_heads, cap, device="cuda", generator=g)
    born = torch.randint(0, 1000, weight.shape, dtype=torch.int32, device="cuda", generator=g)
    since = ints(990, 0, 500)
    after, w, r = sb.paged_evict(k, v, table, lens, weight, keep, born=born, since=since)
    assert after.tolist() == [keep] * b
    for i in range(b):
        for pool, sign in ((k, 1), (v, -1)):
            rows = pool.view(-1, page, kv_heads, dim)[table[i][: -(-keep // page)].long()].flatten(0, 1)[:keep]
            was = (sign * (rows[..., 0].double() + 1024 * rows[..., 1].double())).long().t()
            assert (rows[..., 2].t() == torch.arange(kv_heads, device="cuda")[:, None]).all()
            assert torch.equal(w[i, :, :keep], weight[i].gather(1, was)) and torch.equal(r[i, :, :keep], born[i].gather(1, was))
            assert (was < lens[i]).all() and (was.sort(-1).values.diff(dim=-1) > 0).all()
            stays = torch.zeros(kv_heads, cap, dtype=torch.bool, device="cuda").scatter_(1, was, True)
            guarded = born[i] >= since[i]
            gone = ~stays & (state < lens[i])
            # none that went is before one that stays
            for h in range(kv_heads):
                if gone[h].any():
                    best = (guarded[h].double() * 2 + weight[i, h].double())
                    assert best[gone[h]].max() <= best[stays[h]].min()


@pytest.mark.parametrize("qt,n", [(torch.bfloat16, 3000), (torch.float16, 3000), (torch.bfloat16, 20000), (torch.bfloat16, 200)])
def test_attention_ramps_on_e4m3(qt, n):
    """Scores that rise over one item's e4m3 states and fall over the other's: the running maximum grows with every chunk."""
    import sarbon_b200 as sb
    g = gen(n)
    b, heads, dim, page = 2, 4, 64, 50
    k, v, table = pages_of(g, b, n, page, dim, E4M3)
    q = rand(g, b, 1, heads * dim, by=0.5).abs().to(qt)
    ramp = torch.linspace(-12, 12, table.shape[1] * page, device="cuda")[:, None]
    for i, r in enumerate((ramp, -ramp)):
        rows = (rand(g, table.shape[1] * page, dim) * 0.1 + r).to(E4M3).view(-1, page, dim)
        k.view(torch.uint8)[table[i].long()] = rows.view(torch.uint8)
    lens = ints(n, n)
    scores = (q.double().view(b, heads, dim) @ k.float()[table.long()].flatten(1, 2)[:, :n].double().transpose(1, 2)).argmax(-1)
    assert (scores[0] > n * 0.9).all() and (scores[1] < n * 0.1).all()
    lse, weight = torch.empty(b, heads, 1, device="cuda"), torch.zeros(b, 1, table.shape[1] * page, device="cuda")
    out = sb.paged_attention(q, k, v, table, lens, heads, kv_heads=1, scale=0.25, k_scale=0.5, lse=lse, weight=weight)
    check_attention(out, lse, weight, q, k, v, table, lens, heads, 1, before=torch.zeros_like(weight), scale=0.25, k_scale=0.5)
