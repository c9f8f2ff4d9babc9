"""The operators of a memory that a camera stream keeps between frames, as measured cases.

The memory lies in pages; an item's table says which.  Three operators work on it: new states are
written behind the ones that are there (``write``), a few query tokens attend to all of them and add
up how much each was looked at (``attend``), and when there are more than the budget allows, the states that
were looked at least make room (``evict``).  A frame of the cameras here has 34 x 60 tokens at stride
32, 68 x 120 at stride 16 and 136 x 240 at stride 8 (42,840 in all); streams keep one frame to
sixteen, in 16 bits or in e4m3.

``own`` False runs the plain form (elementary torch operations in fp32), True the kernels.
"""
import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
K_SCALE, V_SCALE = 2.0 ** -6, 2.0 ** -5  # what an e4m3 code of 1 stands for
NEWEST = 1_000_000  # stamp of the first state of the newest frame


def listed():
    return [
        # one track token of two streams on one 384 x 640 frame's stride-32 tokens: a launch
        dict(name="attend_small", op="attend", b=2, tq=1, n=240, heads=8, kv_heads=8, dim=32, page=20, type="f16",
             pages="f16", causal=False, weight=True, lse=False, joint=True),
        # one token of 64 streams that keep a stride-16 frame, key heads shared by four
        dict(name="attend_token", op="attend", b=64, tq=1, n=8160, heads=16, kv_heads=4, dim=128, page=120, type="bf16",
             pages="bf16", causal=False, weight=True, lse=False, joint=False),
        # the same from e4m3 pages
        dict(name="attend_token_e4m3", op="attend", b=64, tq=1, n=8160, heads=16, kv_heads=4, dim=128, page=64,
             type="bf16", pages="e4m3", causal=False, weight=True, lse=False, joint=True),
        # one stream that keeps sixteen stride-16 frames
        dict(name="attend_long", op="attend", b=1, tq=1, n=130560, heads=16, kv_heads=4, dim=128, page=240, type="bf16",
             pages="bf16", causal=False, weight=False, lse=True, joint=False),
        # the last eight tokens of 16 streams, each seeing those before it, three levels of a 1080p frame
        dict(name="attend_tokens", op="attend", b=16, tq=8, n=42840, heads=8, kv_heads=4, dim=64, page=60, type="f16",
             pages="f16", causal=True, weight=True, lse=True, joint=True),
        # one new token of 64 streams
        dict(name="write_token", op="write", b=64, t=1, n=8160, kv_heads=4, dim=128, page=120, type="bf16", pages="bf16",
             ragged=False, joint=False),
        # a new stride-32 frame of 16 streams, images of several heights
        dict(name="write_frame", op="write", b=16, t=2040, n=4080, kv_heads=8, dim=128, page=60, type="bf16",
             pages="bf16", ragged=True, joint=True),
        # a new stride-16 frame of 8 streams into e4m3 pages
        dict(name="write_frame_e4m3", op="write", b=8, t=8160, n=16320, kv_heads=8, dim=64, page=128, type="f16",
             pages="e4m3", ragged=False, joint=False),
        # 64 streams at a budget of 240 states, one too many each
        dict(name="evict_token", op="evict", b=64, n=241, keep=240, recent=1, kv_heads=4, dim=128, page=16, pages="bf16",
             joint=False),
        # 16 streams keep eight stride-32 frames and have got a ninth, whose last quarter stays
        dict(name="evict_frame", op="evict", b=16, n=18360, keep=16320, recent=510, kv_heads=8, dim=128, page=60,
             pages="bf16", joint=True),
        # two streams halve what they keep of sixteen stride-16 frames
        dict(name="evict_half", op="evict", b=2, n=130560, keep=65280, recent=8160, kv_heads=8, dim=64, page=240,
             pages="e4m3", joint=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "write", "evict", "evict"])
    dim, kv_heads, page = rng.choice([32, 64, 128]), rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 7, 16, 20, 60, 64, 128, 240])
    pages = rng.choice(["f16", "bf16", "e4m3"])
    kind = pages if pages != "e4m3" else rng.choice(["f16", "bf16"])
    joint, b = rng.random() < 0.5, _log(rng, 1, 64)
    most = int(2.6e8 / (b * kv_heads * dim))  # values of all keys
    if op == "attend":
        tq = rng.choice([1, 1, 1, 2, 5, 8])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
        n = _log(rng, 1, max(1, min(130560, most, int(4e7 / (b * heads * tq)))))
        return dict(op=op, b=b, tq=tq, n=n, heads=heads, kv_heads=kv_heads, dim=dim, page=page, type=kind, pages=pages,
                    causal=rng.random() < 0.5, weight=rng.random() < 0.7, lse=rng.random() < 0.5, joint=joint)
    if op == "write":
        t = _log(rng, 1, max(1, min(8160, int(3.2e7 / (b * kv_heads * dim)))))
        n = _log(rng, t, max(t, min(42840, int(1e8 / (b * kv_heads * dim)))))
        return dict(op=op, b=b, t=t, n=n, kv_heads=kv_heads, dim=dim, page=page, type=kind, pages=pages,
                    ragged=rng.random() < 0.5, joint=joint)
    n = _log(rng, 2, max(2, min(130560, most // 2)))
    keep = rng.choice([n - 1, max(1, n - page), max(1, n - n // 9), max(1, n // 2)])
    return dict(op=op, b=b, n=n, keep=keep, recent=rng.choice([0, (n - keep + 3) // 4, n - keep]), kv_heads=kv_heads,
                dim=dim, page=page, pages=pages, joint=joint)


# ------------------------------------------------------------------ inputs
def _lens(case):
    """States of each item: the most for the first, down to three quarters of it for others; all alike after a write."""
    n = case["n"]
    return [n if case["op"] == "write" else n - (i * 7919) % max(1, n // 4) for i in range(case["b"])]


def _counts(case):
    """New states of each item."""
    t = case["t"]
    return [t - (i * 613) % max(1, t // 3) if case["ragged"] else t for i in range(case["b"])]


def _normal(gen, *shape, type=torch.float32, by=1.0):
    return (torch.randn(*shape, device="cuda", generator=gen) * by).to(type)


def _codes(gen, shape, type, scale):
    """Standard normal values as pages of `type` hold them."""
    if type != "e4m3":
        return _normal(gen, *shape, type=TYPES[type])
    return _normal(gen, *shape, by=1.0 / scale).clamp_(-448, 448).to(TYPES[type])


def _pages(case, gen):
    """Pools of keys and values, and the items' tables; places of a table that no state needs are -1."""
    page, width = case["page"], case["kv_heads"] * case["dim"]
    need = -(-case["n"] // page)
    pool = case["b"] * need + 3
    if case["joint"]:  # keys and values of a page side by side
        both = torch.cat([_codes(gen, (pool, page, width), case["pages"], x).view(torch.uint8)
                          for x in (K_SCALE, V_SCALE)], -1).view(TYPES[case["pages"]])
        k, v = both[..., :width], both[..., width:]
    else:
        k, v = (_codes(gen, (pool, page, width), case["pages"], x) for x in (K_SCALE, V_SCALE))
    table = torch.randperm(pool, device="cuda", generator=gen)[:case["b"] * need].view(case["b"], need).to(torch.int32)
    lens = torch.tensor(_lens(case), dtype=torch.int32, device="cuda")
    table.masked_fill_(torch.arange(need, device="cuda") * page >= lens[:, None], -1)
    e4m3 = case["pages"] == "e4m3"
    return dict(k_pages=k, v_pages=v, table=table, lens=lens, k_scale=K_SCALE if e4m3 else 1.0,
                v_scale=V_SCALE if e4m3 else 1.0)


def _attend_inputs(case, gen):
    s = _pages(case, gen)
    s["q"] = _normal(gen, case["b"], case["tq"], case["heads"] * case["dim"], type=TYPES[case["type"]])
    places = s["table"].shape[1] * case["page"]
    s["weight"] = _normal(gen, case["b"], case["kv_heads"], places).exp_() if case["weight"] else None
    return s


def _write_inputs(case, gen):
    s, b, t, width = _pages(case, gen), case["b"], case["t"], case["kv_heads"] * case["dim"]
    # keys and values as one projection leaves them; the lengths are those after the call
    kv = _normal(gen, b, t, 2 * width, type=TYPES[case["type"]], by=1.5)
    s["k"], s["v"] = kv[..., :width], kv[..., width:]
    s["count"] = torch.tensor(_counts(case), dtype=torch.int32, device="cuda")
    s["at"] = s.pop("lens") - s["count"]
    places = s["table"].shape[1] * case["page"]
    s["weight"] = _normal(gen, b, case["kv_heads"], places).exp_()
    s["born"] = torch.randint(0, NEWEST, (b, case["kv_heads"], places), dtype=torch.int32, device="cuda", generator=gen)
    s["stamp"] = NEWEST + torch.arange(t, dtype=torch.int32, device="cuda").expand(b, t).contiguous()
    return s


def _evict_inputs(case, gen):
    s, keep = _pages(case, gen), case["keep"]
    j = torch.arange(s["table"].shape[1] * case["page"], device="cuda")
    shape = (case["b"], case["kv_heads"], len(j))
    # what earlier evictions left, in no order, then the newest states in theirs, the last not yet looked at
    s["weight"] = (2 * _normal(gen, *shape)).exp_().masked_fill_(j >= case["n"] - max(1, (case["n"] - keep) // 8), 0.0)
    old = torch.randint(0, NEWEST, shape, device="cuda", generator=gen)
    s["born"] = torch.where(j < keep, old, NEWEST + j - keep).to(torch.int32)
    s["since"] = (NEWEST + s["lens"] - keep - case["recent"]).clamp_(min=NEWEST)
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    make = {"attend": _attend_inputs, "write": _write_inputs, "evict": _evict_inputs}
    return dict(make[case["op"]](case, gen), case=case)


# ------------------------------------------------------------------ plain forms
DECAY = 0.98


def _states(pages, table, heads, scale):
    """Every item's states from its pages, fp32 [B, heads, places, dim]."""
    x = pages[table.long().clamp(min=0)].flatten(1, 2).float() * scale
    return x.unflatten(-1, (heads, -1)).transpose(1, 2)


def _attend(case, s):
    b, tq, kv_heads = case["b"], case["tq"], case["kv_heads"]
    k, v = _states(s["k_pages"], s["table"], kv_heads, s["k_scale"]), _states(s["v_pages"], s["table"], kv_heads, s["v_scale"])
    q = s["q"].float().view(b, tq, kv_heads, -1, case["dim"]).permute(0, 2, 3, 1, 4).flatten(2, 3)  # rows (head, token)
    j = torch.arange(k.shape[2], device="cuda")
    seen = s["lens"][:, None].expand(b, tq)
    if case["causal"]:
        seen = seen - torch.arange(tq - 1, -1, -1, device="cuda")
    seen = (j < seen[..., None]).repeat(1, case["heads"] // kv_heads, 1)[:, None]
    p = (q @ k.transpose(-1, -2) * case["dim"] ** -0.5).masked_fill_(~seen, -math.inf)
    top = p.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(p - top)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)  # a row without states: zeros
    used = j < s["lens"][:, None]
    out = p @ v.masked_fill_(~used[:, None, :, None], 0.0)
    out = out.unflatten(2, (-1, tq)).permute(0, 3, 1, 2, 4).flatten(2).to(s["q"].dtype)
    if s["weight"] is not None:
        w = s["weight"]
        w.copy_(torch.where(used[:, None], DECAY * w + p.sum(2), w))
    lse = (top + torch.log(total)).view(b, case["heads"], tq) if case["lse"] else None
    return dict(out=out, lse=lse, weight=s["weight"])


def _place(s, case, item, pos):
    """(page, row) of positions of items."""
    return s["table"].long()[item, pos // case["page"]], pos % case["page"]


def _write(case, s):
    item, t = (torch.arange(case["t"], device="cuda") < s["count"][:, None]).nonzero(as_tuple=True)
    pos = s["at"].long()[item] + t
    page, row = _place(s, case, item, pos)
    for pages, x, scale in ((s["k_pages"], s["k"], s["k_scale"]), (s["v_pages"], s["v"], s["v_scale"])):
        x = x[item, t].float() / scale
        if case["pages"] == "e4m3":  # as bytes: there is no assignment by index for e4m3
            pages.view(torch.uint8)[page, row] = x.clamp_(-448, 448).to(pages.dtype).view(torch.uint8)
        else:
            pages[page, row] = x.to(pages.dtype)
    s["weight"][item, :, pos] = 0.0
    s["born"][item, :, pos] = s["stamp"][item, t][:, None]
    return dict(k=s["k_pages"], v=s["v_pages"], weight=s["weight"], born=s["born"], after=s["at"] + s["count"])


def _evict(case, s):
    keep, lens, weight, born = case["keep"], s["lens"], s["weight"], s["born"]
    j = torch.arange(weight.shape[-1], device="cuda")
    used, after = j < lens[:, None, None], lens.clamp(max=keep)
    # by weight, then by what is protected, then by what is there at all; equal ones stay in order
    order = torch.sort(weight, dim=-1, descending=True, stable=True).indices
    rank = (born >= s["since"][:, None, None]).long() + 2 * used.expand_as(born).long()
    order = order.gather(-1, torch.sort(rank.gather(-1, order), dim=-1, descending=True, stable=True).indices)
    place = torch.empty_like(order).scatter_(-1, order, j.expand_as(order))
    stays = place < after[:, None, None]
    low = j < after[:, None, None]
    free, moves = (low & ~stays).nonzero(as_tuple=True), (stays & ~low).nonzero(as_tuple=True)
    weight, born = weight.masked_fill(~low, 0.0), born.masked_fill(~low, 0)
    weight[free], born[free] = s["weight"][moves], s["born"][moves]
    to, at = _place(s, case, free[0], free[2]), _place(s, case, moves[0], moves[2])
    for pages in (s["k_pages"], s["v_pages"]):
        rows = pages.view(torch.uint8).unflatten(-1, (case["kv_heads"], -1))
        rows[to[0], to[1], free[1]] = rows[at[0], at[1], moves[1]]
    return dict(k=s["k_pages"], v=s["v_pages"], weight=weight, born=born, after=after)


def run(s):
    case = s["case"]
    if own:
        import sarbon_b200 as sb
        if case["op"] == "attend":
            lse = torch.empty(case["b"], case["heads"], case["tq"], device="cuda") if case["lse"] else None
            out = sb.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], case["heads"],
                                     kv_heads=case["kv_heads"], causal=case["causal"], k_scale=s["k_scale"],
                                     v_scale=s["v_scale"], weight=s["weight"], decay=DECAY, lse=lse)
            return dict(out=out, lse=lse, weight=s["weight"])
        if case["op"] == "write":
            after = sb.paged_write(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["at"], count=s["count"],
                                   k_scale=s["k_scale"], v_scale=s["v_scale"], weight=s["weight"], born=s["born"],
                                   stamp=s["stamp"])
            return dict(k=s["k_pages"], v=s["v_pages"], weight=s["weight"], born=s["born"], after=after)
        after, weight, born = sb.paged_evict(s["k_pages"], s["v_pages"], s["table"], s["lens"], s["weight"], case["keep"],
                                             born=s["born"], since=s["since"])
        return dict(k=s["k_pages"], v=s["v_pages"], weight=weight, born=born, after=after)
    return {"attend": _attend, "write": _write, "evict": _evict}[case["op"]](case, s)


# ------------------------------------------------------------------ in 64 bits
def _exact_attend(case, s):
    """One item and head at a time, its own states only."""
    g, tq, dim = case["heads"] // case["kv_heads"], case["tq"], case["dim"]
    out = torch.zeros(case["b"], tq, case["heads"], dim, dtype=torch.float64, device="cuda")
    lse = torch.full((case["b"], case["heads"], tq), -math.inf, dtype=torch.float64, device="cuda")
    weight = None if s["weight"] is None else s["weight"].double()
    for i, n in enumerate(s["lens"].tolist()):
        pages = s["table"][i, :-(-n // case["page"])].long()
        keys, values = (s[x][pages].flatten(0, 1)[:n].double() for x in ("k_pages", "v_pages"))
        if weight is not None:
            weight[i, :, :n] *= DECAY
        for h in range(case["heads"]):
            at = slice(h // g * dim, h // g * dim + dim)
            scores = (s["q"][i, :, h * dim:(h + 1) * dim].double() @ keys[:, at].T) * (s["k_scale"] / math.sqrt(dim))
            if case["causal"]:
                ends = n - tq + torch.arange(tq, device="cuda")
                scores = scores.masked_fill(torch.arange(n, device="cuda") > ends[:, None], -math.inf)
            lse[i, h] = torch.logsumexp(scores, -1)
            share = torch.exp(scores - lse[i, h][:, None]).nan_to_num(0.0)
            out[i, :, h] = share @ values[:, at] * s["v_scale"]
            if weight is not None:
                weight[i, h // g, :n] += share.sum(0)
    return dict(out=out.flatten(2), lse=lse if case["lse"] else None, weight=weight)


def _exact_write(case, s):
    """One item at a time; values before they are rounded to the pages' type."""
    k, v, weight, born = s["k_pages"].double(), s["v_pages"].double(), s["weight"].double(), s["born"].clone()
    after = []
    for i, (start, n) in enumerate(zip(s["at"].tolist(), s["count"].tolist())):
        at = torch.arange(start, start + n, device="cuda")
        page, row = s["table"][i].long()[at // case["page"]], at % case["page"]
        k[page, row], v[page, row] = s["k"][i, :n].double() / s["k_scale"], s["v"][i, :n].double() / s["v_scale"]
        weight[i, :, start:start + n] = 0
        born[i, :, start:start + n] = s["stamp"][i, :n]
        after.append(start + n)
    return dict(k=k, v=v, weight=weight, born=born, after=torch.tensor(after, dtype=torch.int32, device="cuda"))


def _exact_evict(case, s):
    """One item and head at a time: the states from best to worst, the first of them stay."""
    keep, page = case["keep"], case["page"]
    k, v = (s[x].view(torch.uint8).clone().view(s[x].dtype).unflatten(-1, (case["kv_heads"], -1)) for x in ("k_pages", "v_pages"))
    weight, born = torch.zeros_like(s["weight"], dtype=torch.float64), torch.zeros_like(s["born"])
    lens = s["lens"].tolist()
    for i, n in enumerate(lens):
        table = s["table"][i].long()
        for h in range(case["kv_heads"]):
            left = min(n, keep)
            weight[i, h, :left], born[i, h, :left] = s["weight"][i, h, :left].double(), s["born"][i, h, :left]
            if n <= keep:
                continue
            w, b = s["weight"][i, h, :n].double(), s["born"][i, h, :n]
            ranks, new = torch.argsort(-w, stable=True), b >= s["since"][i]
            best = torch.cat([ranks[new[ranks]], ranks[~new[ranks]]])  # protected states before all others
            stays = torch.zeros(n, dtype=torch.bool, device="cuda").index_fill_(0, best[:keep], True)
            to = (~stays[:keep]).nonzero()[:, 0]
            at = keep + stays[keep:].nonzero()[:, 0]
            weight[i, h, to], born[i, h, to] = w[at], b[at]
            for x in (k, v):
                bytes_ = x.view(torch.uint8)
                bytes_[table[to // page], to % page, h] = bytes_[table[at // page], at % page, h]
    after = torch.tensor([min(n, keep) for n in lens], dtype=torch.int32, device="cuda")
    return dict(k=k.flatten(2).double(), v=v.flatten(2).double(), weight=weight, born=born, after=after)


def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "write": _exact_write, "evict": _exact_evict}[case["op"]](case, s)


# ------------------------------------------------------------------ work
def work(case):
    size = {"f16": 2, "bf16": 2, "e4m3": 1}[case["pages"]]
    b, kv_heads, dim = case["b"], case["kv_heads"], case["dim"]
    places = b * kv_heads * -(-case["n"] // case["page"]) * case["page"]
    if case["op"] == "attend":
        used, rows = sum(_lens(case)), b * case["tq"] * case["heads"]
        return dict(bytes=2 * used * kv_heads * dim * size + 2 * rows * dim * 2 + (8 * used * kv_heads if case["weight"] else 0)
                    + (4 * rows if case["lse"] else 0), flops=4 * used * case["tq"] * case["heads"] * dim)
    if case["op"] == "write":
        new = sum(_counts(case))
        return dict(bytes=2 * new * kv_heads * dim * (2 + size) + 8 * new * kv_heads, flops=2 * new * kv_heads * dim)
    # states that move: the protected ones behind the budget, and of the others there as large a share as of all
    moved = 0.0
    for n in _lens(case):
        tail = max(0, n - case["keep"])
        kept = min(tail, case["recent"])
        moved += min(tail, kept + (tail - kept) * max(0.0, (case["keep"] - kept) / max(1, n - kept)))
    used = sum(_lens(case)) * kv_heads
    return dict(bytes=8 * used + 8 * places + int(4 * moved * kv_heads * dim * size), flops=4 * used)
