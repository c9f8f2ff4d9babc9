"""The operators of a transformer block that reads an encoder's memory, as measured cases.

Three operators, each with its gradient: attention of queries to an encoder's states of another
length (``attend``, ``attend_back``), rotary positions with several axes (``rope``; its gradient
is the inverse rotation) and the gated residual with the norms around it (``norm``,
``norm_back``).  The memory is what the detector sees: 34 x 60, 68 x 120 and 136 x 240 tokens of
a 1080p frame at strides 32, 16 and 8 (42,840 in all), 300 queries, 8 heads of 32 channels, 16
cameras; the wider heads and the longer query lists are those of ordinary video transformers.

``own`` False runs the plain form (elementary torch operations in fp32), True the kernels.
"""
import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # the decoder's 300 queries on the stride-32 tokens of two 384 x 640 frames: a launch
        dict(name="attend_queries_p32", op="attend", b=2, tq=300, tk=240, heads=8, kv_heads=8, dim=32, type="f16",
             mask="none", width=20, lse=False),
        # 300 queries of 16 cameras on all three levels of a 1080p memory, images padded
        dict(name="attend_queries_memory", op="attend", b=16, tq=300, tk=42840, heads=8, kv_heads=8, dim=32,
             type="f16", mask="image", width=120, lse=False),
        # one track token per camera stream on the stride-16 tokens seen so far, shared key heads
        dict(name="attend_one_token", op="attend", b=64, tq=1, tk=8160, heads=16, kv_heads=4, dim=128, type="bf16",
             mask="lens", width=120, lse=False),
        # tokens of two frames on the stride-16 tokens, wide heads, training forward
        dict(name="attend_wide", op="attend", b=2, tq=4096, tk=8160, heads=16, kv_heads=4, dim=128, type="bf16",
             mask="none", width=120, lse=True),
        # a training step of the decoder: 300 queries, ragged memories of 8 images
        dict(name="attend_back_ragged", op="attend_back", b=8, tq=300, tk=2040, heads=8, kv_heads=8, dim=64,
             type="f16", mask="lens", width=60, lse=True),
        # gradients of wide heads that share their keys
        dict(name="attend_back_wide", op="attend_back", b=2, tq=2040, tk=8160, heads=16, kv_heads=4, dim=128,
             type="bf16", mask="none", width=120, lse=True),
        # positions of 300 queries of one image: two axes, a launch
        dict(name="rope_queries", op="rope", b=1, t=300, heads=8, dim=32, sections="8,8", layout="pairs", type="f16",
             inverse=False, pos="float", width=20),
        # a clip of 16 frames of stride-16 tokens, time, height and width
        dict(name="rope_clip", op="rope", b=2, t=65280, heads=8, dim=128, sections="16,24,24", layout="half",
             type="bf16", inverse=False, pos="int", width=120),
        # its gradient, in fp32, heads rotated in part
        dict(name="rope_clip_back", op="rope", b=3, t=8161, heads=12, dim=64, sections="4,6,6", layout="half",
             type="f32", inverse=True, pos="int", width=120),
        # residual and norms of 300 queries, fp32 residual stream
        dict(name="norm_queries", op="norm", b=2, t=300, d=256, kind="layer", xtype="f32", ztype="f16", gate="none",
             scale=True, post=True, pre=True),
        # tokens of 8 frames with one gate per image
        dict(name="norm_tokens", op="norm", b=8, t=8160, d=2048, kind="rms", xtype="bf16", ztype="bf16", gate="image",
             scale=True, post=True, pre=True),
        # the gradients of that
        dict(name="norm_back_tokens", op="norm_back", b=8, t=8160, d=1024, kind="layer", xtype="f32", ztype="bf16",
             gate="image", scale=True, post=True, pre=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend_back", "rope", "norm", "norm_back"])
    if op in ("attend", "attend_back"):
        dim = rng.choice([32, 64, 128])
        kv_heads = rng.choice([1, 2, 3, 4, 8])
        heads = kv_heads * rng.choice([1, 1, 2, 3, 4])
        b, tq = _log(rng, 1, 16), _log(rng, 1, 4096)
        room = (1.2e9 if op == "attend" else 4e8) / (b * heads * tq)  # scores of a pass
        tk = _log(rng, 1, max(1, min(42840, int(room), int(5e8 / (b * kv_heads * dim)))))
        return dict(op=op, b=b, tq=tq, tk=tk, heads=heads, kv_heads=kv_heads, dim=dim, type=rng.choice(["f16", "bf16"]),
                    mask=rng.choice(["none", "lens", "image"]), width=rng.choice([13, 20, 60, 120]),
                    lse=op == "attend_back" or rng.random() < 0.5)
    if op == "rope":
        dim, n = rng.choice([32, 64, 80, 128]), rng.choice([1, 2, 3])
        half = dim // 2 if rng.random() < 0.7 else dim // 4
        cut = sorted(rng.sample(range(1, half), n - 1)) if n > 1 else []
        sections = [y - x for x, y in zip([0] + cut, cut + [half])]
        b, heads = _log(rng, 1, 8), rng.choice([1, 3, 8, 12, 16])
        t = _log(rng, 1, min(65280, int(1.2e8 / (b * heads * dim))))
        return dict(op=op, b=b, t=t, heads=heads, dim=dim, sections=",".join(map(str, sections)),
                    layout=rng.choice(["half", "pairs"]), type=rng.choice(["f16", "bf16", "f32"]),
                    inverse=rng.random() < 0.5, pos=rng.choice(["int", "float"]), width=rng.choice([13, 20, 60, 120]))
    d = rng.choice([64, 96, 100, 255, 256, 384, 768, 1024, 1152, 1536, 2048, 4096])
    b = _log(rng, 1, 16)
    t = _log(rng, 1, max(1, min(32640, int((1.3e8 if op == "norm" else 6.5e7) / (b * d)))))
    post, pre = rng.random() < 0.8, rng.random() < 0.8
    return dict(op=op, b=b, t=t, d=d, kind=rng.choice(["rms", "layer"]), xtype=rng.choice(["f32", "bf16", "f16"]),
                ztype=rng.choice(["bf16", "f16"]), gate=rng.choice(["none", "vector", "image", "row"]),
                scale=rng.random() < 0.7, post=post, pre=pre)


# ------------------------------------------------------------------ inputs
def _lens(case):
    """Number of encoder states of each item: from a quarter of them to all."""
    tk = case["tk"]
    return [tk - (i * 7919) % max(1, tk - tk // 4) for i in range(case["b"])]


def _image(case):
    """(width, rows) of the image inside each item's padded token grid; the second of four or
    more cameras is off."""
    w = case["width"]
    rows = -(-case["tk"] // w)
    return [(0, 0) if case["b"] >= 4 and i == 1 else (w - (3 * i) % max(1, w // 2), rows - (5 * i) % max(1, rows // 2))
            for i in range(case["b"])]


def _used(case):
    """Encoder states that take part, over the batch."""
    if case["mask"] == "lens":
        return sum(_lens(case))
    if case["mask"] == "image":
        w, tk = case["width"], case["tk"]
        return sum(sum(min(c, max(0, tk - y * w)) for y in range(r)) for c, r in _image(case))
    return case["b"] * case["tk"]


def _normal(gen, *shape, type=torch.float32, by=1.0):
    return (torch.randn(*shape, device="cuda", generator=gen) * by).to(type)


def _attend_inputs(case, gen):
    b, tq, tk, dim = case["b"], case["tq"], case["tk"], case["dim"]
    t = TYPES[case["type"]]
    s = dict(q=_normal(gen, b, tq, case["heads"] * dim, type=t), lens=None, valid=None)
    # keys and values as one projection leaves them, side by side
    kv = _normal(gen, b, tk, 2 * case["kv_heads"] * dim, type=t)
    s["k"], s["v"] = kv[..., :case["kv_heads"] * dim], kv[..., case["kv_heads"] * dim:]
    if case["mask"] == "lens":
        s["lens"] = torch.tensor(_lens(case), dtype=torch.int32, device="cuda")
    elif case["mask"] == "image":
        i = torch.arange(tk, device="cuda")
        size = torch.tensor(_image(case), device="cuda")
        s["valid"] = ((i % case["width"] < size[:, :1]) & (i // case["width"] < size[:, 1:])).to(torch.uint8)
    if case["op"] == "attend_back":
        # what the forward pass left behind, and the gradient that comes in
        s["out"], s["lse"] = _attend(case, s)
        s["dout"] = _normal(gen, b, tq, case["heads"] * dim, type=t)
    return s


def _rope_inputs(case, gen):
    b, t, w = case["b"], case["t"], case["width"]
    sections = [int(x) for x in case["sections"].split(",")]
    n = sum(sections)
    i = torch.arange(t, device="cuda")
    # a camera that has run for days: its frame numbers are in the millions
    start = torch.randint(0, 5_000_000, (b, 1), device="cuda", generator=gen)
    axes = [start + i // (68 * w), (i // w % 68).expand(b, t), (i % w).expand(b, t)][-len(sections):]
    pos = torch.stack(axes, -1)
    if case["pos"] == "float":
        pos = pos.float() + torch.rand(b, t, len(sections), device="cuda", generator=gen)
    freq = torch.cat([1e4 ** (-torch.arange(k, dtype=torch.float64) / k) for k in sections])
    axis = torch.cat([torch.full((k,), a, dtype=torch.int32) for a, k in enumerate(sections)])
    return dict(x=_normal(gen, b, t, case["heads"] * case["dim"], type=TYPES[case["type"]]), n=n,
                pos=pos.to(torch.int32) if case["pos"] == "int" else pos, freq=freq.cuda(), axis=axis.cuda())


def _norm_inputs(case, gen):
    b, t, d = case["b"], case["t"], case["d"]
    x, z = TYPES[case["xtype"]], TYPES[case["ztype"]]
    layer = case["kind"] == "layer"

    def weights(on):
        if not on:
            return None
        w = 1 + _normal(gen, d, by=0.2)
        return (w, _normal(gen, d, by=0.2)) if layer else (w, None)

    shape = {"none": None, "vector": (d,), "image": (b, d), "row": (b, t, d)}[case["gate"]]
    s = dict(x=_normal(gen, b, t, d, type=x, by=3.0), z=_normal(gen, b, t, d, type=z),
             gate=None if shape is None else _normal(gen, *shape, type=z),
             scale=_normal(gen, d, by=0.5) if case["scale"] else None, post=weights(case["post"]),
             pre=weights(case["pre"]))
    if case["op"] == "norm_back":
        s["dy"] = _normal(gen, b, t, d, type=x)
        s["dh"] = _normal(gen, b, t, d, type=z) if case["pre"] else None
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    make = {"attend": _attend_inputs, "attend_back": _attend_inputs, "rope": _rope_inputs}
    return dict(make.get(case["op"], _norm_inputs)(case, gen), case=case)


# ------------------------------------------------------------------ plain forms
def _split(x, heads, groups):
    """[B, T, heads * dim] rows -> fp32 [B, groups, heads / groups, T, dim]."""
    return x.float().unflatten(-1, (groups, heads // groups, -1)).permute(0, 2, 3, 1, 4)


def _rows(x):
    """The inverse of _split."""
    return x.permute(0, 3, 1, 2, 4).flatten(2)


def _keep(s):
    """[B, Tk] of the states that take part, or None."""
    if s["lens"] is not None:
        return torch.arange(s["k"].shape[1], device="cuda") < s["lens"][:, None]
    return None if s["valid"] is None else s["valid"] != 0


def _softmax(case, s):
    """Scaled scores' softmax [B, kv_heads, group, Tq, Tk] and the scores' log-sum-exp."""
    q, k = _split(s["q"], case["heads"], case["kv_heads"]), _split(s["k"], case["kv_heads"], case["kv_heads"])
    p = q @ k.transpose(-1, -2) * case["dim"] ** -0.5
    keep = _keep(s)
    if keep is not None:
        p.masked_fill_(~keep[:, None, None, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(p - top)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)  # a row without states: zeros
    return q, k, p, top + torch.log(total)


def _values(case, s):
    v, keep = _split(s["v"], case["kv_heads"], case["kv_heads"]), _keep(s)
    return v if keep is None else v.masked_fill(~keep[:, None, None, :, None], 0.0)


def _attend(case, s):
    _, _, p, lse = _softmax(case, s)
    out = _rows(p @ _values(case, s)).to(s["q"].dtype)
    return out, lse.flatten(1, 2).squeeze(-1)


def _attend_back(case, s):
    q, k, p, _ = _softmax(case, s)
    dout, v = _split(s["dout"], case["heads"], case["kv_heads"]), _values(case, s)
    dp = dout @ v.transpose(-1, -2)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * case["dim"] ** -0.5
    dq = ds @ k
    dk = (ds.transpose(-1, -2) @ q).sum(2, keepdim=True)
    dv = (p.transpose(-1, -2) @ dout).sum(2, keepdim=True)
    t = s["q"].dtype
    return dict(dq=_rows(dq).to(t), dk=_rows(dk).to(t), dv=_rows(dv).to(t))


def _rope(case, s):
    x, n = s["x"].float().unflatten(-1, (case["heads"], case["dim"])), s["n"]
    angle = s["pos"].double()[..., s["axis"].long()] * s["freq"]
    cos, sin = torch.cos(angle).float()[:, :, None], torch.sin(angle).float()[:, :, None]
    sin = -sin if case["inverse"] else sin
    if case["layout"] == "half":
        u, v = x[..., :n], x[..., n:2 * n]
        turned = torch.cat([u * cos - v * sin, u * sin + v * cos], -1)
    else:
        u, v = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        turned = torch.stack([u * cos - v * sin, u * sin + v * cos], -1).flatten(-2)
    return torch.cat([turned, x[..., 2 * n:]], -1).flatten(2).to(s["x"].dtype)


EPS = 1e-6


def _normed(v, w, layer):
    """(normalised rows, 1 / deviation, weighted rows) of v."""
    if layer:
        v = v - v.mean(-1, keepdim=True)
    r = torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS)
    hat = v * r
    return hat, r, hat * w[0] + w[1] if layer else hat * w[0]


def _gate(case, s):
    """The gate as fp32 factors of [B, T, D] rows; [B, D] holds one an image."""
    return s["gate"].float()[:, None] if case["gate"] == "image" else s["gate"].float()


def _norm_parts(case, s):
    layer = case["kind"] == "layer"
    z = s["z"].float()
    zhat, zr, n = _normed(z, s["post"], layer) if s["post"] else (None, None, z)
    factor = 1.0
    if s["gate"] is not None:
        factor = _gate(case, s)
    if s["scale"] is not None:
        factor = factor * s["scale"]
    y = s["x"].float() + factor * n
    return zhat, zr, n, factor, y


def _norm(case, s):
    y = _norm_parts(case, s)[-1]
    h = _normed(y, s["pre"], case["kind"] == "layer")[2].to(s["z"].dtype) if s["pre"] else None
    return dict(y=y.to(s["x"].dtype), h=h)


def _norm_input_grad(d, hat, r, w, layer):
    t = d * w[0]
    g = t - hat * (t * hat).mean(-1, keepdim=True)
    return r * (g - t.mean(-1, keepdim=True) if layer else g)


def _norm_back(case, s):
    layer = case["kind"] == "layer"
    zhat, zr, n, factor, y = _norm_parts(case, s)
    dy, out = s["dy"].float(), {}
    if s["pre"]:
        hat, r, _ = _normed(y, s["pre"], layer)
        dh = s["dh"].float()
        dy = dy + _norm_input_grad(dh, hat, r, s["pre"], layer)
        out["pre_w"], out["pre_b"] = (dh * hat).sum((0, 1)), dh.sum((0, 1)) if layer else None
    out["dx"] = dy.to(s["x"].dtype)
    dn = dy * factor
    if s["scale"] is not None:
        out["scale"] = (dy * n * (1.0 if s["gate"] is None else _gate(case, s))).sum((0, 1))
    if s["gate"] is not None:
        dg = dy * n * (1.0 if s["scale"] is None else s["scale"])
        # a gate of a whole image or of all rows gets its sum in fp32, one of each row its own type
        out["gate"] = {"vector": lambda: dg.sum((0, 1)), "image": lambda: dg.sum(1),
                       "row": lambda: dg.to(s["gate"].dtype)}[case["gate"]]()
    if s["post"]:
        out["post_w"], out["post_b"] = (dn * zhat).sum((0, 1)), dn.sum((0, 1)) if layer else None
        dn = _norm_input_grad(dn, zhat, zr, s["post"], layer)
    out["dz"] = dn.to(s["z"].dtype)
    return out


def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        import sarbon_b200 as sb
        if op == "attend":
            lse = torch.empty(case["b"], case["heads"], case["tq"], device="cuda") if case["lse"] else None
            out = sb.cross_attention(s["q"], s["k"], s["v"], case["heads"], kv_heads=case["kv_heads"], lens=s["lens"],
                                     valid=s["valid"], lse=lse)
            return dict(out=out, lse=lse)
        if op == "attend_back":
            dq, dk, dv = sb.cross_attention_backward(s["dout"], s["q"], s["k"], s["v"], s["out"], s["lse"],
                                                     case["heads"], kv_heads=case["kv_heads"], lens=s["lens"],
                                                     valid=s["valid"])
            return dict(dq=dq, dk=dk, dv=dv)
        if op == "rope":
            return sb.rope_axes(s["x"], s["pos"], case["heads"], s["freq"], s["axis"], layout=case["layout"],
                                inverse=case["inverse"])
        if op == "norm":
            y, h = sb.gated_norm(s["x"], s["z"], gate=s["gate"], scale=s["scale"], post=s["post"], pre=s["pre"],
                                 kind=case["kind"], eps=EPS)
            return dict(y=y, h=h)
        return sb.gated_norm_backward(s["dy"], s["dh"], s["x"], s["z"], gate=s["gate"], scale=s["scale"],
                                      post=s["post"], pre=s["pre"], kind=case["kind"], eps=EPS)
    if op == "attend":
        out, lse = _attend(case, s)
        return dict(out=out, lse=lse if case["lse"] else None)
    return {"attend_back": _attend_back, "rope": _rope, "norm": _norm, "norm_back": _norm_back}[op](case, s)


# ------------------------------------------------------------------ in 64 bits
def _exact_attend(case, s, grads):
    """One image at a time, keys that take part only, gradients by differentiation."""
    h, g, dim = case["heads"], case["heads"] // case["kv_heads"], case["dim"]
    keep = _keep(s)
    found = {"out": [], "lse": [], "dq": [], "dk": [], "dv": []}
    for i in range(case["b"]):
        q, k, v = (s[n][i].double().requires_grad_(grads) for n in ("q", "k", "v"))
        use = slice(None) if keep is None else keep[i].nonzero()[:, 0]
        outs, lses = [], []
        for j in range(h):
            kk, vv = k[use].view(-1, case["kv_heads"], dim), v[use].view(-1, case["kv_heads"], dim)
            scores = torch.einsum("qd,kd->qk", q.view(-1, h, dim)[:, j], kk[:, j // g]) / math.sqrt(dim)
            lse = torch.logsumexp(scores, -1)
            some = kk.shape[0] > 0
            outs.append(torch.exp(scores - lse[:, None]) @ vv[:, j // g] if some else q.view(-1, h, dim)[:, j] * 0)
            lses.append(lse)
            if grads:
                # heads one after the other: the gradients add up in q, k and v
                out = outs.pop()
                out.backward(s["dout"][i].double().view(-1, h, dim)[:, j])
        if grads:
            for n, x in (("dq", q), ("dk", k), ("dv", v)):
                found[n].append(torch.zeros_like(x) if x.grad is None else x.grad)
        else:
            found["out"].append(torch.stack(outs, 1).flatten(1))
            found["lse"].append(torch.stack(lses))
    if grads:
        return {n: torch.stack(found[n]) for n in ("dq", "dk", "dv")}
    return dict(out=torch.stack(found["out"]), lse=torch.stack(found["lse"]) if case["lse"] else None)


def _exact_rope(case, s):
    """Pairs as complex numbers, turned by their angle."""
    n = s["n"]
    x = s["x"].double().view(case["b"], case["t"], case["heads"], case["dim"]).clone()
    at = [(slice(0, n), slice(n, 2 * n)), (slice(0, 2 * n, 2), slice(1, 2 * n, 2))][case["layout"] == "pairs"]
    turn = torch.zeros(case["b"], case["t"], n, dtype=torch.float64, device="cuda")
    for i, (a, f) in enumerate(zip(s["axis"].tolist(), s["freq"].tolist())):
        turn[..., i] = s["pos"][..., a].double() * f
    z = torch.complex(x[..., at[0]].contiguous(), x[..., at[1]].contiguous())
    z = z * torch.polar(torch.ones_like(turn), -turn if case["inverse"] else turn)[:, :, None]
    x[..., at[0]], x[..., at[1]] = z.real, z.imag
    return x.flatten(2)


def _exact_norm(case, s, grads):
    def wide(t):
        return None if t is None else t.double().requires_grad_(grads)

    def norm(v, w):
        if case["kind"] == "layer":
            return torch.nn.functional.layer_norm(v, v.shape[-1:], w[0], w[1], EPS)
        return v / (v.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * w[0]

    x, z, gate, scale = (wide(s[n]) for n in ("x", "z", "gate", "scale"))
    post, pre = (tuple(wide(w) for w in s[n]) if s[n] else None for n in ("post", "pre"))
    part = norm(z, post) if post else z
    if gate is not None:
        part = part * (gate[:, None] if case["gate"] == "image" else gate)
    if scale is not None:
        part = part * scale
    y = x + part
    h = norm(y, pre) if pre else None
    if not grads:
        return dict(y=y, h=h)
    total = (y * s["dy"].double()).sum()
    if pre:
        total = total + (h * s["dh"].double()).sum()
    total.backward()
    out = dict(dx=x.grad, dz=z.grad)
    if gate is not None:
        out["gate"] = gate.grad
    if scale is not None:
        out["scale"] = scale.grad
    for name, w in (("post", post), ("pre", pre)):
        if w:
            out[name + "_w"], out[name + "_b"] = w[0].grad, None if w[1] is None else w[1].grad
    return out


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op in ("attend", "attend_back"):
        return _exact_attend(case, s, op == "attend_back")
    return _exact_rope(case, s) if op == "rope" else _exact_norm(case, s, op == "norm_back")


# ------------------------------------------------------------------ work
def work(case):
    op = case["op"]
    if op in ("attend", "attend_back"):
        b, tq, h, dim, used = case["b"], case["tq"], case["heads"], case["dim"], _used(case)
        rows, keys, stats = b * tq * h * dim * 2, used * case["kv_heads"] * dim * 2, b * h * tq * 4
        masks = {"none": 0, "lens": 4 * b, "image": b * case["tk"]}[case["mask"]]
        if op == "attend":
            return dict(bytes=2 * rows + 2 * keys + masks + (stats if case["lse"] else 0), flops=4 * used * tq * h * dim)
        # q, out, its gradient and the keys and values in; the three gradients out
        all_keys = b * case["tk"] * case["kv_heads"] * dim * 2
        return dict(bytes=4 * rows + 2 * keys + 2 * all_keys + masks + stats, flops=10 * used * tq * h * dim)
    size = {"f16": 2, "bf16": 2, "f32": 4}
    if op == "rope":
        n = case["b"] * case["t"] * case["heads"] * case["dim"]
        axes = case["sections"].count(",") + 1
        return dict(bytes=2 * n * size[case["type"]] + case["b"] * case["t"] * axes * 4, flops=3 * n)
    n, x, z = case["b"] * case["t"] * case["d"], size[case["xtype"]], size[case["ztype"]]
    gate = {"none": 0, "vector": case["d"], "image": case["b"] * case["d"], "row": n}[case["gate"]] * z
    if op == "norm":
        return dict(bytes=n * (2 * x + z + (z if case["pre"] else 0)) + gate, flops=12 * n)
    gate += gate if case["gate"] == "row" else 2 * gate
    return dict(bytes=n * (3 * x + 2 * z + (z if case["pre"] else 0)) + gate, flops=30 * n)
