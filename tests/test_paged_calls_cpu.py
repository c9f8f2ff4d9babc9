"""What the native side of the paged memory's calls takes on: never a call that the Python side would refuse, and
every call in its plain forms.  Looked at on CPU tensors, which the Python side turns down last of all."""
import random

import pytest
import torch

import sarbon_b200 as sb
from sarbon_b200._lib import LIB_PATH

calls = pytest.importorskip("sarbon_b200._paged_calls") if LIB_PATH.exists() else pytest.skip("not built", allow_module_level=True)

F16, BF16, E4M3, I32 = torch.float16, torch.bfloat16, torch.float8_e4m3fn, torch.int32
ORDER = {
    "attend": (sb.paged_attention, "q k_pages v_pages table lens heads kv_heads scale causal k_scale v_scale weight decay out lse"),
    "append": (sb.paged_write, "k v k_pages v_pages table at count k_scale v_scale weight born stamp after kv_heads"),
    "cut": (sb.paged_evict, "k_pages v_pages table lens weight keep born since weight_out born_out after"),
}
DEFAULTS = dict(kv_heads=None, scale=None, causal=False, k_scale=1.0, v_scale=1.0, weight=None, decay=1.0, out=None, lse=None,
                count=None, born=None, stamp=None, after=None, since=None, weight_out=None, born_out=None)


def taken(op, args):
    return getattr(calls, "takes_" + op)(*({**DEFAULTS, **args}[x] for x in ORDER[op][1].split())) is True


def valid(op, args):
    try:
        ORDER[op][0](**args)
    except ValueError as e:
        return "one CUDA device" in str(e)
    except Exception:
        return False
    return True  # (an empty call is done)


def plain(op, r):
    """The arguments of a call that is right."""
    b, n, page, heads, dim = r.randrange(1, 4), r.randrange(1, 4), r.choice([1, 3, 8]), r.choice([1, 2, 3]), r.choice([32, 64, 128])
    t, kind = r.choice([1, 1, 2, 5]), r.choice([F16, BF16])
    pages = r.choice([kind, E4M3])
    pool = torch.zeros(2, r.randrange(1, 6), page, heads * dim, dtype=pages)
    at = dict(k_pages=pool[0], v_pages=pool[1], table=torch.zeros(b, n, dtype=I32))
    if r.random() < 0.5:  # keys and values side by side
        pool = torch.zeros(pool.shape[1], page, 2 * heads * dim, dtype=pages)
        at.update(k_pages=pool[..., :heads * dim], v_pages=pool[..., heads * dim:])
    account = (b, heads, n * page)
    lens = lambda: torch.zeros(b, dtype=I32)
    if op == "attend":
        group = r.choice([1, 2, 4])
        at.update(q=torch.zeros(b, t, group * heads * dim, dtype=kind), lens=lens(), heads=group * heads)
        if group > 1 or r.random() < 0.5:
            at["kv_heads"] = heads
        more = dict(scale=r.choice([1, 0.5]), causal=True, weight=torch.zeros(account), decay=0.5, lse=torch.zeros(b, group * heads, t),
                    out=torch.zeros(b, t, group * heads * dim, dtype=kind))
    elif op == "append":
        at.update(k=torch.zeros(b, t, heads * dim, dtype=kind), v=torch.zeros(b, t, heads * dim, dtype=kind), at=lens(),
                  kv_heads=heads)
        more = dict(count=lens(), weight=torch.zeros(account), after=lens())
        if r.random() < 0.5:
            at.update(born=torch.zeros(account, dtype=I32), stamp=r.choice([torch.zeros(b, t, dtype=I32), lens()]))
    else:
        at.update(lens=lens(), weight=torch.zeros(account), keep=r.choice([0, 5, 1 << 40, lens()]))
        more = dict(weight_out=r.choice([at["weight"], torch.zeros(account)]), after=r.choice([at["lens"], lens()]))
        if r.random() < 0.5:
            at["born"] = torch.zeros(account, dtype=I32)
            more.update(since=lens(), born_out=r.choice([at["born"], torch.zeros(account, dtype=I32)]))
    if pages == E4M3 and op != "cut":
        more.update(k_scale=0.5, v_scale=3)
    at.update({x: y for x, y in more.items() if r.random() < 0.5})
    return at


@pytest.mark.parametrize("op", list(ORDER))
def test_plain_calls_are_taken(op):
    r = random.Random(1)
    for _ in range(300):
        args = plain(op, r)
        assert valid(op, args) and taken(op, args), {x: getattr(y, "shape", y) for x, y in args.items()}


def bent(x, args, r):
    """Another value for an argument, mostly a wrong one."""
    if not isinstance(x, torch.Tensor):
        return r.choice([None, 0, -1, 2, 3, 7, 0.0, -0.5, 1.5, 1e39, float("nan"), True, False, "1", torch.zeros(2, dtype=I32),
                         1 << 31, 1 << 70, 2.0])
    others = [t for t in args.values() if isinstance(t, torch.Tensor)]
    way = r.randrange(13)
    if way == 0:
        return r.choice(others)
    if way == 1:
        return x.to(r.choice([F16, BF16, torch.float32, I32, torch.int64]))
    if way == 2:
        return x[:-1]
    if way == 3:
        return x[..., :-1]
    if way == 4:
        return x.unsqueeze(0)
    if way == 5:
        return x.flatten()
    if way == 6:
        return x.transpose(0, -1).contiguous().transpose(0, -1)
    if way == 7:
        return x[:1].expand(x.shape) if x.shape[0] else x
    if way == 8:
        return torch.cat([x.float(), x.float()], -1).to(x.dtype)[..., :x.shape[-1]]
    if way == 9:
        return x.clone().requires_grad_() if x.dtype in (F16, BF16, torch.float32) else None
    if way == 10:
        return x[:, :1].expand(x.shape) if x.dim() > 1 and x.shape[1] else torch.zeros(0, dtype=x.dtype)
    if way == 11:
        room = torch.zeros(x.numel() + 8, dtype=torch.float32).to(x.dtype)
        return room[r.randrange(8):][:x.numel()].view(x.shape)
    other = r.choice(others)  # memory of another argument, in part or whole
    if other.dtype != x.dtype or not other.is_contiguous() or other.numel() < x.numel():
        return None
    return other.flatten()[other.numel() - x.numel():].view(x.shape)


@pytest.mark.parametrize("op", list(ORDER))
def test_what_is_refused_is_not_taken(op):
    r, kept = random.Random(2), 0
    for _ in range(4000):
        args = plain(op, r)
        for _ in range(r.choice([1, 1, 2])):
            name = r.choice([x for x in ORDER[op][1].split() if x in args or r.random() < 0.2] or list(args))
            args[name] = bent(args.get(name, DEFAULTS.get(name)), args, r)
        if taken(op, args):
            kept += 1
            assert valid(op, args), {x: (y.shape, y.stride(), y.dtype) if isinstance(y, torch.Tensor) else y for x, y in args.items()}
    assert kept > 400  # what stays right after the change is looked at too


def test_what_is_no_plain_tensor_is_left_alone():
    r = random.Random(3)
    args = plain("attend", r)
    assert taken("attend", args)

    class Own(torch.Tensor):
        pass

    assert not taken("attend", {**args, "q": args["q"].as_subclass(Own)})
    assert not taken("attend", {**args, "q": args["q"].to_sparse()})
    grad = args["q"].clone().requires_grad_()
    assert not taken("attend", {**args, "q": grad})
    with torch.no_grad():
        assert taken("attend", {**args, "q": grad})
        assert taken("attend", {**args, "q": torch.nn.Parameter(grad)})
    with pytest.raises(TypeError):
        calls.takes_attend(1, 2)
    seen = []
    torch.func.vmap(lambda q: (seen.append(taken("attend", {**args, "q": q})), q)[1])(args["q"].unsqueeze(0))
    assert seen == [False]
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        assert not taken("attend", args)
