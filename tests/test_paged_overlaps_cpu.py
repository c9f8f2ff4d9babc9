"""What the paged memory's calls write lies apart from all else that they are given: layouts that lie between one another are
taken, such that meet are refused, by both sides of a call alike."""
import random

import pytest
import torch

import sarbon_b200 as sb
from sarbon_b200 import paged_ops
from sarbon_b200._lib import LIB_PATH
from test_paged_ops_cpu import ATTEND, EVICT, WRITE

F16, I32 = torch.float16, torch.int32
P, PAGE, W = 6, 4, 128
OPS = {"attend": sb.paged_attention, "append": sb.paged_write, "cut": sb.paged_evict}
FULL = {"attend": ATTEND, "append": WRITE, "cut": EVICT}


def outcome(op, change):
    """"apart" if a call gets past every check but that of its device, "meet" if it is refused for its memory."""
    with pytest.raises(ValueError) as e:
        OPS[op](**{**FULL[op], **change})
    text = str(e.value)
    assert "one CUDA device" in text or "own memory" in text, text
    return "apart" if "one CUDA device" in text else "meet"


def taken(op, change):
    if not LIB_PATH.exists():
        pytest.skip("not built")
    calls = pytest.importorskip("sarbon_b200._paged_calls")
    from test_paged_calls_cpu import DEFAULTS, ORDER
    return getattr(calls, "takes_" + op)(*({**DEFAULTS, **FULL[op], **change}[x] for x in ORDER[op][1].split())) is True


def pools(*shape):
    return torch.zeros(*shape, dtype=F16)


def side_by_side(off=W, between=2 * W):
    room = pools(P, PAGE, max(between, off + W))
    return room[..., :W], room[..., off:off + W]


def halves():  # all keys of a page, then all values
    room = pools(P, 2, PAGE, W)
    return room[:, 0], room[:, 1]


def of_heads():  # pages of heads of keys and values, a row's in the middle of wider ones
    room = pools(P + 1, PAGE + 3, 3 * W)
    return room[1:, 1:PAGE + 1, W:2 * W], room[1:, 2:PAGE + 2, 2 * W:]


def pages_turned():  # the same row of all pages together; not one of the plain forms
    room = pools(PAGE, P, 2 * W).transpose(0, 1)
    return room[..., :W], room[..., W:]


def layers():  # two layers' pages alternate
    room = pools(2 * P, PAGE, W)
    return room[::2], room[1::2]


def shifted(rows):  # values a few rows behind the keys in the same pages
    room = pools(P, PAGE + rows, W)
    return room[:, :PAGE], room[:, rows:]


def next_page():
    room = pools(P + 1, PAGE, W)
    return room[:-1], room[1:]


APART = [side_by_side(), side_by_side(W, 2 * W + 8), halves(), of_heads(), layers(), shifted(PAGE)]
MEET = [side_by_side(64), side_by_side(W - 8, 2 * W), side_by_side(8, 3 * W), shifted(1), shifted(PAGE - 1), next_page()]


@pytest.mark.parametrize("op", ["append", "cut"])
def test_pools_side_by_side(op):
    for k, v in APART:
        for pair in (dict(k_pages=k, v_pages=v), dict(k_pages=v, v_pages=k)):
            assert outcome(op, pair) == "apart" and taken(op, pair)
    k, v = pages_turned()
    assert outcome(op, dict(k_pages=k, v_pages=v)) == "apart"
    for k, v in MEET:
        for pair in (dict(k_pages=k, v_pages=v), dict(k_pages=v, v_pages=k)):
            assert outcome(op, pair) == "meet" and not taken(op, pair)
            if op == "append":  # what is only read may lie as it likes
                assert outcome("attend", pair) == "apart" and taken("attend", pair)


def test_new_states_from_the_pools():
    room = pools(P + 2, PAGE, 2 * W)
    k, v = room[:P, :, :W], room[:P, :, W:]
    own = dict(k_pages=k, v_pages=v, weight=None, born=None, stamp=None, kv_heads=2)
    for source in (room[1:3, :, :W], room[1:3, 1:3, W:], room[P - 1:P + 1, :, :W], k[:2]):
        for change in (dict(k=source, v=torch.zeros_like(source)), dict(k=torch.zeros_like(source), v=source)):
            assert outcome("append", {**own, **change}) == "meet" and not taken("append", {**own, **change})
    source = room[P:, :, :W]  # behind the pools' pages
    assert outcome("append", {**own, "k": source, "v": room[P:, :, W:]}) == "apart"
    assert taken("append", {**own, "k": source, "v": room[P:, :, W:]})


def test_results_on_other_arguments():
    room = torch.zeros(2 * 2 * 12 + 12)
    weight, beside = room[:48].view(2, 2, 12), room[12:].view(2, 2, 12)
    rows = pools(2, 1, 1024)
    numbers = torch.zeros(64, dtype=I32)
    on_lens = numbers.view(torch.float32)[:48].view(2, 2, 12)
    cases = [
        ("attend", dict(q=rows[..., :256], out=rows[..., 128:384])), ("attend", dict(q=rows[..., :256], out=rows[..., :256])),
        ("attend", dict(weight=weight, lse=room[40:48].view(2, 4, 1))), ("attend", dict(weight=on_lens, lens=numbers[2:4])),
        ("attend", dict(weight=on_lens, table=numbers[:6].view(2, 3))), ("attend", dict(out=ATTEND["v_pages"].view(-1)[512:1024].view(2, 1, 256))),
        ("append", dict(weight=weight, born=beside.view(I32))), ("append", dict(born=weight.view(I32), weight=weight)),
        ("append", dict(at=numbers[:2], after=numbers[1:3])), ("append", dict(table=numbers[:6].view(2, 3), after=numbers[4:6])),
        ("append", dict(stamp=numbers[:10].view(2, 5), after=numbers[8:10])), ("append", dict(weight=on_lens, stamp=numbers[:10].view(2, 5))),
        ("append", dict(weight=WRITE["v_pages"].view(-1).view(torch.float32)[:48].view(2, 2, 12))),
        ("cut", dict(weight=weight, weight_out=beside)), ("cut", dict(weight=weight, born=weight.view(I32), weight_out=weight)),
        ("cut", dict(weight=weight, born_out=weight.view(I32))), ("cut", dict(since=numbers[:2], after=numbers[:2])),
        ("cut", dict(table=numbers[:6].view(2, 3), after=numbers[5:7])), ("cut", dict(keep=numbers[:2], after=numbers[1:3])),
        ("cut", dict(lens=numbers[:2], after=numbers[:2], born_out=numbers[1:49].view(2, 2, 12))),
    ]
    for op, change in cases:
        assert outcome(op, change) == "meet" and not taken(op, change), (op, list(change))
    wide = pools(2, 1, 1024)
    lens = numbers[:2]
    for op, change in [
        ("attend", dict(q=wide[..., :256], out=wide[..., 256:512])), ("attend", dict(weight=weight, lse=room[48:56].view(2, 4, 1))),
        ("cut", dict(weight=weight, weight_out=weight, born_out=EVICT["born"], lens=lens, after=lens)),
        ("cut", dict(lens=lens, after=lens, keep=lens, since=lens)), ("cut", dict(weight=weight, weight_out=room[48:].repeat(4).view(2, 2, 12))),
        ("append", dict(at=numbers[:2], count=numbers[:2], after=numbers[2:4])),
    ]:
        assert outcome(op, change) == "apart" and taken(op, change), (op, list(change))


def bytes_of(t):
    at = torch.arange(t.untyped_storage().nbytes())
    return set(at.as_strided(t.size(), t.stride(), t.storage_offset()).flatten().tolist())


def test_layouts_against_their_bytes():
    """No layout that meets another is let through; what lies apart in steps of two lengths is."""
    r = random.Random(7)
    room = torch.zeros(4000, dtype=torch.uint8)
    met = told = 0
    for _ in range(6000):
        steps = [r.choice([1, 2, 3, 5, 8, 12, 20, 24, 40, 48]) for _ in range(2)]
        both = []
        for _ in range(2):
            own = steps if r.random() < 0.7 else [r.choice([0, 1, 4, 7, 12, 36]) for _ in range(2)]
            shape = (r.randrange(1, 5), r.randrange(1, 7), r.randrange(1, 10))
            both.append(room.as_strided(shape, (*own, 1), r.randrange(0, 120)))
        a, b = both
        lo = [t.storage_offset() for t in both]
        hi = [x + sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1 for x, t in zip(lo, both)]
        if lo[0] >= hi[1] or lo[1] >= hi[0]:
            continue
        meet = bool(bytes_of(a) & bytes_of(b))
        said = paged_ops._meet(a, b)
        met += meet
        assert said or not meet
        if len(paged_ops._steps(a)[1].keys() | paged_ops._steps(b)[1].keys()) <= 2:
            assert said == meet
            told += not meet
    assert met > 1000 and told > 200


def test_both_sides_tell_alike():
    """Results and operands moved over one another in one storage: what the native side takes the Python side does not
    refuse, and of these plain layouts it takes all that the Python side does."""
    r = random.Random(8)
    room = pools(40000)
    count = {"apart": 0, "meet": 0}
    for _ in range(1500):
        row = r.choice([W, W + 8, 2 * W, 3 * W])
        img = row * PAGE + r.choice([0, 0, 8, row, 2 * W])
        views = [room.as_strided((P, PAGE, W), (img, row, 1), r.choice([0, 8, W, 2 * W, row, img, r.randrange(0, 9000) // 8 * 8]))
                 for _ in range(2)]
        source = room.as_strided((2, 5, W), (r.choice([5 * row, img, 9 * row]), row, 1), r.randrange(0, 30000) // 8 * 8)
        change = dict(k_pages=views[0], v_pages=views[1], k=source)
        said = outcome("append", change)
        count[said] += 1
        assert taken("append", change) == (said == "apart")
    assert min(count.values()) > 150, count
