"""CPU: the paged history's geometry -- which keys a block of query rows
reads, how a ragged batch is split over the CTAs -- and the refusals of its
entry points, before any of it touches a GPU."""

import ctypes
import random

import pytest
import torch

from fast_moss_b200 import _lib


def plan(q_start, kv_len, n, *, group=1, hkv=1, page=16, columns=8, context=0, rows=16, tile=64,
         setup=0, ctas=7):
    """[(cta, s, h, block, tile, tiles, lo, hi, begins, ends)] of the split."""
    most = 200000
    out = (ctypes.c_int64 * (9 * most))()
    count = _lib.load().moss_paged_attention_plan(
        _lib.strides(q_start), _lib.strides(kv_len), n, len(kv_len), group, hkv, page, columns,
        context, rows, tile, setup, ctas, out, most)
    assert 0 <= count <= most
    return [tuple(out[9 * i:9 * i + 8]) + (bool(out[9 * i + 8] & 1), bool(out[9 * i + 8] & 2))
            for i in range(count)]


def keys_of(t, length, group, context, rows, block):
    """The union of the positions that the block's rows attend to."""
    seen = set()
    for r in range(block * rows, min((block + 1) * rows, t * group)):
        pos = length - t + r // group
        low = 0 if context == 0 else max(0, pos - context + 1)
        seen.update(range(low, pos + 1))
    return seen


@pytest.mark.parametrize("seed", range(24))
def test_the_split_covers_every_key_of_every_block_once(seed):
    rng = random.Random(seed)
    group, hkv = rng.choice([1, 2, 3, 8]), rng.choice([1, 2, 5])
    rows, tile = rng.choice([(16, 64), (256, 128)])
    context = rng.choice([0, 0, 1, 7, 64, 100])
    ctas, setup = rng.choice([1, 2, 7, 148, 444]), seed % 4
    new = [rng.choice([0, 1, 1, 4, rng.randint(0, 90)]) for _ in range(rng.randint(1, 12))]
    past = [rng.choice([0, 1, 15, 16, 63, 64, 65, rng.randint(0, 900)]) for _ in new]
    length = [a + b for a, b in zip(new, past)]
    q_start = [0]
    for t in new:
        q_start.append(q_start[-1] + t)
    pieces = plan(q_start, length, q_start[-1], group=group, hkv=hkv, columns=70, context=context,
                  rows=rows, tile=tile, setup=setup, ctas=ctas)
    items = {}
    for p in pieces:
        items.setdefault(p[1:4], []).append(p)
    expected = {(s, h, b) for s, t in enumerate(new) for h in range(hkv)
                for b in range(-(-t * group // rows))}
    assert set(items) == expected
    total = sum(p[5] for p in pieces) + setup * len(expected)
    share = max(-(-total // ctas), 1 + setup)
    taken = {}
    for (s, h, b), parts in items.items():
        seen = keys_of(new[s], length[s], group, context, rows, b)
        lo, hi = parts[0][6:8]
        assert (lo, hi) == (min(seen), max(seen) + 1)
        tiles = -(-hi // tile) - lo // tile
        at = 0
        for k, p in enumerate(parts):  # in CTA order, one after the other, no gap
            assert p[4] == at and p[8] == (k == 0) and p[9] == (k == len(parts) - 1)
            if k:
                assert p[0] == parts[k - 1][0] + 1
            at += p[5]
        assert at == tiles
        for p in parts:
            taken[p[0]] = taken.get(p[0], 0) + p[5]
    assert all(v <= share for v in taken.values())
    # at most one cut piece of either kind per CTA: each has one slot
    for kind in (True, False):
        cut = [p[0] for p in pieces if p[8] == kind and not (p[8] and p[9])]
        assert len(cut) == len(set(cut))


def test_arrays_that_lie_stay_inside_the_buffers():
    """Decreasing or too large row numbers, negative and too large lengths:
    the clamped geometry never leaves the packed rows or the table."""
    n, columns, page = 20, 3, 16
    rng = random.Random(1)
    for _ in range(200):
        s = rng.randint(1, 5)
        q_start = [rng.choice([-5, 0, 3, 19, 20, 21, 2 ** 40, -2 ** 40, rng.randint(0, 20)])
                   for _ in range(s + 1)]
        kv_len = [rng.choice([-1, 0, 1, 47, 48, 49, 2 ** 31, 2 ** 40, -2 ** 62]) for _ in range(s)]
        for p in plan(q_start, kv_len, n, columns=columns, page=page, rows=16, tile=64, ctas=3):
            assert 0 <= p[6] <= p[7] <= columns * page
            row0 = min(max(q_start[p[1]], 0), n)
            row1 = min(max(q_start[p[1] + 1], row0), n)
            assert p[3] * 16 < row1 - row0  # the block has rows


def test_rows_without_positions_still_get_a_piece():
    """More new tokens than positions: the rows before position 0 attend to
    nothing, and their block is still visited (its rows are written)."""
    (p,) = plan([0, 5], [0], 5, ctas=4)
    assert p[5] == 1 and p[6] == p[7] == 0 and p[8] and p[9]


def test_plan_rejects_bad_arguments():
    z = _lib.strides([0, 0])
    lib = _lib.load()
    assert lib.moss_paged_attention_plan(None, z, 1, 1, 1, 1, 16, 1, 0, 16, 64, 0, 1, z, 0) == -1
    assert lib.moss_paged_attention_plan(z, z, 1, 1, 1, 1, 24, 1, 0, 16, 64, 0, 1, z, 0) == -1
    assert lib.moss_paged_attention_plan(z, z, 1, 1, 0, 1, 16, 1, 0, 16, 64, 0, 1, z, 0) == -1
    assert lib.moss_paged_attention_plan(z, z, 1, 1, 1, 1, 16, 1, 0, 24, 64, 0, 1, z, 0) == -1
    assert lib.moss_paged_attention_plan(z, z, 1, 1, 1, 1, 16, 1, 0, 16, 64, -1, 1, z, 0) == -1


P = ctypes.c_void_p(4096)  # a pointer that is never followed


def _attention(**kw):
    a = dict(q=P, k=P, v=P, qs=P, kl=P, pt=P, n=4, s=1, hq=4, hkv=2, d=64, pages=2, page=16,
             columns=2, most=0, context=0, scale=0.125, ws=P, size=1 << 40, out=P)
    a.update(kw)
    return _lib.load().moss_paged_attention(
        a["q"], a["k"], a["v"], a["qs"], a["kl"], a["pt"], a["n"], a["s"], a["hq"], a["hkv"],
        a["d"], a["pages"], a["page"], a["columns"], a["most"], a["context"], a["scale"], a["ws"],
        a["size"], a["out"], None)


@pytest.mark.parametrize("kw,status", [
    (dict(n=-1), _lib.ERR_VALUE), (dict(hkv=3), _lib.ERR_VALUE), (dict(hkv=0), _lib.ERR_VALUE),
    (dict(context=-1), _lib.ERR_VALUE), (dict(scale=0.0), _lib.ERR_VALUE),
    (dict(scale=float("nan")), _lib.ERR_VALUE), (dict(scale=float("inf")), _lib.ERR_VALUE),
    (dict(d=96), _lib.ERR_UNSUPPORTED), (dict(page=24), _lib.ERR_UNSUPPORTED),
    (dict(page=8), _lib.ERR_UNSUPPORTED), (dict(page=512), _lib.ERR_UNSUPPORTED),
    (dict(q=None), _lib.ERR_VALUE), (dict(ws=None), _lib.ERR_VALUE), (dict(size=0), _lib.ERR_VALUE),
    (dict(columns=1 << 28), _lib.ERR_UNSUPPORTED), (dict(n=1 << 30), _lib.ERR_UNSUPPORTED),
    (dict(out=ctypes.c_void_p(4104)), _lib.ERR_VALUE),
    (dict(n=0), _lib.OK), (dict(s=0), _lib.OK),
])
def test_attention_refusals(kw, status):
    assert _attention(**kw) == status


def _append(**kw):
    a = dict(q=P, k=P, v=P, dtype=1, qw=None, kw=None, eps=1e-6, qs=P, kl=P, pt=P, period=1e4,
             pairs=1, oq=P, kp=P, vp=P, n=4, s=1, hq=4, hkv=2, d=64, pages=2, page=16, columns=2,
             st=[256, 64, 1])
    a.update(kw)
    st = _lib.strides(a["st"])
    return _lib.load().moss_rope_paged_kv(
        a["q"], a["k"], a["v"], a["dtype"], a["qw"], a["kw"], a["eps"], a["qs"], a["kl"], a["pt"],
        a["period"], a["pairs"], a["oq"], a["kp"], a["vp"], a["n"], a["s"], a["hq"], a["hkv"],
        a["d"], a["pages"], a["page"], a["columns"], st, st, st, None)


@pytest.mark.parametrize("kw,status", [
    (dict(n=-1), _lib.ERR_VALUE), (dict(dtype=2), _lib.ERR_VALUE), (dict(period=0.0), _lib.ERR_VALUE),
    (dict(period=float("inf")), _lib.ERR_VALUE), (dict(eps=-1.0), _lib.ERR_VALUE),
    (dict(d=32), _lib.ERR_UNSUPPORTED), (dict(page=20), _lib.ERR_UNSUPPORTED),
    (dict(k=None), _lib.ERR_VALUE), (dict(st=[256, 64, 2]), _lib.ERR_UNSUPPORTED),
    (dict(st=[256, 60, 1]), _lib.ERR_UNSUPPORTED), (dict(q=ctypes.c_void_p(4104)), _lib.ERR_UNSUPPORTED),
    (dict(qw=ctypes.c_void_p(4104)), _lib.ERR_UNSUPPORTED), (dict(n=0), _lib.OK), (dict(s=0), _lib.OK),
])
def test_append_refusals(kw, status):
    assert _append(**kw) == status


def _norm(**kw):
    a = dict(q=P, k=P, dtype=1, qw=None, kw=None, eps=1e-6, off=P, odt=0, period=1e4, oq=P, ok=P,
             b=1, hq=2, hk=2, t=3, d=64, st=[384, 192, 64, 1])
    a.update(kw)
    st = _lib.strides(a["st"])
    return _lib.load().moss_qk_norm_rope(
        a["q"], a["k"], a["dtype"], a["qw"], a["kw"], a["eps"], a["off"], a["odt"], a["period"], 1,
        a["oq"], a["ok"], a["b"], a["hq"], a["hk"], a["t"], a["d"], st, st, None)


@pytest.mark.parametrize("kw,status", [
    (dict(b=-1), _lib.ERR_VALUE), (dict(hk=0), _lib.ERR_VALUE), (dict(d=63), _lib.ERR_VALUE),
    (dict(dtype=5), _lib.ERR_VALUE), (dict(odt=2), _lib.ERR_VALUE), (dict(period=-1.0), _lib.ERR_VALUE),
    (dict(eps=float("nan")), _lib.ERR_VALUE), (dict(d=96), _lib.ERR_UNSUPPORTED),
    (dict(off=None), _lib.ERR_VALUE), (dict(st=[384, 192, 64, 2]), _lib.ERR_UNSUPPORTED),
    (dict(st=[384, 192, 63, 1]), _lib.ERR_UNSUPPORTED), (dict(b=0), _lib.OK), (dict(t=0), _lib.OK),
])
def test_norm_refusals(kw, status):
    assert _norm(**kw) == status


def test_wrappers_refuse_tensors_that_are_not_on_a_gpu():
    import fast_moss_b200 as fm

    q, k = torch.zeros(1, 2, 3, 64), torch.zeros(1, 1, 3, 64)
    with pytest.raises(ValueError):
        fm.qk_norm_rope(q, k, None, None, torch.zeros(1, dtype=torch.int64), 1e4)
    with pytest.raises(ValueError):
        fm.qk_norm_rope(q, torch.zeros(1, 1, 2, 64), None, None, torch.zeros(1, dtype=torch.int64), 1e4)
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    pages = torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16)
    index = (torch.tensor([0, 3]), torch.tensor([3]), torch.zeros(1, 1, dtype=torch.int32))
    with pytest.raises(ValueError):
        fm.paged_attention(x, pages, pages, *index)
    with pytest.raises(ValueError):
        fm.rope_paged_kv(x, x[:, :1], x[:, :1], *index, 1e4, pages, pages)


@pytest.mark.parametrize("rows,tile", [(16, 64), (256, 128)])
def test_rows_that_are_there_keep_their_positions(rows, tile):
    """A sequence with more rows than were packed: row r is position kv_len -
    (q_start[s + 1] - r) all the same, where rope_paged_kv put it."""
    (p,) = plan([0, 10], [100], 6, rows=rows, tile=tile, ctas=1)
    assert p[6:8] == (0, 96)  # the last row that is there, 5, is position 95
    (p,) = plan([0, 10], [100], 6, rows=rows, tile=tile, ctas=1, context=20)
    assert p[6:8] == (71, 96)
    (p,) = plan([0, 10], [3], 6, rows=rows, tile=tile, ctas=1)  # all before position 0
    assert p[6:8] == (0, 0)
    first, = plan([0, 6, 10], [50, 60], 6, rows=rows, tile=tile, ctas=1)
    assert first[6:8] == (0, 50)
    (p,) = plan([0, 2 ** 63 - 1], [2 ** 63 - 1], 6, rows=rows, tile=tile, ctas=1)
    assert 0 <= p[6] <= p[7] <= 128


@pytest.mark.parametrize("seed", range(12))
@pytest.mark.parametrize("rows,tile,setup,least", [(8, 16, 2, 4), (16, 16, 2, 4), (256, 128, 3, 4)])
def test_the_split_of_the_kernels_own_shapes(rows, tile, setup, least, seed):
    """Blocks, tiles, set-up and least share as the three forms of the kernels
    have them: every key of every block once, shares that are even."""
    rng = random.Random(seed)
    group, hkv = rng.choice([1, 2, 5]), rng.choice([1, 3])
    context = rng.choice([0, 0, 30, 200])
    ctas = rng.choice([3, 148, 148 * 12])
    most = 32 // group if rows < 256 else 700
    new = [rng.choice([0, 1, 1, 4, rng.randint(0, most)]) for _ in range(rng.randint(1, 9))]
    past = [rng.choice([0, 1, 15, 16, 17, 255, 256, rng.randint(0, 3000)]) for _ in new]
    length = [a + b for a, b in zip(new, past)]
    q_start = [sum(new[:i]) for i in range(len(new) + 1)]
    pieces = plan(q_start, length, q_start[-1], group=group, hkv=hkv, columns=400, context=context,
                  rows=rows, tile=tile, setup=setup, ctas=ctas)
    items = {}
    for p in pieces:
        items.setdefault(p[1:4], []).append(p)
    total = sum(p[5] for p in pieces) + setup * len(items)
    share = max(-(-total // ctas), least)
    assert set(items) == {(s, h, b) for s, t in enumerate(new) for h in range(hkv)
                          for b in range(-(-t * group // rows))}
    at = 0  # tiles before the item, its set-up among them
    for s, h, b in sorted(items):
        seen = keys_of(new[s], length[s], group, context, rows, b)
        tiles = -(-(max(seen) + 1) // tile) - min(seen) // tile
        expected, k = [], at
        while k < at + setup + tiles:
            end = min((k // share + 1) * share, at + setup + tiles)
            first, last = max(k - at - setup, 0), end - at - setup
            if last > first:
                expected.append((k // share, first, last - first))
            k = end
        assert [(p[0], p[4], p[5]) for p in items[s, h, b]] == expected
        at += setup + tiles


def test_plan_refuses_what_the_attention_refuses():
    """Sizes beyond the kernels' index arithmetic."""
    lib = _lib.load()
    z = _lib.strides([0, 0])

    def ask(n=1, s=1, group=1, hkv=1, page=16, columns=1, rows=16, tile=64, setup=0, ctas=1):
        return lib.moss_paged_attention_plan(z, z, n, s, group, hkv, page, columns, 0, rows, tile,
                                             setup, ctas, z, 0)

    assert ask(s=0) == 0
    for kw in (dict(n=1 << 30), dict(n=1 << 20, group=1 << 11), dict(s=1 << 30), dict(hkv=1 << 21),
               dict(columns=1 << 28), dict(columns=-1), dict(rows=1 << 31), dict(tile=1 << 31),
               dict(setup=1 << 31), dict(ctas=1 << 31)):
        assert ask(**kw) == -1, kw


@pytest.mark.parametrize("limit", [0, 999, 100_000_001, -5])
def test_wait_limits_out_of_range_are_refused(limit):
    assert _lib.load().moss_test_paged_wait(limit, 1, None) == _lib.ERR_VALUE
