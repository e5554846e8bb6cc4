"""GPU: the softmax of `paged_attention` over scores that leap from tile to
tile, against plain float64 evaluations.

The kernels take weights against a reference that they move late: by the
running maximum once it is exceeded by 2^8 (few rows; d = 64), or raised by a
power of two when a tile's weights passed 2^16 and by the true maximum when
they passed 2^64 (d = 128, many rows).  Every such path is reached here: rows
of all kinds lie side by side in one warp, so that a step takes several of
them at once.

Bars: as in test_gpu_paged.py, a weight is off by 2^-15 of itself (two bf16
terms) or 2^-8 more (one term), the result is rounded by 2^-8 of its value; and
the exponents reach 256 here, see `leaping_scores`.
"""

import math

import pytest
import torch

from test_gpu_paged import History, attention_reference, no_device_error

pytestmark = pytest.mark.gpu

# The exponent (base 2) of all keys of tile 0, 1, ... of 128 positions.
PROFILES = [
    [0] * 12,
    [0, 30, 30, 30, 30, 30, 30, 30, 30, 30, 30, 30],            # passes 2^16 once
    [0, 0, 130, 130, 130, 130, 130, 130, 130, 130, 130, 130],   # passes 2^64 once
    [0, 22, 44, 66, 88, 110, 132, 154, 176, 198, 220, 242],     # 2^16 in every tile
    [0, 120, 0, 0, 120, 121, 0, 0, 0, 120, 0, 121],             # up and down again
    [0, 126, 252, 252, 252, 252, 252, 252, 252, 252, 252, 252],
    [0, -30, -60, -90, -120, -150, -180, -210, -240, -240, -240, -240],
    [0, 60, 60, 190, 190, 220, 250, 250, 250, 250, 250, 250],   # both kinds of leap
    [-250, -250, -130, -100, -70, 30, 40, 170, 200, 200, 201, 250],
    [0, 17, 16, 33, 34, 50, 67, 83, 100, 203, 219, 236],        # at the limits
]


def leaping_scores(h, q_heads, scale, g):
    """Queries that pick a profile each (row % len), keys whose first columns
    hold the profiles' exponents, and unit noise in the others.

    All of it is in bf16: the exponents are integers up to 256, so q . k is
    off by the float32 accumulation alone, at most 8 * 2^-24 of 300 (exponent
    and noise); the product with the scale and the shift by the reference by
    3 * 2^-24 of it.  A weight, and the sum that divides it, is off by ln 2 times
    that: 2 * 11 * 2^-24 * 300 * ln 2 < 2^-11.9."""
    hkv, d = h.k.shape[1], h.k.shape[3]
    count = len(PROFILES)
    device = h.k.device
    table = torch.tensor(PROFILES, device=device, dtype=torch.float32)
    for s, length in enumerate(h.length):
        at = torch.arange(length, device=device)
        page, slot = h.where(s, at)
        column = table[:, (at // 128).clamp(max=11)].T.to(torch.bfloat16)
        for head in range(hkv):
            h.k[page, head, slot, :count] = column
    q = torch.randn(h.n, q_heads, d, generator=g).to(device) * 0.3 / scale / d ** 0.5
    q[..., :count] = 0
    row = torch.arange(h.n * q_heads, device=device).view(h.n, q_heads)
    # with a scale of ln 2 the exponents are those of 2
    q.scatter_(2, (row % count)[..., None], 1.0)
    return q.to(torch.bfloat16)


SCALE = float(torch.tensor(math.log(2.0), dtype=torch.float32))


def check(h, q, got, context, one_term):
    want, size = attention_reference(h, q, context, SCALE)
    weight = 2.0 ** -15 + 2.0 ** -11.9 + (2.0 ** -8 if one_term else 0.0)
    bound = (2.0 ** -8 * want.abs() + weight * size) * 1.001 + 1e-38
    worst = ((got.double() - want).abs() / bound).max().item()
    assert worst <= 1.0, worst


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new,past,hq,hkv,context", [
    ([200], [1100], 2, 2, 0),           # few items: every one cut and joined
    ([200], [1100], 2, 2, 300),         # rows that start late
    ([256], [1000], 150, 150, 0),       # as many items as workers: long pieces
    ([70, 256], [1300, 700], 160, 40, 400),
    ([3], [1400], 4, 2, 0),             # few rows
    ([7] * 30, [40 * i for i in range(30)], 20, 20, 0),
])
def test_leaping_scores(moss, cuda_device, d, new, past, hq, hkv, context):
    g = torch.Generator().manual_seed(d + len(new))
    h = History(new, past, hkv, d, 32, cuda_device, seed=hq)
    q = leaping_scores(h, hq, SCALE, g)
    got = moss.paged_attention(q, h.k, h.v, *h.index, scale=SCALE, context=context or None)
    no_device_error()
    check(h, q, got, context, max(new) * (hq // hkv) > 16)
    again = moss.paged_attention(q, h.k, h.v, *h.index, scale=SCALE, context=context or None)
    assert torch.equal(again, got)


def cancelling(h, hq, g):
    """Queries and values whose results are zero but for rounding: the earlier
    keys' values, taken by their weights, cancel, and the new tokens' keys score
    50 below all others, so that every row of a sequence has the same weights.
    What is left of a result is the error of the weights."""
    hkv, d = h.k.shape[1], h.k.shape[3]
    q = torch.zeros(h.n, hq, d, device=h.k.device, dtype=torch.bfloat16)
    for s, t in enumerate(h.new):
        u = torch.randn(hkv, d, generator=g).to(h.k.device, torch.bfloat16)
        q[h.start[s]:h.start[s] + t] = u.repeat_interleave(hq // hkv, 0)
        page, slot = h.where(s, torch.arange(h.past[s], h.length[s], device=h.k.device))
        h.k[page, :, slot] = (-60 * d ** 0.5 / u.float().pow(2).sum(-1, keepdim=True) * u).to(
            torch.bfloat16)
        k, v = h.dense(s)
        weight = torch.softmax(torch.einsum("hd,hkd->hk", u.double(), k) * d ** -0.5, -1)
        mean = torch.einsum("hk,hkd->hd", weight, v)
        page, slot = h.where(s, torch.arange(h.past[s], device=h.k.device))
        h.v[page, :, slot] = (h.v[page, :, slot].double() - mean).to(torch.bfloat16)
    return q


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [[1], [8], [9], [16], [17], [25], [32], [33],
                                 [32, 1, 17, 8], [1, 200, 9, 32, 16, 33, 2]])
def test_weights_in_two_terms(moss, cuda_device, new, d):
    """The weights of a sequence of up to 32 rows per key head are good to 2^-16,
    alone as beside others, longer ones among them; beyond, to 2^-8."""
    hkv = 3
    g = torch.Generator().manual_seed(d)
    h = History(new, [90 + 11 * i for i in range(len(new))], hkv, d, 16, cuda_device, seed=d)
    q = cancelling(h, hkv, g)
    want, size = attention_reference(h, q, 0, d ** -0.5)
    for hint in (None, max(new)):
        got = moss.paged_attention(q, h.k, h.v, *h.index, max_tokens=hint)
        no_device_error()
        for s, t in enumerate(new):
            rows = slice(h.start[s], h.start[s] + t)
            weight = 2.0 ** -15 + (2.0 ** -8 if t > 32 else 0.0)
            bound = (2.0 ** -8 * want[rows].abs() + weight * size[rows]) * 1.001
            worst = ((got[rows].double() - want[rows]).abs() / bound).max().item()
            assert worst <= 1.0, (t, worst)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("t,length", [(3, 1), (8, 5), (32, 31), (60, 50)])
def test_rows_without_a_position_beside_values_that_are_not_finite(moss, cuda_device, t, length,
                                                                   bad, d):
    """A sequence with more new tokens than positions: its first rows are zero
    whatever the others attend to, in whole pieces and in joined ones."""
    h = History([t] * 3, [0] * 3, 7, d, 16, cuda_device)
    h.kv_len.fill_(length)
    h.v.fill_(bad)
    q = torch.randn(h.n, 7, d, device=cuda_device, dtype=torch.bfloat16)
    for hint in (None, t):
        got = moss.paged_attention(q, h.k, h.v, *h.index, max_tokens=hint).view(3, t, 7, d)
        assert torch.equal(got[:, :t - length], torch.zeros_like(got[:, :t - length]))
        assert not torch.isfinite(got[:, t - length:].float()).any()
    no_device_error()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [[3, 2], [20, 16], [40, 20], [300, 129]])
def test_masked_places_have_no_effect(moss, cuda_device, new, d):
    """Infinities, NaN and the type's extremes in keys and values that no row of
    a sequence attends to, for both widths of head and all forms of the kernels."""
    past, context = [400, 190], 150
    outs = []
    for poison in (0.0, float("nan"), float("inf"), -float("inf"), torch.finfo(torch.bfloat16).min):
        h = History(new, past, 3, d, 32, cuda_device, seed=3, poison=poison)
        for s in range(2):  # positions before every row's window
            page, slot = h.where(s, torch.arange(0, past[s] - context + 1, device=cuda_device))
            h.k[page, :, slot] = poison
            h.v[page, :, slot] = poison
        g = torch.Generator().manual_seed(4)
        q = torch.randn(h.n, 6, d, generator=g).to(cuda_device, torch.bfloat16)
        outs.append(moss.paged_attention(q, h.k, h.v, *h.index, context=context))
    no_device_error()
    assert torch.isfinite(outs[0].float()).all()
    assert all(torch.equal(o, outs[0]) for o in outs)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("leap", [15, 17, 40, 63, 65, 90, 101])
@pytest.mark.parametrize("new", [[5], [200]])
def test_leaps_over_large_values(moss, cuda_device, new, leap, d):
    """Values of 2^40 and a leap of the scores in one tile, of any size: the sums
    that hold both stay finite, as the results are."""
    g = torch.Generator().manual_seed(leap)
    h = History(new, [700], 2, d, 32, cuda_device, seed=leap)
    q = torch.zeros(h.n, 2, d, device=cuda_device)
    q[..., 0] = 1
    q[..., 1:] = 0.3 / SCALE / d ** 0.5 * torch.randn(h.n, 2, d - 1, generator=g).to(cuda_device)
    q = q.to(torch.bfloat16)
    at = torch.arange(h.length[0], device=cuda_device)
    page, slot = h.where(0, at)
    h.k[page, :, slot, 0] = torch.where(at < 400, 0.0, float(leap)).to(torch.bfloat16)[:, None]
    h.v.mul_(2.0 ** 40)
    got = moss.paged_attention(q, h.k, h.v, *h.index, scale=SCALE)
    no_device_error()
    check(h, q, got, 0, new[0] > 16)
