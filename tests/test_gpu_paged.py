"""GPU: the paged key/value history -- per-head norm + rotary embedding, page
writes, attention over the pages -- against plain float64 evaluations.

Bars (half a rounding step is 2^-8 of the value for bf16):
  norm + rotary  a pair (a, b) of magnitude r: the norm's sum (up to 20
      additions in sequence), reciprocal root and products are off by at most
      17 * 2^-24 of r, the reduced angle and its sine and cosine by 6 * 2^-24,
      the rotation's products and sum by 3 * 2^-24: below 2^-19 r in float32,
      and 2^-8 of the value for a bf16 result on top.
  attention  A = sum p |v|: a score is off by some 100 * 2^-24 (its terms sum
      to about 10 before the base-2 scale), an exponential by 2^-22, a weight
      held in two bf16 terms by 2^-16: below 2^-15 A; where more than 16 query
      rows share a key head the weights may be held in one bf16 term, 2^-8 A
      more; and 2^-8 of the value for the result.
"""

import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

PERIOD = 10000.0
EPS = 1e-6


# ------------------------------------------------------------ plain evaluation
def rotated(x, weight, position, interleaved, period=PERIOD):
    """Norm and rotation in float64; position broadcasts against x[..., 0].
    Returns the result and every value's pair magnitude."""
    x = x.double()
    d = x.shape[-1]
    if weight is not None:
        x = x * (x.pow(2).mean(-1, keepdim=True) + EPS).rsqrt() * weight.double()
    j = torch.arange(d // 2, device=x.device, dtype=torch.float64)
    angle = position.double()[..., None] * period ** (-2 * j / d)
    c, s = angle.cos(), angle.sin()
    out, size = torch.empty_like(x), torch.empty_like(x)
    first = slice(0, None, 2) if interleaved else slice(0, d // 2)
    second = slice(1, None, 2) if interleaved else slice(d // 2, None)
    a, b = x[..., first], x[..., second]
    out[..., first], out[..., second] = a * c - b * s, a * s + b * c
    size[..., first] = size[..., second] = torch.hypot(a, b)
    return out, size


def check_rotated(got, want, size):
    step = 2.0 ** -8 if got.dtype == torch.bfloat16 else 0.0
    bound = (step * want.abs() + 2.0 ** -19 * size) * 1.0001 + 1e-38
    worst = ((got.double() - want).abs() / bound).max().item()
    assert worst <= 1.0, worst


class History:
    """A paged history of sequences with `new` tokens on top of `past`."""

    def __init__(self, new, past, hkv, d, page, device, seed=0, spare=3, columns=0, poison=None):
        g = torch.Generator().manual_seed(seed)
        self.new, self.past, self.page, self.device = new, past, page, device
        self.length = [a + b for a, b in zip(new, past)]
        need = [-(-n // page) for n in self.length]
        width = max(max(need), columns, 1)
        pages = sum(need) + spare
        order = torch.randperm(pages, generator=g).to(torch.int32)
        table = torch.full((len(new), width), -1, dtype=torch.int32)
        at = 0
        for s, c in enumerate(need):
            table[s, :c] = order[at:at + c]
            at += c
        self.table = table.to(device)
        start = [0]
        for t in new:
            start.append(start[-1] + t)
        self.start = start
        self.n = start[-1]
        self.q_start = torch.tensor(start, device=device)
        self.kv_len = torch.tensor(self.length, device=device)
        shape = (pages, hkv, page, d)
        self.k = torch.randn(shape, generator=g).to(device, torch.bfloat16)
        self.v = torch.randn(shape, generator=g).to(device, torch.bfloat16)
        if poison is not None:  # everything that no position uses
            used = torch.zeros(pages, page, dtype=torch.bool)
            for s, n in enumerate(self.length):
                p = torch.arange(n)
                used[table[s].long()[p // page], p % page] = True
            free = ~used.to(device)[:, None, :, None].expand(shape)
            self.k[free] = poison
            self.v[free] = poison
        self.index = (self.q_start, self.kv_len, self.table)

    def where(self, s, position):
        return self.table[s].long()[position // self.page], position % self.page

    def dense(self, s):
        """k, v [hkv, length, d] of a sequence in float64."""
        page, slot = self.where(s, torch.arange(self.length[s], device=self.device))
        return (self.k[page, :, slot].double().transpose(0, 1),
                self.v[page, :, slot].double().transpose(0, 1))


def attention_reference(h, q, context, scale):
    """[n, hq, d] outputs and sum p |v| in float64."""
    n, hq, d = q.shape
    out = torch.zeros(q.shape, device=q.device, dtype=torch.float64)
    size = torch.zeros_like(out)
    for s, t in enumerate(h.new):
        if t == 0 or h.length[s] == 0:
            continue
        k, v = h.dense(s)
        group = hq // k.shape[0]
        rows = slice(h.start[s], h.start[s] + t)
        qs = q[rows].double().transpose(0, 1)
        score = torch.einsum("htd,hkd->htk", qs, k.repeat_interleave(group, 0)) * scale
        at = torch.arange(h.length[s], device=q.device)
        pos = torch.arange(h.past[s], h.length[s], device=q.device)[:, None]
        seen = at <= pos
        if context:
            seen &= at > pos - context
        weight = torch.softmax(score.masked_fill(~seen, -math.inf), -1)
        vv = v.repeat_interleave(group, 0)
        out[rows] = torch.einsum("htk,hkd->htd", weight, vv).transpose(0, 1)
        size[rows] = torch.einsum("htk,hkd->htd", weight, vv.abs()).transpose(0, 1)
    return out, size


def check_attention(got, want, size, most_rows):
    weight = 2.0 ** -15 + (2.0 ** -8 if most_rows > 16 else 0.0)
    bound = (2.0 ** -8 * want.abs() + weight * size) * 1.001 + 1e-38
    worst = ((got.double() - want).abs() / bound).max().item()
    assert worst <= 1.0, worst


def no_device_error():
    from fast_moss_b200 import _lib

    _lib.check(_lib.load().moss_check_device_error(torch.cuda.current_stream().cuda_stream), "check")


def take_device_error():
    from fast_moss_b200 import _lib

    return _lib.load().moss_check_device_error(torch.cuda.current_stream().cuda_stream)


# --------------------------------------------------------------- qk_norm_rope
@pytest.mark.parametrize("b,hq,hk,t,d,dtype,interleaved,normed", [
    (1, 1, 1, 1, 64, torch.bfloat16, True, True),
    (64, 20, 20, 4, 64, torch.bfloat16, True, True),
    (3, 5, 2, 7, 128, torch.float32, False, True),
    (2, 8, 1, 333, 128, torch.bfloat16, False, True),
    (2, 3, 3, 17, 32, torch.float32, True, True),
    (1, 4, 2, 65, 256, torch.bfloat16, True, True),
    (1, 2, 2, 40, 256, torch.float32, False, False),
    (2, 4, 4, 1201, 64, torch.float32, True, False),
    (1, 40, 8, 2500, 64, torch.bfloat16, False, True),
])
def test_qk_norm_rope(moss, cuda_device, b, hq, hk, t, d, dtype, interleaved, normed):
    g = torch.Generator().manual_seed(b * 1000 + t)
    # views of one projection's output, [b, t, heads, d]
    qkv = torch.randn(b, t, hq + 2 * hk, d, generator=g).to(cuda_device, dtype)
    q, k = qkv[:, :, :hq].transpose(1, 2), qkv[:, :, hq:hq + hk].transpose(1, 2)
    qw = (1 + 0.3 * torch.randn(d, generator=g)).to(cuda_device) if normed else None
    kw = (1 + 0.3 * torch.randn(d, generator=g)).to(cuda_device) if normed else None
    offset = torch.tensor([(7919 * i * i) % 5000000 for i in range(b)], device=cuda_device)
    oq, ok = moss.qk_norm_rope(q, k, qw, kw, offset, PERIOD, interleaved=interleaved)
    assert oq.shape == q.shape and ok.shape == k.shape and oq.dtype == dtype
    assert oq.is_contiguous() and ok.is_contiguous()
    position = (offset[:, None] + torch.arange(t, device=cuda_device))[:, None]
    check_rotated(oq, *rotated(q, qw, position, interleaved))
    check_rotated(ok, *rotated(k, kw, position, interleaved))


def test_qk_norm_rope_one_weight_strides_and_offsets(moss, cuda_device):
    """Only one of the two normed, int32 and negative offsets, contiguous and
    misaligned inputs, another eps and period."""
    g = torch.Generator().manual_seed(5)
    base = torch.randn(2 * 3 * 9 * 64 + 1, generator=g).to(cuda_device, torch.bfloat16)
    q = base[1:].view(2, 3, 9, 64)          # two bytes off any 16-byte boundary
    k = torch.randn(2, 3, 9, 128, generator=g).to(cuda_device, torch.bfloat16)[..., ::2]
    w = (1 + 0.3 * torch.randn(64, generator=g)).to(cuda_device)
    offset = torch.tensor([-4, 2 ** 31 - 30], device=cuda_device, dtype=torch.int32)
    position = (offset.long()[:, None] + torch.arange(9, device=cuda_device))[:, None]
    for qw, kw in ((w, None), (None, w)):
        oq, ok = moss.qk_norm_rope(q, k, qw, kw, offset, 500.0)
        check_rotated(oq, *rotated(q, qw, position, True, 500.0))
        check_rotated(ok, *rotated(k, kw, position, True, 500.0))
    zero = torch.zeros(2, 3, 9, 64, device=cuda_device, dtype=torch.bfloat16)
    oq, _ = moss.qk_norm_rope(zero, zero, w, w, offset, 500.0, eps=1e-6)
    assert torch.equal(oq, zero)
    empty = zero[:, :, :0]
    oq, ok = moss.qk_norm_rope(empty, empty, w, w, offset, 500.0)
    assert oq.shape == (2, 3, 0, 64)


# -------------------------------------------------------------- rope_paged_kv
@pytest.mark.parametrize("new,past,hq,hkv,d,page,dtype,interleaved,normed", [
    ([1], [0], 1, 1, 64, 16, torch.bfloat16, True, False),
    ([4] * 64, [37 * i for i in range(64)], 20, 20, 64, 16, torch.bfloat16, True, False),
    ([1, 0, 33, 16, 0, 5], [15, 7, 0, 16, 0, 4000000], 8, 2, 128, 32, torch.float32, False, True),
    ([300, 1, 700], [1, 255, 0], 6, 3, 64, 256, torch.bfloat16, False, True),
    ([1] * 40 + [3] * 60 + [0] * 3, [i * 5 for i in range(103)], 4, 1, 128, 64, torch.bfloat16, True, True),
    ([2500, 17], [3, 200], 40, 8, 128, 128, torch.float32, True, False),
])
def test_rope_paged_kv(moss, cuda_device, new, past, hq, hkv, d, page, dtype, interleaved, normed):
    g = torch.Generator().manual_seed(len(new))
    columns = 0
    far = max(past)
    if far > 1000000:  # a far position in a table whose early pages are gone
        small = [p if p < 1000000 else 0 for p in past]
        h = History(new, small, hkv, d, page, cuda_device)
        s = past.index(far)
        first = far // page
        table = torch.full((len(new), first + 2), -1, dtype=torch.int32, device=cuda_device)
        table[:, :h.table.shape[1]] = h.table
        table[s] = -1
        table[s, first] = h.table[s, 0]
        h.table, h.past, h.length = table, past, [a + b for a, b in zip(new, past)]
        h.kv_len = torch.tensor(h.length, device=cuda_device)
        h.index = (h.q_start, h.kv_len, h.table)
    else:
        h = History(new, past, hkv, d, page, cuda_device, columns=columns)
    n = h.n
    qkv = torch.randn(n, hq + 2 * hkv, d, generator=g).to(cuda_device, dtype)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    qw = (1 + 0.3 * torch.randn(d, generator=g)).to(cuda_device) if normed else None
    kw = (1 + 0.3 * torch.randn(d, generator=g)).to(cuda_device) if normed else None
    k_want, v_want = h.k.clone(), h.v.clone()
    k_size = torch.zeros(h.k.shape, device=cuda_device, dtype=torch.float64)
    k_exact = h.k.double()
    oq = moss.rope_paged_kv(q, k, v, *h.index, PERIOD, h.k, h.v, q_weight=qw, k_weight=kw,
                            interleaved=interleaved)
    no_device_error()
    touched = torch.zeros(h.k.shape, dtype=torch.bool, device=cuda_device)
    for s, t in enumerate(new):
        rows = slice(h.start[s], h.start[s] + t)
        position = torch.arange(past[s], past[s] + t, device=cuda_device)
        check = rotated(q[rows], qw, position[:, None], interleaved)
        if t:
            check_rotated(oq[rows], *check)
            where = h.where(s, position)
            k_exact[where[0], :, where[1]], k_size[where[0], :, where[1]] = rotated(
                k[rows], kw, position[:, None], interleaved)
            v_want[where[0], :, where[1]] = v[rows].to(torch.bfloat16)
            touched[where[0], :, where[1]] = True
    assert torch.equal(h.v, v_want)
    assert torch.equal(h.k[~touched], k_want[~touched])
    check_rotated(h.k[touched], k_exact[touched], k_size[touched])


def test_rope_paged_kv_leaves_rows_of_no_sequence(moss, cuda_device):
    """Rows before the first sequence and behind the last write nothing."""
    h = History([3, 2], [5, 20], 2, 64, 16, cuda_device)
    q_start = h.q_start + 2
    k0, v0 = h.k.clone(), h.v.clone()
    x = torch.randn(9, 4, 64, device=cuda_device, dtype=torch.bfloat16)
    kv = torch.randn(9, 2, 64, device=cuda_device, dtype=torch.bfloat16)
    moss.rope_paged_kv(x, kv, kv, q_start, h.kv_len, h.table, PERIOD, h.k, h.v)
    no_device_error()
    for s, (t, p) in enumerate(zip(h.new, h.past)):
        page, slot = h.where(s, torch.arange(p, p + t, device=cuda_device))
        assert torch.equal(h.v[page, :, slot], kv[2 + h.start[s]:2 + h.start[s] + t])
        v0[page, :, slot] = h.v[page, :, slot]
        k0[page, :, slot] = h.k[page, :, slot]
    assert torch.equal(h.v, v0) and torch.equal(h.k, k0)


def test_bad_pages_are_skipped_and_reported(moss, cuda_device):
    """Pages outside the pool and positions outside the table: nothing is
    written there, the error word is set, the other sequences are right."""
    from fast_moss_b200 import _lib

    no_device_error()
    h = History([2, 2, 2, 2], [20, 20, 20, 20], 2, 64, 16, cuda_device)
    h.table[0, 1] = -7
    h.table[1, 1] = h.k.shape[0]
    h.kv_len[2] = 16 * h.table.shape[1] + 2     # past the table's end
    x = torch.randn(8, 4, 64, device=cuda_device, dtype=torch.bfloat16)
    kv = torch.randn(8, 2, 64, device=cuda_device, dtype=torch.bfloat16)
    v0 = h.v.clone()
    moss.rope_paged_kv(x, kv, kv, *h.index, PERIOD, h.k, h.v)
    assert take_device_error() == _lib.ERR_TIMEOUT
    page, slot = h.where(3, torch.arange(20, 22, device=cuda_device))
    assert torch.equal(h.v[page, :, slot], kv[6:8])
    v0[page, :, slot] = kv[6:8]
    assert torch.equal(h.v, v0)
    h.length[2] = 22
    q = torch.randn(8, 4, 64, device=cuda_device, dtype=torch.bfloat16)
    got = moss.paged_attention(q, h.k, h.v, *h.index)
    assert take_device_error() == _lib.ERR_TIMEOUT
    h.table[0, 1] = h.table[1, 1] = 0
    want, size = attention_reference(h, q, 0, 1 / 8)
    check_attention(got[6:8], want[6:8], size[6:8], 16)
    no_device_error()


# ------------------------------------------------------------ paged_attention
CASES = [
    # new, past, hq, hkv, d, page, context
    ([1], [0], 1, 1, 64, 16, 0),
    ([1], [0], 4, 1, 128, 256, 1),
    ([4], [2000], 20, 20, 64, 16, 0),
    ([4] * 64, [47 * i for i in range(64)], 20, 20, 64, 16, 250),
    ([1] * 33, [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257] + [211 * i for i in range(19)],
     32, 8, 128, 64, 0),
    ([1], [20000], 8, 2, 128, 128, 0),
    ([1, 1], [9000, 3], 5, 1, 64, 32, 77),
    ([0, 5, 0, 1, 0], [9, 40, 0, 300, 2000], 6, 2, 64, 16, 0),
    ([7, 3, 16], [0, 100, 513], 2, 2, 128, 16, 20),
    # more rows than one block
    ([40], [0], 4, 4, 64, 16, 0),
    ([129, 1, 257, 64], [0, 700, 31, 500], 6, 2, 128, 32, 0),
    ([300], [1000], 3, 1, 64, 64, 100),
    ([513, 1, 1, 2], [77, 900, 0, 31], 16, 2, 64, 128, 0),
    ([256], [256], 8, 8, 128, 256, 0),
    ([1000], [24], 2, 1, 128, 16, 300),
    ([33, 90], [4000, 10], 20, 20, 64, 16, 0),
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_paged_attention(moss, cuda_device, case):
    new, past, hq, hkv, d, page, context = CASES[case]
    h = History(new, past, hkv, d, page, cuda_device, seed=case, poison=float("nan"))
    g = torch.Generator().manual_seed(100 + case)
    q = torch.randn(h.n, hq, d, generator=g).to(cuda_device, torch.bfloat16)
    got = moss.paged_attention(q, h.k, h.v, *h.index, context=context or None)
    no_device_error()
    assert got.shape == q.shape and got.dtype == torch.bfloat16
    want, size = attention_reference(h, q, context, d ** -0.5)
    most = max(new) * (hq // hkv)
    check_attention(got, want, size, most)
    # a hint of the most tokens chooses between kernels, the bar is the same
    hinted = moss.paged_attention(q, h.k, h.v, *h.index, context=context or None,
                                  max_tokens=max(new))
    check_attention(hinted, want, size, most)
    # the same call twice: the same bits
    assert torch.equal(hinted, moss.paged_attention(q, h.k, h.v, *h.index,
                                                    context=context or None,
                                                    max_tokens=max(new)))


@pytest.mark.parametrize("sequences,d,hint", [
    (32, 64, True), (33, 128, True), (128, 64, True), (129, 128, True), (700, 64, True),
    (40, 64, False), (128, 128, False), (130, 64, False), (700, 128, False),
])
def test_batches_of_many_sequences(moss, cuda_device, sequences, d, hint):
    """However the workers find their runs: single tokens and, without the
    hint, prompts and sequences with nothing to do among them; append and
    attention agree with the reference."""
    rng = random.Random(sequences)
    new = [1] * sequences if hint else [rng.choice([0, 1, 1, 2, 9, 17, 40]) for _ in range(sequences)]
    past = [rng.choice([0, 15, 16, 100, 333]) for _ in new]
    h = History(new, past, 2, d, 16, cuda_device, seed=sequences, poison=float("nan"))
    g = torch.Generator().manual_seed(sequences)
    x = torch.randn(h.n, 8, d, generator=g).to(cuda_device, torch.bfloat16)
    q = moss.rope_paged_kv(x[:, :4], x[:, 4:6], x[:, 6:], *h.index, PERIOD, h.k, h.v)
    got = moss.paged_attention(q, h.k, h.v, *h.index, context=90, max_tokens=1 if hint else None)
    no_device_error()
    position = torch.cat([torch.arange(p, p + t) for t, p in zip(new, past)]).to(cuda_device)
    check_rotated(q, *rotated(x[:, :4], None, position[:, None], True))
    for s in range(0, sequences, 7):
        if new[s]:
            page, slot = h.where(s, torch.arange(past[s], h.length[s], device=cuda_device))
            assert torch.equal(h.v[page, :, slot], x[h.start[s]:h.start[s] + new[s], 6:])
    want, size = attention_reference(h, q, 90, d ** -0.5)
    check_attention(got, want, size, 1 if hint else 80)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [15, 16, 17, 31, 32, 33])
def test_either_side_of_the_choice_of_kernels(moss, cuda_device, rows, d):
    """Sequences of as many query rows as the kernels part at, by themselves
    and beside others."""
    for new, past in (([rows], [70]), ([rows, 1, rows, rows + 30], [70, 3, 0, 200])):
        h = History(new, past, 2, d, 32, cuda_device, seed=rows, poison=float("nan"))
        g = torch.Generator().manual_seed(rows)
        q = torch.randn(h.n, 2, d, generator=g).to(cuda_device, torch.bfloat16)
        want, size = attention_reference(h, q, 0, d ** -0.5)
        for hint in (None, max(new)):
            got = moss.paged_attention(q, h.k, h.v, *h.index, max_tokens=hint)
            check_attention(got, want, size, rows + 30)
        # a hint below the truth: computed all the same
        got = moss.paged_attention(q, h.k, h.v, *h.index, max_tokens=1)
        check_attention(got, want, size, rows + 30)
    no_device_error()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("t", [3, 50])
def test_values_that_are_not_finite_stay_in_their_rows(moss, cuda_device, t, d):
    """A query, or a key that only the last token attends to, with infinities
    or NaN makes that row NaN and no other."""
    for bad in (float("inf"), float("nan")):
        h = History([t, t], [300, 20], 1, d, 16, cuda_device, seed=t)
        g = torch.Generator().manual_seed(t)
        q = torch.randn(h.n, 2, d, generator=g).to(cuda_device, torch.bfloat16)
        want, size = attention_reference(h, q, 0, d ** -0.5)
        q[1, 1] = bad
        page, slot = h.where(1, torch.tensor([20 + t - 1], device=cuda_device))
        h.k[page, :, slot] = float("nan")
        got = moss.paged_attention(q, h.k, h.v, *h.index)
        broken = torch.zeros(h.n, 2, dtype=torch.bool, device=cuda_device)
        broken[1, 1] = broken[2 * t - 1] = True
        assert torch.isnan(got[broken].float()).any(-1).all()
        check_attention(got[~broken], want[~broken], size[~broken], 2 * t)
    no_device_error()


@pytest.mark.parametrize("new", [[3, 2], [40, 20]])
def test_values_in_masked_places_have_no_effect(moss, cuda_device, new):
    """Infinities, NaN and the type's extremes in keys and values that no row
    of a sequence attends to -- freed pages before the window, the rest of
    the last page, unused pages -- change nothing."""
    past, context = [200, 90], 30
    outs = []
    for poison in (0.0, float("nan"), float("inf"), -float("inf"), torch.finfo(torch.bfloat16).min):
        h = History(new, past, 2, 64, 16, cuda_device, seed=3, poison=poison)
        for s in range(2):  # positions before every row's window
            old = torch.arange(0, past[s] - context + 1, device=cuda_device)
            page, slot = h.where(s, old)
            h.k[page, :, slot] = poison
            h.v[page, :, slot] = poison
        g = torch.Generator().manual_seed(4)
        q = torch.randn(h.n, 4, 64, generator=g).to(cuda_device, torch.bfloat16)
        outs.append(moss.paged_attention(q, h.k, h.v, *h.index, context=context))
    # whole pages before the window may be gone from the table
    for s in range(2):
        h.table[s, :(past[s] - context + 1) // 16] = -1
    outs.append(moss.paged_attention(q, h.k, h.v, *h.index, context=context))
    no_device_error()
    assert torch.isfinite(outs[0].float()).all()
    assert all(torch.equal(o, outs[0]) for o in outs)


@pytest.mark.parametrize("scale", [0.01, 3.0])
@pytest.mark.parametrize("t", [2, 70])
def test_large_and_constant_scores(moss, cuda_device, scale, t):
    """Sharp and flat softmaxes; scores that rise along the history (every
    tile brings a new maximum) and that are all equal."""
    h = History([t], [600], 1, 64, 16, cuda_device)
    k, _ = h.dense(0)
    ramp = torch.linspace(-1, 1, 600 + t, device=cuda_device)[:, None].expand(-1, 64)
    page, slot = h.where(0, torch.arange(600 + t, device=cuda_device))
    h.k[page, 0, slot] = ramp.to(torch.bfloat16)
    q = torch.ones(t, 1, 64, device=cuda_device, dtype=torch.bfloat16)
    q[1::2] = -1
    got = moss.paged_attention(q, h.k, h.v, *h.index, scale=scale)
    want, size = attention_reference(h, q, 0, scale)
    # scores up to 64 * scale: their float32 rounding (the product, the scale,
    # the shift by the maximum: 4 * 2^-24 of 64 * scale * log2(e)) is a
    # relative error of the weights of ln(2) times that
    extra = 4 * 2.0 ** -24 * 64 * scale * 2
    weight = 2.0 ** -15 + (2.0 ** -8 if t > 16 else 0.0) + extra
    bound = 2.0 ** -8 * want.abs() + weight * size
    assert ((got.double() - want).abs() / bound).max().item() <= 1.001
    q.zero_()
    got = moss.paged_attention(q, h.k, h.v, *h.index)
    want, size = attention_reference(h, q, 0, 1 / 8)
    check_attention(got, want, size, t)


def test_rows_that_attend_to_nothing_are_zero(moss, cuda_device):
    """A sequence with more new tokens than positions: its first rows have
    none; and rows of no sequence stay as they are."""
    h = History([6, 3], [0, 40], 2, 64, 16, cuda_device)
    h.kv_len[0] = 4
    q = torch.randn(12, 2, 64, device=cuda_device, dtype=torch.bfloat16)
    out = torch.full((12, 2, 64), 7.0, device=cuda_device, dtype=torch.bfloat16)
    got = moss.paged_attention(q, h.k, h.v, *h.index, out=out)
    assert got.data_ptr() == out.data_ptr()
    assert torch.equal(out[:2], torch.zeros_like(out[:2]))
    assert torch.equal(out[9:], torch.full_like(out[9:], 7.0))
    assert torch.isfinite(out[2:9].float()).all()
    h.kv_len[0] = 0
    out.fill_(7.0)
    moss.paged_attention(q, h.k, h.v, *h.index, out=out)
    assert torch.equal(out[:6], torch.zeros_like(out[:6]))
    h.kv_len[0] = 4
    k, v = h.dense(0)
    # row 2 is position 0: its only key is its own
    out.fill_(7.0)
    moss.paged_attention(q, h.k, h.v, *h.index, out=out)
    assert torch.equal(out[2], v[:, 0].to(torch.bfloat16))


def test_a_long_history_past_32_bits(moss, cuda_device):
    """A pool of more than 2^31 values: pages at its far end."""
    page, d, hkv = 256, 128, 8
    pages = (1 << 31) // (page * d * hkv) + 64
    k = torch.zeros(pages, hkv, page, d, device=cuda_device, dtype=torch.bfloat16)
    v = torch.zeros_like(k)
    g = torch.Generator(device=cuda_device).manual_seed(0)
    k[-40:].normal_(generator=g)
    v[-40:].normal_(generator=g)
    for new in ([1], [50]):
        h = History(new, [5000], 1, d, page, cuda_device)
        h.k, h.v = k, v
        columns = h.table.shape[1]
        h.table[0] = torch.arange(pages - columns, pages, dtype=torch.int32, device=cuda_device).flip(0)
        x = torch.randn(h.n, 16 + 2 * hkv, d, device=cuda_device, generator=g).to(torch.bfloat16)
        q = moss.rope_paged_kv(x[:, :16], x[:, 16:16 + hkv], x[:, 16 + hkv:], *h.index, PERIOD, k, v)
        position = torch.arange(5000, 5000 + h.n, device=cuda_device)
        where = h.where(0, position)
        assert torch.equal(v[where[0], :, where[1]], x[:, 16 + hkv:])
        got = moss.paged_attention(q, k, v, *h.index)
        want, size = attention_reference(h, q, 0, d ** -0.5)
        check_attention(got, want, size, 2 * new[0])
    no_device_error()


def test_strided_queries_and_other_streams(moss, cuda_device):
    """Queries as a view of a wider tensor; two streams at once with a
    workspace each; results as on the default stream."""
    h = History([4, 60], [700, 300], 2, 64, 16, cuda_device)
    wide = torch.randn(h.n, 10, 64, device=cuda_device, dtype=torch.bfloat16)
    q = wide[:, 3:7]
    want = moss.paged_attention(q.contiguous(), h.k, h.v, *h.index)
    assert torch.equal(moss.paged_attention(q, h.k, h.v, *h.index), want)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i].append(moss.paged_attention(q, h.k, h.v, *h.index))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for part in outs for o in part)


def test_captured_calls_follow_their_index_tensors(moss, cuda_device):
    """A graph of append + attention, replayed for single tokens as the
    history grows page by page: lengths and tables are read on the device.
    Two captured graphs replayed in turn do not disturb one another."""
    hq, hkv, d, page = 4, 2, 64, 16
    device = cuda_device
    h = History([1, 1, 1], [60, 14, 30], hkv, d, page, device, spare=20, columns=8)
    free = [p for p in range(h.k.shape[0]) if p not in set(h.table.flatten().tolist())]
    x = torch.zeros(3, hq + 2 * hkv, d, device=device, dtype=torch.bfloat16)

    def step():
        q = moss.rope_paged_kv(x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], *h.index, PERIOD,
                               h.k, h.v)
        return q, moss.paged_attention(q, h.k, h.v, *h.index, max_tokens=1)

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            made = step()
        graphs.append((graph, made))
    g = torch.Generator().manual_seed(1)
    for i in range(24):
        x.copy_(torch.randn(x.shape, generator=g).to(device, torch.bfloat16))
        graph, (q, out) = graphs[i % 2]
        graph.replay()
        want, size = attention_reference(h, q, 0, d ** -0.5)
        check_attention(out, want, size, 2)
        # the next position, on a new page where the last one is full
        for s in range(3):
            if h.length[s] % page == 0:
                h.table[s, h.length[s] // page] = free.pop()
            h.past[s] += 1
            h.length[s] += 1
        h.kv_len.add_(1)
    no_device_error()


@pytest.mark.parametrize("t", [1, 50])
def test_shared_pages(moss, cuda_device, t):
    """Sequences with the same pages for their beginning."""
    h = History([t, t, t], [64, 64, 70], 2, 64, 16, cuda_device, seed=9)
    h.table[1:, :4] = h.table[0, :4]
    q = torch.randn(h.n, 4, 64, device=cuda_device, dtype=torch.bfloat16)
    got = moss.paged_attention(q, h.k, h.v, *h.index)
    want, size = attention_reference(h, q, 0, 1 / 8)
    check_attention(got, want, size, 2 * t)
    # the output may take the queries' place
    assert moss.paged_attention(q, h.k, h.v, *h.index, out=q) is q
    assert torch.equal(q, got)
    no_device_error()


def test_lengths_past_the_table_are_reported(moss, cuda_device):
    from fast_moss_b200 import _lib

    no_device_error()
    for t in (1, 50):
        h = History([t, t], [100, 30], 2, 64, 16, cuda_device, seed=t)
        room = 16 * h.table.shape[1]
        q = torch.randn(h.n, 2, 64, device=cuda_device, dtype=torch.bfloat16)
        h.table[0, -1] = 0
        h.kv_len[0] = room
        moss.paged_attention(q, h.k, h.v, *h.index)
        no_device_error()
        h.kv_len[0] = room + 1
        got = moss.paged_attention(q, h.k, h.v, *h.index)
        assert take_device_error() == _lib.ERR_TIMEOUT
        h.new[0] = 0
        want, size = attention_reference(h, q, 0, 1 / 8)
        check_attention(got[t:], want[t:], size[t:], t)
    no_device_error()


def test_a_captured_batch_takes_other_splits(moss, cuda_device):
    """One graph over 90 packed rows of six sequences, replayed as the rows
    are shared out anew: all in one, none at all, few and many side by side."""
    device = cuda_device
    splits = [[90, 0, 0, 0, 0, 0], [15, 15, 15, 15, 15, 15], [1, 1, 60, 1, 20, 7],
              [0, 0, 0, 0, 0, 0], [40, 3, 2, 0, 0, 33], [1, 1, 1, 1, 1, 1]]
    past = [30, 0, 500, 16, 129, 8]
    columns = 40
    h = History([90] * 6, past, 2, 128, 16, device, columns=columns)
    q = torch.randn(90, 4, 128, device=device, dtype=torch.bfloat16)
    out = torch.zeros_like(q)
    moss.paged_attention(q, h.k, h.v, *h.index, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        moss.paged_attention(q, h.k, h.v, *h.index, context=200, out=out)
    for new in splits:
        h.new, h.length = new, [a + b for a, b in zip(new, past)]
        h.start = [sum(new[:i]) for i in range(7)]
        h.q_start.copy_(torch.tensor(h.start))
        h.kv_len.copy_(torch.tensor(h.length))
        out.fill_(7.0)
        graph.replay()
        n = h.start[-1]
        want, size = attention_reference(h, q, 200, 128 ** -0.5)
        check_attention(out[:n], want[:n], size[:n], 180) if n else None
        assert (out[n:] == 7).all()
    no_device_error()


def test_wrappers_refuse_bad_tensors(moss, cuda_device):
    from fast_moss_b200._lib import UnsupportedError

    h = History([2], [10], 2, 64, 16, cuda_device)
    q = torch.zeros(2, 4, 64, device=cuda_device, dtype=torch.bfloat16)
    for bad in (q.float(), q[:, :3], q[0], q.cpu()):
        with pytest.raises(ValueError):
            moss.paged_attention(bad, h.k, h.v, *h.index)
    for kw in (dict(context=0), dict(context=-3), dict(scale=0.0), dict(scale=-1.0),
               dict(max_tokens=0), dict(out=q[:1]), dict(out=q.float())):
        with pytest.raises(ValueError):
            moss.paged_attention(q, h.k, h.v, *h.index, **kw)
    with pytest.raises(ValueError):
        moss.paged_attention(q, h.k, h.v, h.q_start.int(), h.kv_len, h.table)
    with pytest.raises(ValueError):
        moss.paged_attention(q, h.k, h.v, h.q_start, h.kv_len, h.table.long())
    with pytest.raises(ValueError):
        moss.paged_attention(q, h.k.transpose(1, 2), h.v.transpose(1, 2), *h.index)
    with pytest.raises(UnsupportedError):
        moss.paged_attention(q, torch.zeros(3, 2, 24, 64, device=cuda_device, dtype=torch.bfloat16),
                             torch.zeros(3, 2, 24, 64, device=cuda_device, dtype=torch.bfloat16), *h.index)
    kv = q[:, :2]
    with pytest.raises(ValueError):
        moss.rope_paged_kv(q, kv[:, :1], kv, *h.index, PERIOD, h.k, h.v)
    with pytest.raises(ValueError):
        moss.rope_paged_kv(q, kv.float(), kv, *h.index, PERIOD, h.k, h.v)
    with pytest.raises(ValueError):
        moss.rope_paged_kv(q, kv, kv, *h.index, 0.0, h.k, h.v)
    with pytest.raises(ValueError):
        moss.rope_paged_kv(q, kv, kv, *h.index, PERIOD, h.k, h.v,
                           q_weight=torch.ones(32, device=cuda_device))
    # nothing to do
    none = torch.zeros(0, 4, 64, device=cuda_device, dtype=torch.bfloat16)
    zero = torch.zeros(2, device=cuda_device, dtype=torch.int64)
    assert moss.paged_attention(none, h.k, h.v, zero, h.kv_len, h.table).shape == (0, 4, 64)


def test_calls_survive_odd_arguments(moss, cuda_device):
    """What is no tensor, or none that the library can read, is an error and
    not the end of the process; single entries may have any stride; an output
    in inference mode and one outside of it."""
    h = History([2], [10], 2, 64, 16, cuda_device)
    q = torch.randn(2, 4, 64, device=cuda_device, dtype=torch.bfloat16)
    want = moss.paged_attention(q, h.k, h.v, *h.index)
    for bad in (None, 3, "q", [q], q.to_sparse(), torch.zeros(2, 4, 64, device="meta")):
        with pytest.raises((ValueError, RuntimeError)):
            moss.paged_attention(bad, h.k, h.v, *h.index)
        with pytest.raises((ValueError, RuntimeError)):
            moss.rope_paged_kv(bad, q[:, :2], q[:, :2], *h.index, PERIOD, h.k, h.v)
        with pytest.raises((ValueError, RuntimeError)):
            moss.qk_norm_rope(bad, bad, None, None, h.kv_len, PERIOD)
    with pytest.raises(TypeError):
        moss.paged_attention(q, h.k, h.v, *h.index, scale="1")
    with pytest.raises(TypeError):
        moss.paged_attention(q, h.k, h.v, *h.index, context=2.5)
    with torch.inference_mode():
        assert moss.paged_attention(q, h.k, h.v, *h.index).is_inference()
    assert torch.equal(moss.paged_attention(q, h.k, h.v, *h.index), want)
    # a batch and a head of one, their strides those of nothing
    x = torch.randn(5, 64, device=cuda_device, dtype=torch.bfloat16)
    view = x.as_strided((1, 1, 5, 64), (7, 3, 64, 1))
    offset = torch.tensor([9], device=cuda_device)
    a, _ = moss.qk_norm_rope(view, view, None, None, offset, PERIOD)
    b, _ = moss.qk_norm_rope(x[None, None], x[None, None], None, None, offset, PERIOD)
    assert torch.equal(a, b)
    no_device_error()


def test_calls_from_two_threads(moss, cuda_device):
    """Two host threads, a stream each, at the same time (a call lets go of
    the interpreter's lock while it launches)."""
    import threading

    h = History([4, 60, 1], [300, 100, 777], 2, 64, 16, cuda_device)
    q = torch.randn(h.n, 4, 64, device=cuda_device, dtype=torch.bfloat16)
    w = torch.ones(64, device=cuda_device)
    x = torch.randn(2, 3, 50, 64, device=cuda_device, dtype=torch.bfloat16)
    offset = torch.tensor([5, 90000], device=cuda_device)
    want = moss.paged_attention(q, h.k, h.v, *h.index)
    turned, _ = moss.qk_norm_rope(x, x, w, w, offset, PERIOD)
    torch.cuda.synchronize()
    wrong = []

    def work():
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                outs = [(moss.paged_attention(q, h.k, h.v, *h.index),
                         moss.qk_norm_rope(x, x, w, w, offset, PERIOD)[0]) for _ in range(60)]
                torch.cuda.current_stream().synchronize()
            wrong.extend(1 for a, b in outs if not (torch.equal(a, want) and torch.equal(b, turned)))
        except Exception as e:  # noqa: BLE001 (seen by the test's thread)
            wrong.append(e)

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert wrong == []
    no_device_error()


@pytest.mark.parametrize("hq,hkv,d", [(64, 1, 128), (71, 1, 64), (40, 8, 128), (300, 3, 64)])
def test_wide_groups_of_query_heads(moss, cuda_device, hq, hkv, d):
    """Many query heads a key head, powers of two and not: a token's rows lie
    across blocks and tiles."""
    new, past = [1, 5, 0, 13], [500, 0, 9, 70]
    h = History(new, past, hkv, d, 16, cuda_device, seed=hq, poison=float("nan"))
    q = torch.randn(h.n, hq, d, device=cuda_device, dtype=torch.bfloat16)
    for context in (0, 40):
        want, size = attention_reference(h, q, context, d ** -0.5)
        for hint in (None, 13):
            got = moss.paged_attention(q, h.k, h.v, *h.index, context=context or None,
                                       max_tokens=hint)
            check_attention(got, want, size, 13 * (hq // hkv))
    no_device_error()


@pytest.mark.parametrize("t", [4, 50])
def test_rows_beyond_the_packed_ones_are_reported(moss, cuda_device, t):
    """Index tensors that promise more rows than there are: the rows that are
    there are what they would be beside the others, and the append, whose keys
    are missing, sets the error word; also where a whole sequence is missing."""
    from fast_moss_b200 import _lib

    no_device_error()
    for n in (2 * t - 3, t):
        h = History([t, t], [100, 30], 2, 64, 16, cuda_device, seed=t)
        x = torch.randn(h.n, 6, 64, device=cuda_device, dtype=torch.bfloat16)
        q = moss.rope_paged_kv(x[:, :2], x[:, 2:4], x[:, 4:], *h.index, PERIOD, h.k, h.v)
        want, size = attention_reference(h, q, 0, 1 / 8)
        no_device_error()
        k, v = h.k.clone(), h.v.clone()
        part = moss.rope_paged_kv(x[:n, :2], x[:n, 2:4], x[:n, 4:], *h.index, PERIOD, k, v)
        assert take_device_error() == _lib.ERR_TIMEOUT
        assert torch.equal(part, q[:n]) and torch.equal(k, h.k) and torch.equal(v, h.v)
        for hint in (None, t):
            got = moss.paged_attention(q[:n], h.k, h.v, *h.index, max_tokens=hint)
            check_attention(got, want[:n], size[:n], t)
    no_device_error()
