"""GPU: the split that the attention kernels work by is the one that
moss_paged_attention_plan gives for the same index arrays."""

import pytest
import torch

from test_gpu_paged import History, no_device_error
from test_paged_plan import plan

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new,past,group,hkv,context", [
    ([4] * 9, [500 * i for i in range(9)], 2, 3, 0),     # 8 rows
    ([4] * 150, [37 * i for i in range(150)], 2, 20, 250),
    ([1], [100000], 1, 2, 0),
    ([9, 3, 1, 0, 16], [40, 0, 9000, 5, 700], 2, 8, 0),  # up to 32 rows
    ([300], [5000], 2, 3, 0),                            # one long sequence
    ([700], [3000], 1, 40, 900),
])
def test_the_plan_is_the_split_that_runs(moss, cuda_device, d, new, past, group, hkv, context):
    """The notes that workers leave about the items that they begin and others
    end: worker, last worker, key head and block."""
    from fast_moss_b200 import _lib

    lib = _lib.load()
    h = History(new, past, hkv, d, 16, cuda_device)
    hq = group * hkv
    q = torch.randn(h.n, hq, d, device=cuda_device, dtype=torch.bfloat16)
    most = max(new) * group
    size = lib.moss_paged_attention_workspace(d, most)
    space = torch.zeros(size, device=cuda_device, dtype=torch.uint8)
    out = torch.empty_like(q)
    _lib.call("moss_paged_attention", q.data_ptr(), h.k.data_ptr(), h.v.data_ptr(),
              h.q_start.data_ptr(), h.kv_len.data_ptr(), h.table.data_ptr(), h.n, len(new), hq, hkv,
              d, h.k.shape[0], 16, h.table.shape[1], max(new), context, d ** -0.5,
              space.data_ptr(), size, out.data_ptr(), torch.cuda.current_stream().cuda_stream)
    no_device_error()
    if most > 32:
        rows, tile, setup, each = 256, 128, 3, 1
    elif most > 8:
        rows, tile, setup, each = 16, 16, 2, 16 if d == 64 else 8
    else:
        rows, tile, setup, each = 8, 16, 2, 16 if d == 64 else 12
    workers = each * torch.cuda.get_device_properties(cuda_device).multi_processor_count
    # a note: eight int32, the first 1 where an item begins, then last worker,
    # key head, first packed row, block and its rows
    notes = space[:32 * workers].view(torch.int32).view(workers, 8).cpu()
    got = {(w, n[1], n[2], n[3], n[4]) for w, n in enumerate(notes.tolist()) if n[0] == 1}
    pieces = plan(h.start, h.length, h.n, group=group, hkv=hkv, page=16, columns=h.table.shape[1],
                  context=context, rows=rows, tile=tile, setup=setup, ctas=workers)
    ends = {p[1:4]: p[0] for p in pieces if p[9]}
    want = {(p[0], ends[p[1:4]], p[2], h.start[p[1]], p[3]) for p in pieces if p[8] and not p[9]}
    assert got == want and want
