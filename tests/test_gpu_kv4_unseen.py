"""What a row of the 4-bit cache's attention does not see leaves no trace in it,
whatever bits lie there: positions below the sequence's length that no store
has written (their rows cut off by the batch, or behind a window) hold scales that
are infinite or no numbers.  The oracle and the tolerances are those of test_gpu_kv4.py."""
import numpy as np
import pytest

import kv4_ref as R
from test_gpu_kv4 import NP, Setup, attend, check, kv4, say  # noqa: F401

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

CASES = [
    # heads, group, d, page, lens, rows, rows kept, window
    (2, 2, 64, 16, [60, 37, 20], [9, 5, 6], 3, 0),         # a workgroup per tile and head
    (1, 4, 96, 32, [90, 133], [20, 40], 11, 0),
    (2, 5, 256, 16, [50, 41], [16, 3], 2, 0),
    (2, 2, 64, 64, [90, 133, 40], [3, 1, 1], 3, 24),
    (1, 4, 128, 16, [300, 70], [2, 5], 2, 33),
    (2, 4, 64, 64, [5000, 40], [6, 7], 3, 0),              # steps shared by workgroups
    (1, 8, 128, 16, [4100, 2222], [5, 2], 2, 3000),
    (1, 3, 256, 128, [2500], [4], 1, 1700),
    (4, 64, 64, 16, [230, 233], [230, 215], 200, 0),      # the prompts' kernel
    (4, 64, 96, 16, [230, 233], [230, 215], 200, 0),
    (4, 64, 128, 16, [230, 233], [230, 215], 200, 0),
    (4, 64, 256, 16, [230, 233], [230, 215], 200, 0),
    (4, 32, 64, 64, [400, 270], [250, 250], 250, 70),
    (4, 64, 128, 64, [400, 270], [250, 250], 240, 81),
]


@pytest.mark.parametrize("dtype,bits", [("f16", 0x7c00), ("f32", 0xffff)])
@pytest.mark.parametrize("heads,group,d,page,lens,rows,kept,window", CASES)
def test_unwritten_positions(kv4, heads, group, d, page, lens, rows, kept, window, dtype, bits):
    say(f"unwritten {heads}x{group}x{d} page {page} {lens} {rows} kept {kept} window {window} {dtype} {bits:#x}")
    rng = np.random.default_rng(sum(lens) + d + window)
    s = Setup(kv4, rng, heads, d, page, lens, rows)
    s.fill(rng)
    nb, holes = d // 32, 0
    scales = np.full(nb, bits, np.uint16).view(np.float16)
    for i, n in enumerate(lens):
        first, last = n - rows[i], n - rows[i] + min(kept, rows[i]) - 1  # positions of the rows kept
        unseen = list(range(last + 1, n))
        if window:
            unseen += [j for j in range(first - window + 1) if j >= 0]
        holes += len(unseen)
        for j in unseen:
            p, o = s.place(i, j)
            code = rng.integers(-7, 8, (heads, 2, d))
            for h in range(heads):
                R.put(s.data, page, d, p, h, o, code[h, 0], scales, code[h, 1], scales)
    assert holes
    s.dev.copy_(torch.from_numpy(s.data))
    nh = heads * group
    q = rng.standard_normal((s.m, nh, d), dtype=np.float32).astype(NP[dtype])
    want, tol = s.expect(q, nh, True, window, d ** -0.5, dtype)
    s.batch = kv4.Batch(s.batch.table, s.batch.lens, rows=kept, row_off=torch.from_numpy(s.off).cuda(), m=s.m)
    got = attend(s, q, nh, dtype, True, window)
    own = [s.off[i] + r for i in range(len(lens)) for r in range(min(kept, rows[i]))]
    check(got[own], want[own], tol[own], dtype)
    left = [r for r in range(s.m) if r not in own]
    assert (got[left] == 77).all()
    if s.batch.work is not None:
        s.batch._c.work, s.batch._c.work_bytes = None, 0
        check(attend(s, q, nh, dtype, True, window, reserve=False)[own], want[own], tol[own], dtype, "one share:")
