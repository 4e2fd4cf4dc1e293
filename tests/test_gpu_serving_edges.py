"""The serving operators where a caller's numbers are out of the ordinary: values on
the device that no host check sees, bounds that are too small, and batches so long that
the kernels' loops go round more than once."""
import kv4_oracle as O
import numpy as np
import pytest
import torch
from test_gpu_kv4 import _batch, _cache, _close, _i32

from kernels.kv4 import kv4_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("starts,total,rows", [
    ([0, 3, 1, 4, 4, 2, 9], 12, 3),
    ([5, 2, 9, -7, 2**31 - 1, 30, -2**31], 33, 40),
    ([0, 70, 0, 70, 10, 140], 140, 70),                       # tiles
    ([0, 2] * 70 + [150], 150, 20),                           # the largest start so far passes from 64 requests on to the next
])
def test_starts_that_go_down(gpu, starts, total, rows):
    """A start below an earlier one counts as that one."""
    rng = np.random.default_rng(len(starts))
    lengths, _, table, pages = _batch(rng, [(int(rng.integers(0, 90)), 0) for _ in starts[1:]], 16)
    cache, k, v = _cache(rng, pages, 16, 2, 64, 64, gpu)
    q = torch.from_numpy(rng.standard_normal((total, 8 * 64)).astype(np.float32)).half()
    args = (q.to(gpu), cache, _i32(table, gpu), _i32(lengths, gpu))
    meant = np.maximum.accumulate(np.clip(starts, 0, total))
    rows = max(rows, int(np.diff(meant).max()))
    y = kv4_attention(*args, _i32(starts, gpu), rows)
    _close(y, O.attend(q.double().numpy().reshape(-1, 8, 64), k, v, lengths, meant, table, 16), "fp16", "starts that go down")
    assert torch.equal(y, kv4_attention(*args, _i32(meant, gpu), rows))
