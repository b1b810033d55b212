"""The 8-bit paged KV cache on the GPU where a call is unusual: batches whose
tiles alternate in size, workspaces and streams left to the call, exponents at
the ends of their range, queries that are not numbers. The batch, the 64-bit
answer and the derived tolerance are those of test_gpu_kv8 and kv8_ref."""
import numpy as np
import pytest

from test_gpu_kv8 import Batch, clean_status, dtype_of, fmt_id, torch, values64  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,hd", [("bf16", 64), ("fp16", 128)])
def test_full_and_half_tiles_in_turn(nv, torch, dtype, hd):
    """Several tiles for each CTA, some of more than 128 rows and some of fewer
    with one or two key tiles: each must be answered with its own queries, every
    time."""
    rng = np.random.default_rng(hd)
    seqs = []
    for i in range(360):
        if i % 3 == 0:
            new = int(rng.integers(33, 64))                 # 132 .. 252 packed rows
            seqs.append((new, new + int(rng.integers(0, 150))))
        else:
            new = int(rng.integers(1, 33))                  # 4 .. 128
            seqs.append((new, int(rng.integers(new, 129))))
    b = Batch(nv, torch, [seqs[i] for i in rng.permutation(360)], 8, 2, hd, dtype=dtype, seed=hd, layers=1)
    b.call()
    b.check()
    first = b.out.clone()
    for _ in range(30):
        b.out.fill_(9.0)
        b.call()
        assert torch.equal(first, b.out)
