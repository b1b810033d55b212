"""The 8-bit paged KV cache on the GPU where a call is unusual: batches whose
tiles alternate in size, workspaces and streams left to the call, exponents at
the ends of their range, queries that are not numbers. The batch, the 64-bit
answer and the derived tolerance are those of test_gpu_kv8 and kv8_ref."""
import numpy as np
import pytest

import kv8_ref as ref
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


@pytest.mark.parametrize("raw", [False, True], ids=["stream", "handle"])
def test_default_workspaces_on_two_streams(nv, torch, raw):
    """Calls without a workspace on a side stream, while the current stream keeps
    allocating, filling and freeing tensors of the workspace's size."""
    seqs = [(1, 2500), (1, 900), (1, 1700), (1, 40)]
    b = Batch(nv, torch, seqs, 8, 2, 128, dtype="bf16", seed=31)
    size = nv.kv8_workspace_size(len(seqs), b.max_new, b.max_ctx, 8, b.arena.layout)
    st = torch.cuda.Stream()
    outs = [torch.full_like(b.out, 9.0) for _ in range(40)]
    st.wait_stream(torch.cuda.current_stream())
    for out in outs:
        junk = torch.empty(size, dtype=torch.uint8, device="cuda").fill_(255)
        b.call(out=out, stream=st.cuda_stream if raw else st)
        del junk
        junk = torch.empty(size, dtype=torch.uint8, device="cuda").fill_(255)
        del junk
    torch.cuda.synchronize()
    b.check(outs[0])
    assert all(torch.equal(o, outs[0]) for o in outs)


@pytest.mark.parametrize("handle", [0, None], ids=["legacy", "current"])
def test_default_workspace_on_the_default_streams(nv, torch, handle):
    b = Batch(nv, torch, [(1, 2500), (3, 40)], 4, 2, 64, seed=32)
    torch.cuda.synchronize()
    b.call(stream=handle)
    torch.cuda.synchronize()
    b.check()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype,hd", [("bf16", 64), ("fp16", 128)])
@pytest.mark.parametrize("by", [20, 28, 30, 32, 34])
def test_keys_far_below_a_later_one(nv, torch, fmt, dtype, hd, by):
    """The last key of a prompt is 2^by larger than the others of its 64: the rows
    before it, which do not see it, are answered as if it were not there."""
    seqs = [(40, 60), (1, 7), (70, 130)]
    b = Batch(nv, torch, seqs, 8, 2, hd, fmt=fmt, dtype=dtype, seed=by)
    for s, (_, ctx) in enumerate(seqs):
        blk = int(b.tables[s, (ctx - 1) // 16])
        b.arena.k_exp[blk, b.layer, :, (ctx - 1) % 16] += by
        b.k[s][ctx - 1] *= 2.0 ** by
    b.call()
    out, q = (values64(x).reshape(-1, 8, hd) for x in (b.out, b.query))
    at = 0
    for s, (new, ctx) in enumerate(seqs):
        rows = slice(at, at + new - 1)
        at += new
        if new > 1:
            want, sizes = ref.attention(q[rows], b.k[s], b.v[s], ctx - new, 4, hd ** -0.5)
            assert (np.abs(out[rows] - want) <= ref.tolerance(want, sizes, hd, dtype)).all()
