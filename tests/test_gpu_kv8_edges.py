"""The 8-bit paged KV cache on the GPU where a call is unusual: batches whose
tiles alternate in size, workspaces and streams left to the call, exponents at
the ends of their range, queries that are not numbers. The batch, the 64-bit
answer and the derived tolerance are those of test_gpu_kv8 and kv8_ref."""
import threading

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


class Rows:
    """One sequence whose K and V are given: written by kv8_write, read back for the
    64-bit answer."""

    def __init__(self, nv, torch, q, k, v, dtype, fmt="e4m3", group=1, block=16):
        ctx, kv, hd = k.shape
        self.nv, self.torch, self.dtype, self.group = nv, torch, dtype, group
        lay = nv.KVLayout(-(-ctx // block), 1, block, kv, hd)
        self.arena = nv.KV8Arena.alloc(lay, fmt_id(nv, fmt))
        slots = torch.arange(ctx, dtype=torch.int32, device="cuda")
        rows = [torch.from_numpy(x.astype(np.float32)).cuda().reshape(ctx, kv * hd) for x in (k, v)]
        nv.kv8_write(*rows, self.arena, slots, 0)
        back = [torch.empty_like(x) for x in rows]
        nv.kv8_read(*back, self.arena, slots, 0)
        self.k, self.v = (values64(x).reshape(k.shape) for x in back)
        self.q = torch.from_numpy(q.astype(np.float32)).cuda().reshape(len(q), -1).to(dtype_of(torch, dtype))
        self.out = torch.full_like(self.q, 9.0)
        ints = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (range(-(-ctx // block)), [0, len(q)], [ctx])]
        nv.kv8_attention(self.out, self.q, self.arena, ints[0][None].contiguous(), ints[1], ints[2], len(q), ctx, 0,
                         num_heads=kv * group)

    def check(self):
        n, (ctx, kv, hd) = len(self.q), self.k.shape
        heads = kv * self.group
        want, sizes = ref.attention(values64(self.q).reshape(n, heads, hd), self.k, self.v, ctx - n, self.group, 1 / np.sqrt(hd))
        off = np.abs(values64(self.out).reshape(n, heads, hd) - want)
        tol = ref.tolerance(want, sizes, hd, self.dtype)
        assert np.isfinite(off).all() and (off <= tol).all(), float((off / tol).max())


def normal(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("rows,ctx", [(1, 300), (1, 5000), (60, 300)], ids=["one", "long", "chunk"])
@pytest.mark.parametrize("power", [-90, 60, 112, 124])
def test_values_at_the_ends_of_the_range(nv, torch, dtype, rows, ctx, power):
    """Value rows of 2^power and so exponents of that size: small weights still count."""
    if power == 124 and rows > 1 and dtype != "fp32":
        pytest.skip("sums of 300 such values are beyond 32 bits")
    Rows(nv, torch, normal(1, rows, 4, 64) * 1.5, normal(2, ctx, 2, 64), normal(3, ctx, 2, 64) * 2.0 ** power, dtype, group=2).check()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("rows,ctx", [(1, 100), (1, 400), (1, 6000), (60, 400)], ids=["short", "one", "long", "chunk"])
@pytest.mark.parametrize("first", [False, True])
@pytest.mark.parametrize("power", [30, 60, 100])
def test_rows_of_zeros_beside_large_values(nv, torch, dtype, rows, ctx, first, power):
    """Half the positions hold value rows of zeros, with nearly all of the weight; the
    other half's values are about 2^power."""
    q, k, v = (np.zeros((n, 1, 64)) for n in (rows, ctx, ctx))
    q[:, :, 0], q[:, :, 1:] = 8.0, normal(4, rows, 1, 63) * 0.1
    k[:, :, 1:] = normal(5, ctx, 1, 63)
    heavy = (np.arange(ctx) < ctx // 2) == first
    k[:, 0, 0] = np.where(heavy, 8.0, 0.0)              # a score of 8 more
    v[~heavy] = normal(6, int((~heavy).sum()), 1, 64) * 2.0 ** power
    Rows(nv, torch, q, k, v, dtype).check()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("rows", [1, 60])
def test_large_values_whose_scores_grow_slowly(nv, torch, dtype, rows):
    """Scores that rise by less than the step at which a kernel moves its reference,
    with values near the end of the range."""
    ctx = 700
    q, k = np.zeros((rows, 1, 64)), np.zeros((ctx, 1, 64))
    q[:, :, 0], k[64:, :, 0] = 1.0, 8 * 7.5 * np.log(2.0)  # 2^7.5 times the weight of the first 64
    Rows(nv, torch, q, k, np.abs(normal(7, ctx, 1, 64)) * 2.0 ** 116, dtype).check()


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,ctx", [(1, 40), (1, 3000), (60, 200)], ids=["short", "long", "chunk"])
@pytest.mark.parametrize("power", [14, 28, 60])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_far_beyond_each_other(nv, torch, dtype, rows, ctx, power, sign):
    """Scores some 2^power apart: the whole weight is on the largest, exactly."""
    if dtype == "fp16" and power > 14:
        power = 15  # the type's range
    q, k, v = np.zeros((rows, 1, 64)), np.zeros((ctx, 1, 64)), normal(11, ctx, 1, 64)
    q[:, 0, 0] = sign * 1.3 * 2.0 ** power
    k[:, 0, 0] = [13 + 2 * (j % 2) + 4 * (j % 5) + (200 if j == ctx // 3 else 0) for j in range(ctx)]
    k[:, 0, 0] *= 2.0 ** (12 if dtype == "fp16" else 0)
    x = Rows(nv, torch, q, k, v, dtype, fmt="int8")
    for r in range(rows):
        seen = sign * x.k[: ctx - rows + r + 1, 0, 0]
        best = x.v[: len(seen)][seen == seen.max()].mean(0)
        off = np.abs(values64(x.out[r]) - best[0])
        half = {"fp32": 2.0 ** -24, "bf16": 2.0 ** -8, "fp16": 2.0 ** -11}[dtype]
        n = int((seen == seen.max()).sum())
        mean = np.abs(x.v[: len(seen)][seen == seen.max()]).mean(0)[0]
        # equal weights, which the product with V may take rounded: that, the sums' n
        # additions and the output's rounding
        assert (off <= half * np.abs(best[0]) + ((2 * n + 16) * 2.0 ** -23 + ref.WEIGHT[dtype]) * mean).all(), r


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("rows", [1, 60])
@pytest.mark.parametrize("power", [-85, 60, 124])
def test_large_keys_and_small_queries(nv, torch, dtype, rows, power):
    """Scores of ordinary size from factors far from it."""
    Rows(nv, torch, normal(8, rows, 2, 128) * 2.0 ** -power, normal(9, 300, 2, 128) * 2.0 ** power, normal(10, 300, 2, 128), dtype).check()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("block", [8, 16])
@pytest.mark.parametrize("seqs", [[(1, 100), (1, 50)], [(30, 100), (1, 50)]], ids=["decodes", "chunks"])
def test_bad_block_ids_beside_small_values(nv, torch, dtype, block, seqs):
    """They count as zero rows whatever the size of the others."""
    b = Batch(nv, torch, seqs, 2, 1, 64, dtype=dtype, block=block, seed=4)
    b.arena.v_exp.copy_((b.arena.v_exp.int() - 80).clamp(min=-100))
    b.v = [v * 2.0 ** -80 for v in b.v]
    b.tables[0, 2] = -1
    b.k[0][2 * block : 3 * block] = 0.0
    b.v[0][2 * block : 3 * block] = 0.0
    b.call()
    assert nv.get_last_error() == nv.ERR_BOUNDS
    b.check()


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("seqs", [[(1, 1), (1, 70), (1, 700), (1, 3000)], [(40, 200), (1, 40), (90, 90)]], ids=["decodes", "chunks"])
@pytest.mark.parametrize("window", [0, 50])
def test_queries_that_are_not_numbers(nv, torch, dtype, seqs, window):
    """A NaN or an infinity makes its own row and head NaN and leaves the others."""
    b = Batch(nv, torch, seqs, 4, 2, 64, dtype=dtype, seed=14, window=window, sinks=3)
    q = b.query.reshape(-1, 4, 64)
    clean = b.query.clone()
    rows = q.shape[0]
    bad = [(0, 1, np.nan), (rows // 2, 3, np.inf), (rows - 1, 0, -np.inf)]
    for r, h, x in bad:
        q[r, h, 5] = x
    b.call()
    out = b.out.reshape(-1, 4, 64)
    for r, h, _ in bad:
        assert out[r, h].isnan().all()
    b.query.copy_(clean)
    good = b.out.clone()
    b.out.fill_(9.0)
    b.call()
    b.check()
    for r, h, _ in bad:
        good.reshape(-1, 4, 64)[r, h] = out[r, h]
    assert torch.equal(good, b.out)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("by", [12, 40, 90])
def test_prompts_with_some_large_value_exponents(nv, torch, hd, by):
    """E4M3 exponents above 7 at some positions of a key tile, at all, and at none."""
    b = Batch(nv, torch, [(40, 200), (130, 130)], 8, 2, hd, dtype="bf16", seed=hd)
    for s, (_, ctx) in enumerate(b.seqs):
        for j in [*range(3, 64, 7), *range(64, 128)]:
            blk = int(b.tables[s, j // 16])
            b.arena.v_exp[blk, b.layer, :, j % 16] += by + (3 if j % 2 else 0)
            b.v[s][j] *= 2.0 ** (by + (3 if j % 2 else 0))
    assert int(b.arena.v_exp[int(b.tables[0, 4]), b.layer].min()) > 0
    b.call()
    b.check()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_fp16_prompts_keep_two_terms_of_a_weight(nv, torch, hd, fmt, monkeypatch):
    """Two bf16 terms leave at most 2^-8 of 2^-8 of a weight, not one fp16's 2^-11."""
    monkeypatch.setitem(ref.WEIGHT, "fp16", 2.0 ** -16)
    b = Batch(nv, torch, [(70, 300), (40, 40), (9, 900)], 8, 2, hd, fmt=fmt, dtype="fp16", seed=3)
    b.call()
    b.check()


@pytest.mark.parametrize("dtype,hd", [("fp16", 64), ("fp16", 128), ("fp32", 32), ("bf16", 32), ("fp32", 256), ("fp16", 256)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (33, 4), (100, 70)])
@pytest.mark.parametrize("seqs", [[(1, 1), (1, 130), (1, 513)], [(5, 5), (33, 70), (130, 300)]], ids=["decodes", "chunks"])
def test_windows_of_other_types_and_head_dims(nv, torch, dtype, hd, window, sinks, seqs):
    b = Batch(nv, torch, seqs, 4, 2, hd, dtype=dtype, window=window, sinks=sinks, seed=window)
    b.call()
    b.check()


def test_two_host_threads(nv, torch):
    """Calls from two threads, each with its stream and workspace."""
    bs = [Batch(nv, torch, s, 4, 2, 64, dtype=d, seed=21 + i)
          for i, (s, d) in enumerate([([(1, 900), (1, 40)], "bf16"), ([(60, 300), (1, 700)], "fp16")])]
    for b in bs:
        b.call()
    torch.cuda.synchronize()
    want = [b.out.clone() for b in bs]
    errors = []

    def work(b, w):
        try:
            st = torch.cuda.Stream()
            ws = nv.kv8_alloc_workspace(len(b.seqs), b.max_new, b.max_ctx, 4, b.arena.layout)
            torch.cuda.synchronize()
            for _ in range(50):
                out = torch.full_like(w, 9.0)
                st.wait_stream(torch.cuda.current_stream())
                b.call(out=out, stream=st, workspace=ws)
                st.synchronize()
                assert torch.equal(out, w)
        except BaseException as e:  # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=work, args=x) for x in zip(bs, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for b in bs:
        b.check()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("window,sinks", [(1500, 0), (2000, 700), (3000, 5)])
@pytest.mark.parametrize("seqs", [[(1, 6000), (1, 1400), (1, 2300)], [(90, 5000), (1, 4000), (300, 300)]], ids=["decodes", "chunks"])
def test_windows_that_are_cut(nv, torch, dtype, window, sinks, seqs):
    """Windows of many chunks, shared out over CTAs and merged, the sinks' part among them."""
    b = Batch(nv, torch, seqs, 4, 1, 64, dtype=dtype, window=window, sinks=sinks, seed=sinks)
    b.call()
    b.check()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("ctx", [40, 900])
def test_rows_of_zeros_alone_at_large_scores(nv, torch, dtype, ctx):
    """All values 0 (exponent -100, the largest weights that there are) at scores near the
    stated limit, rising by less than the step at which the reference moves."""
    q, k, v = np.zeros((1, 1, 64)), np.zeros((ctx, 1, 64)), np.zeros((ctx, 1, 64))
    q[:, :, 0], k[:, 0, 0] = 2.0 ** 20, 127.0
    q[:, :, 1], k[:, 0, 1] = 1.0, np.linspace(0, 16, ctx)
    v[-1] = 2.0 ** -60
    Rows(nv, torch, q, k, v * 0, dtype, fmt="int8").check()
    out = Rows(nv, torch, q, k, v, dtype, fmt="int8").out
    assert torch.isfinite(out).all() and (out >= 0).all() and (out <= 2.0 ** -60).all()
