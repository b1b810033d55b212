"""The 8-bit paged KV cache on the GPU: the quantising write and the read back
against the definition bit for bit, the attention against 64-bit numpy within
the derived tolerance (kv8_ref.tolerance)."""
import math

import numpy as np
import pytest

import kv8_ref as ref

pytestmark = pytest.mark.gpu

DT = {"fp32": "float32", "bf16": "bfloat16", "fp16": "float16"}


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


@pytest.fixture(autouse=True)
def clean_status(nv):
    assert nv.get_last_error() == nv.OK
    yield
    assert nv.get_last_error() == nv.OK


def dtype_of(torch, name):
    return getattr(torch, DT[name])


def fmt_id(nv, fmt):
    return nv.KV8_E4M3 if fmt == "e4m3" else nv.KV8_INT8


def arena_bytes(torch, arena):
    """(k codes, v codes, k exps, v exps) as numpy, codes as bytes."""
    return (arena.k.view(torch.uint8).cpu().numpy(), arena.v.view(torch.uint8).cpu().numpy(),
            arena.k_exp.cpu().numpy(), arena.v_exp.cpu().numpy())


def values64(t):
    return t.detach().double().cpu().numpy()


# ---------------------------------------------------------------- write, read
def rows_for_write(torch, n, heads, hd, dtype, seed):
    """K rows as a strided slice of a fused buffer: normal rows of many
    magnitudes, and first the ones where a quantiser goes wrong."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    fused = torch.randn((n, 2 * heads * hd + 16), generator=g, device="cuda")
    fused *= torch.exp2(torch.randint(-18, 14, (n, 1), generator=g, device="cuda").float())
    x = fused[:, : heads * hd]
    edge = [
        lambda r: r.zero_(),
        lambda r: r.fill_(448.0),                       # the largest code, exactly
        lambda r: r.fill_(448.0).mul_(1.0009765625),    # just above it: the next exponent
        lambda r: r.fill_(127.0),
        lambda r: r.copy_(torch.arange(hd, device="cuda") * 0.5 - 16.25),  # ties
        lambda r: r.copy_((torch.arange(hd, device="cuda") % 17 - 8) * 2.0 ** -9),
        lambda r: r[3:4].fill_(math.nan),
        lambda r: r[:2].copy_(torch.tensor([math.inf, -math.inf])),
        lambda r: r.fill_(math.nan),
        lambda r: r.fill_(1e-40),                       # subnormal in fp32
        lambda r: r.mul_(1e30),
        lambda r: r[5:6].fill_(-0.0),
        lambda r: r.fill_(3.4e38),
    ]
    for i, f in enumerate(edge):
        if i < n:
            f(x[i, (i % heads) * hd : (i % heads + 1) * hd])
    fused = fused.to(dtype_of(torch, dtype))
    return fused[:, : heads * hd], fused[:, heads * hd : 2 * heads * hd]


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("hd,heads,block,n", [(128, 4, 16, 40), (64, 3, 24, 31), (32, 5, 1, 17),
                                              (256, 1, 8, 20), (128, 1, 16, 1)])
def test_write_codes_are_the_definitions(nv, torch, fmt, dtype, hd, heads, block, n):
    blocks = -(-n // block) + 2
    lay = nv.KVLayout(blocks, 3, block, heads, hd)
    arena = nv.KV8Arena.alloc(lay, fmt_id(nv, fmt))
    arena.k.view(torch.uint8).fill_(0x5A)
    arena.k_exp.fill_(77)
    before = arena_bytes(torch, arena)
    key, value = rows_for_write(torch, n, heads, hd, dtype, seed=hd + n)
    rng = np.random.default_rng(n)
    slots = rng.permutation(blocks * block)[:n].astype(np.int32)
    if n > 6:
        slots[[2, 6]] = -1
    nv.kv8_write(key, value, arena, torch.from_numpy(slots).cuda(), 1)
    after = arena_bytes(torch, arena)
    want = [b.copy() for b in before]
    for which, x in ((0, key), (1, value)):
        codes, exps = ref.quantise(values64(x).reshape(n, heads, hd), fmt)
        for t in range(n):
            if slots[t] >= 0:
                b, i = divmod(int(slots[t]), block)
                want[which][b, 1, i] = codes[t].reshape(-1)
                want[2 + which][b, 1, :, i] = exps[t]
    for got, w in zip(after, want):
        assert np.array_equal(got, w)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_write_and_read_of_unaligned_rows(nv, torch, dtype):
    """Rows whose address or stride is not a multiple of 16 bytes."""
    n, heads, hd = 9, 2, 64
    lay = nv.KVLayout(4, 1, 16, heads, hd)
    t = dtype_of(torch, dtype)
    base = torch.randn((n, heads * hd + 3), device="cuda").to(t)
    key, value = base[:, 1 : 1 + heads * hd], base[:, 3:]
    arena = nv.KV8Arena.alloc(lay, nv.KV8_INT8)
    slots = torch.arange(n, dtype=torch.int32, device="cuda") + 5
    nv.kv8_write(key, value, arena, slots, 0)
    back = torch.full((n, heads * hd + 1), 7.0, device="cuda", dtype=t)
    back2 = torch.full((n, heads * hd + 5), 7.0, device="cuda", dtype=t)
    nv.kv8_read(back[:, 1:], back2[:, 2 : 2 + heads * hd], arena, slots, 0)
    for x, y in ((key, back[:, 1:]), (value, back2[:, 2 : 2 + heads * hd])):
        c, e = ref.quantise(values64(x).reshape(n, heads, hd), "int8")
        assert np.array_equal(values64(y).reshape(n, heads, hd), ref.dequantise(c, e, "int8"))
    assert (back[:, 0] == 7).all() and (back2[:, :2] == 7).all() and (back2[:, 2 + heads * hd :] == 7).all()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("hd,heads,block,n", [(128, 4, 16, 33), (64, 3, 24, 20), (32, 5, 1, 9), (256, 2, 8, 7)])
def test_read_gives_code_times_power(nv, torch, fmt, dtype, hd, heads, block, n):
    blocks = 70
    lay = nv.KVLayout(blocks, 2, block, heads, hd)
    arena = nv.KV8Arena.alloc(lay, fmt_id(nv, fmt))
    rng = np.random.default_rng(hd)
    codes = rng.integers(0, 256, (2, *lay.arena_shape())).astype(np.uint8)
    if fmt == "e4m3":
        codes[(codes & 127) == 127] = 0
    exps = rng.integers(-100, 120, (2, blocks, 2, heads, block)).astype(np.int8)
    if dtype == "fp16":
        exps = np.clip(exps, -12, 3)  # the type's range
    for t, c in ((arena.k, codes[0]), (arena.v, codes[1])):
        t.view(torch.uint8).copy_(torch.from_numpy(c))
    arena.k_exp.copy_(torch.from_numpy(exps[0]))
    arena.v_exp.copy_(torch.from_numpy(exps[1]))
    slots = rng.permutation(blocks * block)[:n].astype(np.int32)
    slots[1] = -1
    slots[3] = slots[2]  # the same slot twice
    outs = [torch.full((n, heads * hd), 3.0, device="cuda", dtype=dtype_of(torch, dtype)) for _ in "kv"]
    nv.kv8_read(*outs, arena, torch.from_numpy(slots).cuda(), 1)
    for i, o in enumerate(outs):
        for t in range(n):
            if slots[t] < 0:
                assert (o[t] == 3.0).all()
                continue
            b, s = divmod(int(slots[t]), block)
            want = ref.dequantise(codes[i][b, 1, s].reshape(heads, hd), exps[i][b, 1, :, s], fmt).reshape(-1)
            if dtype == "fp16":
                want = want.astype(np.float16)  # round to nearest
            assert np.array_equal(values64(o[t]), want.astype(np.float64))


def test_slots_beyond_the_arena_are_skipped_and_reported(nv, torch):
    lay = nv.KVLayout(3, 1, 16, 2, 64)
    arena = nv.KV8Arena.alloc(lay)
    x = torch.ones((3, 128), device="cuda")
    slots = torch.tensor([0, 48, 47], dtype=torch.int32, device="cuda")
    nv.kv8_write(x, x, arena, slots, 0)
    assert nv.get_last_error() == nv.ERR_BOUNDS
    y, z = torch.zeros_like(x), torch.zeros_like(x)
    nv.kv8_read(y, z, arena, slots, 0)
    assert nv.get_last_error() == nv.ERR_BOUNDS
    for t in (y, z):
        assert t[:, 0].tolist() == [1.0, 0.0, 1.0]
    n = torch.zeros(0, dtype=torch.int32, device="cuda")
    nv.kv8_write(x[:0], x[:0], arena, n, 0)


# ------------------------------------------------------------------ attention
class Batch:
    """Random cached rows in an arena (every other byte of it garbage that must
    not matter), random queries, and the 64-bit answer."""

    def __init__(self, nv, torch, seqs, heads, kv_heads, hd, block=16, fmt="e4m3", dtype="bf16", window=0, sinks=0,
                 seed=0, pad_rows=0, layers=2, q_scale=1.0, spread=2, width=0):
        self.nv, self.torch, self.seqs, self.dtype, self.fmt = nv, torch, seqs, dtype, fmt
        self.heads, self.kv, self.hd, self.window, self.sinks, self.layer = heads, kv_heads, hd, window, sinks, layers - 1
        rng = np.random.default_rng(seed)
        need = [-(-c // block) for _, c in seqs]
        blocks = sum(need) + 5
        lay = nv.KVLayout(blocks, layers, block, kv_heads, hd)
        arena = self.arena = nv.KV8Arena.alloc(lay, fmt_id(nv, fmt))
        ctxs = sum(c for _, c in seqs)
        codes, exps = [], []
        for _ in "kv":
            x = rng.standard_normal((ctxs, kv_heads, hd)) * 2.0 ** rng.integers(-spread, spread + 1, (ctxs, kv_heads, 1))
            c, e = ref.quantise(x, fmt)
            codes.append(c)
            exps.append(e)
        raw = [np.full(lay.arena_shape(), 0xFF, np.uint8) for _ in "kv"]
        rexp = [np.full((blocks, layers, kv_heads, block), 127, np.int8) for _ in "kv"]
        order = rng.permutation(blocks)
        tables = np.full((len(seqs), max(max(need), 1) + width), -7, np.int32)
        at = used = 0
        self.k, self.v = [], []
        for s, (new, ctx) in enumerate(seqs):
            tables[s, : need[s]] = order[used : used + need[s]]
            for j in range(ctx):
                b, i = tables[s, j // block], j % block
                for w in range(2):
                    raw[w][b, self.layer, i] = codes[w][at + j].reshape(-1)
                    rexp[w][b, self.layer, :, i] = exps[w][at + j]
            self.k.append(ref.dequantise(codes[0][at : at + ctx], exps[0][at : at + ctx], fmt))
            self.v.append(ref.dequantise(codes[1][at : at + ctx], exps[1][at : at + ctx], fmt))
            used += need[s]
            at += ctx
        for t, c in ((arena.k, raw[0]), (arena.v, raw[1])):
            t.view(torch.uint8).copy_(torch.from_numpy(c))
        arena.k_exp.copy_(torch.from_numpy(rexp[0]))
        arena.v_exp.copy_(torch.from_numpy(rexp[1]))
        self.tables = torch.from_numpy(tables).cuda()
        self.cu = torch.tensor([0, *np.cumsum([n for n, _ in seqs])], dtype=torch.int32, device="cuda")
        self.ctx = torch.tensor([c for _, c in seqs], dtype=torch.int32, device="cuda")
        self.max_new, self.max_ctx = max(1, max(n for n, _ in seqs)), max(1, max(c for _, c in seqs))
        rows = sum(n for n, _ in seqs) + pad_rows
        g = torch.Generator(device="cuda").manual_seed(seed)
        t = dtype_of(torch, dtype)
        self.query = (torch.randn((rows, heads * hd), generator=g, device="cuda") * q_scale).to(t)
        self.out = torch.full((rows, heads * hd), 9.0, device="cuda", dtype=t)

    def call(self, **kw):
        kw = {"num_heads": self.heads, "window": self.window, "sinks": self.sinks, **kw}
        self.nv.kv8_attention(kw.pop("out", self.out), kw.pop("query", self.query), self.arena, self.tables, self.cu,
                              self.ctx, kw.pop("max_new", self.max_new), kw.pop("max_ctx", self.max_ctx), self.layer, **kw)

    def check(self, out=None, skip=()):
        out = values64(self.out if out is None else out).reshape(-1, self.heads, self.hd)
        q = values64(self.query).reshape(-1, self.heads, self.hd)
        at = 0
        for s, (new, ctx) in enumerate(self.seqs):
            if new and s not in skip:
                want, sizes = ref.attention(q[at : at + new], self.k[s], self.v[s], ctx - new, self.heads // self.kv,
                                                   1.0 / math.sqrt(self.hd), self.window, self.sinks)
                tol = ref.tolerance(want, sizes, self.hd, self.dtype)
                off = np.abs(out[at : at + new] - want)
                i = np.unravel_index(np.argmax(off / tol), off.shape)
                far = bool(off[i] > tol[i]) or not np.isfinite(off).all()
                assert not far, (s, new, ctx, i, float(out[at : at + new][i]), float(want[i]), float(tol[i]))
            at += new
        assert (out[at:] == 9.0).all()  # rows of no sequence


DECODES = [(1, 1), (1, 2), (1, 15), (1, 16), (1, 17), (1, 64), (1, 130), (1, 513)]
CHUNKS = [(5, 5), (1, 40), (33, 70), (2, 257), (17, 17), (0, 0), (130, 300), (0, 12)]


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("seqs", [DECODES, CHUNKS], ids=["decodes", "chunks"])
@pytest.mark.parametrize("heads,kv,hd", [(4, 4, 128), (8, 2, 64), (3, 1, 32), (4, 2, 256), (16, 2, 128)])
def test_attention(nv, torch, fmt, dtype, seqs, heads, kv, hd):
    b = Batch(nv, torch, seqs, heads, kv, hd, fmt=fmt, dtype=dtype, seed=heads * hd, pad_rows=3)
    b.call()
    b.check()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (16, 0), (33, 4), (100, 17), (64, 600), (1000, 2)])
@pytest.mark.parametrize("seqs", [DECODES, CHUNKS, [(200, 700)]], ids=["decodes", "chunks", "late"])
@pytest.mark.parametrize("heads,kv,hd", [(4, 1, 128), (2, 2, 64)])
def test_window_and_sinks(nv, torch, dtype, window, sinks, seqs, heads, kv, hd):
    b = Batch(nv, torch, seqs, heads, kv, hd, dtype=dtype, window=window, sinks=sinks, seed=window)
    b.call()
    b.check()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("window", [513, 1 << 20, 2 ** 31 - 1])
@pytest.mark.parametrize("seqs", [DECODES, CHUNKS], ids=["decodes", "chunks"])
def test_windows_no_context_outgrows(nv, torch, dtype, window, seqs):
    b = Batch(nv, torch, seqs, 2, 1, 128, dtype=dtype, window=window, sinks=2 ** 31 - 1, seed=9)
    b.call()
    b.check()


def test_more_sequences_than_one_launch_counts(nv, torch):
    """Over 512 decodes in one call, some without rows, ragged."""
    seqs = [(1 if i % 5 else 0, 1 + (i * 37) % 90) for i in range(1100)] + [(1, 2000)]
    b = Batch(nv, torch, seqs, 2, 1, 64, dtype="bf16", seed=4)
    b.call()
    b.check()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_one_workspace_serves_smaller_calls(nv, torch, dtype):
    """Sized once for the largest step, used for all kinds after one another."""
    ws = None
    for seqs in ([(300, 900), (1, 2000), (5, 5)], [(1, 2000), (1, 700)], [(2, 2000)], [(9, 40), (1, 600)], [(64, 2000)], [(1, 1)]):
        b = Batch(nv, torch, seqs, 4, 2, 128, dtype=dtype, seed=len(seqs))
        if ws is None:
            ws = nv.kv8_alloc_workspace(3, 300, 2000, 4, b.arena.layout)
        b.call(workspace=ws)
        b.check()


@pytest.mark.parametrize("block", [1, 8, 16, 24, 32])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("seqs", [[(1, 700), (1, 90)], [(7, 400), (90, 600)]], ids=["decodes", "chunks"])
def test_blocks_behind_the_window_are_not_read(nv, torch, block, dtype, seqs):
    """Table entries of blocks that no row sees any part of may hold anything."""
    b = Batch(nv, torch, seqs, 4, 2, 128, block=block, dtype=dtype, window=70, sinks=5, seed=block)
    for s, (new, ctx) in enumerate(seqs):
        first = ctx - new - 70 + 1  # of the first row's window
        for i in range(-(-5 // block), max(0, first) // block):
            b.tables[s, i] = -9 if i % 2 else 1 << 30
    b.call()
    b.check()


@pytest.mark.parametrize("block", [1, 3, 8, 24, 32, 100])
@pytest.mark.parametrize("seqs", [DECODES, CHUNKS], ids=["decodes", "chunks"])
@pytest.mark.parametrize("hd", [64, 128])
def test_block_sizes(nv, torch, block, seqs, hd):
    b = Batch(nv, torch, seqs, 4, 2, hd, block=block, fmt="int8", window=90, sinks=5, seed=block, width=2)
    b.call()
    b.check()


@pytest.mark.parametrize("heads,kv", [(5, 1), (7, 1), (6, 2), (20, 1), (40, 1), (130, 1)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("seqs", [[(1, 300), (1, 77)], [(3, 40), (1, 9)], [(40, 200)]], ids=["one", "few", "chunk"])
def test_group_sizes(nv, torch, heads, kv, dtype, seqs):
    b = Batch(nv, torch, seqs, heads, kv, 64, dtype=dtype, seed=heads)
    b.call()
    b.check()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("seqs", [[(1, 9000)], [(1, 4000), (1, 1), (1, 2500)], [(3, 5000)], [(64, 6000), (1, 3000)]])
def test_long_contexts_are_split_and_joined(nv, torch, dtype, seqs):
    b = Batch(nv, torch, seqs, 2, 1, 128, dtype=dtype, seed=5)
    b.call()
    b.check()


@pytest.mark.parametrize("seqs", [[(1024, 5000)], [(300, 4900), (700, 5000)]], ids=["one", "two"])
def test_the_last_round_of_tiles_is_cut(nv, torch, seqs):
    """A few more tiles of nearly one length than CTAs: the last ones are shared out
    and merged, the same way every time."""
    heads = 40
    b = Batch(nv, torch, seqs, heads, heads, 64, dtype="bf16", seed=21)
    b.call()
    first = b.out.clone()
    b.out.fill_(9.0)
    b.call()
    assert torch.equal(first, b.out)
    q = values64(b.query).reshape(-1, heads, 64)
    out = values64(b.out).reshape(-1, heads, 64)
    some = [0, 39]
    at = 0
    for s, (new, ctx) in enumerate(seqs):
        want, sizes = ref.attention(q[at : at + new, some], b.k[s][:, some], b.v[s][:, some], ctx - new, 1, 0.125)
        assert (np.abs(out[at : at + new, some] - want) <= ref.tolerance(want, sizes, 64, "bf16")).all()
        at += new


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("seqs", [DECODES, CHUNKS], ids=["decodes", "chunks"])
def test_wide_magnitudes(nv, torch, dtype, seqs):
    """Rows whose exponents are far apart (2^-24 .. 2^24 around one), and sharp
    softmaxes: weights that underflow must not disturb the others."""
    b = Batch(nv, torch, seqs, 4, 2, 128, dtype=dtype, seed=8, spread=12, q_scale=2.0 ** -6)
    b.call()
    b.check()


def test_largest_exponents(nv, torch):
    """Value rows whose exponents are far above those of their keys."""
    b = Batch(nv, torch, [(1, 40), (20, 50)], 2, 1, 128, dtype="fp32", seed=2)
    b.arena.v_exp.copy_(self_shift(b.arena.v_exp, 20))
    b.v = [v * 2.0 ** 20 for v in b.v]
    b.call()
    b.check()


def self_shift(e, by):
    return (e.int() + by).clamp(max=119).to(e.dtype)


@pytest.mark.parametrize("seqs", [DECODES, CHUNKS], ids=["decodes", "chunks"])
def test_strided_rows_and_bounds_that_are_not_tight(nv, torch, seqs):
    b = Batch(nv, torch, seqs, 4, 2, 64, dtype="bf16", seed=1, pad_rows=2, width=9)
    rows = b.query.shape[0]
    wide_q = torch.full((rows, 3 * 256 + 8), 5.0, device="cuda", dtype=torch.bfloat16)
    wide_o = torch.full((rows, 256 + 24), 9.0, device="cuda", dtype=torch.bfloat16)
    wide_q[:, 256:512] = b.query
    ctx = max(c for _, c in seqs) + 16 * 9
    ws = nv.kv8_alloc_workspace(len(seqs), 140, ctx, 4, b.arena.layout)
    b.call(out=wide_o[:, 8:264], query=wide_q[:, 256:512], max_new=140, max_ctx=ctx, workspace=ws)
    b.check(wide_o[:, 8:264])
    assert (wide_o[:, :8] == 9.0).all() and (wide_o[:, 264:] == 9.0).all()


@pytest.mark.parametrize("seqs", [[(1, 40), (1, 70), (1, 33)], [(4, 40), (60, 200), (1, 33)]], ids=["decodes", "chunks"])
def test_bad_metadata_skips_its_sequence(nv, torch, seqs):
    b = Batch(nv, torch, seqs, 2, 1, 64, seed=3)
    b.ctx[1] = b.max_ctx + 1000  # beyond the declared maximum
    b.call()
    assert nv.get_last_error() == nv.ERR_INVALID
    b.check(skip=(1,))
    at = int(b.cu[1])
    assert (b.out[at : at + seqs[1][0]] == 9.0).all()


@pytest.mark.parametrize("seqs", [[(1, 100), (1, 50)], [(30, 100), (1, 50)]], ids=["decodes", "chunks"])
@pytest.mark.parametrize("bad", [-1, 1 << 20])
def test_bad_block_ids_count_as_zero_rows(nv, torch, seqs, bad):
    b = Batch(nv, torch, seqs, 2, 1, 64, seed=4)
    b.tables[0, 2] = bad
    b.k[0][32:48] = 0.0
    b.v[0][32:48] = 0.0
    b.call()
    assert nv.get_last_error() == nv.ERR_BOUNDS
    b.check()


def test_no_sequence_and_no_rows(nv, torch):
    b = Batch(nv, torch, [(0, 0), (0, 5)], 2, 1, 64, pad_rows=2)
    b.call()
    b.check()
    nv.kv8_attention(b.out, b.query, b.arena, b.tables[:0], b.cu[:1], b.ctx[:0], 1, 1, 0, num_heads=2)
    b.check()


@pytest.mark.parametrize("seqs", [DECODES, CHUNKS], ids=["decodes", "chunks"])
def test_runs_repeat_bit_for_bit(nv, torch, seqs):
    b = Batch(nv, torch, seqs + [(1, 3000)], 8, 2, 128, dtype="fp32", seed=6)
    b.call()
    first = b.out.clone()
    for _ in range(3):
        b.out.fill_(9.0)
        b.call()
        assert torch.equal(first, b.out)


@pytest.mark.parametrize("seqs", [DECODES, CHUNKS], ids=["decodes", "chunks"])
def test_captured_and_replayed_with_other_lengths(nv, torch, seqs):
    """Two graphs with a workspace each, replayed beside one another on two
    streams, the lengths changed between replays; then an eager call."""
    bs = [Batch(nv, torch, seqs, 4, 2, 128, dtype="bf16", seed=s) for s in (11, 12)]
    ws = [nv.kv8_alloc_workspace(len(seqs), b.max_new, b.max_ctx, 4, b.arena.layout) for b in bs]
    graphs = []
    for b, w in zip(bs, ws):
        b.call(workspace=w)
        torch.cuda.synchronize()
        b.out.fill_(9.0)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            b.call(workspace=w)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(3):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for b in bs:
        b.check()
        short = [(n, max(n, c - 9)) for n, c in seqs]
        b.ctx.copy_(torch.tensor([c for _, c in short], dtype=torch.int32))
        b.k, b.v, b.seqs = [k[: c] for k, (_, c) in zip(b.k, short)], [v[: c] for v, (_, c) in zip(b.v, short)], short
        b.out.fill_(9.0)
    torch.cuda.synchronize()
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    for b in bs:
        b.check()
        b.out.fill_(9.0)
        b.call()
        b.check()


def test_other_streams(nv, torch):
    b = Batch(nv, torch, CHUNKS, 4, 2, 128, seed=13)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    b.call(stream=st)
    st.synchronize()
    b.check()
    b.out.fill_(9.0)
    st.wait_stream(torch.cuda.current_stream())
    b.call(stream=st.cuda_stream, workspace=nv.kv8_alloc_workspace(len(CHUNKS), b.max_new, b.max_ctx, 4, b.arena.layout))
    st.synchronize()
    b.check()


@pytest.mark.parametrize("dtype,hd", [("bf16", 128), ("fp32", 64)])
def test_offsets_beyond_32_bits(nv, torch, dtype, hd):
    """Blocks past 4 GiB of codes, rows written, read and attended there."""
    heads, block = 4096 // hd, 16
    blocks = (1 << 32) // (block * 4096) + 70
    lay = nv.KVLayout(blocks, 1, block, heads, hd)
    arena = nv.KV8Arena(lay, *(torch.empty(lay.arena_shape(), dtype=torch.int8, device="cuda") for _ in "kv"),
                        *(torch.empty((blocks, 1, heads, block), dtype=torch.int8, device="cuda") for _ in "kv"))
    t = dtype_of(torch, dtype)
    n = 60 * block
    x = torch.randn((n, 2 * 4096), device="cuda").to(t)
    key, value = x[:, :4096], x[:, 4096:]
    table = torch.arange(blocks - 60, blocks, dtype=torch.int32, device="cuda").flip(0)
    pos = torch.arange(n, device="cuda")
    slots = (table[pos // block].long() * block + pos % block).int()
    nv.kv8_write(key, value, arena, slots, 0)
    back = [torch.empty((n, 4096), device="cuda") for _ in "kv"]
    nv.kv8_read(*back, arena, slots, 0)
    for got, x in zip(back, (key, value)):
        c, e = ref.quantise(values64(x[::97]).reshape(-1, heads, hd), "int8")
        assert np.array_equal(values64(got[::97]).reshape(-1, heads, hd), ref.dequantise(c, e, "int8"))
    for new in (1, 20):
        q = torch.randn((new, 4096), device="cuda").to(t)
        out = torch.empty_like(q)
        nv.kv8_attention(out, q, arena, table[None].contiguous(), torch.tensor([0, new], dtype=torch.int32, device="cuda"),
                         torch.tensor([n], dtype=torch.int32, device="cuda"), new, n, 0)
        k, v = (values64(b).reshape(n, heads, hd) for b in back)
        want, sizes = ref.attention(values64(q).reshape(new, heads, hd), k, v, n - new, 1, 1 / math.sqrt(hd))
        off = np.abs(values64(out).reshape(new, heads, hd) - want)
        assert (off <= ref.tolerance(want, sizes, hd, dtype)).all()


# --------------------------------------------------------------- run together
@pytest.mark.parametrize("dtype,fmt", [("fp32", "e4m3"), ("bf16", "int8")])
@pytest.mark.parametrize("window,sinks", [(0, 0), (48, 4)])
def test_prompt_in_chunks_then_decode(nv, torch, dtype, fmt, window, sinks):
    """Two sequences served as an engine would: the prompt written and attended
    in chunks beside the other's decode, then token by token, all captured rows
    checked against the whole context's attention over what the cache reads
    back."""
    heads, kv, hd, block = 8, 2, 64, 16
    lay = nv.KVLayout(40, 1, block, kv, hd)
    arena = nv.KV8Arena.alloc(lay, fmt_id(nv, fmt))
    t = dtype_of(torch, dtype)
    total = [150, 90]
    qkv = [torch.randn((n, (heads + 2 * kv) * hd), device="cuda").to(t) for n in total]
    rng = np.random.default_rng(0)
    order = rng.permutation(40)
    tables = np.zeros((2, 12), np.int32)
    tables[0], tables[1] = order[:12], order[12:24]
    dt = torch.from_numpy(tables).cuda()
    done = [0, 0]
    outs = [torch.zeros((n, heads * hd), device="cuda", dtype=t) for n in total]
    ws = nv.kv8_alloc_workspace(2, 150, 150, heads, lay)
    steps = [(64, 0), (50, 70), (30, 1)] + [(1, 1)] * 6
    for a, b in steps:
        new = [min(a, total[0] - done[0]), min(b, total[1] - done[1])]
        rows = torch.cat([x[d : d + n] for x, d, n in zip(qkv, done, new)])
        slots = np.concatenate([tables[s][(done[s] + np.arange(new[s])) // block] * block + (done[s] + np.arange(new[s])) % block
                                for s in range(2)]).astype(np.int32)
        nv.kv8_write(rows[:, heads * hd : (heads + kv) * hd], rows[:, (heads + kv) * hd :], arena, torch.from_numpy(slots).cuda(), 0)
        ctx = [d + n for d, n in zip(done, new)]
        out = torch.empty((sum(new), heads * hd), device="cuda", dtype=t)
        nv.kv8_attention(out, rows[:, : heads * hd], arena, dt, torch.tensor([0, new[0], sum(new)], dtype=torch.int32, device="cuda"),
                         torch.tensor(ctx, dtype=torch.int32, device="cuda"), max(new), max(ctx), 0, num_heads=heads,
                         window=window, sinks=sinks, workspace=ws)
        outs[0][done[0] : ctx[0]], outs[1][done[1] : ctx[1]] = out[: new[0]], out[new[0] :]
        done = ctx
    assert done == [150, 77]
    for s in range(2):
        n = done[s]
        pos = np.arange(n)
        back = [torch.empty((n, kv * hd), device="cuda") for _ in "kv"]
        nv.kv8_read(*back, arena, torch.from_numpy((tables[s][pos // block] * block + pos % block).astype(np.int32)).cuda(), 0)
        for got, x in zip(back, (qkv[s][:n, heads * hd : (heads + kv) * hd], qkv[s][:n, (heads + kv) * hd :])):
            c, e = ref.quantise(values64(x).reshape(n, kv, hd), fmt)
            assert np.array_equal(values64(got).reshape(n, kv, hd), ref.dequantise(c, e, fmt))
        k, v = (values64(b).reshape(n, kv, hd) for b in back)
        want, sizes = ref.attention(values64(qkv[s][:n, : heads * hd]).reshape(n, heads, hd), k, v, 0, heads // kv,
                                             1 / math.sqrt(hd), window, sinks)
        off = np.abs(values64(outs[s][:n]).reshape(n, heads, hd) - want)
        assert (off <= ref.tolerance(want, sizes, hd, dtype)).all()
