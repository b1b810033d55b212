"""The 8-bit paged KV cache without a GPU: refusals before any launch, workspace
sizes, and the reference quantiser against torch's casts."""
import ctypes

import numpy as np
import pytest

import kv8_ref as ref

VP = ctypes.c_void_p


@pytest.fixture(scope="module")
def lib(nv):
    from nvllm import kv8
    return kv8._lib()


def arena(fmt=0, **kw):
    from nvllm import kv8
    a = kv8._Arena(256, 256, 256, 256, fmt)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


MOVE = dict(key=VP(256), value=VP(256), dtype=0, ks=128, vs=128, arena=arena(), slots=VP(256), n=4, layer=0)


@pytest.mark.parametrize("which", ["nvllm_kv8_write", "nvllm_kv8_read"])
@pytest.mark.parametrize("change,status", [
    (dict(dtype=3), "INVALID"), (dict(dtype=-1), "INVALID"), (dict(ks=127), "INVALID"), (dict(vs=0), "INVALID"),
    (dict(key=None), "INVALID"), (dict(value=None), "INVALID"), (dict(slots=None), "INVALID"),
    (dict(n=-1), "INVALID"), (dict(n=1 << 40), "INVALID"), (dict(n=1 << 31), "INVALID"), (dict(layer=2), "INVALID"), (dict(layer=-1), "INVALID"),
    (dict(arena=arena(2)), "INVALID"), (dict(arena=arena(k_codes=264)), "INVALID"), (dict(arena=arena(v_exps=None)), "INVALID"),
    (dict(n=0, key=None), "OK")])
def test_moves_refuse(nv, lib, which, change, status):
    a = {**MOVE, **change}
    lay = nv.KVLayout(16, 2, 16, 2, 64)
    rc = getattr(lib, which)(a["key"], a["value"], a["dtype"], a["ks"], a["vs"], ctypes.byref(a["arena"]), a["slots"], a["n"],
                             a["layer"], ctypes.byref(lay), None)
    assert rc == (nv.OK if status == "OK" else nv.ERR_INVALID)


def test_moves_refuse_layouts(nv, lib):
    a = MOVE
    for lay, want in ((nv.KVLayout(16, 2, 16, 2, 48), nv.ERR_UNSUPPORTED), (nv.KVLayout(0, 2, 16, 2, 64), nv.ERR_INVALID)):
        assert lib.nvllm_kv8_write(a["key"], a["value"], 0, 128, 128, ctypes.byref(arena()), a["slots"], 4, 0, ctypes.byref(lay),
                                   None) == want
    assert lib.nvllm_kv8_write(a["key"], a["value"], 0, 128, 128, None, a["slots"], 4, 0,
                               ctypes.byref(nv.KVLayout(16, 2, 16, 2, 64)), None) == nv.ERR_INVALID


ATT = dict(out=VP(256), os=256, q=VP(256), qs=256, dtype=1, arena=arena(), tables=VP(256), width=4, cu=VP(256), ctx=VP(256),
           seqs=2, max_q=8, max_ctx=64, heads=4, layer=1, scale=0.1, window=0, sinks=0, ws=VP(256), bytes=1 << 40)


@pytest.mark.parametrize("change,status", [
    (dict(dtype=5), "INVALID"), (dict(os=255), "INVALID"), (dict(qs=260), "INVALID"), (dict(out=VP(264)), "INVALID"),
    (dict(q=None), "INVALID"), (dict(tables=None), "INVALID"), (dict(cu=None), "INVALID"), (dict(ctx=None), "INVALID"),
    (dict(heads=3), "INVALID"), (dict(heads=1), "INVALID"), (dict(heads=0), "INVALID"), (dict(layer=2), "INVALID"),
    (dict(max_q=0), "INVALID"), (dict(max_q=65), "INVALID"), (dict(max_ctx=65), "INVALID"), (dict(width=0), "INVALID"),
    (dict(window=-1), "INVALID"), (dict(sinks=-1), "INVALID"), (dict(scale=0.0), "INVALID"), (dict(scale=float("nan")), "INVALID"),
    (dict(scale=float("inf")), "INVALID"), (dict(seqs=-1), "INVALID"), (dict(seqs=1 << 20), "INVALID"), (dict(arena=arena(7)), "INVALID"),
    (dict(arena=arena(v_codes=8)), "INVALID"), (dict(ws=None), "WORKSPACE"), (dict(ws=VP(128)), "WORKSPACE"),
    (dict(bytes=0), "WORKSPACE"), (dict(seqs=0, out=None, q=None), "OK")])
def test_attention_refuses(nv, lib, change, status):
    a = {**ATT, **change}
    lay = nv.KVLayout(16, 2, 16, 2, 64)
    rc = lib.nvllm_kv8_attention(a["out"], a["os"], a["q"], a["qs"], a["dtype"], ctypes.byref(a["arena"]), a["tables"], a["width"],
                                 a["cu"], a["ctx"], a["seqs"], a["max_q"], a["max_ctx"], a["heads"], a["layer"], a["scale"],
                                 a["window"], a["sinks"], a["ws"], a["bytes"], ctypes.byref(lay), None)
    assert rc == (nv.OK if status == "OK" else getattr(nv, "ERR_" + status))


def test_workspace_sizes(nv):
    lay = nv.KVLayout(1024, 1, 16, 8, 128)
    sizes = [nv.kv8_workspace_size(s, q, c, 32, lay) for s, q, c in ((1, 1, 1), (64, 1, 4096), (64, 300, 4096), (1, 4096, 16384))]
    assert all(n > 0 and n % 256 == 0 for n in sizes)
    assert nv.kv8_workspace_size(1, 1, 1, 9, lay) == 0
    assert nv.kv8_workspace_size(1, 2, 1, 8, lay) == 0
    assert nv.kv8_workspace_size(1, 1, 1, 8, nv.KVLayout(4, 1, 16, 8, 96)) == 0


@pytest.mark.parametrize("kv,heads,hd", [(1, 1, 64), (8, 32, 128), (32, 32, 128), (2, 32, 256), (4, 4, 32), (600, 600, 64)])
def test_a_workspace_serves_every_smaller_call(nv, kv, heads, hd):
    lay = nv.KVLayout(1 << 16, 1, 16, kv, hd)
    sizes = [(s, q, c) for s in (1, 3, 64, 700) for q in (1, 2, 7, 33, 300, 4096) for c in (1, 300, 512, 513, 1280, 5000, 70000) if q <= c]
    size = {k: nv.kv8_workspace_size(*k, heads, lay) for k in sizes}
    for a in sizes:
        for b in sizes:
            if all(x <= y for x, y in zip(a, b)):
                assert size[a] <= size[b], (a, b)


def test_arena_checks_its_tensors(nv):
    import torch
    lay = nv.KVLayout(2, 1, 16, 2, 64)
    k = torch.zeros(lay.arena_shape(), dtype=torch.int8)
    e = torch.zeros((2, 1, 2, 16), dtype=torch.int8)
    with pytest.raises(ValueError, match="CUDA"):
        nv.KV8Arena(lay, k, k, e, e)
    with pytest.raises(ValueError, match="float8_e4m3fn or int8"):
        nv.KV8Arena(lay, k.float(), k, e, e)
    with pytest.raises(ValueError, match="shape"):
        nv.KV8Arena(lay, k[:1], k, e, e)
    with pytest.raises(ValueError, match="int8"):
        nv.KV8Arena(lay, k, k.view(torch.float8_e4m3fn), e, e)
    with pytest.raises(ValueError, match="unknown format"):
        nv.KV8Arena.alloc(lay, 5)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_reference_quantiser(fmt):
    """The reference against torch's own casts of the scaled rows."""
    import torch
    rng = np.random.default_rng(1)
    x = rng.standard_normal((50, 64)).astype(np.float32) * 2.0 ** rng.integers(-30, 30, (50, 1)).astype(np.float32)
    c, e = ref.quantise(x.astype(np.float64), fmt)
    y = torch.from_numpy(x * np.exp2(-e.astype(np.float32))[:, None])
    want = y.to(torch.float8_e4m3fn).view(torch.uint8) if fmt == "e4m3" else y.round().to(torch.int8).view(torch.uint8)
    assert np.array_equal(c, want.numpy())
    top = np.abs(ref.code_values(c, fmt)).max(-1)
    assert (top <= ref.MAX[fmt]).all() and (top > ref.MAX[fmt] / 2 * 0.9).all()
