"""The Python binding of the 8-bit cache without a GPU: which stream and device a
call and its default workspace are on, with stand-ins for tensors and torch.cuda;
and the errors that the header states of the formats."""
import contextlib
from types import SimpleNamespace

import pytest


class Tensor:
    """What the binding asks of a CUDA tensor."""

    def __init__(self, *shape, dtype, device=0, stride=None, contiguous=True, size=None):
        self.shape, self.dtype, self.device, self.contiguous = shape, dtype, device, contiguous
        self.strides = stride or (shape[-1], 1)[-len(shape):]
        self.size = size if size is not None else 4

    def get_device(self):
        return self.device

    def dim(self):
        return len(self.shape)

    def stride(self, i):
        return self.strides[i]

    def numel(self):
        n = 1
        for s in self.shape:
            n *= s
        return n

    def element_size(self):
        return self.size

    def is_contiguous(self):
        return self.contiguous

    def data_ptr(self):
        return 4096

    def record_stream(self, stream):
        pass


class World:
    """torch.cuda as the binding sees it, and the calls that reach the library."""

    def __init__(self, monkeypatch, nv):
        import torch
        from nvllm import kv8
        self.current, self.device, self.allocated, self.calls = 1000, 0, [], []
        self.kv8, self.torch, self.layout = kv8, torch, nv.KVLayout(8, 1, 16, 2, 64)

        def library(name):
            def f(*args):
                self.calls.append(SimpleNamespace(name=name, args=args, stream=args[-1], device=self.device))
                return 0
            return f

        @contextlib.contextmanager
        def use(stream):
            before, self.current = self.current, stream.cuda_stream
            yield
            self.current = before

        @contextlib.contextmanager
        def on(index):
            before, self.device = self.device, index
            yield
            self.device = before

        def alloc(*args, **kw):
            self.allocated.append(self.current)
            return Tensor(1 << 20, dtype=torch.uint8, size=1, device=args[-1] if isinstance(args[-1], int) else 0)

        def external(handle, device=None):
            return SimpleNamespace(cuda_stream=handle)
        names = ("nvllm_kv8_attention", "nvllm_kv8_write", "nvllm_kv8_read")
        lib = SimpleNamespace(**{n: library(n) for n in names})
        monkeypatch.setattr(kv8, "_lib", lambda: lib)
        monkeypatch.setattr(kv8, "_DTYPES", {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2})
        monkeypatch.setattr(kv8, "_INT32", torch.int32)
        monkeypatch.setattr(kv8, "_RAW_STREAM", lambda index: self.current + index)
        monkeypatch.setattr(kv8, "_CURRENT_DEVICE", lambda: self.device)
        monkeypatch.setattr(kv8, "kv8_alloc_workspace", alloc)
        monkeypatch.setattr(torch.cuda, "stream", use)
        monkeypatch.setattr(torch.cuda, "device", on)
        monkeypatch.setattr(torch.cuda, "ExternalStream", external)
        monkeypatch.setattr(torch.cuda, "default_stream", lambda device=None: SimpleNamespace(cuda_stream=0))

    def arena(self, index=0):
        return SimpleNamespace(layout=self.layout, index=index, device=index, _ref=None, _lay=None)

    def attention(self, index=0, rows=3, **kw):
        t = self.torch
        x = dict(device=index)
        q, out = (kw.pop(n, Tensor(rows, 128, dtype=t.bfloat16, size=2, **x)) for n in ("query", "out"))
        return self.kv8.kv8_attention(
            out, q, self.arena(index), Tensor(2, 4, dtype=t.int32, **x), Tensor(3, dtype=t.int32, **x),
            Tensor(2, dtype=t.int32, **x), kw.pop("max_query_len", 2), kw.pop("max_context_len", 20), kw.pop("layer", 0), **kw)


@pytest.fixture
def world(monkeypatch, nv):
    return World(monkeypatch, nv)


def test_default_workspace_is_allocated_on_the_calls_stream(world):
    """The allocator orders a block's reuse on the stream that it was allocated on."""
    for stream, handle in ((None, 1000), (2048, 2048), (SimpleNamespace(cuda_stream=4096), 4096), (0, 0)):
        world.attention(stream=stream)
        assert world.calls[-1].stream == handle
        assert world.allocated[-1] == handle
    assert world.current == 1000


def test_calls_run_on_their_tensors_device(world):
    t = world.torch
    world.attention(index=1)
    assert (world.calls[-1].device, world.calls[-1].stream) == (1, 1001)
    rows = Tensor(2, 128, dtype=t.float32, device=1)
    for f in (world.kv8.kv8_write, world.kv8.kv8_read):
        f(rows, rows, world.arena(1), Tensor(2, dtype=t.int32, device=1), 0)
        assert (world.calls[-1].device, world.calls[-1].stream) == (1, 1001)
    assert world.device == 0
    with pytest.raises(ValueError, match="device"):
        world.kv8.kv8_write(rows, rows, world.arena(0), Tensor(2, dtype=t.int32, device=1), 0)


def test_a_workspace_must_be_the_bytes_it_counts(world):
    """An expanded tensor counts elements that it has no memory for."""
    t = world.torch
    good = Tensor(1 << 16, dtype=t.uint8, size=1)
    world.attention(workspace=good)
    assert world.calls[-1].args[-3] == 1 << 16
    n = len(world.calls)
    with pytest.raises(ValueError, match="workspace.*contiguous"):
        world.attention(workspace=Tensor(1 << 16, dtype=t.uint8, size=1, contiguous=False))
    assert len(world.calls) == n


BIG = 1 << 32


@pytest.mark.parametrize("arg", ["max_query_len", "max_context_len", "layer", "window", "sinks"])
@pytest.mark.parametrize("value", [BIG, BIG + 5, 1 << 31, -BIG + 5])
def test_attention_refuses_what_32_bits_do_not_hold(world, arg, value):
    """The C ABI takes int32, and ctypes drops the rest without a word."""
    with pytest.raises(ValueError, match="32 bits"):
        world.attention(**{arg: value})
    assert not world.calls
    world.attention(window=(1 << 31) - 1, sinks=(1 << 31) - 1)
    world.attention(layer=-1)  # the library's to refuse
    assert len(world.calls) == 2


@pytest.mark.parametrize("value", [BIG, -BIG + 1])
def test_moves_and_sizes_refuse_what_32_bits_do_not_hold(world, value):
    t = world.torch
    rows, slots = Tensor(2, 128, dtype=t.float32), Tensor(2, dtype=t.int32)
    for f in (world.kv8.kv8_write, world.kv8.kv8_read):
        with pytest.raises(ValueError, match="32 bits"):
            f(rows, rows, world.arena(), slots, value)
    for i in range(4):
        args = [1, 1, 1, 2]
        args[i] = value
        with pytest.raises(ValueError, match="32 bits"):
            world.kv8.kv8_workspace_size(*args, world.layout)
    assert not world.calls


def test_a_lone_row_has_no_stride(world):
    """One row sliced out of a buffer whose rows are not a multiple of 16 bytes apart."""
    t = world.torch
    q, out = (Tensor(1, 128, dtype=t.bfloat16, size=2, stride=(s, 1)) for s in (387, 1))
    world.attention(query=q, out=out)
    assert (world.calls[-1].args[1], world.calls[-1].args[3]) == (128, 128)
    q, out = (Tensor(2, 128, dtype=t.bfloat16, size=2, stride=(s, 1)) for s in (384, 136))
    world.attention(query=q, out=out)
    assert (world.calls[-1].args[1], world.calls[-1].args[3]) == (136, 384)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_the_stated_errors_of_the_formats(fmt):
    """What include/nvllm.h says of each format's error, over rows whose elements are
    far apart; for E4M3 a relative error alone is not true of the small ones."""
    import numpy as np
    import kv8_ref as ref
    rng = np.random.default_rng(5)
    x = rng.standard_normal((400, 64)) * 2.0 ** rng.integers(-20, 1, (400, 64)) * 2.0 ** rng.integers(-40, 40, (400, 1))
    codes, e = ref.quantise(x, fmt)
    off, step = np.abs(ref.dequantise(codes, e, fmt) - x), 2.0 ** e[:, None].astype(np.float64)
    if fmt == "e4m3":
        assert (off <= np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10 * step)).all()
        assert (off[np.abs(x) >= 2.0 ** -6 * step] <= 2.0 ** -4 * np.abs(x)[np.abs(x) >= 2.0 ** -6 * step]).all()
        assert (off > 2.0 ** -4 * np.abs(x)).any()
    else:
        assert (off <= np.abs(x).max(1, keepdims=True) / 127).all()
