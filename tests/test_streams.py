"""Sequences on a stream of their own: the loader's work, the copies, the model's
calls and the outputs are ordered one behind the other, whatever stream the
caller has current.

On the CPU the streams are stand-ins that note who waited for whom and which one
was current at each call; on the GPU a loader makes every frame anew (non-
contiguous, out of pinned memory, dropped at once) while the caller's stream is
busy, and the outputs equal those of one stream.
"""
import contextlib
import importlib

import numpy as np
import pytest
import torch

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def S(pkg):
    return importlib.import_module(pkg.__name__ + ".sharding")


class FakeStream:
    device, cuda_stream = None, 0

    def __init__(self, name):
        self.name, self.waited_for = name, []

    def wait_stream(self, other):
        self.waited_for.append(other.name)


@pytest.fixture
def streams(monkeypatch):
    """A caller's stream, which is current, and a side stream."""
    main, side = FakeStream("main"), FakeStream("side")
    now = [main]

    @contextlib.contextmanager
    def use(s):
        now.append(s if s is not None else now[-1])
        yield
        now.pop()

    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: now[-1])
    monkeypatch.setattr(torch.cuda, "stream", use)
    return main, side, now


class FakeModel:
    """Notes the stream that is current at each call, and the one it is given."""

    def __init__(self, T, now):
        self.slots, self.now, self.calls = [None] * T, now, []

    def note(self, stream):
        self.calls.append((self.now[-1].name, None if stream is None else stream.name))

    def encode_frame(self, x, slot, stream=None):
        assert x.is_contiguous()
        self.note(stream)
        self.slots[slot] = float(x.ravel()[0])

    def decode_window(self, slots, beauty, stream=None):
        assert beauty.is_contiguous()
        self.note(stream)
        return beauty.new_tensor([[self.slots[s] for s in slots]])

    def __call__(self, x, stream=None):
        assert x.is_contiguous()
        self.note(stream)
        return x.flatten(1)[:, :1]


class FakeStore:
    def __init__(self, model, h, w):
        self.model, self.held, self.h, self.w = model, {}, h, w

    def park(self, slot, entry, stream=None):
        self.model.note(stream)
        self.held[entry] = self.model.slots[slot]

    def restore(self, entry, slot, stream=None):
        self.model.note(stream)
        self.model.slots[slot] = self.held[entry]


def loader(now, seen, base=0.0):
    def frames(f):
        seen.append(now[-1].name)
        return torch.full((2, 4, 3), base + f).permute(2, 0, 1)  # a copy makes it contiguous
    return frames


def test_clips_in_turn_run_on_the_stream_that_they_are_given(S, streams):
    main, side, now = streams
    m, seen, done = FakeModel(3, now), [], []
    clips = [(loader(now, seen, 100.0 * k), n) for k, n in enumerate((4, 2))]
    got = S.denoise_streams(m, clips, 3, store=FakeStore(m, 2, 4), stream=side,
                            on_frame=lambda k, i, y: done.append(now[-1].name))
    assert set(seen) == {"side"} and set(done) == {"side"} and set(m.calls) == {("side", "side")}
    assert side.waited_for == ["main"] and main.waited_for == [] and now == [main]
    assert len(got) == 6
    for k, i, y in got:
        assert y.tolist() == [100.0 * k + f for f in S.window(i, 3, (4, 2)[k])]
    m.calls.clear(), seen.clear()
    S.denoise_streams(m, clips, 3, store=FakeStore(m, 2, 4))
    assert set(seen) == {"main"} and set(m.calls) == {("main", None)} and main.waited_for == []


@pytest.mark.parametrize("T,cache", [(1, True), (3, True), (3, False)])
def test_a_sequence_runs_on_the_stream_that_it_is_given(S, streams, T, cache):
    main, side, now = streams
    for stream, name in ((side, "side"), (None, "main"), (main, "main")):
        m, seen, done = FakeModel(T, now), [], []
        got = S.denoise_segment(m, loader(now, seen), 5, 1, 0, num_frames=T, stream=stream, cache=cache)
        assert [i for i, _ in got] == list(range(5))
        S.denoise_range(m, loader(now, seen), 5, 1, 3, T, stream, cache, on_frame=lambda i, y: done.append(now[-1].name))
        assert set(seen) == {name} and done == [name] * 2 and {c for c, _ in m.calls} == {name}
        assert now == [main] and main.waited_for == []
    assert side.waited_for == ["main"] * 2


class NoKernels:
    """The library's launchers, not called."""

    def __getattr__(self, name):
        return lambda *args: None


class Noted(torch.Tensor):
    """A tensor that notes the streams that are current when it is copied."""

    def contiguous(self):
        self.seen.append(self.now[-1].name)
        return self.as_subclass(torch.Tensor).contiguous()


@pytest.mark.parametrize("tile", [0, 8])
@pytest.mark.parametrize("flip", [False, True])
def test_whole_sequences_and_tiles_run_on_the_stream_that_they_are_given(pkg, streams, monkeypatch, tile, flip):
    infer = importlib.import_module(pkg.__name__ + ".infer")
    monkeypatch.setattr(infer, "lib", NoKernels)
    monkeypatch.setattr(infer, "check", lambda rc: None)
    main, side, now = streams
    stacked, stack = [], torch.stack
    monkeypatch.setattr(torch, "stack", lambda *a, **k: stacked.append(now[-1].name) or stack(*a, **k))
    m = FakeModel(3, now)
    m.decode_window = lambda slots, beauty, stream=None: m.note(stream) or beauty
    m.__class__ = type("Whole", (FakeModel,), {"__call__": lambda s, x, stream=None: s.note(stream) or x[:, 0]})
    frames = [torch.rand(2, 4, 12).permute(0, 2, 1) for _ in range(4)]
    assert len(infer.denoise_temporal_sequence(m, frames, 3, flip, tile, stream=side)) == 4
    assert set(m.calls) == {("side", "side")} and set(stacked) <= {"side"} and bool(stacked) == (tile > 0)
    assert side.waited_for == ["main"] and now == [main]
    x = torch.rand(1, 3, 16, 12).transpose(2, 3).as_subclass(Noted)
    x.seen, x.now = [], now
    infer.tile_inference(m, x, 8, stream=side)
    assert x.seen == ["side"] and side.waited_for == ["main"] * 2 and main.waited_for == [] and now == [main]


def test_a_cache_is_made_when_its_constructor_returns(pkg, streams, monkeypatch):
    """Its zeros, on the stream that is current, are waited for: later calls may
    be on any stream."""
    Q = importlib.import_module(pkg.__name__ + ".quant")
    main, side, now = streams
    order, zeros = [], torch.zeros

    def filled(*size, device=None, **k):
        order.append("zeros")
        return zeros(*size, **k)

    monkeypatch.setattr(torch, "zeros", filled)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    main.synchronize = lambda: order.append("synchronize")
    capturing = False
    Q.RowCache(2, 3, 8)
    assert order == ["zeros"] * 3 + ["synchronize"]
    order.clear()
    capturing = True  # where it would end the capture
    Q.RowCache(2, 3, 8)
    assert order == ["zeros"] * 3


def temporal(pkg, tmp_path, T=3):
    synth = importlib.import_module(pkg.__name__ + ".synth")
    cfg = synth.NAFConfig(base_channels=8, enc_blocks=(1, 1), middle_blocks=1, dec_blocks=(1, 1))
    return pkg.Model(synth.make_model_dir(str(tmp_path), cfg, 4, "py", T, True)[0])


def host_clip(seed, n, h=62, w=74):
    """Frames (H, W, 3) in pinned memory, as a decoder leaves them."""
    rng = np.random.default_rng(seed)
    return [torch.from_numpy(rng.uniform(0, 1, (h, w, 3)).astype(np.float16)).pin_memory() for _ in range(n)]


def fresh(clip):
    """A loader whose frames nobody else holds."""
    return lambda f: clip[f].to("cuda", non_blocking=True).permute(2, 0, 1)


@gpu
def test_clips_in_turn_with_frames_that_are_loaded_and_dropped(pkg, S, tmp_path):
    m = temporal(pkg, tmp_path)
    clips = [host_clip(s, 5) for s in (1, 2)]
    take = [(fresh(c), 5) for c in clips]
    want = [y.clone() for _, _, y in S.denoise_streams(m, take, 3)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        torch.cuda._sleep(20_000_000)  # the caller's stream is busy when the loop begins
        got = S.denoise_streams(m, take, 3, stream=side, on_frame=lambda k, i, y: torch.zeros(3, 62, 74, device="cuda"))
        side.synchronize()
        for (k, i, y), w in zip(got, want):
            assert torch.equal(y, w), (k, i)
    m.sync()


@gpu
@pytest.mark.parametrize("cache", [True, False])
def test_a_sequence_with_frames_that_are_loaded_and_dropped(pkg, S, tmp_path, cache):
    m = temporal(pkg, tmp_path)
    clip = host_clip(3, 6)
    want = [y.clone() for _, y in S.denoise_segment(m, fresh(clip), 6, 1, 0, num_frames=3, cache=cache)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        torch.cuda._sleep(20_000_000)
        got = S.denoise_segment(m, fresh(clip), 6, 1, 0, num_frames=3, stream=side, cache=cache)
        side.synchronize()
        for (i, y), w in zip(got, want):
            assert torch.equal(y, w), i
    m.sync()


@gpu
def test_a_cache_used_on_another_stream_than_it_was_made_on(pkg):
    Q = importlib.import_module(pkg.__name__ + ".quant")
    side = torch.cuda.Stream()
    x = torch.full((300, 64), 127.0, dtype=torch.float16, device="cuda")
    slots = torch.tensor([300] * 300, device="cuda")  # behind the cache
    for bits in (8, 4):
        torch.cuda.synchronize()
        torch.cuda._sleep(40_000_000)
        cache = Q.RowCache(1, 300, 64, bits=bits)
        cache.write(x, stream=side)
        cache.write(x, slots=slots, stream=side)
        with torch.cuda.stream(side):
            back = cache.read_rows(rows=300)
        with pytest.raises(pkg.DenoiserError):
            cache.sync(stream=side)
        torch.cuda.synchronize()
        assert bool((back == 127).all()) and bool((cache.scales > 0).all())


@gpu
def test_a_cache_made_in_a_capture(pkg):
    Q = importlib.import_module(pkg.__name__ + ".quant")
    x = torch.ones(5, 32, dtype=torch.float16, device="cuda")
    Q.RowCache(2, 5, 32).write(x)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cache = Q.RowCache(2, 5, 32)
        cache.write(x, row0=2)
        out = cache.read_rows(rows=10)
    for _ in range(2):
        x += 1
        g.replay()
        torch.cuda.synchronize()
        assert bool((out[2:7] == x).all()) and not bool(out[:2].any()) and not bool(out[7:].any())
