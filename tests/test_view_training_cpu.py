"""What a Trainer asks of the library around an iteration's views, without a GPU: a stand-in for the library that works on host memory
and notes every call with its stream.  Its views' gradients are functions of the arrays that the views are given, its dropout calls are
the oracle's."""
import contextlib
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import view_ops_oracle as O  # noqa: E402
from spirula_studio_b200 import lib as L, scenes, trainer as T  # noqa: E402
from spirula_studio_b200.trainer import DropoutOptions, Trainer  # noqa: E402

N = 37


def floats(address, count):
    address = getattr(address, "value", address)
    return np.ctypeslib.as_array((C.c_float * count).from_address(address))


def handle(stream):
    return getattr(stream, "value", stream) or 0


class StandIn:
    """Entry points without a method of their own succeed and do nothing."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            own = getattr(self, "_" + name, None) if not name.startswith("_") else None
            if own is not None:
                own(*args)
            self.calls.append((name, args))
            return 0
        if name.startswith("_"):
            raise AttributeError(name)
        return call

    def names(self):
        return [n for n, _ in self.calls]

    def _ssb_step_views(self, step, params, shq, vm, K, gt, views, grads, accumulate, losses, stream):
        self._ssb_step_views_gated(step, params, shq, vm, K, gt, views, None, grads, accumulate, losses, stream)

    def _ssb_step_views_gated(self, step, params, shq, vm, K, gt, views, ready, grads, accumulate, losses, stream):
        if views == 0:
            return
        p, g = params._obj, grads._obj
        for k, w in (("means", 3), ("quats", 4), ("scales", 3), ("opacities", 1), ("features_dc", 3), ("features_sh", 45)):
            out = floats(getattr(g, k), N * w)
            value = views * view_gradient(k, floats(getattr(p, k), N * w))
            out[:] = out + value if accumulate else value

    def _ssb_dropout(self, x, first, count, group, d, y, stream):
        d = d._obj
        floats(y, count)[:] = O.dropout(floats(x, count).copy(), first, group, d.rate, d.seed, d.offset)

    def _ssb_dropout_opacities(self, x, first, count, d, y, stream):
        d = d._obj
        floats(y, count)[:] = O.dropout_opacities(floats(x, count).copy(), first, d.rate, d.seed, d.offset)[0]

    def _ssb_dropout_opacities_bwd(self, x, v, first, count, d, out, stream):
        d = d._obj
        floats(out, count)[:] = O.dropout_opacities(floats(x, count).copy(), first, d.rate, d.seed, d.offset)[1] * floats(v, count)


def view_gradient(name, read):
    """One view's gradient of the array that it reads."""
    return (0.5 * read + 1.0) if name in ("opacities", "features_sh") else np.full_like(read, 2.0)


@pytest.fixture
def fake(monkeypatch):
    lib = StandIn()
    monkeypatch.setattr(L, "load", lambda: lib)
    monkeypatch.setattr(Trainer, "_on", lambda self, stream: contextlib.nullcontext(), raising=False)
    return lib


def make(fake, kinds=1, **kw):
    cfg = scenes.scaled(scenes.CONFIGS["plumbing_50k" if kinds == 1 else "wide_5m"], n_splats=N, width=64, height=48, n_views=2)
    tr = Trainer(cfg, scenes.make_splats(cfg), device="cpu", **kw)
    assert len(tr.handles) == kinds
    fake.calls.clear()
    return tr


def views(tr, count=2, **kw):
    tr.views_fwd_bwd(torch.zeros(count, 16), torch.zeros(count, 4), torch.zeros(count, 1), count, **kw)


OPTS = DropoutOptions(splat_rate=0.3, sh_rate=0.4, sh_group=3, seed=21)


def stored_gradients(tr, count, opts=OPTS):
    """The chain rule through both dropouts, in 64 bits."""
    i, p = tr.iteration, {k: v.numpy().copy() for k, v in tr.params.items()}
    want = {k: count * view_gradient(k, v).astype(np.float64) for k, v in p.items()}
    if opts.splat_rate:
        y, slope, _ = O.dropout_opacities(p["opacities"], 0, opts.splat_rate, 2 * opts.seed, i)
        want["opacities"] = slope * (count * view_gradient("opacities", y))
    if opts.sh_rate:
        mask = O.dropout(np.ones(N * 45, np.float32), 0, opts.sh_group, opts.sh_rate, 2 * opts.seed + 1, i)
        want["features_sh"] = mask * (count * view_gradient("features_sh", mask * p["features_sh"]))
    return want


def same(got, want):
    """A handful of roundings: the copy the views read, the view's own two, the mask's, the slope's, a sum."""
    for k in want:
        assert np.allclose(got[k].numpy(), want[k], rtol=16 * O.U, atol=16 * O.U * np.abs(want[k]).max()), k


def test_conversion_runs_in_the_views_call_on_its_stream(fake):
    """A caller who orders two streams by an event between the calls must find the gradients complete at that event."""
    tr = make(fake, dropout=OPTS, view_sh_bits=4)
    want = stored_gradients(tr, 2)
    views(tr, stream=0x10)
    launched = [n for n in fake.names() if "dropout" in n]
    assert sorted(launched) == ["ssb_dropout", "ssb_dropout", "ssb_dropout_opacities", "ssb_dropout_opacities_bwd"]
    assert all(handle(a[-1]) == 0x10 for n, a in fake.calls)
    same(tr.grads, want)
    fake.calls.clear()
    tr.allreduce_grads()
    tr.optimizer_step(2, stream=0x20)
    assert not [n for n in fake.names() if "dropout" in n] and all(handle(a[-1]) == 0x20 for n, a in fake.calls)
    same(tr.grads, want)


@pytest.mark.parametrize("opts", [OPTS, DropoutOptions(splat_rate=0.5, seed=3), DropoutOptions(sh_rate=0.5, sh_group=45, seed=4)])
def test_accumulation_leaves_the_other_terms_alone(fake, opts):
    tr = make(fake, dropout=opts)
    want = stored_gradients(tr, 2, opts)
    for k, g in tr.grads.items():
        g.copy_(torch.linspace(-3, 3, g.numel()))
    base = {k: g.numpy().astype(np.float64) for k, g in tr.grads.items()}
    views(tr, accumulate=True)                                      # into what the caller put there
    same(tr.grads, {k: base[k] + want[k] for k in want})
    tr.allreduce_grads()
    views(tr, accumulate=True)                                      # after the exchange of the first part
    same(tr.grads, {k: base[k] + 2 * want[k] for k in want})
    for g in tr.grads.values():
        g += 1.0                                                    # a regulariser of the caller's
    tr.optimizer_step(2)
    same(tr.grads, {k: base[k] + 2 * want[k] + 1.0 for k in want})
    again = stored_gradients(tr, 2, opts)                           # the next iteration draws its own masks
    views(tr)
    same(tr.grads, again)


def test_accumulating_views_read_the_parameters_as_they_are(fake):
    tr = make(fake, dropout=OPTS)
    first = stored_gradients(tr, 2)
    views(tr)
    tr.params["features_sh"].mul_(-2.0)
    tr.params["opacities"].add_(0.25)
    second = stored_gradients(tr, 2)
    views(tr, accumulate=True)
    same(tr.grads, {k: first[k] + second[k] for k in first})


def test_camera_kinds_of_an_iteration_share_one_copy_and_one_conversion(fake):
    tr = make(fake, kinds=2, dropout=OPTS)
    want = stored_gradients(tr, 5)
    batch = lambda kind, n: (kind, torch.zeros(n, 16), torch.zeros(n, 4), torch.zeros(n, 1), n)
    tr.step_device_kinds([batch(0, 2), batch(1, 0), batch(1, 3)], 5)
    assert fake.names().count("ssb_dropout") == 2 and fake.names().count("ssb_dropout_opacities_bwd") == 1
    same(tr.grads, want)
    tr.step_device_kinds([], 5)
    assert not any(g.any() for g in tr.grads.values())


@pytest.mark.parametrize("accumulate", [False, True])
def test_a_call_without_views_leaves_the_gradients(fake, accumulate):
    tr = make(fake, dropout=OPTS)
    want = stored_gradients(tr, 2)
    views(tr)
    views(tr, count=0, accumulate=accumulate)
    same(tr.grads, want)


def test_buffers_are_allocated_on_the_stream_that_writes_them(fake, monkeypatch):
    """torch's allocator orders the reuse of memory by the stream it is asked on."""
    tr = make(fake, dropout=OPTS, view_sh_bits=4)
    current, asked = [None], []

    @contextlib.contextmanager
    def on(self, stream):
        before, current[0] = current[0], handle(stream)
        yield
        current[0] = before
    monkeypatch.setattr(Trainer, "_on", on, raising=False)
    for name in ("empty", "empty_like"):
        real = getattr(torch, name)
        monkeypatch.setattr(torch, name, lambda *a, real=real, **kw: asked.append(current[0]) or real(*a, **kw))
    views(tr, stream=0x10)
    assert asked == [0x10] * 3                       # opacities, SH values, rows
    del asked[:]
    views(tr, accumulate=True, stream=0x20)
    assert asked == [0x20] * 2                       # their gradients
    del asked[:]
    views(tr, accumulate=True, stream=0x20)
    assert not asked


def test_rows_of_renders_on_several_streams(fake, monkeypatch):
    """A camera kind's renders share a buffer and are ordered by an event; those of another kind have their own."""
    tr = make(fake, kinds=2)
    log = fake.calls

    class Stream:
        def __init__(self, handle):
            self.cuda_stream = handle

        def wait_event(self, event):
            log.append(("wait", (event.recorded, self.cuda_stream)))

    class Event:
        recorded = None

        def record(self, stream):
            self.recorded = (stream.cuda_stream, len(log))
            log.append(("record", (stream.cuda_stream,)))

    a, b = Stream(0x10), Stream(0x20)
    monkeypatch.setattr(torch.cuda, "Event", Event)
    encoded = []
    for stream, kind in ((a, 0), (b, 1), (b, 0), (a, 1), (a, 0)):
        monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None, stream=stream: stream)
        del log[:]
        tr.render(np.eye(4), np.ones(4), kind=kind, sh_bits=4)
        names = fake.names()
        first = kind not in [k for k, _, _ in encoded]
        assert names == ([] if first else ["wait"]) + ["ssb_quant_encode", "ssb_step_render", "record"]
        if not first:
            last = [s for k, s, _ in encoded if k == kind][-1]
            assert log[0][1][0][0] == last.cuda_stream
        assert all(handle(args[-1]) == stream.cuda_stream for _, args in log)
        encoded.append((kind, stream, handle(dict(log)["ssb_quant_encode"][3])))
    assert len({p for _, _, p in encoded}) == 2 and len({(k, p) for k, _, p in encoded}) == 2


@pytest.mark.parametrize("bad", [dict(splat_rate=1.0 - 1e-9), dict(sh_rate=1.0 - 2.0 ** -26), dict(sh_rate=float("nan")), dict(splat_rate=1e300),
                                 dict(sh_rate=0.1, sh_group=2 ** 31), dict(sh_rate=0.1, sh_group=2 ** 32 + 3), dict(sh_rate=0.1, sh_group=0)])
def test_options_that_the_library_cannot_take_are_refused_when_they_are_set(fake, bad):
    """A rate that is one in fp32, a group that 32 bits would cut off: refused here, not in the middle of a run, nor taken for another."""
    with pytest.raises(ValueError):
        make(fake, dropout=DropoutOptions(**bad))
    make(fake, dropout=DropoutOptions(splat_rate=1.0 - 2.0 ** -24, sh_rate=0.0, sh_group=2 ** 31 - 1))


def test_every_rank_draws_the_masks_of_the_whole_array(fake, monkeypatch):
    """Ranks hold the same parameters and see other views: what their views read must be the same copies."""
    monkeypatch.setattr(torch.distributed, "all_reduce", lambda *a, **kw: None)
    drawn = []
    for rank in range(2):
        tr = make(fake, dropout=OPTS, world_size=2, rank=rank, grad_sync="nccl")
        for _ in range(2):
            fake.calls.clear()
            views(tr, count=1 + rank)
            tr.allreduce_grads()
            tr.optimizer_step(3)
            for name, args in fake.calls:
                if "dropout" in name:
                    d = [a._obj for a in args if isinstance(getattr(a, "_obj", None), L.SsbDropout)][0]
                    plain = [handle(a) for a in args if not hasattr(a, "_obj")]
                    sizes = [a for a in plain if a in (0, N, 45 * N, OPTS.sh_group)]
                    drawn.append((rank, name, d.rate, d.seed, d.offset, tuple(sizes)))
    mine = [[c[1:] for c in drawn if c[0] == r] for r in range(2)]
    assert mine[0] == mine[1] and len(mine[0]) == 8
    assert [c[3] for c in mine[0]] == [0] * 4 + [1] * 4               # the iteration's number
    assert {(c[1], c[2]) for c in mine[0]} == {(float(np.float32(OPTS.splat_rate)), 2 * OPTS.seed), (float(np.float32(OPTS.sh_rate)), 2 * OPTS.seed + 1)}
    assert all(0 in c[4] and (N in c[4] or 45 * N in c[4]) for c in mine[0])
