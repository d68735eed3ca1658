"""Dropout and 4-bit SH rows in a trainer whose calls are spread over streams, parts of an iteration, camera kinds and a densifier."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import view_ops_oracle as O  # noqa: E402
from spirula_studio_b200 import lib as L, scenes  # noqa: E402
from spirula_studio_b200.trainer import DropoutOptions, Trainer  # noqa: E402

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
OPTS = DropoutOptions(splat_rate=0.2, sh_rate=0.4, seed=9)


@pytest.fixture(scope="module", autouse=True)
def device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def scene(n=2500, views=3, w=160, h=112, of="plumbing_50k"):
    cfg = scenes.scaled(scenes.CONFIGS[of], n_splats=n, width=w, height=h, n_views=views)
    cfg.log_scale_mu = -3.0
    cfg.rig = "ring"
    sp = scenes.make_splats(cfg)
    vm, K = scenes.make_cameras(cfg)
    gt = np.stack([scenes.make_target(cfg, v) for v in range(views)]) if not cfg.view_kinds else None
    return cfg, sp, vm, K, gt


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def close(a, b):
    """Rasteriser gradients are summed by reductions in no fixed order: the parity tests' own tolerance."""
    a, b = a.double(), b.double()
    bad = (a - b).abs() > 2e-5 * float(b.abs().max()) + 1e-3 * b.abs()
    return float(bad.double().mean()) <= 1e-3


def raw(stream):
    return C.c_void_p(stream.cuda_stream)


def gradients(cfg, sp, vm, K, gt, **kw):
    tr = Trainer(cfg, sp, device=DEV, **kw)
    tr.views_fwd_bwd(dev(vm), dev(K), dev(gt), len(vm))
    torch.cuda.synchronize()
    out = {k: v.clone() for k, v in tr.grads.items()}
    tr.close()
    return out


def test_views_on_one_stream_and_the_optimiser_on_another():
    cfg, sp, vm, K, gt = scene()
    ref = gradients(cfg, sp, vm, K, gt, view_sh_bits=4, dropout=OPTS)
    tr = Trainer(cfg, sp, device=DEV, view_sh_bits=4, dropout=OPTS)
    d = dev(vm), dev(K), dev(gt)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    tr.views_fwd_bwd(*d, 3, stream=raw(a))
    ready = torch.cuda.Event()
    ready.record(a)
    b.wait_event(ready)
    tr.optimizer_step(3, stream=raw(b))
    torch.cuda.synchronize()
    for k in ref:
        assert close(tr.grads[k], ref[k]), k
        if k not in ("opacities", "features_sh"):        # the dropped arrays; the rotations, e.g., are moved off their gradient (unit norm)
            continue
        # their first moments are a tenth of the gradients' mean that the optimiser read: 1 - 0.9 in fp32 (4 U off), three products, a sum
        want = 0.1 * tr.grads[k].double() / 3
        assert bool(((tr.m1[k].double() - want).abs() <= 16 * O.U * want.abs() + 2.0 ** -126).all()), k
    tr.close()


def test_accumulation_over_parts_streams_and_foreign_terms():
    cfg, sp, vm, K, gt = scene()
    ref = gradients(cfg, sp, vm, K, gt, view_sh_bits=4, dropout=OPTS)
    tr = Trainer(cfg, sp, device=DEV, view_sh_bits=4, dropout=OPTS)
    base = {k: torch.randn(v.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)) * float(ref[k].abs().max()) for k, v in tr.grads.items()}
    for k, v in base.items():
        tr.grads[k].copy_(v)
    d = dev(vm), dev(K), dev(gt)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    last = None
    for i in range(3):                                   # a view at a time, on alternating streams, into what is there
        s = streams[i % 2]
        if last is not None:
            s.wait_event(last)
        tr.views_fwd_bwd(*(t[i:i + 1] for t in d), 1, accumulate=True, stream=raw(s))
        last = torch.cuda.Event()
        last.record(s)
        tr.allreduce_grads()
    torch.cuda.synchronize()
    for k in ref:
        assert close(tr.grads[k], base[k] + ref[k]), k
    tr.close()


def test_renders_from_rows_on_several_streams():
    """Two camera kinds and two streams taking turns while the values change: each image is that of a trainer with its values."""
    cfg, sp, vm, K, _ = scene(n=4000, views=2, of="wide_5m")
    tr = Trainer(cfg, sp, device=DEV)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    start = tr.params["features_sh"].clone()
    torch.cuda.synchronize()
    images, last = [], None
    for i in range(12):
        s = streams[i // 2 % 2]
        if last is not None:
            s.wait_event(last)                           # the change of values waits for the renders of the ones before
        with torch.cuda.stream(s):
            tr.params["features_sh"].copy_(start * (1 + i // 4))
            images.append((i % 2, 1 + i // 4, tr.render(vm[i % 2], K[i % 2], kind=i % 2, sh_bits=4)[0]))
        last = torch.cuda.Event()
        last.record(s)
    torch.cuda.synchronize()
    assert len(tr._render_rows) == 2
    for kind, factor, image in images:
        ref = Trainer(cfg, {**sp, "features_sh": sp["features_sh"] * np.float32(factor)}, device=DEV)
        assert torch.equal(image, ref.render(vm[kind], K[kind], kind=kind, sh_bits=4)[0])
        ref.close()
    tr.close()
