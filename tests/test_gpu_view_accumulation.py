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


def test_densification_under_dropout_works_on_the_stored_parameters():
    """Relocation and growth happen between iterations whose views read dropped copies and rows: the parameters stay those of a
    trainer that keeps its logits itself, unused slots stay unused."""
    from spirula_studio_b200.densify import DensifyConfig, Densifier
    cfg, sp, vm, K, gt = scene(n=3000)
    start = 2000
    sp["opacities"][:start:17] = -8.0                    # some dead splats among the ones in use
    host = [torch.from_numpy(np.ascontiguousarray(a)).pin_memory() for a in (vm, K, gt)]
    tr = Trainer(cfg, sp, device=DEV, view_sh_bits=4, dropout=OPTS)
    dc = DensifyConfig(refine_start_iter=1, refine_stop_iter=1000, refine_every=3, growth_factor=1.1, noise_lr=0.0)
    dn = Densifier(tr, dc, start)
    grown = 0
    for step in range(8):
        dn.before_step()
        before = {k: v.clone() for k, v in tr.params.items()}
        count = dn.count
        tr.train_step(*host, 3)
        drop = dev(O.dropped(0, cfg.n_splats, 1, OPTS.splat_rate, 2 * OPTS.seed, step))
        assert not tr.grads["means"].view(-1, 3)[drop].any() and not dn.radii[drop].any()      # out of this iteration's views
        assert not any(g.view(cfg.n_splats, -1)[count:].any() for g in tr.grads.values())      # nor do unused slots appear in them
        # Adam moves a logit by at most its bias-corrected rate: none has become the logit of a dropped splat, none was compensated
        # for the rate (0.22 of a logit and more)
        moved = (tr.params["opacities"] - before["opacities"]).abs()[:count]
        assert float(moved.max()) <= 3.2 * cfg.lrs["lr_opacities"]
        stepped = {k: v.clone() for k, v in tr.params.items()}
        added = dn.after_step(step, 8)
        grown += added
        refined = step > dc.refine_start_iter and step % dc.refine_every == 0
        assert (added > 0) == refined
        if refined:
            op = tr.params["opacities"][:dn.count]
            assert float(op.min()) > -10.0               # relocated and new splats start from stored logits, none from a dropped one
            assert float((torch.sigmoid(op) <= dc.min_opacity).double().mean()) < 0.01
        else:
            assert torch.equal(tr.params["features_sh"], stepped["features_sh"])
        assert bool((tr.params["opacities"][dn.count:] == -30.0).all())
    assert grown > 0
    for k, v in tr.params.items():
        assert bool(torch.isfinite(v.view(cfg.n_splats, -1)[:dn.count]).all()), k
    tr.close()


def test_splat_dropout_over_sixteen_bit_sh_values():
    """Opacities are fp32 whatever the SH values are stored in."""
    cfg, sp, vm, K, gt = scene()
    cfg.sh_value_bits, cfg.sh_optim_bits = 16, 8
    opts = DropoutOptions(splat_rate=0.3, seed=5)
    got = gradients(cfg, sp, vm, K, gt, dropout=opts)
    op, slope, _ = O.dropout_opacities(sp["opacities"], 0, 0.3, 10, 0)
    ref = gradients(cfg, {**sp, "opacities": op.astype(np.float32)}, vm, K, gt)
    ref["opacities"] = ref["opacities"] * dev(slope).float()
    drop = dev(O.dropped(0, cfg.n_splats, 1, 0.3, 10, 0))
    for k in got:
        assert close(got[k], ref[k]), k
        assert not got[k].view(cfg.n_splats, -1)[drop].any(), k
