"""Dropout and 4-bit SH rows where a user meets them: the projection calls, the step, the trainer, splat.ply."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import view_ops_oracle as O  # noqa: E402
from spirula_studio_b200 import lib as L, scenes  # noqa: E402
from spirula_studio_b200.trainer import DropoutOptions, OptimOptions, Trainer  # noqa: E402

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(scope="module")
def lib():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return L.load()


def scene(n=3001, views=3, w=160, h=112):
    cfg = scenes.scaled(scenes.CONFIGS["plumbing_50k"], n_splats=n, width=w, height=h, n_views=views)
    cfg.log_scale_mu = -3.0
    cfg.rig = "ring"
    sp = scenes.make_splats(cfg)
    vm, K = scenes.make_cameras(cfg)
    gt = np.stack([scenes.make_target(cfg, v) for v in range(views)])
    return cfg, sp, vm, K, gt


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def rows_of(lib, sh):
    rows = torch.zeros(sh.shape[0], 32, dtype=torch.uint8, device=DEV)
    L.check(lib.ssb_quant_encode(L.ptr(sh), sh.shape[0] * 45, 4, L.ptr(rows), None, None))
    vals = torch.empty(sh.shape[0], 45, device=DEV)
    L.check(lib.ssb_quant_decode(L.ptr(rows), None, sh.shape[0] * 45, 4, L.ptr(vals), None))
    return rows, vals


@pytest.mark.parametrize("n", [1, 128, 3001])
@pytest.mark.parametrize("model,degree", [(0, 3), (0, 1), (1, 3), (3, 3)])
def test_projection_of_rows_equals_projection_of_their_values(lib, n, model, degree):
    """Decoding is exact, so both read the same numbers and every output is the same bit for bit."""
    cfg, sp, vm, K, _ = scene(n)
    t = {k: dev(v) for k, v in sp.items()}
    rows, vals = rows_of(lib, t["features_sh"])
    d_vm, d_K = dev(vm), dev(K)
    views = 3
    cams = L.cameras_struct(d_vm, d_K, cfg.width, cfg.height, model=model, sh_degree=degree)
    shq = L.shq_struct(rows, None, 4, 0)
    outs = []
    for struct, q in ((L.splats_struct({**t, "features_sh": vals}), None), (L.splats_struct({**t, "features_sh": None}), C.byref(shq))):
        aabb, depths, rec = (torch.zeros(views * n, k, device=DEV) for k in (4, 1, 12))
        L.check(lib.ssb_project_fwd(C.byref(struct), q, n, C.byref(cams), L.ptr(aabb), L.ptr(depths), None, L.ptr(rec), None))
        v_rec = torch.randn(views * n, 12, device=DEV, generator=torch.Generator(device=DEV).manual_seed(5))
        grads = {k: torch.zeros_like(v) for k, v in t.items()}
        g = L.splats_struct(grads)
        L.check(lib.ssb_project_bwd(C.byref(struct), q, n, C.byref(cams), L.ptr(aabb), L.ptr(v_rec), C.byref(g), 0, None))
        one = L.cameras_struct(d_vm, d_K, cfg.width, cfg.height, model=model, sh_degree=degree, count=1)
        single = {k: torch.zeros_like(v) for k, v in t.items()}
        g1 = L.splats_struct(single)
        L.check(lib.ssb_project_bwd(C.byref(struct), q, n, C.byref(one), L.ptr(aabb), L.ptr(v_rec), C.byref(g1), 0, None))
        ws = torch.zeros(lib.ssb_project_fwd_packed_workspace_bytes(n, views), dtype=torch.uint8, device=DEV)
        paabb, pdep, prec = (torch.zeros(views * n, k, device=DEV) for k in (4, 1, 12))
        ci, gi = (torch.zeros(views * n, dtype=torch.int32, device=DEV) for _ in range(2))
        cnt = torch.zeros(1, dtype=torch.int64, device=DEV)
        L.check(lib.ssb_project_fwd_packed(C.byref(struct), q, n, C.byref(cams), L.ptr(ws), ws.numel(), L.ptr(paabb), L.ptr(pdep), None, L.ptr(prec),
                                           L.ptr(ci), L.ptr(gi), views * n, L.ptr(cnt), None, None))
        pgrads = {k: torch.zeros_like(v) for k, v in t.items()}
        gp = L.splats_struct(pgrads)
        ws2 = torch.zeros(lib.ssb_project_bwd_packed_workspace_bytes(n, views), dtype=torch.uint8, device=DEV)
        L.check(lib.ssb_project_bwd_packed(C.byref(struct), q, n, C.byref(cams), L.ptr(paabb), L.ptr(v_rec), L.ptr(ci), L.ptr(gi), L.ptr(cnt), views * n,
                                           L.ptr(ws2), ws2.numel(), C.byref(gp), 0, None))
        torch.cuda.synchronize()
        outs.append([aabb, depths, rec, *grads.values(), *single.values(), *pgrads.values(), paabb, pdep, prec, cnt])
    assert n == 1 or int(outs[0][-1]) > n // 4
    for a, b in zip(*outs):
        assert torch.equal(a.reshape(-1).view(torch.int32 if a.dtype == torch.float32 else a.dtype), b.reshape(-1).view(torch.int32 if b.dtype == torch.float32 else b.dtype))


def test_projected_colour_is_the_product_plus_half(lib):
    """ssb_sh_eval_fwd against the colours inside the projection's records."""
    cfg, sp, vm, K, _ = scene(2000)
    t = {k: dev(v) for k, v in sp.items()}
    rows, vals = rows_of(lib, t["features_sh"])
    shq = L.shq_struct(rows, None, 4, 0)
    struct = L.splats_struct({**t, "features_sh": None})
    d_vm, d_K = dev(vm), dev(K)
    cams = L.cameras_struct(d_vm, d_K, cfg.width, cfg.height)
    aabb, depths, rec = (torch.zeros(3 * 2000, k, device=DEV) for k in (4, 1, 12))
    L.check(lib.ssb_project_fwd(C.byref(struct), C.byref(shq), 2000, C.byref(cams), L.ptr(aabb), L.ptr(depths), None, L.ptr(rec), None))
    out = torch.empty(3 * 2000, 3, device=DEV)
    L.check(lib.ssb_sh_eval_fwd(C.byref(struct), C.byref(shq), 2000, C.byref(cams), L.ptr(out), None))
    keep = aabb[:, 2] > aabb[:, 0]
    assert int(keep.sum()) > 1000
    # both are fp32 evaluations with the oracle's bound around the same number (the projection takes the direction from
    # mean + R^T t with |R^T t| <= 4 in one float, another 4 U of 3 units of distance); values stay below 4
    _, tol = O.sh_eval(sp["means"], sp["features_dc"], vals.cpu().numpy().reshape(-1, 15, 3), vm)
    tol = torch.from_numpy(3 * tol + 4 * O.U).reshape(-1, 3).to(DEV)
    want = (out.double() + 0.5).clamp_min(0)
    assert bool(((rec[:, 8:11].double() - want).abs() <= tol)[keep].all())


def pinned(*arrays):
    return [torch.from_numpy(np.ascontiguousarray(a)).pin_memory() for a in arrays]


def grads_of(tr, gt, vm, K):
    tr.views_fwd_bwd(dev(vm), dev(K), dev(gt), len(vm))
    tr.allreduce_grads()
    torch.cuda.synchronize()
    return {k: v.clone() for k, v in tr.grads.items()}


def close(a, b, scale=None):
    """Rasteriser gradients are summed by reductions in no fixed order: the parity tests' own tolerance."""
    a, b = a.double(), b.double()
    s = float(b.abs().max()) if scale is None else scale
    bad = (a - b).abs() > 2e-5 * s + 1e-3 * b.abs()
    return float(bad.double().mean()) <= 1e-3


def test_trainer_dropout_is_training_on_the_dropped_parameters(lib):
    cfg, sp, vm, K, gt = scene()
    n = cfg.n_splats
    tr = Trainer(cfg, sp, device=DEV, dropout=DropoutOptions(splat_rate=0.3, sh_rate=0.2, sh_group=3, seed=77))
    tr.iteration = 5
    before = {k: v.clone() for k, v in tr.params.items()}
    got = grads_of(tr, gt, vm, K)
    for k in before:
        assert torch.equal(before[k], tr.params[k])                       # the stored parameters are read only
    # the same step by a plain trainer on the dropped parameters, and the chain rule on its gradients
    op, slope, _ = O.dropout_opacities(sp["opacities"], 0, 0.3, 154, 5)
    sh = O.dropout(sp["features_sh"].reshape(-1), 0, 3, 0.2, 155, 5)
    plain = Trainer(cfg, {**sp, "opacities": op.astype(np.float32), "features_sh": sh.astype(np.float32)}, device=DEV)
    ref = grads_of(plain, gt, vm, K)
    drop = O.dropped(0, n, 1, 0.3, 154, 5)
    assert 0.25 < drop.mean() < 0.35
    ref["opacities"] = ref["opacities"] * dev(slope).float()
    ref["features_sh"] = dev(O.dropout(ref["features_sh"].cpu().numpy(), 0, 3, 0.2, 155, 5)).float()
    for k in got:
        assert close(got[k], ref[k]), k
        assert not got[k].view(n, -1)[dev(drop)].any(), k                 # a dropped splat gets no gradient at all
    assert abs(float(tr.losses[2]) - float(plain.losses[2])) <= 1e-5 * abs(float(plain.losses[2]))
    # the optimiser works on the stored parameters
    tr.optimizer_step(3)
    moved = (tr.params["means"] - before["means"]).view(n, 3).abs().sum(1) > 0
    assert not bool(moved[dev(drop)].any()) and int(moved.sum()) > n // 4
    # render() drops nothing
    base = Trainer(cfg, {k: tr.params[k].cpu().numpy().reshape(np.shape(sp[k])) for k in sp}, device=DEV)
    assert torch.equal(tr.render(vm[0], K[0])[0], base.render(vm[0], K[0])[0])
    for t in (tr, plain, base):
        t.close()


def test_trainer_dropout_masks_follow_the_iteration_and_the_schedule(lib):
    cfg, sp, vm, K, gt = scene(n=2000)
    tr = Trainer(cfg, sp, device=DEV, dropout=DropoutOptions(splat_rate=0.5, seed=3), optim=OptimOptions())
    h = pinned(vm, K, gt)
    for it in range(3):
        tr.train_step(*h, 3)
        # an unseen splat gets no gradient; a dropped one is unseen
        drop = O.dropped(0, 2000, 1, 0.5, 6, it)
        assert not tr.grads["means"].view(2000, 3)[dev(drop)].any()
        assert int((tr.grads["means"].view(2000, 3)[dev(~drop)].abs().sum(1) > 0).sum()) > 500
    tr.set_dropout(0.0)
    tr.train_step(*h, 3)
    assert int((tr.grads["means"].view(2000, 3).abs().sum(1) > 0).sum()) > 1500
    tr.close()


def test_trainer_reads_rows_and_updates_values(lib):
    cfg, sp, vm, K, gt = scene()
    tr = Trainer(cfg, sp, device=DEV, view_sh_bits=4)
    got = grads_of(tr, gt, vm, K)
    values = O.row_values(*O.encode_rows(sp["features_sh"])).astype(np.float32)
    plain = Trainer(cfg, {**sp, "features_sh": values}, device=DEV)
    ref = grads_of(plain, gt, vm, K)
    for k in got:
        assert close(got[k], ref[k]), k
    assert np.array_equal(tr.params["features_sh"].cpu().numpy().reshape(values.shape), sp["features_sh"])
    assert torch.equal(tr.render(vm[0], K[0])[0], plain.render(vm[0], K[0])[0])
    assert torch.equal(tr.render(vm[0], K[0])[0], tr.render(vm[0], K[0], sh_bits=4)[0])
    full = Trainer(cfg, sp, device=DEV)
    assert torch.equal(tr.render(vm[0], K[0], sh_bits=32)[0], full.render(vm[0], K[0])[0])
    assert torch.equal(full.render(vm[0], K[0], sh_bits=4)[0], plain.render(vm[0], K[0])[0])
    tr.optimizer_step(3)
    # Adam's first step has the size of the rate wherever there is a gradient; it starts from the fp32 values
    step = (tr.params["features_sh"].double() - dev(sp["features_sh"].reshape(-1)).double()).abs()
    lr = cfg.lrs["lr_features_sh"]
    assert float(step.max()) <= lr * (1 + 1e-3) and int((step > 0.9 * lr).sum()) > 1000
    for t in (tr, plain, full):
        t.close()


def test_rows_with_dropout_and_with_the_fused_backward(lib):
    cfg, sp, vm, K, gt = scene(n=2500)
    # dropout first, then the rows
    tr = Trainer(cfg, sp, device=DEV, view_sh_bits=4, dropout=DropoutOptions(splat_rate=0.2, sh_rate=0.3, sh_group=45, seed=1))
    got = grads_of(tr, gt, vm, K)
    op, slope, _ = O.dropout_opacities(sp["opacities"], 0, 0.2, 2, 0)
    sh = O.dropout(sp["features_sh"].reshape(-1), 0, 45, 0.3, 3, 0).astype(np.float32).reshape(-1, 15, 3)
    plain = Trainer(cfg, {**sp, "opacities": op.astype(np.float32), "features_sh": O.row_values(*O.encode_rows(sh)).astype(np.float32)}, device=DEV)
    ref = grads_of(plain, gt, vm, K)
    ref["opacities"] = ref["opacities"] * dev(slope).float()
    ref["features_sh"] = dev(O.dropout(ref["features_sh"].cpu().numpy(), 0, 45, 0.3, 3, 0)).float()
    for k in got:
        assert close(got[k], ref[k]), k
    # rows through the fused backward + optimiser equal rows through the per-view one
    h = pinned(vm, K, gt)
    a = Trainer(cfg, sp, device=DEV, view_sh_bits=4, fused_backward=True)
    b = Trainer(cfg, sp, device=DEV, view_sh_bits=4)
    for t in (a, b):
        t.train_step(*h, 3)
    for k in a.params:
        # an update is at most the rate, in the direction of a gradient whose sums may round differently: where that is nearly
        # zero the sign may differ
        diff = (a.params[k] - b.params[k]).abs()
        lr = cfg.lrs["lr_" + k]
        assert float((diff > 1e-2 * lr).double().mean()) <= 1e-2 and float(diff.max()) <= 2.01 * lr, k
    with pytest.raises(NotImplementedError):
        a.set_dropout(0.1)
    for t in (tr, plain, a, b):
        t.close()


def test_rendering_between_the_views_of_an_iteration_changes_nothing(lib):
    cfg, sp, vm, K, gt = scene(n=2500)
    opts = DropoutOptions(splat_rate=0.2, sh_rate=0.4, seed=9)
    grads = []
    for render in (False, True):
        tr = Trainer(cfg, sp, device=DEV, view_sh_bits=4, dropout=opts)
        tr.views_fwd_bwd(dev(vm[:1]), dev(K[:1]), dev(gt[:1]), 1)
        if render:
            tr.render(vm[0], K[0])
        tr.views_fwd_bwd(dev(vm[1:]), dev(K[1:]), dev(gt[1:]), 2, accumulate=True)
        tr.optimizer_step(3)              # without allreduce_grads: the step itself ends the views
        torch.cuda.synchronize()
        grads.append({k: v.clone() for k, v in tr.grads.items()})
        tr.close()
    for k in grads[0]:
        assert close(grads[1][k], grads[0][k]), k
    drop = O.dropped(0, 2500 * 45, 3, 0.4, 19, 0)
    assert not grads[0]["features_sh"][dev(drop)].any()
    # gradient accumulation into a caller's own zeroed buffer, the first call already accumulating
    tr = Trainer(cfg, sp, device=DEV, view_sh_bits=4, dropout=opts)
    tr.views_fwd_bwd(dev(vm), dev(K), dev(gt), 3, accumulate=True)
    tr.allreduce_grads()
    torch.cuda.synchronize()
    for k in grads[0]:
        assert close(tr.grads[k], grads[0][k]), k
    tr.close()


def test_dropout_with_a_densifier_and_a_checkpoint(lib, tmp_path):
    """The stored parameters, not the dropped ones, are densified, saved and resumed; a resumed trainer draws the same masks."""
    from spirula_studio_b200 import checkpoint as ck
    cfg, sp, vm, K, gt = scene(n=2000)
    opts = DropoutOptions(splat_rate=0.3, sh_rate=0.3, seed=4)
    h = pinned(vm, K, gt)
    a = Trainer(cfg, sp, device=DEV, view_sh_bits=4, dropout=opts)
    for _ in range(2):
        a.train_step(*h, 3)
    ck.save_checkpoint(a, str(tmp_path))
    b = Trainer(cfg, sp, device=DEV, view_sh_bits=4, dropout=opts)
    ck.load_checkpoint(b, str(tmp_path))
    assert b.iteration == 2 and torch.equal(a.params["opacities"], b.params["opacities"])
    la, lb = a.train_step(*h, 3), b.train_step(*h, 3)
    assert abs(la[2] - lb[2]) <= 1e-5 * abs(la[2])
    drop = O.dropped(0, 2000, 1, 0.3, 8, 2)
    for t in (a, b):
        assert not t.grads["means"].view(2000, 3)[dev(drop)].any()
    for k in a.grads:
        assert close(a.grads[k], b.grads[k]), k
    a.close(); b.close()


def test_first_calls_inside_a_capture():
    """A fresh process whose first call of every entry point happens while a stream is being captured."""
    import os
    import subprocess
    import sys
    code = """
import ctypes as C, torch
from spirula_studio_b200 import lib as L
lib = L.load()
n, V = 500, 20
x = torch.randn(n * 45, device="cuda"); y = torch.zeros_like(x); rows = torch.zeros(n, 32, dtype=torch.uint8, device="cuda")
m = torch.randn(n, 3, device="cuda"); vm = torch.eye(4, device="cuda").reshape(1, 16).repeat(V, 1).contiguous()
out = torch.zeros(V, n, 3, device="cuda"); g = torch.zeros(n, 45, device="cuda"); gm = torch.zeros(n, 3, device="cuda")
d = L.dropout_struct(0.3, 1, 2)
sp = L.splats_struct(dict(means=m)); spf = L.splats_struct(dict(means=m, features_sh=y)); gr = L.splats_struct(dict(means=gm, features_sh=g))
q = L.shq_struct(rows, None, 4, 0)
cams = L.cameras_struct(vm, vm, 1, 1); one, three = (L.cameras_struct(vm, vm, 1, 1, count=k) for k in (1, 3))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    st = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    L.check(lib.ssb_dropout(L.ptr(x), 0, n * 45, 3, C.byref(d), L.ptr(y), st))
    L.check(lib.ssb_dropout(L.ptr(y), 0, n * 45, 1, C.byref(d), L.ptr(y), st))
    L.check(lib.ssb_dropout_opacities(L.ptr(x), 0, n, C.byref(d), L.ptr(gm), st))
    L.check(lib.ssb_dropout_opacities_bwd(L.ptr(x), L.ptr(x), 0, n, C.byref(d), L.ptr(gm), st))
    L.check(lib.ssb_quant_encode(L.ptr(y), n * 45, 4, L.ptr(rows), None, st))
    L.check(lib.ssb_quant_decode(L.ptr(rows), None, n * 45, 4, L.ptr(g), st))
    for s, shq in ((sp, C.byref(q)), (spf, None)):
        for c in (one, three, cams):
            L.check(lib.ssb_sh_eval_fwd(C.byref(s), shq, n, C.byref(c), L.ptr(out), st))
            L.check(lib.ssb_sh_eval_bwd(C.byref(s), shq, n, C.byref(c), L.ptr(out), C.byref(gr), 0, st))
graph.replay()
torch.cuda.synchronize()
assert torch.isfinite(out).all() and out.abs().sum() > 0 and torch.isfinite(g).all()
print("captured")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_trainer_refusals(lib):
    cfg, sp, _, _, _ = scene(n=300)
    for kw in (dict(dropout=DropoutOptions(splat_rate=1.0)), dict(dropout=DropoutOptions(sh_rate=-0.1)), dict(dropout=DropoutOptions(sh_rate=0.1, sh_group=0)),
               dict(view_sh_bits=8)):
        with pytest.raises(ValueError):
            Trainer(cfg, sp, device=DEV, **kw)
    cfg.sh_value_bits = 16
    for kw in (dict(dropout=DropoutOptions(sh_rate=0.1)), dict(view_sh_bits=4)):
        with pytest.raises(ValueError):
            Trainer(cfg, sp, device=DEV, **kw)
    tr = Trainer(cfg, sp, device=DEV, dropout=DropoutOptions(splat_rate=0.1))       # opacities are fp32 in every storage
    with pytest.raises(ValueError):
        tr.render(np.eye(4), np.ones(4), sh_bits=4)
    tr.close()


def test_ply_holds_the_values_of_the_rows(lib, tmp_path):
    _, sp, _, _, _ = scene(n=700)
    t = {k: dev(v) for k, v in sp.items()}
    rows, vals = rows_of(lib, t["features_sh"])
    shq = L.shq_struct(rows, None, 4, 0)
    a, b = str(tmp_path / "rows.ply"), str(tmp_path / "values.ply")
    s = L.splats_struct({**t, "features_sh": None})
    L.check(lib.ssb_ply_write(a.encode(), C.byref(s), C.byref(shq), 700, None, None))
    s = L.splats_struct({**t, "features_sh": vals})
    L.check(lib.ssb_ply_write(b.encode(), C.byref(s), None, 700, None, None))
    da, db = open(a, "rb").read(), open(b, "rb").read()
    assert da == db
