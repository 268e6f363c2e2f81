"""Shared rows and the budget where the trainer uses them: lookup before the render, the table's gradient after its
backward, Adam on the table; blend weights accumulated over views, eviction to a budget, training on."""
import dataclasses

import numpy as np
import pytest
import torch

import gsx_b200 as gb
from gsx_b200 import scenes, train
from gsx_b200.train import GaussianModel, SharedRows, Trainer
from oracle import pyoracle as po

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
W, H = 96, 80


def _ocam(cam):
    return po.Camera(cam.width, cam.height, cam.fx, cam.fy, cam.cx, cam.cy, cam.rot_xyzw, cam.transl, cam.near_plane, cam.far_plane)


def _trainer(n=3000, rows=50, sh_degree=0, fields=("sh0",)):
    g, cam = scenes.small_scene(3, n, W, H, sh_degree)
    gen = torch.Generator(device="cuda").manual_seed(1)
    model = GaussianModel(g, sh_degree=sh_degree)
    shared = {}
    for f in fields:
        cols = model.params[f].view(n, -1).shape[1]
        shared[f] = SharedRows(torch.randn(rows, cols, generator=gen, device="cuda") * 0.3,
                               torch.randint(0, rows, (n,), generator=gen, device="cuda", dtype=torch.int32), scale=0.5)
    target = torch.rand(3, H, W, generator=gen, device="cuda")
    return Trainer(model, W, H, shared=shared), cam, target


@pytest.mark.parametrize("sh_degree,fields", [(0, ("sh0",)), (1, ("sh0", "sh1"))])
def test_a_step_with_shared_rows(cuda_device, sh_degree, fields):
    tr, cam, target = _trainer(sh_degree=sh_degree, fields=fields)
    m = tr.model
    tr.gradients(cam, target)
    for f in fields:
        rows = tr.shared[f]
        n = m.n
        assert torch.equal(m.params[f].view(n, -1), rows.table[rows.index.long()] * 0.5)
        grad = m.grads[f].view(n, -1).double()
        want = torch.zeros_like(rows.table, dtype=torch.float64).index_add_(0, rows.index.long(), grad) * 0.5
        size = torch.zeros_like(want).index_add_(0, rows.index.long(), grad.abs()) * 0.5
        count = torch.bincount(rows.index.long(), minlength=rows.table.shape[0]).double()[:, None]
        assert bool(((rows.grad.double() - want).abs() <= 1.01 * size * (count + 2) * U).all())
        assert float(rows.grad.abs().max()) > 0
    before = {f: tr.shared[f].table.clone() for f in fields}
    other = m.params["mean3d"].clone()
    tr.update()
    for f in fields:  # the table took the place of the field in Adam
        alone = before[f].clone()
        gb.Adam([gb.ParamGroup(f, alone, tr.shared[f].grad, tr.lr[f])]).step()
        assert torch.equal(alone, tr.shared[f].table)
    assert not torch.equal(other, m.params["mean3d"])


def test_blend_weights_are_the_colour_gradient_of_the_oracle(cuda_device):
    tr, cam, _ = _trainer()
    for rows in tr.shared.values():
        rows.expand(tr.model.params["sh0"])
    score = torch.full((tr.model.n,), 2.0, device="cuda")
    assert tr.blend_weights(cam, score, decay=0.0) is score
    g = {k: v.cpu().numpy() for k, v in tr.model.params.items()}
    g["sh0"] = np.zeros_like(g["sh0"])
    ref = po.render_forward(g, _ocam(cam))
    grad = np.zeros((3, H, W), np.float32)
    grad[0] = np.float32(1.0 / 0.28209479177387814)
    want = po.render_backward(g, _ocam(cam), ref, grad)["sh0"][:, 0].astype(np.float64)
    got = score.cpu().numpy().astype(np.float64)
    assert np.linalg.norm(got - want) <= 1e-3 * np.linalg.norm(want)
    assert (got >= 0).all() and got.max() > 1
    once = score.clone()
    tr.blend_weights(cam, score, decay=0.5)
    # the backward adds up with atomics, so a second run differs by its order (the bar above); the decay is exact
    assert float((score - 1.5 * once).norm()) <= 2e-3 * float(once.norm())


def test_train_evict_and_train_on(cuda_device):
    tr, cam, target = _trainer(n=4001, sh_degree=1, fields=("sh1",))
    for _ in range(3):
        tr.step(cam, target)
    m = tr.model
    score = torch.zeros(m.n, device="cuda")
    for _ in range(2):
        tr.blend_weights(cam, score, decay=0.9)
    old = {f: v.clone() for f, v in m.params.items()}
    m1 = [t.clone() for t in tr.optim.m1]
    m2 = [t.clone() for t in tr.optim.m2]
    index, table = tr.shared["sh1"].index.clone(), tr.shared["sh1"].table.clone()
    left = tr.keep_budget(score, 1500, first=10, recent=200)
    s = score.cpu().numpy().astype(np.float64)
    middle = np.arange(10, 4001 - 200)
    best = middle[np.lexsort((middle, -s[middle]))][:1500 - 210]
    keep = torch.from_numpy(np.sort(np.concatenate([np.arange(10), best, np.arange(3801, 4001)]))).cuda()
    assert m.n == 1500 and torch.equal(left, score[keep])
    for f in m.fields:
        assert torch.equal(m.params[f], old[f][keep]), f
    assert torch.equal(tr.shared["sh1"].index, index[keep]) and torch.equal(tr.shared["sh1"].table, table)
    assert tr.optim.steps == [3] * len(m.fields)
    for i, f in enumerate(m.fields):
        rows = slice(None) if f == "sh1" else keep
        assert torch.equal(tr.optim.m1[i], m1[i][rows]) and torch.equal(tr.optim.m2[i], m2[i][rows])
    assert tr.keep_budget(left, 1500) is left
    for _ in range(2):
        loss = tr.step(cam, target)
    assert bool(torch.isfinite(loss).all()) and tr.optim.steps[0] == 5


def test_a_table_set_between_renders_is_seen(cuda_device):
    tr, cam, _ = _trainer(n=500)
    rows, m = tr.shared["sh0"], tr.model
    tr.blend_weights(cam, torch.zeros(500, device="cuda"))
    assert torch.equal(m.params["sh0"].view(500, -1), rows.table[rows.index.long()] * 0.5)
    rows.table.add_(1.0)
    tr.keep_budget(torch.arange(500, device="cuda").float(), 100)
    assert torch.equal(m.params["sh0"].view(100, -1), rows.table[rows.index.long()] * 0.5)


def test_refusals(cuda_device):
    tr, cam, target = _trainer(n=200)
    m = tr.model
    rows = tr.shared["sh0"]
    for bad in (SharedRows(rows.table.half(), rows.index), SharedRows(rows.table, rows.index[:-1])):
        with pytest.raises(gb.GsxError) as e:
            Trainer(m, W, H, shared={"sh0": bad})
        assert e.value.code == gb.NOT_SUPPORTED
    with pytest.raises(gb.GsxError) as e:
        Trainer(m, W, H, shared={"sh2": rows})
    assert e.value.code == gb.NOT_SUPPORTED
    for call in (lambda: tr.keep_budget(torch.zeros(199, device="cuda"), 10), lambda: tr.keep_budget(torch.zeros(200, device="cuda"), 0),
                 lambda: tr.keep_budget(torch.zeros(200, device="cuda", dtype=torch.float16), 10),
                 lambda: tr.keep_budget(torch.zeros(200, device="cuda"), 10, first=6, recent=5)):
        with pytest.raises(gb.GsxError) as e:
            call()
        assert e.value.code == gb.INVALID_ARGUMENT
        assert m.n == 200


def _follows(tr, fields):
    for f in fields:
        rows, n = tr.shared[f], tr.model.n
        assert torch.equal(tr.model.params[f].view(n, -1), rows.table[rows.index.long()] * 0.5), f


def _image(tr, cam):
    out = torch.empty(3, H, W, device="cuda")
    tr.renderer.render(tr.ctx, tr.model.params, cam, out, sh_degree=tr.model.sh_degree, forward_type=gb.FORWARD_INFERENCE)
    return out


@pytest.mark.parametrize("sh_degree,fields", [(0, ("sh0",)), (1, ("sh0", "sh1"))])
def test_a_shared_field_follows_its_table(cuda_device, sh_degree, fields):
    """model.params holds the table's rows whenever a call of the trainer has returned, for renders outside of it."""
    tr, cam, target = _trainer(sh_degree=sh_degree, fields=fields)
    _follows(tr, fields)
    for _ in range(2):
        tr.step(cam, target)
        _follows(tr, fields)
    seen = _image(tr, cam)
    for f in fields:
        tr.shared[f].expand(tr.model.params[f])
    assert torch.equal(seen, _image(tr, cam))
    tr.keep_budget(torch.rand(tr.model.n, device="cuda"), 700)
    _follows(tr, fields)


def test_an_eviction_keeps_the_optimizer_and_its_settings(cuda_device):
    tr, cam, target = _trainer(n=900, fields=("sh0",))
    tr.step(cam, target)
    optim, groups = tr.optim, list(tr.optim.groups)
    for i, g in enumerate(groups):
        g.learning_rate = 1e-4 * (i + 1)
        g.beta1, g.beta2, g.weight_decay, g.epsilon, g.max_grad = 0.8, 0.99, 0.01, 1e-6, 0.5
    tr.keep_budget(torch.rand(900, device="cuda"), 300)
    assert tr.optim is optim and all(a is b for a, b in zip(optim.groups, groups))
    m = tr.model
    for i, (f, g) in enumerate(zip(m.fields, groups)):
        assert g.role == f and g.learning_rate == 1e-4 * (i + 1)
        assert (g.beta1, g.beta2, g.weight_decay, g.epsilon, g.max_grad) == (0.8, 0.99, 0.01, 1e-6, 0.5)
        if f != "sh0":
            assert g.parameter.data_ptr() == m.params[f].data_ptr() and g.gradient.data_ptr() == m.grads[f].data_ptr()
            assert optim.m1[i].shape == optim.m2[i].shape == m.params[f].shape
    tr.gradients(cam, target)
    alone = gb.Adam([dataclasses.replace(g, parameter=g.parameter.clone()) for g in groups])
    alone.steps = list(optim.steps)
    for i in range(len(groups)):
        alone.m1[i].copy_(optim.m1[i])
        alone.m2[i].copy_(optim.m2[i])
    alone.step()
    tr.update()
    for a, b in zip(alone.groups, groups):
        assert torch.equal(a.parameter, b.parameter), b.role


def test_an_eviction_with_an_optimizer_of_some_fields(cuda_device):
    """The caller's own Adam, over a few fields in any order: its moments go with their Gaussians."""
    tr, cam, target = _trainer(n=900, fields=("sh0",))
    m = tr.model
    tr.optim = gb.Adam([gb.ParamGroup("opacity", m.params["opacity"], m.grads["opacity"], 1e-2),
                        gb.ParamGroup("sh0", tr.shared["sh0"].table, tr.shared["sh0"].grad, 1e-2),
                        gb.ParamGroup("mean3d", m.params["mean3d"], m.grads["mean3d"], 1e-3)])
    tr.step(cam, target)
    m1 = [t.clone() for t in tr.optim.m1]
    old = {f: v.clone() for f, v in m.params.items()}
    score = torch.arange(900, device="cuda").float()  # the last 300 stay
    tr.keep_budget(score, 300)
    for f in m.fields:
        assert torch.equal(m.params[f], old[f][600:])
    assert torch.equal(tr.optim.m1[0], m1[0][600:]) and torch.equal(tr.optim.m1[1], m1[1]) and torch.equal(tr.optim.m1[2], m1[2][600:])
    before = m.params["logscale"].clone()
    tr.step(cam, target)
    assert torch.equal(m.params["logscale"], before) and not torch.equal(m.params["mean3d"], old["mean3d"][600:])


@pytest.mark.parametrize("where", ["_allocate", "budget_gather"])
def test_an_eviction_that_fails_changes_nothing(cuda_device, monkeypatch, where):
    """Out of memory, or a refused gather: the model, its optimizer and the row numbers stay as they were."""
    tr, cam, target = _trainer(n=900, fields=("sh0",))
    tr.step(cam, target)
    m, rows = tr.model, tr.shared["sh0"]
    held = [m.flat_param, m.flat_grad, *m.params.values(), *m.grads.values(), *tr.optim.m1, *tr.optim.m2, rows.index, rows.table]
    copies = [t.clone() for t in held]
    layout = (m.n, m.numel, dict(m.offsets), dict(m.field_ranges), list(tr.optim.steps))

    def fail(*args, **kw):
        raise torch.OutOfMemoryError("no memory")

    with monkeypatch.context() as patch:
        patch.setattr(train.GaussianModel, where, fail) if where == "_allocate" else patch.setattr(train, where, fail)
        with pytest.raises(torch.OutOfMemoryError):
            tr.keep_budget(torch.rand(900, device="cuda"), 300)
    now = [m.flat_param, m.flat_grad, *m.params.values(), *m.grads.values(), *tr.optim.m1, *tr.optim.m2, rows.index, rows.table]
    assert all(a is b for a, b in zip(held, now)) and all(torch.equal(a, b) for a, b in zip(copies, now))
    assert layout == (m.n, m.numel, m.offsets, m.field_ranges, tr.optim.steps)
    tr.step(cam, target)
    tr.keep_budget(torch.rand(900, device="cuda"), 300)
    assert m.n == 300 and bool(torch.isfinite(tr.step(cam, target)).all())


def test_a_table_serves_one_field(cuda_device):
    """Two groups of one Adam launch over the same table would race; the row numbers may be shared."""
    tr, _, _ = _trainer(n=300, fields=())
    m = tr.model
    table = torch.randn(20, 3, device="cuda")
    index = torch.randint(0, 10, (300,), device="cuda")
    rows = SharedRows(table, index)
    for other in (rows, SharedRows(table, index), SharedRows(table[10:], index), SharedRows(table[:10].view(10, 3), index.clone())):
        with pytest.raises(gb.GsxError) as e:
            Trainer(m, W, H, shared={"sh0": rows, "logscale": other})
        assert e.value.code == gb.INVALID_ARGUMENT
    two = Trainer(m, W, H, shared={"sh0": SharedRows(table[:10], index), "logscale": SharedRows(table[10:], index)})
    two.keep_budget(torch.arange(300, device="cuda").float(), 50)
    for rows in two.shared.values():
        assert torch.equal(rows.index, index[250:])
    with pytest.raises(gb.GsxError) as e:  # Adam walks a table as one array
        Trainer(two.model, W, H, shared={"sh0": SharedRows(torch.randn(3, 20, device="cuda").t(), index[:50].clone())})
    assert e.value.code == gb.INVALID_ARGUMENT


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_row_numbers_outside_the_table_are_reported(cuda_device, dtype):
    tr, cam, target = _trainer(n=300, fields=())
    table = torch.randn(20, 3, device="cuda")
    fine = torch.randint(0, 20, (300,), device="cuda", dtype=dtype)
    for number in (20, -1, 2 ** 31 - 1):
        index = fine.clone()
        index[7] = number
        with pytest.raises(gb.GsxError) as e:
            Trainer(tr.model, W, H, shared={"sh0": SharedRows(table, index)})
        assert e.value.code == gb.OUT_OF_RANGE and "sh0" in str(e.value)
    rows = SharedRows(table, fine)
    tr = Trainer(tr.model, W, H, shared={"sh0": rows})
    tr.step(cam, target)
    rows.check()
    rows.index[299] = 20  # changed while training: reported by the next check, once
    tr.step(cam, target)
    with pytest.raises(gb.GsxError) as e:
        rows.check()
    assert e.value.code == gb.OUT_OF_RANGE
    rows.check()
    rows.index[299] = 0
    tr.step(cam, target)
    rows.check()


def test_blend_weights_leave_the_density_statistics_alone(cuda_device):
    """Its render and backward are no training view: statistics that the context has bound see neither, and stay bound."""
    tr, cam, target = _trainer(n=800, fields=("sh0",))
    stats = [torch.full((800,), 3.0, device="cuda") for _ in range(4)]
    tr.ctx.bind_aux(*stats)
    tr.blend_weights(cam, torch.zeros(800, device="cuda"))
    assert all(bool((t == 3.0).all()) for t in stats)
    tr.step(cam, target)
    assert all(bool((t != 3.0).any()) for t in stats)
    tr.ctx.bind_aux()
    tr.blend_weights(cam, torch.zeros(800, device="cuda"))


def test_a_trainer_that_is_refused_leaves_its_model_alone(cuda_device):
    tr, _, _ = _trainer(n=300, fields=(), sh_degree=1)
    m = tr.model
    before = m.flat_param.clone()
    good = SharedRows(torch.randn(20, 3, device="cuda"), torch.zeros(300, dtype=torch.int32, device="cuda"))
    table, index = torch.randn(20, 9, device="cuda"), torch.zeros(300, dtype=torch.int64, device="cuda")
    for code, other in [(gb.INVALID_ARGUMENT, SharedRows(table[:, :8].contiguous(), index)),
                        (gb.INVALID_ARGUMENT, SharedRows(table[:, 0].contiguous(), index)),
                        (gb.INVALID_ARGUMENT, SharedRows(table, index.cpu())), (gb.INVALID_ARGUMENT, SharedRows(table.cpu(), index)),
                        (gb.INVALID_ARGUMENT, SharedRows(table, index.repeat(2)[::2])), (gb.NOT_SUPPORTED, SharedRows(table, index.short())),
                        (gb.OUT_OF_RANGE, SharedRows(table, index + 20)), (gb.OUT_OF_RANGE, SharedRows(table, index - 1))]:
        with pytest.raises(gb.GsxError) as e:
            Trainer(m, W, H, shared={"sh0": good, "sh1": other})
        assert e.value.code == code, e.value
        assert torch.equal(m.flat_param, before)
