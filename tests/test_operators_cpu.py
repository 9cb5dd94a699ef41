"""Layer norm, filtered draws and gradient norms without a GPU: what is refused, and the host logic around the kernels with the
kernels replaced by their definitions."""
import copy
import ctypes
import math

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

import asdl_amd
from asdl_amd import (FISHER_EMP, FISHER_EXACT, FISHER_MC, FisherConfig, FusedLayerNorm, KfacGradientMaker, LOSS_CROSS_ENTROPY, LOSS_MSE,
                      PreconditioningConfig, SHAPE_KRON, ShampooGradientMaker, get_fisher_maker, kernels)
from tests import cpu_backend


def test_cpu_tensors_are_refused():
    x, w = torch.randn(4, 8), torch.ones(8)
    for call in (lambda: kernels.layer_norm(x, w), lambda: kernels.layer_norm_backward(x, x, w, w), lambda: kernels.sample_filtered(x, torch.rand(4)),
                 lambda: kernels.grad_norm([x]), lambda: kernels.clip_grad_norm([x], 1.0), lambda: FusedLayerNorm(8)(x)):
        with pytest.raises(RuntimeError, match='ROCm device'):
            call()
    with pytest.raises(ValueError):
        kernels.grad_norm([])


def test_entry_points_refuse_bad_arguments():
    """Before anything is launched: return codes of the C interface."""
    from asdl_amd import _lib
    lib = _lib.load()
    a = 4096                                   # stands for an address; nothing reads it
    f32, bf16, f16, bad = 0, 1, 4, 7

    def norm(x=a, xt=f32, ldx=64, wt=f32, rows=4, F=64, eps=1e-5, y=a, yt=f32, ldy=64, mean=a, rstd=a):
        return lib.ak_layer_norm(x, xt, ldx, a, a, wt, rows, F, eps, y, yt, ldy, mean, rstd, None)
    assert norm(rows=0) == 0
    for kw in (dict(x=None), dict(y=None), dict(mean=None), dict(rstd=None), dict(xt=bad), dict(yt=bad), dict(wt=bad), dict(xt=bf16, yt=f16, wt=f32),
               dict(xt=bf16, yt=bf16, wt=f16), dict(rows=-1), dict(F=0), dict(ldx=63), dict(ldy=63), dict(eps=-1.0), dict(eps=math.nan)):
        assert norm(**kw) == -1, kw
    assert norm(rows=1 << 31) == -3 and norm(F=(1 << 30) + 1, ldx=1 << 31, ldy=1 << 31) == -3

    def back(g=a, gt=f32, ldg=64, x=a, xt=f32, ldx=64, wt=f32, rows=4, F=64, dx=a, lddx=64, dw=a, db=a, blocks=None, ws=a, need=1 << 40):
        return lib.ak_layer_norm_backward(g, gt, ldg, x, xt, ldx, a, a, a, wt, rows, F, dx, lddx, dw, db, blocks, 1.0, 0.0, ws, need, None)
    for kw in (dict(g=None), dict(x=None), dict(gt=bad), dict(gt=bf16), dict(xt=bad), dict(wt=bf16), dict(rows=-1), dict(F=0), dict(ldg=1), dict(lddx=1)):
        assert back(**kw) == -1, kw
    assert back(ws=None) == -2 and back(need=8) == -2 and back(blocks=a, need=lib.ak_layer_norm_backward_ws_bytes(4, 64, 0)) == -2
    assert back(dx=None, dw=None, db=None, ws=None) == 0          # nothing is asked for
    assert lib.ak_layer_norm_backward_ws_bytes(0, 64, 1) == 0 and lib.ak_layer_norm_backward_ws_bytes(4, 64, 1) > lib.ak_layer_norm_backward_ws_bytes(4, 64, 0) > 0

    def draw(logits=a, dtype=f32, rows=4, classes=10, ld=10, u=a, t=1.0, ts=None, targets=a):
        return lib.ak_sample_filtered(logits, dtype, rows, classes, ld, u, 0, t, ts, 0, None, 1.0, None, 0.0, None, targets, None, None)
    assert draw(rows=0) == 0
    for kw in (dict(logits=None), dict(dtype=bad), dict(rows=-1), dict(classes=0), dict(ld=9), dict(u=None), dict(t=-1.0), dict(t=math.nan), dict(targets=None)):
        assert draw(**kw) == -1, kw
    assert draw(rows=1 << 31) == -5 and draw(classes=(1 << 30) + 1, ld=1 << 31) == -5

    def clip(rows, kind=0, most=1.0, norm=a, ws=a, need=1 << 20):
        table = (ctypes.c_int64 * len(rows))(*rows)
        return lib.ak_clip_grad_norm(table, len(rows) // 5, kind, most, norm, ws, need, None)
    good = [a, a, 10, f32, f32]
    for rows, kw in ((good, dict(kind=3)), (good, dict(kind=-1)), (good, dict(most=-1.0)), (good, dict(most=math.nan)), (good, dict(norm=None)),
                     ([0, a, 10, f32, f32], {}), ([a, 0, 10, f32, f32], {}), ([a, a, -1, f32, f32], {}), ([a, a, 10, bad, bad], {}),
                     ([a, a, 10, f32, bf16], {}), ([a, a, 10, bf16, f16], {})):
        assert clip(rows, **kw) == -1, (rows, kw)
    assert clip(good, ws=None) == -2 and clip(good, need=64) == -2 and clip([a, a, 1 << 46, f32, f32]) == -5
    assert lib.ak_grad_norm_ws_bytes(1000) > lib.ak_grad_norm_ws_bytes(0) > 0 and lib.ak_grad_norm_ws_bytes(-1) == 0


@pytest.mark.parametrize('filters', [dict(mc_temperature=0.5), dict(mc_top_k=3), dict(mc_top_p=0.9), dict(mc_min_p=0.1)])
def test_filters_are_for_the_sampled_fisher_of_a_cross_entropy(filters):
    model = nn.Sequential(nn.Linear(3, 4))
    for fisher_type, loss in ((FISHER_EMP, LOSS_CROSS_ENTROPY), (FISHER_EXACT, LOSS_CROSS_ENTROPY), (FISHER_MC, LOSS_MSE)):
        with pytest.raises(ValueError, match='mc_temperature'):
            get_fisher_maker(model, FisherConfig(fisher_type, [SHAPE_KRON], loss_type=loss, **filters))
    get_fisher_maker(model, FisherConfig(FISHER_MC, [SHAPE_KRON], loss_type=LOSS_CROSS_ENTROPY, **filters))
    maker = KfacGradientMaker(model, PreconditioningConfig(data_size=2), **filters)
    assert all(getattr(maker.fisher_maker.config, k) == v for k, v in filters.items())
    assert not FisherConfig(FISHER_MC, [SHAPE_KRON]).mc_filtered


def test_layer_norm_checks_its_shapes():
    x = torch.randn(2, 3, 4)
    for args in ((5,), ((2, 3),), ((),)):
        with pytest.raises(ValueError, match='has to end'):
            asdl_amd.layer_norm(x, *args)
    with pytest.raises(ValueError, match='weight has to have the shape'):
        asdl_amd.layer_norm(x, 4, torch.ones(3))
    with pytest.raises(ValueError, match='bias has to have the shape'):
        asdl_amd.layer_norm(x, (3, 4), torch.ones(3, 4), torch.ones(12))


def test_fuse_layer_norms_keeps_parameters_and_subclasses():
    class Mine(nn.LayerNorm):
        pass
    model = nn.Sequential(nn.LayerNorm(4), nn.Linear(4, 4), nn.Sequential(nn.LayerNorm(4, elementwise_affine=False)), Mine(4), FusedLayerNorm(4))
    state = {k: v.clone() for k, v in model.state_dict().items()}
    params = [id(p) for p in model.parameters()]
    assert asdl_amd.fuse_layer_norms(model) == 2 and asdl_amd.fuse_layer_norms(model) == 0
    assert [type(m) for m in (model[0], model[2][0], model[3])] == [FusedLayerNorm, FusedLayerNorm, Mine]
    assert params == [id(p) for p in model.parameters()] and all(torch.equal(state[k], v) for k, v in model.state_dict().items())


# ------------------------------------------------------------------------------------------------ hooks, with stand-ins for the kernels
def _layer_norm(x, weight=None, bias=None, eps=1e-5, out_dtype=None):
    m = x.mean(-1, keepdim=True)
    r = ((x - m).square().mean(-1, keepdim=True) + eps).rsqrt()
    h = (x - m) * r
    y = h if weight is None else h * weight
    return (y if bias is None else y + bias), m.squeeze(-1), r.squeeze(-1)


class _Backward:
    """layer_norm_backward() by its formula; counts who asks for what."""

    def __init__(self):
        self.fused = self.alone = 0

    def __call__(self, g, x, mean, rstd, weight=None, blocks=None, alpha=1.0, beta=0.0, need_x=True, need_weight=True, need_bias=True, weight_dtype=None):
        h = (x - mean.unsqueeze(-1)) * rstd.unsqueeze(-1)
        gw = g if weight is None else g * weight
        dx = rstd.unsqueeze(-1) * (gw - gw.mean(-1, keepdim=True) - h * (gw * h).mean(-1, keepdim=True))
        g2, h2 = g.reshape(-1, g.shape[-1]), h.reshape(-1, h.shape[-1])
        if blocks is not None:
            self.fused, self.alone = self.fused + bool(need_x), self.alone + (not need_x)
            a, b = g2 * h2, g2
            new = torch.stack([(a * a).sum(0), (a * b).sum(0), (a * b).sum(0), (b * b).sum(0)], -1).view(-1, 2, 2)
            blocks.copy_(alpha * new if beta == 0 else beta * blocks + alpha * new)
        return dx if need_x else None, (g2 * h2).sum(0) if need_weight else None, g2.sum(0) if need_bias else None


class _Net(nn.Module):
    """Layer norms in front (its input needs no gradient), in the middle, and over two dimensions."""

    def __init__(self):
        super().__init__()
        self.first, self.a, self.middle = nn.LayerNorm(6), nn.Linear(6, 6), nn.LayerNorm(6)
        self.square, self.b = nn.LayerNorm((2, 3)), nn.Linear(6, 4)

    def forward(self, x):
        x = self.middle(self.a(self.first(x)).tanh())
        return self.b(self.square(x.view(-1, 2, 3)).flatten(1))


@pytest.mark.parametrize('ema', [-1, 0.3])
@pytest.mark.parametrize('fisher_type', [FISHER_EMP, FISHER_MC, FISHER_EXACT])
def test_blocks_of_fused_layer_norms_are_those_of_plain_ones(fisher_type, ema, monkeypatch):
    cpu_backend.install(monkeypatch)
    backward = _Backward()
    monkeypatch.setattr(kernels, 'layer_norm', _layer_norm)
    monkeypatch.setattr(kernels, 'layer_norm_backward', backward)
    torch.manual_seed(1)
    plain = _Net()
    for m in plain.modules():
        if isinstance(m, nn.LayerNorm):
            nn.init.normal_(m.weight, 1.0, 0.1)
            nn.init.normal_(m.bias, 0.0, 0.1)
    fused = copy.deepcopy(plain)
    assert asdl_amd.fuse_layer_norms(fused) == 3
    x, t = torch.randn(5, 6), torch.randint(4, (5,))
    makers = []
    for model in (plain, fused):
        maker = KfacGradientMaker(model, PreconditioningConfig(data_size=5, damping=1e-2, ema_decay=ema), fisher_type=fisher_type, seed=3)
        for _ in range(3):
            model.zero_grad()
            maker.setup_loss_call(F.cross_entropy, maker.setup_model_call(model, x), t)
            maker.forward_and_backward()
        makers.append(maker)
    # float32 blocks of up to 50 with a damping of 1e-2: their inverses, and what is multiplied by them, magnify the 2^-24 of some ten
    # roundings by up to 5000
    def off(a, b):
        return float((a - b).norm() / b.norm())
    for (name, p), q in zip(plain.named_parameters(), fused.parameters()):
        assert off(q.grad, p.grad) < 5000 * 10 * 2.0 ** -24, name
    for m, n in zip(plain.modules(), fused.modules()):
        if isinstance(m, nn.LayerNorm):
            a, b = m.fisher.unit, n.fisher.unit
            assert off(b.inv, a.inv) < 5000 * 10 * 2.0 ** -24
            assert (a.data is None) == (b.data is None) and (a.data is None or off(b.data, a.data) < 64 * 2.0 ** -24)
    # the first layer's backward pass does not run where only the edges to the hooked outputs are differentiated
    assert backward.fused > 0 and (fisher_type == FISHER_EMP or backward.alone > 0)


def test_a_layer_norm_called_twice_adds_the_blocks_of_both_calls(monkeypatch):
    """Each from its own input.  (Of torch.nn.LayerNorm, as in the reference, the output of the last call stands for all.)"""
    cpu_backend.install(monkeypatch)
    monkeypatch.setattr(kernels, 'layer_norm', _layer_norm)
    monkeypatch.setattr(kernels, 'layer_norm_backward', _Backward())
    from asdl_amd import OP_COV_UNIT_WISE, OP_COV_UNIT_WISE_INV, extend
    ln = FusedLayerNorm(4)
    x = torch.randn(7, 4, requires_grad=True)
    want = 0
    y1 = ln(x)
    y2 = ln(y1.sin())
    y1.retain_grad()
    y2.retain_grad()
    (y2 ** 3).sum().backward()
    for inp, g in ((x, y1.grad), (y1.sin(), y2.grad)):
        h = _layer_norm(inp.detach())[0]
        a, b = g * h, g
        want = want + torch.stack([(a * a).sum(0), (a * b).sum(0), (a * b).sum(0), (b * b).sum(0)], -1).view(-1, 2, 2)
    for op, key in ((OP_COV_UNIT_WISE, 'data'), (OP_COV_UNIT_WISE_INV, 'inv')):
        with extend(ln, op) as cxt:
            cxt.set_damping(1.0)
            (ln(ln(x).sin()) ** 3).sum().backward()
            cxt.flush_inverses()
            got = cxt.get_result(ln, OP_COV_UNIT_WISE, key)
        expect = want if key == 'data' else torch.inverse(want + torch.eye(2))
        assert torch.allclose(got, expect, rtol=1e-3, atol=1e-5), key


def test_a_gradient_that_another_hook_replaces_does_not_reach_the_blocks(monkeypatch):
    cpu_backend.install(monkeypatch)
    backward = _Backward()
    monkeypatch.setattr(kernels, 'layer_norm', _layer_norm)
    monkeypatch.setattr(kernels, 'layer_norm_backward', backward)
    from asdl_amd import OP_COV_UNIT_WISE, extend
    ln = FusedLayerNorm(4)
    pre = nn.Linear(4, 4)
    x = torch.randn(7, 4)
    with extend(ln, OP_COV_UNIT_WISE) as cxt:
        y = ln(pre(x))
        y.register_hook(lambda g: 2 * g)
        (y ** 2).sum().backward()
        got = cxt.get_result(ln, OP_COV_UNIT_WISE, 'data')
    assert backward.alone == 1 and backward.fused == 0
    h, g = _layer_norm(pre(x).detach())[0], 2 * y.detach()
    assert torch.allclose(got[:, 1, 1], (g * g).sum(0)) and torch.allclose(got[:, 0, 0], (g * h * g * h).sum(0), rtol=1e-4)


@pytest.mark.parametrize('maker_class', [KfacGradientMaker, ShampooGradientMaker])
def test_makers_clip_what_the_step_leaves(maker_class, monkeypatch):
    calls = []

    def clip(grads, max_norm, norm_type=2.0, outs=None):
        calls.append((len(grads), max_norm, norm_type))
        norm = torch.stack([g.norm() for g in grads]).norm()
        for g in grads:
            g.mul_(min(1.0, max_norm / (float(norm) + 1e-6)))
        return norm
    cpu_backend.install(monkeypatch)
    monkeypatch.setattr(kernels, 'clip_grad_norm', clip)
    if maker_class is ShampooGradientMaker:
        pytest.importorskip('torch')
        monkeypatch.setattr(ShampooGradientMaker, '__init__', lambda self, model, config: asdl_amd.PreconditionedGradientMaker.__init__(self, model, config))
        for stage in ('update_curvature', 'update_preconditioner', 'precondition'):
            monkeypatch.setattr(ShampooGradientMaker, stage, lambda self: None)
    torch.manual_seed(0)
    model = nn.Sequential(nn.Linear(5, 6), nn.Tanh(), nn.Linear(6, 4))
    x, t = torch.randn(8, 5), torch.randint(4, (8,))
    got = {}
    for most in (None, 1e-3, 1e6):
        kwargs = dict(fisher_type=FISHER_EMP) if maker_class is KfacGradientMaker else {}
        maker = maker_class(model, PreconditioningConfig(data_size=8, damping=1e-2, max_grad_norm=most), **kwargs)
        model.zero_grad()
        maker.setup_loss_call(F.cross_entropy, maker.setup_model_call(model, x), t)
        maker.forward_and_backward()
        got[most] = [p.grad.clone() for p in model.parameters()]
        assert (maker.grad_norm is None) == (most is None)
    norm = float(torch.stack([g.norm() for g in got[None]]).norm())
    assert calls == [(4, 1e-3, 2.0), (4, 1e6, 2.0)] and norm > 1e-3
    for a, b, c in zip(got[None], got[1e-3], got[1e6]):
        assert torch.equal(a, c) and torch.allclose(b, a * (1e-3 / norm), rtol=1e-4)


def test_clip_grad_norm_of_parameters_without_gradients():
    p = nn.Parameter(torch.ones(3))
    assert float(asdl_amd.clip_grad_norm_([p], 1.0)) == 0 and float(asdl_amd.clip_grad_norm_(p, 1.0)) == 0
    p.grad = torch.ones(3)
    with pytest.raises(ValueError, match='max_norm'):
        asdl_amd.clip_grad_norm_([p], -1.0)
    with pytest.raises(RuntimeError, match='ROCm device'):
        asdl_amd.clip_grad_norm_([p], 1.0)


def test_calls_in_one_step_leave_the_unusual_to_the_others():
    """The module of host_calls.cpp says None to what it does not take, whatever it is."""
    from asdl_amd import _lib
    host = _lib.load_host()
    x, w = torch.randn(4, 8), torch.ones(8)
    assert host.layer_norm(x, w, None, 1e-5, False, 0) is None and host.layer_norm('x', w, None, 1e-5, False, 0) is None and host.layer_norm() is None
    assert host.layer_norm_backward(x, x, w, w, None, None, 1.0, 0.0, 7, 0) is None and host.layer_norm_backward(1, 2) is None
    assert host.sample_filtered(x, torch.rand(4), 1.0, None, None, None, 0) is None and host.sample_filtered(x, None, 1.0, None, None, None, 0) is None
    assert host.gradient_norm([x], None, 0, 0.0, 0) is None and host.gradient_norm([], None, 0, 0.0, 0) is None and host.gradient_norm((x,), None, 0, 0.0, 0) is None
    with pytest.raises(TypeError):
        host.bind(1)
    with pytest.raises(ValueError):
        host.bind(0, 0, 0, 0, 0, 0, 0)
    assert _lib.load_host() is host


def test_sums_over_rows_refuse_more_features_than_a_launch_has_threads_for():
    from asdl_amd import _lib
    lib, a, F = _lib.load(), 4096, (1 << 24) + 1
    for dw, blocks in ((a, None), (None, a)):
        assert lib.ak_layer_norm_backward(a, 0, F, a, 0, F, a, a, a, 0, 4, F, a, F, dw, None, blocks, 1.0, 0.0, a, 1 << 40, None) == -3


class _Dropped(nn.Module):
    """A layer norm whose result nothing uses."""

    def __init__(self):
        super().__init__()
        self.a, self.ln, self.b = nn.Linear(6, 6), nn.LayerNorm(6), nn.Linear(6, 4)

    def forward(self, x):
        x = self.a(x)
        self.ln(x)
        return self.b(x.tanh())


@pytest.mark.parametrize('fisher_type', [FISHER_EMP, FISHER_MC, FISHER_EXACT])
def test_a_fused_layer_norm_whose_result_is_dropped(fisher_type, monkeypatch):
    """The pass differentiates with respect to its output, too, which is gone: no blocks, and the factors of the others."""
    cpu_backend.install(monkeypatch)
    monkeypatch.setattr(kernels, 'layer_norm', _layer_norm)
    monkeypatch.setattr(kernels, 'layer_norm_backward', _Backward())
    torch.manual_seed(1)
    plain = _Dropped()
    fused = copy.deepcopy(plain)
    assert asdl_amd.fuse_layer_norms(fused) == 1
    x, t = torch.randn(5, 6), torch.randint(4, (5,))
    for model in (plain, fused):
        shapes = [(nn.Linear, SHAPE_KRON), (nn.LayerNorm, asdl_amd.SHAPE_UNIT_WISE)]
        maker = get_fisher_maker(model, FisherConfig(fisher_type, shapes, loss_type=LOSS_CROSS_ENTROPY, data_size=5, seed=1))
        maker.setup_loss_call(F.cross_entropy, maker.setup_model_call(model, x), t)
        maker.forward_and_backward()
    assert getattr(plain.ln, 'fisher', None) is None and getattr(fused.ln, 'fisher', None) is None
    for m, n in ((plain.a, fused.a), (plain.b, fused.b)):
        assert torch.equal(m.fisher.kron.A, n.fisher.kron.A) and torch.equal(m.fisher.kron.B, n.fisher.kron.B)


# ------------------------------------------------------------------------------------------------ blocks and what else users do with a pass
class _Block(nn.Module):
    def __init__(self, d=6, layer_norm_first=False):
        super().__init__()
        self.a, self.ln, self.b = nn.Linear(d, d), nn.LayerNorm(d), nn.Linear(d, d)
        self.layer_norm_first = layer_norm_first

    def forward(self, x):
        return self.b((self.a(self.ln(x)) if self.layer_norm_first else self.ln(self.a(x))).tanh())


class _Checkpointed(nn.Module):
    def __init__(self, checkpointed, layer_norm_first):
        super().__init__()
        self.blocks = nn.ModuleList([_Block(layer_norm_first=layer_norm_first and i == 0) for i in range(2)])
        self.head = nn.Linear(6, 4)
        self.checkpointed = checkpointed

    def forward(self, x):
        from torch.utils.checkpoint import checkpoint
        for block in self.blocks:
            x = checkpoint(block, x, use_reentrant=False) if self.checkpointed else block(x)
        return self.head(x)


def _stand_ins(monkeypatch):
    cpu_backend.install(monkeypatch)
    backward = _Backward()
    monkeypatch.setattr(kernels, 'layer_norm', _layer_norm)
    monkeypatch.setattr(kernels, 'layer_norm_backward', backward)
    return backward


@pytest.mark.parametrize('layer_norm_first', [False, True])
def test_blocks_under_checkpointing_are_those_without(layer_norm_first, monkeypatch):
    """Saved tensors are unpacked once a pass, as torch.utils.checkpoint asks for."""
    from asdl_amd import OP_COV_UNIT_WISE, extend
    _stand_ins(monkeypatch)
    torch.manual_seed(1)
    plain = _Checkpointed(False, layer_norm_first)
    x, t = torch.randn(5, 6), torch.randint(4, (5,))
    got = []
    for checkpointed in (False, True):
        model = copy.deepcopy(plain)
        model.checkpointed = checkpointed
        assert asdl_amd.fuse_layer_norms(model) == 2
        with extend(model, (nn.LayerNorm, OP_COV_UNIT_WISE)) as cxt:
            F.cross_entropy(model(x), t, reduction='sum').backward()
            got.append([cxt.get_result(b.ln, OP_COV_UNIT_WISE, 'data').clone() for b in model.blocks] + [p.grad for p in model.parameters() if p.grad is not None])
    assert len(got[0]) == len(got[1]) > 2 and all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize('layer_norm_first', [False, True])
@pytest.mark.parametrize('config', [dict(ema_decay=0.3), dict(ignore_modules=[nn.Linear])])
@pytest.mark.parametrize('fisher_type,samples', [(FISHER_EMP, 1), (FISHER_MC, 1), (FISHER_MC, 2), (FISHER_EXACT, 1)])
def test_a_checkpointed_step_with_fused_layer_norms_is_the_plain_one(fisher_type, samples, config, layer_norm_first, monkeypatch):
    """The same factors and gradients as with torch.nn.LayerNorm, whatever the checkpoint runs again for the blocks.  float32 and a damping
    of 1e-2, as above."""
    _stand_ins(monkeypatch)
    torch.manual_seed(2)
    plain = _Checkpointed(True, layer_norm_first)
    fused = copy.deepcopy(plain)
    assert asdl_amd.fuse_layer_norms(fused) == 2
    x, t = torch.randn(5, 6), torch.randint(4, (5,))
    for model in (plain, fused):
        maker = KfacGradientMaker(model, PreconditioningConfig(data_size=5, damping=1e-2, **config), fisher_type=fisher_type, n_mc_samples=samples, seed=3)
        for _ in range(2):
            model.zero_grad()
            maker.setup_loss_call(F.cross_entropy, maker.setup_model_call(model, x), t)
            maker.forward_and_backward()

    def off(a, b):
        return float((a - b).norm() / b.norm())
    for (name, p), q in zip(plain.named_parameters(), fused.named_parameters()):
        assert (p.grad is None) == (q[1].grad is None) and (p.grad is None or off(q[1].grad, p.grad) < 5000 * 10 * 2.0 ** -24), name
    held = 0
    for m, n in zip(plain.modules(), fused.modules()):
        if hasattr(m, 'fisher'):
            a, b = (m.fisher.unit, n.fisher.unit) if isinstance(m, nn.LayerNorm) else (m.fisher.kron, n.fisher.kron)
            for key in ('data', 'A', 'B'):
                if isinstance(getattr(a, key, None), torch.Tensor):
                    held += 1
                    assert off(getattr(b, key), getattr(a, key)) < 64 * 2.0 ** -24, (m, key)
            for key in ('inv', 'A_inv', 'B_inv'):
                if getattr(a, key, None) is not None:
                    held += 1
                    assert off(getattr(b, key), getattr(a, key)) < 5000 * 10 * 2.0 ** -24, (m, key)
    assert held >= 2


def test_blocks_outlive_the_graph_of_a_pass_that_left_the_layer_norm_out(monkeypatch):
    """A pass as far as the layer norm's output only: its blocks are computed when they are asked for, whatever is left of the graph."""
    from asdl_amd import OP_COV_UNIT_WISE, extend
    backward = _stand_ins(monkeypatch)
    torch.manual_seed(3)
    ln, x = FusedLayerNorm(6), torch.randn(5, 6)
    with extend(ln, OP_COV_UNIT_WISE) as cxt:
        y = ln(x)
        loss = (y ** 3).sum()
        (g,) = torch.autograd.grad(loss, y)
        g, h = g.clone(), _layer_norm(x)[0]
        del y, loss
        got = cxt.get_result(ln, OP_COV_UNIT_WISE, 'data')
    assert backward.alone == 1 and torch.allclose(got[:, 1, 1], (g * g).sum(0)) and torch.allclose(got[:, 0, 0], (g * h * g * h).sum(0))


def test_blocks_of_two_passes_that_left_the_layer_norm_out(monkeypatch):
    """Each pass ends with its blocks: a later forward pass, and new values in what the first one saved, do not reach them."""
    from asdl_amd import OP_COV_UNIT_WISE, extend
    backward = _stand_ins(monkeypatch)
    torch.manual_seed(3)
    ln, x = FusedLayerNorm(6), torch.randn(5, 6)
    want = 0
    with extend(ln, OP_COV_UNIT_WISE) as cxt:
        for turn in range(2):
            y = ln(x)
            (g,) = torch.autograd.grad((y ** 3).sum(), y)
            h = _layer_norm(x)[0]
            want = want + torch.stack([(g * h * g * h).sum(0), (g * g).sum(0)])
            del y
            g.mul_(100)
            x.normal_()
            with torch.no_grad():
                ln.weight.mul_(1.5)
        got = cxt.get_result(ln, OP_COV_UNIT_WISE, 'data')
    assert backward.alone == 2 and torch.allclose(got[:, 0, 0], want[0]) and torch.allclose(got[:, 1, 1], want[1])


@pytest.mark.parametrize('where', ['tensor', 'two calls', 'checkpoint', 'full'])
def test_a_gradient_that_another_hook_scales_in_place_does_not_reach_the_blocks(where, monkeypatch):
    """The blocks are those of the gradient that the framework's hook sees, as with torch.nn.LayerNorm."""
    from torch.utils.checkpoint import checkpoint
    from asdl_amd import OP_COV_UNIT_WISE, extend
    _stand_ins(monkeypatch)
    torch.manual_seed(4)
    pre = nn.Linear(6, 6)
    x, got, grads = torch.randn(5, 6), [], []

    def scale(g):
        g.mul_(10)

    def scale_of_module(module, grads, out_grads):
        out_grads[0].mul_(10)
    for ln in (nn.LayerNorm(6), FusedLayerNorm(6)):
        pre.zero_grad()
        with extend(ln, OP_COV_UNIT_WISE) as cxt:
            if where == 'full':
                ln.register_full_backward_hook(scale_of_module)
            y = checkpoint(lambda z: ln(pre(z)), x, use_reentrant=False) if where == 'checkpoint' else ln(pre(x))
            if where != 'full':
                y.register_hook(scale)
            if where == 'two calls':
                y.register_hook(lambda g: g * 2)
            (y ** 3).sum().backward()          # (of y ** 2 the sum is a constant, and the gradients in front all rounding)
            got.append(cxt.get_result(ln, OP_COV_UNIT_WISE, 'data').clone())
            grads.append(pre.weight.grad.clone())
    assert torch.allclose(got[0], got[1], rtol=1e-4, atol=1e-5) and torch.allclose(grads[0], grads[1], rtol=1e-4, atol=1e-5)


def test_a_gradient_that_changes_behind_all_hooks_is_refused(monkeypatch):
    """A hook on the autograd node itself runs behind those on the tensor, unseen: what it writes to the gradient is noticed."""
    from asdl_amd import OP_COV_UNIT_WISE, extend
    _stand_ins(monkeypatch)
    ln, pre, x = FusedLayerNorm(6), nn.Linear(6, 6), torch.randn(5, 6)
    with pytest.raises(RuntimeError, match='in place'):
        with extend(ln, OP_COV_UNIT_WISE):
            y = ln(pre(x))

            def scale(grads):
                grads[0].mul_(10)
            y.grad_fn.register_prehook(scale)
            (y ** 2).sum().backward()


@pytest.mark.parametrize('limited', [False, True])
def test_two_sets_of_hooks_on_one_layer_norm_have_their_blocks_each(limited, monkeypatch):
    from asdl_amd import OP_COV_UNIT_WISE, extend
    backward = _stand_ins(monkeypatch)
    torch.manual_seed(5)
    ln, x = FusedLayerNorm(6), torch.randn(5, 6)
    with extend(ln, OP_COV_UNIT_WISE) as first, extend(ln, OP_COV_UNIT_WISE) as second:
        second.set_cov_scale(0.5)
        y = ln(x)
        loss = (y ** 3).sum()
        torch.autograd.grad(loss, y) if limited else loss.backward()
        got = [cxt.get_result(ln, OP_COV_UNIT_WISE, 'data').clone() for cxt in (first, second)]
    h, g = _layer_norm(x)[0], 3 * y.detach() ** 2
    assert torch.allclose(got[0][:, 1, 1], (g * g).sum(0)) and torch.allclose(got[0][:, 0, 0], (g * h * g * h).sum(0)) and torch.allclose(got[1], 0.5 * got[0])
    assert backward.alone == 2          # (the input needs no gradient)


@pytest.mark.parametrize('how', ['attribute', 'subclass'])
@pytest.mark.parametrize('filters', [dict(mc_temperature=0.5), dict(mc_top_k=3), dict(mc_top_p=0.9), dict(mc_min_p=0.1)])
def test_filters_with_replaced_targets_are_refused(filters, how, monkeypatch):
    """sample_targets() gets the whole distribution: filters would be dropped.  Before the forward pass, so that no factor has changed."""
    from asdl_amd import fisher
    cpu_backend.install(monkeypatch)
    model = nn.Sequential(nn.Linear(3, 4))
    x, ran = torch.randn(2, 3), []
    model.register_forward_pre_hook(lambda *_: ran.append(1))

    class Mine(fisher.FisherMCCrossEntropy):
        def sample_targets(self, dist, i):
            return torch.zeros(2, dtype=torch.long)
    for more in (filters, {}):
        config = FisherConfig(FISHER_MC, [SHAPE_KRON], loss_type=LOSS_CROSS_ENTROPY, data_size=2, **more)
        maker = Mine(model, config) if how == 'subclass' else get_fisher_maker(model, config)
        if how == 'attribute':
            maker.sample_targets = lambda dist, i: torch.zeros(2, dtype=torch.long)
        maker.setup_model_call(model, x)
        if more:
            with pytest.raises(ValueError, match='sample_targets'):
                maker.forward_and_backward()
            assert not ran
        else:
            maker.forward_and_backward()


@pytest.mark.parametrize('loss', ['cubes', 'linear'])
def test_a_second_derivative_of_layer_norm_raises(loss, monkeypatch):
    """However it is asked for: a graph that ends at the gradient would give zeros."""
    _stand_ins(monkeypatch)
    torch.manual_seed(6)
    ln, x, c = FusedLayerNorm(6), torch.randn(5, 6), torch.randn(5, 6)

    def f(x):
        return (ln(x) ** 3).sum() if loss == 'cubes' else (ln(x) * c).sum()
    with pytest.raises(RuntimeError, match='differentiable once'):
        torch.autograd.functional.hessian(f, x)
    x.requires_grad_()
    for ask in (lambda dx: torch.autograd.grad(dx.square().sum(), x, allow_unused=True), lambda dx: dx.square().sum().backward(),
                lambda dx: torch.autograd.grad(dx.square().sum(), ln.weight, allow_unused=True)):
        (dx,) = torch.autograd.grad(f(x), x, create_graph=True)
        with pytest.raises(RuntimeError, match='differentiable once'):
            ask(dx)
    (dx, db) = torch.autograd.grad(f(x), (x, ln.bias), create_graph=True)
    (want,) = torch.autograd.grad(f(x), x)
    assert torch.equal(dx.detach(), want) and db.shape == (6,)
    plain = nn.LayerNorm(6)
    assert torch.allclose(want, torch.autograd.grad((plain(x) ** 3).sum() if loss == 'cubes' else (plain(x) * c).sum(), x)[0], rtol=1e-4, atol=1e-5)
