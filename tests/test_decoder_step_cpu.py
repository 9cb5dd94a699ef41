"""The cross entropy of a linear layer, embeddings and activations in 8 bits without a GPU: what is refused, and the host logic around the
kernels with the kernels replaced by their definitions."""
import copy

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

import asdl_amd
from asdl_amd import (FISHER_EMP, FISHER_MC, FisherConfig, FusedEmbedding, GELU8bit, GradientMaker, LOSS_CROSS_ENTROPY, Linear8bit, SHAPE_KRON,
                      get_fisher_maker, kernels, module_wise_assignments)
from asdl_amd import layers
from tests import cpu_backend

F32, BF16, F16, I32, I64, BAD = 0, 1, 4, 5, 6, 9


def test_cpu_tensors_are_refused():
    x, w, t = torch.randn(4, 8), torch.randn(10, 8, requires_grad=True), torch.zeros(4, dtype=torch.int64)
    kept = kernels.Quantized8(x.to(torch.float8_e4m3fn), torch.zeros(4, 1, dtype=torch.int8))
    for call in (lambda: kernels.linear_cross_entropy(x, w, t), lambda: kernels.linear_cross_entropy_backward(x, x, w, t, x), lambda: kernels.embedding(t, w),
                 lambda: kernels.embedding_backward(x, t, 10), lambda: kernels.quantize_8bit(x), lambda: kernels.dequantize_8bit(kept), lambda: kernels.gelu_8bit(x),
                 lambda: kernels.gelu_8bit_backward(x, kept), lambda: kernels.weight_grad_8bit(x, kept), lambda: asdl_amd.linear_cross_entropy(x, w, t),
                 lambda: asdl_amd.embedding(t, w), lambda: asdl_amd.gelu_8bit(w), lambda: asdl_amd.linear_8bit(x, w)):
        with pytest.raises(RuntimeError, match='ROCm device'):
            call()


def test_entry_points_refuse_bad_arguments():
    """Before anything is launched: return codes of the C interface."""
    from asdl_amd import _lib
    lib = _lib.load()
    a, room = 4096, 1 << 44                    # stands for an address; nothing reads it

    def loss(h=a, dtype=F32, ldh=64, w=a, ldw=64, bias=a, bias_dtype=F32, targets=a, rows=8, classes=100, width=64, reduction=2, out=a, lse=a, ws=a, need=room):
        return lib.ak_linear_cross_entropy(h, dtype, ldh, w, ldw, bias, bias_dtype, targets, rows, classes, width, -100, reduction, out, lse, ws, need, None)
    for kw in (dict(h=None), dict(w=None), dict(targets=None), dict(out=None), dict(lse=None), dict(dtype=BAD), dict(dtype=I64), dict(bias_dtype=BF16),
               dict(ldh=63), dict(ldw=63), dict(rows=-1), dict(classes=0), dict(width=0), dict(reduction=3), dict(reduction=-1), dict(rows=0)):
        assert loss(**kw) == -1, kw
    assert loss(rows=0, reduction=0) == 0
    for kw in (dict(rows=(1 << 28) + 1), dict(classes=(1 << 28) + 1), dict(width=(1 << 20) + 1, ldh=1 << 21, ldw=1 << 21), dict(ldh=(1 << 21) + 1), dict(ldw=(1 << 21) + 1)):
        assert loss(**kw) == -5, kw
    need = lib.ak_linear_cross_entropy_ws_bytes(F32, 8, 100, 64, 0)
    assert loss(ws=None) == -2 and loss(need=64) == -2 and need > 0
    for args in ((BAD, 8, 100, 64), (F32, 0, 100, 64), (F32, 8, 0, 64), (F32, 8, 100, 0), (F32, 1 << 29, 100, 64)):
        assert lib.ak_linear_cross_entropy_ws_bytes(*args, 1) == 0, args
    assert lib.ak_linear_cross_entropy_ws_bytes(BF16, 8192, 50257, 768, 1) < 2 * (512 << 20) + 8 * 8192 * 768 * 4 + (8192 + 50257) * 768 * 2

    def back(g=a, h=a, dtype=BF16, bias_dtype=F32, targets=a, lse=a, rows=8, width=64, reduction=2, dh=a, dw=a, db=a, ws=a, need=room):
        return lib.ak_linear_cross_entropy_backward(g, h, dtype, 64, a, 64, a, bias_dtype, targets, lse, rows, 100, width, -100, reduction, dh, dw, db, ws, need, None)
    for kw in (dict(g=None), dict(h=None), dict(targets=None), dict(lse=None), dict(dtype=BAD), dict(bias_dtype=F16), dict(rows=0), dict(width=65), dict(reduction=7)):
        assert back(**kw) == -1, kw
    assert back(dh=None, dw=None, db=None) == 0 and back(ws=None) == -2 and back(need=1000) == -2

    def rows_of(tokens=a, kind=I64, count=5, table=a, dtype=F32, ld=64, rows=10, width=64, out=a, out_dtype=F32):
        return lib.ak_embedding(tokens, kind, count, table, dtype, ld, rows, width, 1.0, out, out_dtype, None)
    for kw in (dict(tokens=None), dict(table=None), dict(out=None), dict(kind=F32), dict(dtype=BAD), dict(dtype=I32), dict(out_dtype=BF16), dict(ld=63), dict(count=-1),
               dict(rows=-1), dict(width=0)):
        assert rows_of(**kw) == -1, kw
    assert rows_of(count=0, tokens=None, out=None) == 0
    for kw in (dict(count=(1 << 30) + 1), dict(rows=(1 << 30) + 1), dict(width=(1 << 24) + 1, ld=1 << 25)):
        assert rows_of(**kw) == -5, kw

    def grad(g=a, dtype=F32, ldg=64, tokens=a, kind=I64, count=5, rows=10, width=64, out=a, out_dtype=F32, ldo=64, ws=a, need=room):
        return lib.ak_embedding_backward(g, dtype, ldg, tokens, kind, count, rows, width, 1.0, -1, 0.0, out, out_dtype, ldo, ws, need, None)
    for kw in (dict(g=None), dict(tokens=None), dict(out=None), dict(dtype=BAD), dict(out_dtype=I64), dict(kind=BF16), dict(ldg=63), dict(ldo=63), dict(count=-1),
               dict(width=0)):
        assert grad(**kw) == -1, kw
    assert grad(rows=0) == 0 and grad(ws=None) == -2 and grad(need=100) == -2 and grad(count=(1 << 30) + 1) == -5
    assert lib.ak_embedding_backward_ws_bytes(-1, 10, 64) == 0 and lib.ak_embedding_backward_ws_bytes(0, 10, 64) > 0

    def keep(x=a, dtype=F32, ld=64, rows=4, width=64, gelu=-1, y=a, codes=a, exponents=a):
        return lib.ak_quantize_8bit(x, dtype, ld, rows, width, gelu, y, codes, exponents, None)
    for kw in (dict(x=None), dict(codes=None), dict(exponents=None), dict(gelu=0, y=None), dict(dtype=BAD), dict(ld=63), dict(rows=-1), dict(width=0), dict(gelu=2),
               dict(gelu=-2)):
        assert keep(**kw) == -1, kw
    assert keep(rows=0) == 0 and keep(rows=1 << 40) == -5 and keep(width=(1 << 24) + 1, ld=1 << 25) == -5

    def values(codes=a, exponents=a, rows=4, width=64, gelu=0, g=a, ldg=64, y=a, dtype=F32):
        return lib.ak_dequantize_8bit(codes, exponents, rows, width, gelu, g, ldg, y, dtype, None)
    for kw in (dict(codes=None), dict(exponents=None), dict(y=None), dict(g=None), dict(ldg=63), dict(dtype=BAD), dict(gelu=2), dict(rows=-1), dict(width=0)):
        assert values(**kw) == -1, kw
    assert values(rows=0) == 0

    def weight(g=a, dtype=F32, ldg=64, codes=a, exponents=a, rows=4, width=64, out=64, dw=a, db=a, grad_dtype=F32, ws=a, need=room):
        return lib.ak_weight_grad_8bit(g, dtype, ldg, codes, exponents, rows, width, out, dw, db, grad_dtype, ws, need, None)
    for kw in (dict(g=None), dict(codes=None), dict(exponents=None), dict(dtype=BAD), dict(grad_dtype=BAD), dict(ldg=63), dict(rows=0), dict(width=0), dict(out=0)):
        assert weight(**kw) == -1, kw
    assert weight(codes=None, exponents=None, dw=None, width=0, need=64) == -2
    assert 0 < lib.ak_weight_grad_8bit_ws_bytes(F32, 4, 0, 64) < lib.ak_weight_grad_8bit_ws_bytes(F32, 4, 64, 64)
    assert weight(dw=None, db=None) == 0 and weight(ws=None) == -2 and weight(need=64) == -2 and weight(width=(1 << 20) + 1) == -5
    assert lib.ak_weight_grad_8bit_ws_bytes(F32, 0, 64, 64) == 0


def test_calls_in_one_step_leave_the_unusual_to_the_others():
    from asdl_amd import _lib
    host = _lib.load_host()
    x, w, t = torch.randn(4, 8), torch.randn(10, 8), torch.zeros(4, dtype=torch.int64)
    codes, exps = x.to(torch.float8_e4m3fn), torch.zeros(4, 1, dtype=torch.int8)
    assert host.linear_cross_entropy(x, w, t, None, -100, 0, 0) is None and host.linear_cross_entropy(x, 'w', t, None, -100, 0, 0) is None
    assert host.linear_cross_entropy() is None and host.linear_cross_entropy_backward(x, w, t, None, -100, 0, x, x, 7, 0) is None
    assert host.embedding(t, w, 1.0, False, 0) is None and host.embedding(t, None, 1.0, False, 0) is None and host.embedding_backward(x, t, 10, 1.0, -1, 0) is None
    assert host.embedding_backward(x, t, 2.5, 1.0, -1, 0) is None and host.quantize_8bit(x, -1, 0) is None and host.quantize_8bit(1, 2, 3) is None
    assert host.dequantize_8bit(codes, exps, -1, None, 0, 0) is None and host.weight_grad_8bit(codes, exps, x, 3, 0, 0) is None and host.weight_grad_8bit() is None
    with pytest.raises(TypeError):
        host.bind_step(1)
    with pytest.raises(ValueError):
        host.bind_step(*[0] * 10)


# ------------------------------------------------------------------------------------------------ with stand-ins for the kernels
class Stand:
    """The kernels by their definitions; what each call was asked for."""

    def __init__(self):
        self.calls = []

    def linear_cross_entropy(self, h, weight, targets, bias=None, ignore_index=-100, reduction='mean'):
        logits = F.linear(h, weight, bias).float()
        self.calls.append(('loss', h.dtype, weight.dtype))
        return F.cross_entropy(logits.reshape(-1, logits.shape[-1]), targets.reshape(-1), ignore_index=ignore_index, reduction=reduction).reshape(
            targets.shape if reduction == 'none' else ()).clone(), torch.logsumexp(logits, -1)

    def linear_cross_entropy_backward(self, g, h, weight, targets, lse, bias=None, ignore_index=-100, reduction='mean', need_h=True, need_weight=True, need_bias=True):
        self.calls.append(('loss back', need_h, need_weight, need_bias))
        with torch.enable_grad():
            leaves = [t.detach().requires_grad_() if t is not None else None for t in (h, weight, bias)]
            loss, _ = Stand().linear_cross_entropy(leaves[0], leaves[1], targets, leaves[2], ignore_index, reduction)
            grads = iter(torch.autograd.grad(loss, [t for t in leaves if t is not None], g))
        return tuple(next(grads) if t is not None else None for t in leaves)

    def embedding(self, tokens, weight, scale=1.0, out_dtype=None):
        return weight.detach()[tokens.long()] * scale

    def embedding_backward(self, g, tokens, num_embeddings, scale=1.0, padding_idx=None, out=None, beta=0.0, dtype=None):
        self.calls.append(('embed back', padding_idx, dtype))
        grad = torch.zeros(num_embeddings, g.shape[-1]).index_add_(0, tokens.reshape(-1).long(), g.reshape(-1, g.shape[-1]).float()) * scale
        if padding_idx is not None:
            grad[padding_idx] = 0
        return grad.to(dtype)

    def quantize_8bit(self, x):
        self.calls.append(('keep', x.dtype))
        return kernels.Quantized8(x.detach().to(torch.float8_e4m3fn), torch.zeros(1, dtype=torch.int8))

    def gelu_8bit(self, x, approximate='none'):
        return F.gelu(x.detach(), approximate=approximate), self.quantize_8bit(x)

    def gelu_8bit_backward(self, g, kept, approximate='none'):
        with torch.enable_grad():
            x = kept.codes.float().requires_grad_()
            return torch.autograd.grad(F.gelu(x, approximate=approximate), x, g)[0]

    def weight_grad_8bit(self, g, kept, need_weight=True, need_bias=True, dtype=None):
        self.calls.append(('weight', need_weight, need_bias))
        g = g.flatten(0, -2).float()
        return (g.t() @ kept.codes.float().flatten(0, -2)).to(dtype) if need_weight else None, g.sum(0).to(dtype) if need_bias else None


@pytest.fixture
def stand(monkeypatch):
    stand = Stand()
    for name in ('linear_cross_entropy', 'linear_cross_entropy_backward', 'embedding', 'embedding_backward', 'quantize_8bit', 'gelu_8bit', 'gelu_8bit_backward',
                 'weight_grad_8bit'):
        monkeypatch.setattr(kernels, name, getattr(stand, name))
    return stand


def coarse(*shape, seed):
    """Numbers that 8 bits hold exactly."""
    return torch.randint(-7, 8, shape, generator=torch.Generator().manual_seed(seed)).float() / 4


class Decoder(nn.Module):
    def __init__(self, vocab=20, d=6):
        super().__init__()
        self.wte, self.a, self.act, self.b, self.head = nn.Embedding(vocab, d, padding_idx=2), nn.Linear(d, 10), nn.GELU(), nn.Linear(10, d), nn.Linear(d, vocab)

    def features(self, idx):
        return self.b(self.act(self.a(self.wte(idx))))

    def forward(self, idx):
        return self.head(self.features(idx))


def test_gradients_are_those_of_torch(stand):
    torch.manual_seed(0)
    model = Decoder()
    for p in model.parameters():
        p.data = coarse(*p.shape, seed=p.numel())
    fused = copy.deepcopy(model)
    state, params = list(fused.state_dict()), [id(p) for p in fused.parameters()]
    assert asdl_amd.fuse_embeddings(fused) == 1 and asdl_amd.keep_activations_8bit(fused) == 4
    assert asdl_amd.fuse_embeddings(fused) == 0 and asdl_amd.keep_activations_8bit(fused) == 0
    assert list(fused.state_dict()) == state and [id(p) for p in fused.parameters()] == params
    assert [type(m) for m in (fused.wte, fused.a, fused.act, fused.head)] == [FusedEmbedding, Linear8bit, GELU8bit, Linear8bit]
    idx, t = torch.randint(0, 20, (3, 4)), torch.randint(0, 20, (3, 4))
    t[0, 0] = -100
    for reduction in ('mean', 'sum', 'none'):
        model.zero_grad()
        fused.zero_grad()
        want = F.cross_entropy(model(idx).view(-1, 20), t.view(-1), reduction=reduction)
        got = asdl_amd.linear_cross_entropy(fused.features(idx), fused.head.weight, t, fused.head.bias, reduction=reduction)
        assert torch.allclose(got.view(-1), want.view(-1), atol=1e-5) and got.shape == (t.shape if reduction == 'none' else ())
        want.sum().backward()
        got.sum().backward()
        for (name, p), q in zip(model.named_parameters(), fused.parameters()):
            exact = name not in ('a.weight', 'a.bias', 'b.weight', 'wte.weight')        # (behind a kept value that 8 bits do not hold)
            assert torch.allclose(p.grad, q.grad, rtol=1e-4 if exact else 0.1, atol=1e-4 if exact else 0.1 * float(p.grad.abs().max())), name


def test_only_what_a_pass_takes_is_computed(stand):
    w, x, b = (coarse(*s, seed=i).requires_grad_() for i, s in enumerate(((5, 4), (7, 4), (5,))))
    t = torch.randint(0, 5, (7,))

    def last():
        calls, stand.calls[:] = [c for c in stand.calls if c[0] in ('loss back', 'weight')], []
        return calls
    asdl_amd.linear_cross_entropy(x, w, t, b).backward()
    assert last() == [('loss back', True, True, True)]
    for inputs, needs in (([x], (True, False, False)), ([w], (False, True, False)), ([b, x], (True, False, True))):
        torch.autograd.grad(asdl_amd.linear_cross_entropy(x, w, t, b), inputs)
        assert last() == [('loss back', *needs)], inputs
    asdl_amd.linear_cross_entropy(x, w.detach(), t).backward()
    assert last() == [('loss back', True, False, False)]
    y = asdl_amd.linear_8bit(x, w, b)
    torch.autograd.grad(y.sum(), [x], retain_graph=True)
    assert last() == []
    torch.autograd.grad(y.sum(), [b], retain_graph=True)
    assert last() == [('weight', False, True)]
    y.sum().backward()
    assert last() == [('weight', True, True)]
    asdl_amd.linear_8bit(x, w.detach(), None).sum().backward()
    assert ('keep', torch.float32) not in stand.calls and last() == []
    with torch.no_grad():
        assert torch.equal(asdl_amd.gelu_8bit(x), F.gelu(x)) and not stand.calls


def test_a_second_derivative_raises(stand):
    w, x, e = coarse(5, 4, seed=1).requires_grad_(), coarse(7, 4, seed=2).requires_grad_(), coarse(9, 4, seed=3).requires_grad_()
    t = torch.randint(0, 5, (7,))
    for make, leaf in ((lambda: asdl_amd.linear_cross_entropy(x, w, t), x), (lambda: asdl_amd.linear_8bit(x, w).square().sum(), x),
                       (lambda: asdl_amd.gelu_8bit(x).square().sum(), x), (lambda: asdl_amd.embedding(t, e).square().sum(), e)):
        g, = torch.autograd.grad(make(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match='differentiable once'):
            torch.autograd.grad(g.sum(), leaf)
        with pytest.raises(RuntimeError, match='differentiable once'):
            g.square().sum().backward()


def test_embedding_modules(stand):
    made = FusedEmbedding(10, 4, padding_idx=3, scale=2.0)
    idx = torch.tensor([[1, 3], [3, 9]], dtype=torch.int32)
    assert torch.equal(made(idx), 2 * made.weight[idx.long()])
    made(idx).sum().backward()
    assert float(made.weight.grad[3].abs().sum()) == 0 and torch.equal(made.weight.grad[9], torch.full((4,), 2.0))
    assert stand.calls == [('embed back', 3, torch.float32)]
    for option in (dict(max_norm=1.0), dict(scale_grad_by_freq=True), dict(sparse=True)):
        with pytest.raises(ValueError, match='max_norm'):
            FusedEmbedding(10, 4, **option)
        assert asdl_amd.fuse_embeddings(nn.Sequential(nn.Embedding(10, 4, **option))) == 0

    class Mine(nn.Embedding):
        pass
    assert asdl_amd.fuse_embeddings(nn.Sequential(Mine(10, 4))) == 0


def test_stand_ins_take_the_rules_of_their_classes():
    model = nn.Sequential(nn.Linear(4, 4), nn.LayerNorm(4), nn.Linear(4, 3))
    asdl_amd.keep_activations_8bit(model)
    got = {m: v for m, v in module_wise_assignments(model, 'common', (nn.Linear, 'kron'))}
    assert got[model[0]] == got[model[2]] == ['kron'] and got[model[1]] == ['common']
    assert not list(module_wise_assignments(model, 'common', ignore_modules=[nn.Linear, nn.LayerNorm]))


def test_a_maker_takes_the_loss(stand, monkeypatch):
    """GradientMaker, and FisherEmp, which asks for the sum: factors and gradients are those of the model with its head."""
    for name in ('syrk_tn', 'kron_damping', 'chol_inv_batched', 'chol_inv_grouped'):
        monkeypatch.setattr(kernels, name, getattr(cpu_backend, name))
    torch.manual_seed(1)
    model = Decoder()
    with torch.no_grad():
        model.wte.weight[2] = 0
    idx, t = torch.randint(0, 20, (3, 4)), torch.randint(0, 20, (3, 4))
    other = copy.deepcopy(model)

    def flat(y, target, reduction='mean'):
        return F.cross_entropy(y.reshape(-1, y.shape[-1]), target.reshape(-1), reduction=reduction)
    plain = GradientMaker(model)
    plain.setup_loss_call(flat, plain.setup_model_call(model, idx), t)
    _, want = plain.forward_and_backward()
    maker = GradientMaker(other)
    maker.setup_loss_call(asdl_amd.linear_cross_entropy, maker.setup_model_call(other.features, idx), other.head.weight, t, other.head.bias)
    _, got = maker.forward_and_backward()
    assert torch.allclose(got, want) and all(torch.allclose(p.grad, q.grad, atol=1e-6) for p, q in zip(model.parameters(), other.parameters()))
    made = []
    for net, call in ((model, lambda m, net: m.setup_loss_call(flat, m.setup_model_call(net, idx), t)),
                      (other, lambda m, net: m.setup_loss_call(asdl_amd.linear_cross_entropy, m.setup_model_call(net.features, idx), net.head.weight, t, net.head.bias))):
        fisher = get_fisher_maker(net, FisherConfig(FISHER_EMP, [SHAPE_KRON], data_size=12, ignore_modules=['head', 'wte']))
        call(fisher, net)
        net.zero_grad()
        _, loss = fisher.forward_and_backward(calc_loss_grad=True)
        made.append((loss, [p.grad.clone() for p in net.parameters()], [m.fisher.kron for m in (net.a, net.b)]))
    assert torch.allclose(made[0][0], made[1][0])
    assert all(torch.allclose(a, b, atol=1e-6) for a, b in zip(made[0][1], made[1][1]))
    assert all(torch.allclose(a.A, b.A) and torch.allclose(a.B, b.B, atol=1e-6) for a, b in zip(made[0][2], made[1][2]))


def test_a_sampled_fisher_leaves_the_weights_of_8_bit_layers_out(stand, monkeypatch):
    for name in ('syrk_tn', 'kron_damping', 'chol_inv_batched', 'chol_inv_grouped'):
        monkeypatch.setattr(kernels, name, getattr(cpu_backend, name))
    torch.manual_seed(2)
    model = nn.Sequential(nn.Linear(6, 8), nn.GELU(), nn.Linear(8, 5))
    asdl_amd.keep_activations_8bit(model)
    maker = get_fisher_maker(model, FisherConfig(FISHER_MC, [SHAPE_KRON], loss_type=LOSS_CROSS_ENTROPY, data_size=4))
    maker.setup_model_call(model, torch.randn(4, 6))
    maker.forward_and_backward()
    assert model[0].fisher.has_kron and not [c for c in stand.calls if c[0] == 'weight']


def test_public_names():
    for name in layers.__all__:
        assert getattr(asdl_amd, name) is getattr(layers, name)


def test_embedding_refuses_a_padding_outside_the_table():
    for padding in (7, -8):
        with pytest.raises(ValueError, match='within 7 rows'):
            asdl_amd.embedding(torch.zeros(3, dtype=torch.int64), torch.zeros(7, 4), padding)


def test_weight_gradient_refuses_to_go_without_the_input():
    with pytest.raises(ValueError, match='kept input'):
        kernels.weight_grad_8bit(torch.zeros(3, 4), None)
