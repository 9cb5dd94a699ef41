"""A decoder's training step with the cross entropy of its head, its embeddings and 8-bit activations, together: under autograd and
autocast, with tied weights, under the hooks of the gradient makers, checkpointed and captured."""
import copy

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

import asdl_amd
from asdl_amd import (FISHER_EMP, FISHER_MC, FusedEmbedding, GELU8bit, GradientMaker, KfacGradientMaker, Linear8bit, PreconditioningConfig,
                      ShampooGradientMaker, kernels)

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF16 = torch.bfloat16


def off(got, want):
    want = want.double()
    return float((got.detach().double() - want).norm() / want.norm().clamp_min(1e-300))


def rand(*shape, seed, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, device='cuda', generator=torch.Generator('cuda').manual_seed(seed)) * scale).to(dtype)


def ints(high, *shape, seed):
    return torch.randint(0, high, shape, device='cuda', generator=torch.Generator('cuda').manual_seed(seed))


def kept(x):
    return kernels.dequantize_8bit(kernels.quantize_8bit(x), torch.float32)


class _Kept(torch.autograd.Function):
    """A linear layer by torch's products whose weight gradient reads the kept input."""

    @staticmethod
    def forward(ctx, x, w, b):
        ctx.save_for_backward(kept(x), w)
        return F.linear(x, w, b)

    @staticmethod
    def backward(ctx, g):
        x, w = ctx.saved_tensors
        return g @ w, (g.flatten(0, -2).float().t() @ x.flatten(0, -2)).to(w.dtype), g.flatten(0, -2).float().sum(0).to(w.dtype) if ctx.needs_input_grad[2] else None


class _KeptGELU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        ctx.save_for_backward(kept(x))
        return F.gelu(x)

    @staticmethod
    def backward(ctx, g):
        with torch.enable_grad():
            x = ctx.saved_tensors[0].double().requires_grad_()
            return torch.autograd.grad(F.gelu(x), x, g.double())[0].to(g.dtype)


class Linear(nn.Linear):
    def forward(self, x):
        if not self.of_kept:
            return super().forward(x)
        dtype = torch.get_autocast_dtype('cuda') if torch.is_autocast_enabled('cuda') else x.dtype
        return _Kept.apply(x.to(dtype), self.weight.to(dtype), None if self.bias is None else self.bias.to(dtype))


class Decoder(nn.Module):
    def __init__(self, vocab=211, d=48, layers=2, heads=4, n=32, of_kept=False):
        super().__init__()
        Linear.of_kept = of_kept
        self.wte, self.wpe, self.heads, self.act = nn.Embedding(vocab, d), nn.Embedding(n, d), heads, nn.GELU()
        self.layers = nn.ModuleList(nn.ModuleList([nn.LayerNorm(d), nn.Linear(d, 3 * d), nn.Linear(d, d), nn.LayerNorm(d), nn.Linear(d, 4 * d), nn.Linear(4 * d, d)])
                                    for _ in range(layers))
        self.ln, self.head = nn.LayerNorm(d), nn.Linear(d, vocab, bias=False)

    def features(self, idx):
        x = self.wte(idx) + self.wpe(torch.arange(idx.shape[1], device=idx.device))
        for ln1, qkv, proj, ln2, up, down in self.layers:
            b, t, d = x.shape
            q, k, v = (z.view(b, t, self.heads, -1).transpose(1, 2) for z in qkv(ln1(x)).split(d, 2))
            x = x + proj(F.scaled_dot_product_attention(q, k, v, is_causal=True).transpose(1, 2).reshape(b, t, d))
            x = x + down(self.act(up(ln2(x))))
        return self.ln(x)

    def forward(self, idx):
        return self.head(self.features(idx))


class OfKept(nn.GELU):
    def forward(self, x):
        return _KeptGELU.apply(x)


def decoders(tied=False, seed=1):
    """A decoder of torch's operators that reads kept inputs on the way back, and the same one with the framework's."""
    torch.manual_seed(seed)
    plain = Decoder().cuda()
    if tied:
        plain.head.weight = plain.wte.weight
    fused = copy.deepcopy(plain)
    Linear.of_kept = True
    for m in plain.modules():
        if type(m) is nn.Linear and m is not plain.head:
            m.__class__ = Linear
        elif type(m) is nn.GELU:
            m.__class__ = OfKept
    assert asdl_amd.fuse_layer_norms(fused) == 5 and asdl_amd.fuse_embeddings(fused) == 2 and asdl_amd.keep_activations_8bit(fused) == 10
    assert type(fused.wte) is FusedEmbedding and type(fused.act) is GELU8bit and type(fused.head) is Linear8bit
    return plain, fused


def flat_loss(y, target, reduction='mean'):
    return F.cross_entropy(y.reshape(-1, y.shape[-1]).float(), target.reshape(-1), reduction=reduction)


@pytest.mark.parametrize('reduction', ['mean', 'sum', 'none'])
def test_gradients_of_the_loss(reduction):
    """Against the gradients of the definition in 64 bits and its differences along one direction (as for layer norm: off by some 1e-8 at a
    step of 1e-4).  Scores of 64 products are off by (2 * 64 u + 2^-21) a, a < 30 the sum of magnitudes: 2.4e-4 at most, of the
    shares and so of the gradients; 1e-4 is allowed in the 2-norm, where signs cancel."""
    h, w, b = rand(3, 50, 64, seed=1).requires_grad_(), rand(900, 64, seed=2, scale=0.3).requires_grad_(), rand(900, seed=3).requires_grad_()
    t = ints(900, 3, 50, seed=4)
    t[1, ::7] = -100
    loss = asdl_amd.linear_cross_entropy(h, w, t, b, reduction=reduction)
    g = rand(*loss.shape, seed=5)
    got = torch.autograd.grad(loss, (h, w, b), g)
    doubles = [x.detach().double().requires_grad_() for x in (h, w, b)]

    def f(h, w, b):
        return F.cross_entropy((h @ w.t() + b).flatten(0, 1), t.flatten(), reduction=reduction).view(loss.shape)
    want = torch.autograd.grad(f(*doubles), doubles, g.double())
    assert off(loss, f(*doubles).detach()) < 1e-5
    for i, (x, y) in enumerate(zip(got, want)):
        assert x.shape == y.shape and off(x, y) < 1e-4
        v = rand(*doubles[i].shape, seed=6).double()
        ends = [(f(*[d + s * 1e-4 * v if j == i else d for j, d in enumerate(doubles)]).detach() * g.double()).sum() for s in (1, -1)]
        assert abs(float((x.double() * v).sum()) - float((ends[0] - ends[1]) / 2e-4)) < 2e-4 * float(y.norm() * v.norm())


def test_gradients_of_embeddings_and_gelu():
    """Differences of the definitions; the gradient of a GELU is that of the kept input."""
    e, g = rand(70, 40, seed=1).requires_grad_(), rand(5, 9, 40, seed=2)
    idx = ints(70, 5, 9, seed=3)
    y = asdl_amd.embedding(idx, e, 4, 1.5)
    assert torch.equal(y, F.embedding(idx, e) * 1.5)
    de, = torch.autograd.grad(y, e, g)
    want, = torch.autograd.grad(F.embedding(idx, e, 4) * 1.5, e, g)
    assert off(de, want) < 8 * U and float(de[4].abs().sum()) == 0
    for way in ('none', 'tanh'):
        x, g = rand(50, 300, seed=4, scale=2.0).requires_grad_(), rand(50, 300, seed=5)
        dx, = torch.autograd.grad(asdl_amd.gelu_8bit(x, way), x, g)
        at = kept(x.detach()).double()
        v = 1e-4
        want = (F.gelu(at + v, approximate=way) - F.gelu(at - v, approximate=way)) / (2 * v) * g.double()
        assert off(dx, want) < 1e-6


def test_types_under_autocast():
    x, w, b = rand(6, 30, 96, seed=1).requires_grad_(), rand(500, 96, seed=2, scale=0.1).requires_grad_(), rand(500, seed=3).requires_grad_()
    t = ints(500, 6, 30, seed=4)
    with torch.autocast('cuda', dtype=BF16):
        loss = asdl_amd.linear_cross_entropy(x, w, t, b)
        y = asdl_amd.linear_8bit(x, w, b)
        z = asdl_amd.gelu_8bit(y)
        want = F.cross_entropy(F.linear(x, w, b).flatten(0, 1), t.flatten())
        assert torch.equal(y, F.linear(x, w, b))
    assert loss.dtype == torch.float32 and y.dtype == z.dtype == BF16 and asdl_amd.embedding(t, w).dtype == torch.float32
    # (torch's logits are rounded to bfloat16: 2^-8 of scores of about 1 each, of which a mean over 180 rows is left with far less)
    assert abs(float(loss.detach() - want.detach())) < 2 ** -8
    for out in (loss, z.float().square().mean()):
        grads = torch.autograd.grad(out, (x, w, b), retain_graph=True)
        assert [g.dtype for g in grads] == [torch.float32] * 3 and all(bool(g.isfinite().all()) for g in grads)
    with torch.autocast('cuda', dtype=torch.float16):
        assert asdl_amd.linear_8bit(x, w, b).dtype == torch.float16


@pytest.mark.parametrize('autocast', [False, True])
@pytest.mark.parametrize('tied', [False, True])
def test_a_step_of_a_decoder(tied, autocast):
    """Loss and all gradients against torch's operators with the same kept inputs.  float32: sums of up to 250 terms in another order
    through two blocks, 1e-4 in the 2-norm with room.  bfloat16: every intermediate is rounded to 2^-8 on both sides, and a share that
    the softmax or a norm magnifies is another kept value here and there (2^-4 of it, one in some 2^4 values): 5e-2."""
    plain, fused = decoders(tied)
    idx, t = ints(211, 8, 25, seed=2), ints(211, 8, 25, seed=3)
    t[0, :5] = -100
    losses = []
    for model in (plain, fused):
        with torch.autocast('cuda', dtype=BF16, enabled=autocast):
            loss = flat_loss(model(idx), t) if model is plain else asdl_amd.linear_cross_entropy(model.features(idx), model.head.weight, t)
        loss.backward()
        losses.append(float(loss.detach()))
    tol = 5e-2 if autocast else 1e-4
    assert abs(losses[0] - losses[1]) < (2 ** -8 if autocast else 1e-5) * losses[0]
    for (name, p), q in zip(plain.named_parameters(), fused.named_parameters()):
        assert off(q[1].grad, p.grad) < tol, name


@pytest.mark.parametrize('ema', [-1, 0.5])
@pytest.mark.parametrize('fisher_type', [FISHER_EMP, FISHER_MC])
def test_kfac_steps_of_a_decoder(fisher_type, ema):
    """Two steps.  Condition numbers as in the tests of layer norm and clipping: 1e-2 is allowed for float32 curvature with a damping of 1e-2."""
    plain, fused = decoders()
    idx, t = ints(211, 8, 25, seed=2), ints(211, 8, 25, seed=3)
    emp = fisher_type == FISHER_EMP
    if not emp:
        plain.head.__class__ = Linear           # (both heads are called)
    for model in (plain, fused):
        config = PreconditioningConfig(data_size=200, damping=1e-2, ema_decay=ema, ignore_modules=[nn.Embedding, model.head])
        maker = KfacGradientMaker(model, config, fisher_type=fisher_type, mc_temperature=1.0 if emp else 0.0)
        for _ in range(2):
            model.zero_grad()
            if model is fused and emp:
                maker.setup_loss_call(asdl_amd.linear_cross_entropy, maker.setup_model_call(model.features, idx), model.head.weight, t)
            else:       # (a sampled Fisher matrix draws from the logits)
                maker.setup_loss_call(F.cross_entropy, maker.setup_model_call(lambda i, m=model: m(i).flatten(0, 1), idx), t.flatten())
            maker.forward_and_backward()
    for (name, p), q in zip(plain.named_parameters(), fused.parameters()):
        if p.grad is not None:
            assert off(q.grad, p.grad) < 1e-2, name


def test_shampoo_step_of_a_decoder():
    """Its statistics of the new gradients; the same allowance."""
    plain, fused = decoders()
    idx, t = ints(211, 8, 25, seed=2), ints(211, 8, 25, seed=3)
    for model in (plain, fused):
        for p in (model.wte.weight, model.wpe.weight, model.head.weight):
            p.requires_grad_(False)
        maker = ShampooGradientMaker(model, PreconditioningConfig(damping=1e-2))
        if model is fused:
            maker.setup_loss_call(asdl_amd.linear_cross_entropy, maker.setup_model_call(model.features, idx), model.head.weight, t)
        else:
            maker.setup_loss_call(flat_loss, maker.setup_model_call(model, idx), t)
        maker.forward_and_backward()
    for (name, p), q in zip(plain.named_parameters(), fused.parameters()):
        if p.grad is not None:
            assert off(q.grad, p.grad) < 1e-2, name


def test_a_checkpointed_decoder():
    """The forward pass run again gives the same kept values: the same bits."""
    from torch.utils.checkpoint import checkpoint
    _, fused = decoders()
    idx, t = ints(211, 8, 25, seed=2), ints(211, 8, 25, seed=3)
    grads = []
    for again in (False, True):
        fused.zero_grad()
        h = checkpoint(fused.features, idx, use_reentrant=False) if again else fused.features(idx)
        asdl_amd.linear_cross_entropy(h, fused.head.weight, t).backward()
        grads.append([p.grad.clone() for p in fused.parameters()])
    assert all(off(a, b) < 1e-5 for a, b in zip(*grads))
    # (attention's own gradient may add in another order; what lies behind it is the same)
    assert torch.equal(grads[0][-1], grads[1][-1])


def test_what_a_step_keeps():
    """The loss takes a tenth of the logits' memory forward; a layer keeps a byte a value."""
    h, w, t = rand(8192, 64, seed=1, dtype=BF16).requires_grad_(), rand(50257, 64, seed=2, dtype=BF16).requires_grad_(), ints(50257, 8192, seed=3)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    loss = asdl_amd.linear_cross_entropy(h, w, t)
    assert torch.cuda.max_memory_allocated() - before < 0.1 * 8192 * 50257 * 2
    before = torch.cuda.memory_allocated()
    loss.backward()
    assert torch.cuda.max_memory_allocated() - before < 8192 * 50257 * 2 + 300e6
    model = nn.Sequential(*(m for _ in range(8) for m in (nn.Linear(1024, 1024), nn.GELU()))).cuda().bfloat16()
    x = rand(4096, 1024, seed=4, dtype=BF16).requires_grad_()
    sizes = []
    for kept_8bit in (False, True):
        if kept_8bit:
            asdl_amd.keep_activations_8bit(model)
        before = torch.cuda.memory_allocated()
        y = model(x)
        sizes.append(torch.cuda.memory_allocated() - before)
        del y
    # 16 inputs (the first of them x itself) of a byte a value and one for 128 of them, and the result
    values = 4096 * 1024
    assert sizes[0] >= 16 * values * 2 and sizes[1] <= 16 * (values + values // 128) + values * 2 + 16 * 4096


def test_a_captured_step():
    """Captured on inputs that are no leaves of an eager graph; replayed several times with new values, against the eager pass."""
    table, w, b = rand(300, 96, seed=1), rand(96, 96, seed=2, scale=0.1), rand(96, seed=3)
    idx, t = ints(300, 500, seed=4), ints(300, 500, seed=5)

    def passes(table, w, b):
        leaves = [x.detach().requires_grad_() for x in (table, w, b)]
        h = asdl_amd.gelu_8bit(asdl_amd.linear_8bit(asdl_amd.embedding(idx, leaves[0], None, 2.0), leaves[1], leaves[2]))
        loss = asdl_amd.linear_cross_entropy(h, leaves[0], t)
        return [loss.detach(), *torch.autograd.grad(loss, leaves)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        passes(table, w, b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = passes(table, w, b)
    for turn in range(4):
        table.mul_(0.9).add_(0.01)
        w.mul_(1.1)
        idx.copy_(idx.roll(3) // 2)
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        assert all(off(o, e) < 1e-6 for o, e in zip(got, passes(table, w, b))), turn


def test_a_plain_maker_with_the_loss():
    plain, fused = decoders()
    idx, t = ints(211, 4, 25, seed=2), ints(211, 4, 25, seed=3)
    maker = GradientMaker(fused)
    maker.setup_loss_call(asdl_amd.linear_cross_entropy, maker.setup_model_call(fused.features, idx), fused.head.weight, t)
    _, loss = maker.forward_and_backward()
    assert abs(float(loss) - float(flat_loss(plain(idx), t))) < 1e-4
    assert all(p.grad is not None for p in fused.parameters())
