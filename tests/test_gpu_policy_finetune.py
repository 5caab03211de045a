"""GPU: the training operators together, as examples/policy_finetune.py uses them; and the
gradient of its whole network against 64-bit automatic differentiation."""
import importlib.util
import os

import pytest
import torch

import volta_amd
from volta_amd import nn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
_PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "policy_finetune.py")
_spec = importlib.util.spec_from_file_location("policy_finetune", _PATH)
example = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(example)


def test_learns():
    """Every step moves the loss down or the reward up in the large: halves the one, doubles the other."""
    losses, rewards = example.train(steps=20, rows=128, vocab=200, width=128, log=lambda line: None)
    assert losses[-1] < 0.5 * losses[0] and rewards[-1] > 2 * rewards[0]


def test_network_gradients():
    """fp32 through eleven layers: each adds a few 2^-24 of its sums, 1e-4 of the largest entry in all."""
    width, vocab, rows = 96, 333, 50
    model = example.Model(width, vocab, device=DEV, generator=torch.Generator().manual_seed(3))
    g = torch.Generator(device=DEV).manual_seed(4)
    x = torch.randn((rows, width), generator=g, device=DEV)
    tokens = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    adv = torch.randn((rows,), generator=g, device=DEV)
    logits, saved = model.forward(x)
    old = volta_amd.ops.gpu_token_logprobs(logits, tokens) + 0.05
    _, _, grad = nn.PolicyLoss(0.5, 0.5, 0.3)(logits, tokens, old, adv, old)
    matrices, vectors = model.backward(grad, saved)

    leaf = lambda t: t.double().cpu().requires_grad_()  # noqa: E731
    mats, vecs = [leaf(t) for t in model.matrices()], [leaf(t) for t in model.vectors()]
    y = n = x.double().cpu()
    rms = lambda v: v / (v.square().mean(1, keepdim=True) + 1e-6).sqrt()  # noqa: E731
    for i in range(len(model.blocks)):
        b1, b2, gate, post, nxt = vecs[5 * i:5 * i + 5]
        b = torch.relu(n @ mats[2 * i] + b1) @ mats[2 * i + 1] + b2
        y = y + 0.5 * gate * rms(b) * post
        n = rms(y) * nxt
    logp = (n @ mats[-1] + vecs[-1]).log_softmax(1).gather(1, tokens.cpu()[:, None])[:, 0]
    o, a = old.double().cpu(), adv.double().cpu()
    r, d = (logp - o).exp(), o - logp
    (0.3 * (d.exp() - d - 1) - torch.minimum(r * a, r.clamp(0.5, 1.5) * a)).mean().backward()
    for got, want in zip(matrices + vectors, mats + vecs):
        w = want.grad.reshape(got.shape)
        assert float((got.double().cpu() - w).abs().max()) <= 1e-4 * float(w.abs().max())


def test_layers_refuse_host_tensors_and_vectors():
    x = torch.ones((2, 8))
    for call in (lambda: nn.ResidualNorm(8, device="cpu")(x, x), lambda: nn.PolicyLoss()(x, x[:, 0].long(), x[:, 0], x[:, 0]),
                 lambda: nn.PreferenceLoss()(x, x[:, 0].long(), torch.tensor([0, 1, 2]), x[0, :2]),
                 lambda: nn.Muon([x]).step([x]), lambda: nn.Muon([x[0]])):
        with pytest.raises(volta_amd.VoltaHipError):
            call()
    with pytest.raises(ValueError):
        nn.Muon([x]).step([])


def test_muon_takes_kernels():
    """A convolution's weight as the matrix [out, in * k * k]."""
    g = torch.Generator(device=DEV).manual_seed(5)
    w, dw = (torch.randn((24, 6, 3, 3), generator=g, device=DEV) for _ in range(2))
    flat = w.reshape(24, -1).clone()
    opt = nn.Muon([w], lr=0.1, nesterov=False)
    opt.step([dw])
    m = torch.zeros_like(flat)
    volta_amd.ops.gpu_muon_step(flat, dw.reshape(24, -1), m, 0.1, nesterov=False)
    assert torch.equal(w.reshape(24, -1), flat) and torch.equal(opt.momentum[0].reshape(24, -1), m)


def test_muon_refuses_before_it_updates():
    """A gradient of another shape (a transposed one has as many elements), type or layout, wherever in the list:
    no parameter and no momentum has changed."""
    g = torch.Generator(device=DEV).manual_seed(6)
    n = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    params = [n(48, 32), n(24, 6, 3, 3), n(784, 512)]
    good = [n(*p.shape) for p in params]
    E = volta_amd.VoltaHipError
    bad = ((0, n(32, 48), E), (1, n(6, 24, 3, 3), E), (1, n(54, 24), E), (2, n(512, 784), E), (2, n(784 * 512), E),
           (2, n(784, 512).bfloat16(), TypeError), (2, n(512, 784).t(), ValueError),
           (1, n(24, 6, 3, 3).to(memory_format=torch.channels_last), ValueError), (2, n(784, 512).cpu(), E), (2, None, TypeError))
    for at, wrong, kind in bad:
        opt = nn.Muon(params, lr=0.1)
        before = [t.clone() for t in params + opt.momentum]
        grads = list(good)
        grads[at] = wrong
        with pytest.raises(kind):
            opt.step(grads)
        assert all(torch.equal(a, b) for a, b in zip(params + opt.momentum, before))
    good[1] = good[1].view(24, 54)  # a kernel's matrix
    opt.step(good)
    assert not any(torch.equal(a, b) for a, b in zip(params + opt.momentum, before))


def _steps_of(u):
    x = u.mT.contiguous() if u.shape[-2] > u.shape[-1] else u
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + 1e-7)
    for _ in range(5):
        gram = x @ x.mT.contiguous()
        x = 3.4445 * x + (-4.7750 * gram + 2.0315 * (gram @ gram)) @ x
    return x.mT.contiguous() if u.shape[-2] > u.shape[-1] else x


@pytest.mark.parametrize("inputs,outputs", [(96, 400), (400, 96), (784, 512), (64, 64), (10, 300)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_muon_steps_go_by_inputs_and_outputs(inputs, outputs, dtype):
    """A layer's update is scaled by sqrt(max(1, outputs / inputs)) however its weight lies: a Linear's [in, out], a
    Conv2d's [out, in, k, k], a ConvTranspose2d's [in, out, k, k].  Tolerances: the parameters' own rounding, and
    the update's error, 1e-4 of it in fp32 and 4e-3 in bf16."""
    lr, wd, beta = 0.05, 0.1, 0.9
    gen = torch.Generator().manual_seed(7)
    c_in, c_out = max(1, inputs // 8), max(1, outputs // 8)
    layers = ((nn.Linear(inputs, outputs, device=DEV, dtype=dtype, generator=gen), None, inputs, outputs),
              (nn.Conv2d(c_in, c_out, 3, device=DEV, dtype=dtype, generator=gen), None, c_in * 9, c_out),
              (nn.ConvTranspose2d(c_in, c_out, 3, device=DEV, dtype=dtype, generator=gen), True, c_in, c_out * 9))
    for layer, in_first, ins, outs in layers:
        w = layer.weight
        grad = torch.randn(w.shape, generator=torch.Generator(device=DEV).manual_seed(8), device=DEV).to(dtype)
        opt = nn.Muon([w], lr=lr, beta=beta, weight_decay=wd, in_first=in_first)
        for _ in range(2):
            old, m64 = w.double(), beta * opt.momentum[0].double() + grad.double()
            rows = w.shape[0]
            u = (grad.double() + beta * m64).view(rows, -1)
            update = (lr * max(1.0, outs / ins) ** 0.5 * _steps_of(u)).view(w.shape)
            opt.step([grad])
            want = old * (1 - lr * wd) - update
            off = float(torch.linalg.vector_norm(w.double() - want))
            own, step = float(torch.linalg.vector_norm(want)), float(torch.linalg.vector_norm(update))
            assert off <= (2.0 ** -8 * own + 4e-3 * step if dtype == torch.bfloat16 else 2.0 ** -23 * own + 1e-4 * step), \
                (type(layer).__name__, off, own, step)


def test_muon_takes_an_orientation_for_each_parameter():
    g = torch.Generator(device=DEV).manual_seed(9)
    w = torch.randn((20, 80), generator=g, device=DEV)
    dw = torch.randn((20, 80), generator=g, device=DEV)
    apart = []
    for in_first in (True, False):
        p = w.clone()
        nn.Muon([p], lr=0.1, in_first=in_first).step([dw])
        apart.append(p)
    assert torch.allclose((w - apart[0]) / 2, w - apart[1], rtol=0, atol=1e-6)  # sqrt(80 / 20) = 2
    a, b = w.clone(), w.clone()
    nn.Muon([a, b], lr=0.1, in_first=[True, False]).step([dw, dw])
    assert torch.equal(a, apart[0]) and torch.equal(b, apart[1])
    with pytest.raises(ValueError):
        nn.Muon([a, b], in_first=[True])
