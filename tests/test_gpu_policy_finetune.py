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
