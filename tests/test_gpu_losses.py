"""GPU: losses over a vocabulary (token log-probabilities, the clipped policy loss, the
preference loss) and their gradients against a plain implementation in 64 bits.

Tolerances.  z - m of a logit is one rounding of a difference of at most ~40 here, so an
exponential is off by 40 * 2^-24 * (1 + log2 e) < 6e-6 of itself, a log-probability by
40 * 2^-24 * 3 < 8e-6; a row's gradient is its coefficient times (1[token] - p), where the
coefficient's terms (the ratio's and the KL's, which may cancel) are each off by what
exp(logp - old) is: 2e-5 of the sum of the terms' sizes, times the row's largest |1[token] - p|,
covers both.  bf16 outputs add one rounding, 2^-8 of the value at most."""
import pytest
import torch

import volta_amd
from volta_amd import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INF = float("inf")


def make(rows, vocab, dtype, seed=0, spread=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = (torch.randn((rows, vocab), generator=g, device=DEV) * spread).to(dtype)
    tokens = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    noise = torch.randn((3, rows), generator=g, device=DEV)
    logp = x.double().log_softmax(1).gather(1, tokens[:, None])[:, 0].float()
    return x, tokens, logp + 0.3 * noise[0], noise[1].contiguous(), logp + 0.2 * noise[2]


def ref_logp64(x, tokens, temperature=1.0):
    z = x.double() / temperature
    return z, z.log_softmax(1).gather(1, tokens[:, None])[:, 0]  # the maximum taken off first: 64 bits hold no 6 beside 1e38


def ref_policy(x, tokens, old, adv, ref, mask, lo, hi, kl, temperature=1.0, scale=1.0):
    keep = torch.ones(x.shape[0], dtype=torch.bool, device=x.device) if mask is None else mask.bool()
    safe = torch.where(keep[:, None], x.double(), torch.zeros((), dtype=torch.float64, device=x.device))
    z, logp = ref_logp64(safe, torch.where(keep, tokens, 0), temperature)
    count = max(1, int(keep.sum()))
    r, a = (logp - old.double()).exp(), adv.double()
    plain, clipped = r * a, r.clamp(1 - lo, 1 + hi) * a
    term, c = -torch.minimum(plain, clipped), torch.where(plain <= clipped, -plain, 0.0)
    size = c.abs()
    if kl:
        d = ref.double() - logp
        term, c = term + kl * (d.exp() - d - 1), c + kl * (1 - d.exp())
        size = size + kl * (1 + d.exp())
    term, c = torch.where(keep, term, 0.0), torch.where(keep, c, 0.0)
    onehot = torch.zeros_like(z).scatter_(1, torch.where(keep, tokens, 0)[:, None], 1.0)
    step = (onehot - z.softmax(1)) * (scale / temperature / count)
    grad, size = c[:, None] * step, torch.where(keep, size, 0.0)[:, None] * step.abs().amax(1, keepdim=True)
    return term.sum() / count, torch.where(keep, logp, 0.0), torch.where(keep[:, None], grad, 0.0), size


def check_grad(got, want, size, dtype):
    tol = 2e-5 * size + (2.0 ** -8 * want.abs() if dtype == torch.bfloat16 else 0)
    assert got.dtype == dtype
    off = (got.double() - want).abs() - tol
    assert float(off.max()) <= 1e-37, f"gradient off by {float(off.max()):.3g} over the tolerance"


def check_policy(x, tokens, old, adv, ref, mask, lo=0.2, hi=0.3, kl=0.1, temperature=1.0, scale=1.0, out=None):
    source = x.clone()
    loss, logp, grad = ops.gpu_policy_loss(x, tokens, old, adv, ref, mask, lo, hi, kl, temperature, scale, True, out)
    l64, p64, g64, size = ref_policy(source, tokens, old, adv, ref, mask, lo, hi, kl, temperature, scale)
    assert torch.allclose(logp.double(), p64, rtol=0, atol=8e-6)
    assert abs(float(loss) - float(l64)) <= 2e-5 * max(1.0, abs(float(l64)))
    check_grad(grad, g64, size, x.dtype)
    return loss, grad


# one unit and less, the register variants' edges, rows longer than a block's registers
@pytest.mark.parametrize("vocab", [1, 3, 8, 257, 1000, 2049, 4099, 16389, 40003, 70001, 140001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_policy_loss(vocab, dtype):
    rows = 7 if vocab < 70000 else 3
    x, tokens, old, adv, ref = make(rows, vocab, dtype)
    mask = torch.tensor([1, 0, 1, 1, 0, 1, 1][:rows], dtype=torch.uint8, device=DEV)
    check_policy(x, tokens, old, adv, ref, mask)
    check_policy(x, tokens, old, adv, ref, mask.bool(), temperature=0.7, scale=3.0)
    check_policy(x, tokens, old, adv, None, None, kl=0.0)


@pytest.mark.parametrize("rows", [1, 2, 300, 4096, 5001])
def test_policy_loss_rows(rows):
    x, tokens, old, adv, ref = make(rows, 65, torch.bfloat16, seed=rows)
    g = torch.Generator(device=DEV).manual_seed(1)
    check_policy(x, tokens, old, adv, ref, torch.rand((rows,), generator=g, device=DEV) < 0.6)


def test_policy_loss_nothing_left():
    x, tokens, old, adv, ref = make(5, 33, torch.float32)
    x[1], tokens[2] = float("nan"), -100  # masked rows are not looked at
    loss, logp, grad = ops.gpu_policy_loss(x, tokens, old, adv, ref, torch.zeros(5, dtype=torch.bool, device=DEV), 0.2, 0.2, 0.1)
    assert float(loss) == 0 and not logp.any() and not grad.any()
    loss, logp, grad = ops.gpu_policy_loss(x[:0], tokens[:0], old[:0], adv[:0], ref[:0], None, 0.2, 0.2, 0.1)
    assert float(loss) == 0 and logp.shape == (0,) and grad.shape == (0, 33)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_policy_loss_masked_places(dtype):
    """NaN, infinities and the type's lowest value where a mask puts them."""
    x, tokens, old, adv, ref = make(6, 515, dtype, seed=3)
    mask = torch.tensor([1, 0, 1, 0, 1, 1], dtype=torch.bool, device=DEV)
    x[1], x[3], tokens[3] = float("nan"), INF, 1 << 40
    tokens[[0, 2, 4, 5]] %= 400
    x[0, 400:], x[2, 400:] = -INF, torch.finfo(dtype).min
    x[4], x[5, 1:] = torch.finfo(dtype).min, -INF  # a row of lowest values is uniform; one entry left is certain
    tokens[5] = 0
    old[4], old[5], ref[4], ref[5] = -6.0, 0.0, -6.5, 0.0
    _, grad = check_policy(x, tokens, old, adv, ref, mask)
    assert not grad[0, 400:].any() and not grad[2, 400:].any() and not grad[1].any() and not grad[3].any()


def test_policy_loss_is_nan_where_the_formula_is():
    x, tokens, old, adv, ref = make(4, 100, torch.float32)
    x[0, 5], x[1, 7], x[2] = float("nan"), INF, -INF
    tokens[3] = 100  # outside the vocabulary
    _, logp, grad = ops.gpu_policy_loss(x, tokens, old, adv, ref)
    assert torch.isnan(logp).all() and torch.isnan(grad[:3]).any(1).all() and torch.isnan(grad[3]).all()


def test_policy_loss_clips():
    """Ratios far outside the clip range pass no gradient on the side that the minimum cuts off."""
    x, tokens, _, _, _ = make(4, 50, torch.float32)
    logp = ops.gpu_token_logprobs(x, tokens)
    old = logp + torch.tensor([-1.0, -1.0, 1.0, 1.0], device=DEV)  # ratios e, e, 1/e, 1/e
    adv = torch.tensor([1.0, -1.0, 1.0, -1.0], device=DEV)
    _, grad = check_policy(x, tokens, old, adv, None, None, kl=0.0)
    assert [bool(r.any()) for r in grad] == [False, True, True, False]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_policy_loss_strides_and_places(dtype):
    x, tokens, old, adv, ref = make(9, 2067, dtype)
    wide = torch.full((9, 2311), float("nan"), dtype=dtype, device=DEV)
    wide[:, 3:2070] = x
    loss, grad = check_policy(wide[:, 3:2070], tokens, old, adv, ref, None)  # a slice, off any alignment
    l2, g2 = check_policy(x, tokens, old, adv, ref, None)
    assert torch.equal(grad, g2) and torch.equal(loss, l2)
    out = torch.full((9, 2100), 5.0, dtype=dtype, device=DEV)
    _, g3 = check_policy(x, tokens, old, adv, ref, None, out=out[:, 1:2068])
    assert torch.equal(g3, g2) and bool((out[:, 0] == 5).all()) and bool((out[:, 2068:] == 5).all())
    _, g4 = check_policy(x, tokens, old, adv, ref, None, out=x)  # in place
    assert g4.data_ptr() == x.data_ptr() and torch.equal(g4, g2)


@pytest.mark.parametrize("vocab", [1001, 70003])
def test_gradients_against_differences(vocab):
    """The loss moves along a direction as the gradient says: h = 1e-2 leaves h^2 / 6 of a third
    derivative of order 1, 2e-5, and 2e-7 / h of the losses' rounding."""
    x, tokens, old, adv, ref = make(6, vocab, torch.float32, seed=5, spread=1.0)
    old = ops.gpu_token_logprobs(x, tokens) + 0.05  # off the kinks of the clip range
    g = torch.Generator(device=DEV).manual_seed(9)
    v = torch.randn(x.shape, generator=g, device=DEV)
    offsets = torch.tensor([0, 2, 2, 3, 6], device=DEV)
    refs = torch.tensor([-20.0, 0.0, -5.0, -28.0], device=DEV)
    calls = (lambda y: ops.gpu_policy_loss(y, tokens, old, adv, ref, None, 0.5, 0.5, 0.2),
             lambda y: ops.gpu_preference_loss(y, tokens, offsets, refs, None, 0.3, 0.1))
    h = 1e-2
    for call in calls:
        slope = float((call(x)[2].double() * v.double()).sum())
        diff = (float(call(x + h * v)[0]) - float(call(x - h * v)[0])) / (2 * h)
        assert abs(slope - diff) <= 2e-4 + 2e-3 * abs(slope)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 777, 16385, 50021])
def test_token_logprobs(vocab, dtype):
    x, tokens, *_ = make(5, vocab, dtype)
    assert torch.allclose(ops.gpu_token_logprobs(x, tokens).double(), ref_logp64(x, tokens)[1], rtol=0, atol=8e-6)
    assert torch.allclose(ops.gpu_token_logprobs(x, tokens, 1.7).double(), ref_logp64(x, tokens, 1.7)[1], rtol=0, atol=8e-6)
    assert ops.gpu_token_logprobs(x[:0], tokens[:0]).shape == (0,)


def ref_preference(x, tokens, offsets, refs, mask, beta, smooth):
    z, logp = ref_logp64(x, tokens)
    keep = torch.ones_like(logp) if mask is None else mask.double()
    n = refs.numel() // 2
    o = offsets.tolist()
    total = torch.stack([(logp * keep)[o[s]:o[s + 1]].sum() for s in range(2 * n)])
    gain = total - refs.double()
    d = beta * (gain[:n] - gain[n:])
    ls = torch.nn.functional.logsigmoid
    loss = (-(1 - smooth) * ls(d) - smooth * ls(-d)).mean()
    c = beta / n * (torch.sigmoid(d) - (1 - smooth))
    rows = torch.zeros_like(logp)
    for s in range(2 * n):
        rows[o[s]:o[s + 1]] = c[s] if s < n else -c[s - n]
    onehot = torch.zeros_like(z).scatter_(1, tokens[:, None], 1.0)
    return loss, total, (rows * keep)[:, None] * (onehot - z.softmax(1))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab,lens", [
    (5, [1, 1]), (1000, [3, 0, 5, 1]), (2051, [0, 0, 0, 0]), (333, [70, 2, 129, 64, 1, 30]), (70001, [2, 1, 3, 2])])
def test_preference_loss(vocab, lens, dtype):
    offsets = torch.tensor([0] + lens, device=DEV).cumsum(0)
    rows = sum(lens) + 2  # two rows of no sequence
    x, tokens, *_ = make(rows, vocab, dtype, seed=vocab)
    g = torch.Generator(device=DEV).manual_seed(2)
    mask = torch.rand((rows,), generator=g, device=DEV) < 0.8
    for m in (None, mask):
        _, total, _ = ref_preference(x, tokens, offsets, torch.zeros(len(lens), device=DEV), m, 1.0, 0.0)
        refs = (total + torch.randn(len(lens), generator=g, device=DEV)).float()
        loss, seq, grad = ops.gpu_preference_loss(x, tokens, offsets, refs, m, 0.3, 0.1)
        l64, s64, g64 = ref_preference(x, tokens, offsets, refs, m, 0.3, 0.1)
        # a sum of up to 129 log-probabilities, each off by 8e-6 at most
        assert torch.allclose(seq.double(), s64, rtol=1e-6, atol=2e-4)
        assert abs(float(loss) - float(l64)) <= 1e-4
        tol = 1e-4 * g64.abs().amax(1, keepdim=True) + (2.0 ** -8 * g64.abs() if dtype == torch.bfloat16 else 0)
        assert float(((grad.double() - g64).abs() - tol).max()) <= 1e-37
        again = ops.gpu_preference_loss(x, tokens, offsets, refs, m, 0.3, 0.1, grad=False)
        assert again[2] is None and torch.equal(again[0], loss) and torch.equal(again[1], seq)
    y = x.clone()
    _, _, g2 = ops.gpu_preference_loss(y, tokens, offsets, refs, mask, 0.3, 0.1, out=y)
    assert torch.equal(g2, grad)


def test_preference_loss_certain():
    """Margins of hundreds of nats: no overflow, the gradient of a lost pair is beta."""
    x, tokens, *_ = make(2, 10, torch.float32)
    offsets = torch.tensor([0, 1, 2], device=DEV)
    loss, _, grad = ops.gpu_preference_loss(x, tokens, offsets, torch.tensor([5000.0, 0.0], device=DEV), None, 1.0)
    assert 4900 < float(loss) < 5100 and torch.isfinite(grad).all() and grad.abs().max() > 0.1
    loss, _, grad = ops.gpu_preference_loss(x, tokens, offsets, torch.tensor([-5000.0, 0.0], device=DEV), None, 1.0)
    assert float(loss) == 0 and not grad.any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_sequences_do_not_drift(dtype):
    """4000 rows against 40, the reference's sums as large as theirs, so that the loss shows the sums' difference:
    its slope in it is 1/2 there.  A row may be off the same way as every other by a quarter of fp32's last place
    (of its sum of exponentials, 2.5e-8 in all, of any sign) and by 4e-7 at random."""
    rows, few = 4000, 40
    x, tokens, _, _, _ = make(rows + few, 20000, dtype, seed=5, spread=1.0)
    offsets = torch.tensor([0, rows, rows + few], device=DEV)
    _, logp = ref_logp64(x, tokens)
    refs = torch.stack((logp[:rows].sum(), logp[rows:].sum())).float()
    loss, _, _ = ops.gpu_preference_loss(x, tokens, offsets, refs, beta=1.0)
    z = (logp[:rows].sum() - refs[0].double()) - (logp[rows:].sum() - refs[1].double())
    want = float(torch.nn.functional.softplus(-z))
    assert abs(float(loss) - want) <= 0.5 * (2.5e-8 * rows + 4e-7 * rows ** 0.5) + 2.0 ** -24


def test_logits_past_32_bits():
    """Rows whose offsets pass 2^31 elements."""
    rows, vocab = 33001, 65100
    x = torch.zeros((rows, vocab), dtype=torch.bfloat16, device=DEV)
    x[-3:] = make(3, vocab, torch.bfloat16)[0]
    tokens = torch.full((rows,), 7, device=DEV)
    logp = ops.gpu_token_logprobs(x, tokens)
    assert torch.allclose(logp[-3:].double(), ref_logp64(x[-3:], tokens[-3:])[1], rtol=0, atol=8e-6)
    mask = torch.zeros(rows, dtype=torch.bool, device=DEV)
    mask[-3:] = True
    adv, last = torch.ones(rows, device=DEV), x[-3:].clone()
    _, _, grad = ops.gpu_policy_loss(x, tokens, logp, adv, None, mask, out=x)
    check_grad(grad[-3:], *ref_policy(last, tokens[-3:], logp[-3:], adv[-3:], None, None, 0.2, 0.2, 0.0)[2:], x.dtype)
    assert not grad[:1000].any()


def test_another_stream():
    x, tokens, old, adv, ref = make(64, 3001, torch.bfloat16)
    want = ops.gpu_policy_loss(x, tokens, old, adv, ref)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = ops.gpu_policy_loss(x, tokens, old, adv, ref)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_graph_replays():
    x, tokens, old, adv, ref = make(40, 1003, torch.bfloat16)
    offsets, refs = torch.tensor([0, 9, 20, 31, 40], device=DEV), torch.zeros(4, device=DEV)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        ops.gpu_policy_loss(x, tokens, old, adv, ref)  # the stream's workspace
        ops.gpu_preference_loss(x, tokens, offsets, refs)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        a = ops.gpu_policy_loss(x, tokens, old, adv, ref)
        b = ops.gpu_preference_loss(x, tokens, offsets, refs)
    for seed in range(3):
        x.copy_(make(40, 1003, torch.bfloat16, seed=seed)[0])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = ops.gpu_policy_loss(x, tokens, old, adv, ref) + ops.gpu_preference_loss(x, tokens, offsets, refs)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(a + b, want))


def test_refusals():
    x, tokens, old, adv, ref = make(4, 30, torch.float32)
    offsets, refs = torch.tensor([0, 2, 4], device=DEV), torch.zeros(2, device=DEV)
    bad = lambda call, *kinds: pytest.raises(kinds or (volta_amd.VoltaHipError, ValueError, TypeError), call)  # noqa: E731
    bad(lambda: ops.gpu_policy_loss(x[0], tokens, old, adv))
    bad(lambda: ops.gpu_policy_loss(x.t(), tokens, old, adv), ValueError)
    bad(lambda: ops.gpu_policy_loss(x.half(), tokens, old, adv), TypeError)
    bad(lambda: ops.gpu_policy_loss(x, tokens.int(), old, adv), TypeError)
    bad(lambda: ops.gpu_policy_loss(x, tokens[:3], old, adv), volta_amd.VoltaHipError)
    bad(lambda: ops.gpu_policy_loss(x, tokens, old.double(), adv), TypeError)
    bad(lambda: ops.gpu_policy_loss(x, tokens, old, adv, None, None, 0.2, 0.2, 0.1), volta_amd.VoltaHipError)  # KL without ref
    bad(lambda: ops.gpu_policy_loss(x, tokens, old, adv, temperature=0.0), volta_amd.VoltaHipError)
    bad(lambda: ops.gpu_policy_loss(x, tokens, old, adv, clip_low=-0.1), volta_amd.VoltaHipError)
    bad(lambda: ops.gpu_policy_loss(x, tokens, old, adv, mask=old), TypeError)
    bad(lambda: ops.gpu_policy_loss(x, tokens, old, adv, out=x[:2]), volta_amd.VoltaHipError)
    wide = torch.zeros((4, 40), device=DEV)
    bad(lambda: ops.gpu_policy_loss(wide[:, :30], tokens, old, adv, out=wide[:, 5:35]), volta_amd.VoltaHipError)  # overlap
    bad(lambda: ops.gpu_preference_loss(x, tokens, offsets[:2], refs), volta_amd.VoltaHipError)
    bad(lambda: ops.gpu_preference_loss(x, tokens, offsets, refs[:1]), volta_amd.VoltaHipError)
    bad(lambda: ops.gpu_preference_loss(x, tokens, offsets.int(), refs), TypeError)
    bad(lambda: ops.gpu_preference_loss(x, tokens, offsets, refs, label_smoothing=1.5), volta_amd.VoltaHipError)
    assert ops.gpu_policy_loss(x.cpu(), tokens.cpu(), old.cpu(), adv.cpu()) is None
    lib = _lib.lib()
    s = ops.stream_ptr(x.device)
    assert lib.vh_token_logprobs(0, None, 30, tokens.data_ptr(), old.data_ptr(), 4, 30, 1.0, s) == _lib.VH_ERR_BAD_ARG
    assert lib.vh_token_logprobs(7, x.data_ptr(), 30, tokens.data_ptr(), old.data_ptr(), 4, 30, 1.0, s) == _lib.VH_ERR_BAD_ARG
    assert lib.vh_token_logprobs(0, x.data_ptr(), 29, tokens.data_ptr(), old.data_ptr(), 4, 30, 1.0, s) == _lib.VH_ERR_BAD_SHAPE
    assert lib.vh_token_logprobs(0, x.data_ptr() + 1, 30, tokens.data_ptr(), old.data_ptr(), 3, 30, 1.0, s) == _lib.VH_ERR_BAD_ARG


@pytest.mark.parametrize("rows,vocab", [((1 << 26) - 15, 512), ((1 << 24) - 15, 1000), ((1 << 22) - 15, 40000)])
def test_refuses_more_rows_than_a_launch_has_threads(rows, vocab):
    """By the sizes alone, before anything is read."""
    x, tokens, old, adv, ref = make(4, 30, torch.float32)
    lib, s = _lib.lib(), ops.stream_ptr(x.device)
    a, t, f = x.data_ptr(), tokens.data_ptr(), old.data_ptr()
    assert lib.vh_token_logprobs(0, a, vocab, t, f, rows, vocab, 1.0, s) == _lib.VH_ERR_UNSUPPORTED
    assert lib.vh_policy_loss(0, a, vocab, t, f, f, None, None, f, f, None, vocab, rows, vocab, 0.2, 0.2, 0.0, 1.0, 1.0, s) == _lib.VH_ERR_UNSUPPORTED
    assert lib.vh_preference_loss(0, a, vocab, t, t, f, None, f, f, None, vocab, rows, vocab, 1, 0.1, 0.0, 1.0, 1.0, s) == _lib.VH_ERR_UNSUPPORTED
    assert lib.vh_preference_loss(0, a, 30, t, t, f, None, f, f, None, 30, 4, 30, (1 << 25) - 15, 0.1, 0.0, 1.0, 1.0, s) == _lib.VH_ERR_UNSUPPORTED


@pytest.mark.parametrize("vocab", [5, 15, 16, 17, 600, 5003])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_preference_loss_wherever_its_rows_lie(vocab, dtype):
    """Rows of every alignment, in a wider table, their gradient elsewhere and in place: the same bits, nothing beside them."""
    x, tokens, *_ = make(9, vocab, dtype)
    tokens[3] = 0  # in the elements before a boundary
    offsets = torch.tensor([0, 4, 5, 8, 8], device=DEV)  # row 8 in no sequence
    refs = torch.tensor([-3.0, -2.0, -4.0, 0.0], device=DEV)
    mask = torch.tensor([1, 0, 1, 1, 1, 1, 1, 1, 1], dtype=torch.bool, device=DEV)
    want = ops.gpu_preference_loss(x, tokens, offsets, refs, mask)
    for at in range(9):
        wide = torch.full((9, vocab + 17), 7.0, dtype=dtype, device=DEV)
        wide[:, at:at + vocab] = x
        out = torch.full((9, vocab + 11), 7.0, dtype=dtype, device=DEV)
        other = (at * 5) % 11
        got = ops.gpu_preference_loss(wide[:, at:at + vocab], tokens, offsets, refs, mask, out=out[:, other:other + vocab])
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        assert (out[:, :other] == 7).all() and (out[:, other + vocab:] == 7).all()
        got = ops.gpu_preference_loss(wide[:, at:at + vocab], tokens, offsets, refs, mask, out=wide[:, at:at + vocab])
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        assert (wide[:, :at] == 7).all() and (wide[:, at + vocab:] == 7).all()


@pytest.mark.parametrize("rows,vocab,dtype", [(1025, 8193, torch.float32), (1300, 16383, torch.float32), (1100, 16385, torch.bfloat16),
                                              (1025, 32003, torch.bfloat16)])
def test_policy_loss_many_rows(rows, vocab, dtype):
    x, tokens, old, adv, ref = make(rows, vocab, dtype)
    mask = torch.arange(rows, device=DEV) % 5 != 3
    check_policy(x, tokens, old, adv, ref, mask)


@pytest.mark.parametrize("vocab,dtype", [(9001, torch.float32), (16384, torch.float32), (32003, torch.bfloat16)])
def test_policy_loss_rows_are_the_same_among_many(vocab, dtype):
    x, tokens, old, adv, ref = make(1030, vocab, dtype)
    logp = ops.gpu_policy_loss(x, tokens, old, adv)[1]
    assert torch.equal(logp[:1024], ops.gpu_policy_loss(x[:1024], tokens[:1024], old[:1024], adv[:1024])[1])
    a, b = (ops.gpu_policy_loss(x[:n], tokens[:n], old[:n], adv[:n], mask=torch.arange(n, device=DEV) < 9)[2] for n in (1030, 1024))
    assert torch.equal(a[:1024], b) and not b[9:].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,temperature", [(9, 203, 1.0), (300, 2067, 0.9), (40, 5003, 1.0), (300, 32003, 0.9), (20, 65533, 1.3), (3, 140001, 0.9)])
def test_policy_gradient_is_one_function_of_the_logit(rows, vocab, temperature, dtype):
    """Entries of a row with the same logit have the same gradient bit for bit, whichever thread writes them (the last
    unit of an odd row is written by two), and every call gives the same."""
    x, tokens, old, adv, ref = make(rows, vocab, dtype, seed=21)
    same = torch.arange(vocab, device=DEV) % 5 == 0
    x[:, same] = x[:, :1]
    tokens = (tokens // 5 * 5 + 1) % (vocab // 5 * 5)  # none of them
    old = ops.gpu_token_logprobs(x, tokens, temperature) + 0.1
    call = lambda: ops.gpu_policy_loss(x, tokens, old, adv, old, None, 0.2, 0.2, 0.1, temperature)  # noqa: E731
    first = call()
    assert torch.equal(first[2][:, same], first[2][:, :1].expand(-1, int(same.sum())))
    for _ in range(10):
        assert all(torch.equal(a, b) for a, b in zip(call(), first))


@pytest.mark.parametrize("smooth", [0.0, 1.0, 0.3])
@pytest.mark.parametrize("margin", [-80.0, -45.0, -30.0, -3.0, 3.0, 30.0, 36.0, 45.0, 80.0])
def test_preference_gradient_of_a_decided_pair(margin, smooth):
    """The slope e sigmoid(z) - (1 - e) sigmoid(-z) to fp32's accuracy where sigmoid(z) is all but 0 or 1: a
    log-probability off by 8e-6 changes it by as much of itself, the row's own terms add 2e-5."""
    x, tokens, *_ = make(3, 70, torch.float32, seed=11)
    offsets = torch.tensor([0, 1, 3], device=DEV)
    _, logp = ref_logp64(x, tokens)
    refs = torch.stack((logp[0] - margin, logp[1:].sum())).float()
    _, _, grad = ops.gpu_preference_loss(x, tokens, offsets, refs, None, 1.0, smooth)
    z = (logp[0] - refs[0].double()) - (logp[1:].sum() - refs[1].double())
    c = smooth * torch.sigmoid(z) - (1 - smooth) * torch.sigmoid(-z)
    onehot = torch.zeros_like(x, dtype=torch.float64).scatter_(1, tokens[:, None], 1.0)
    want = torch.stack((c, -c, -c))[:, None] * (onehot - x.double().softmax(1))
    off = (grad.double() - want).abs().amax(1)
    assert bool((off <= 1e-4 * want.abs().amax(1)).all()), (off / want.abs().amax(1)).tolist()


def test_preference_loss_of_impossible_answers():
    """A sequence that holds a token of probability 0 has lost (a loss of 0 if it is the rejected one, of infinity if
    the preferred one); labels that name one side only do not look at the other's logarithm."""
    x, tokens, *_ = make(4, 40, torch.float32, seed=12)
    tokens[1], x[1, 3] = 3, -INF
    offsets = torch.tensor([0, 2, 4], device=DEV)  # sequence 0 has the row, sequence 1 not
    swap = torch.tensor([2, 3, 0, 1], device=DEV)
    refs = torch.tensor([-5.0, -6.0], device=DEV)
    for smooth, lost in ((0.0, True), (1.0, False)):
        loss, seq, _ = ops.gpu_preference_loss(x, tokens, offsets, refs, None, 0.5, smooth)
        assert float(seq[0]) == -INF and float(loss) == (INF if lost else 0.0)
        loss, seq, grad = ops.gpu_preference_loss(x[swap], tokens[swap], offsets, refs, None, 0.5, smooth)
        assert float(seq[1]) == -INF and float(loss) == (0.0 if lost else INF)
        assert torch.isfinite(grad).all() and (not lost or not grad.any())
    loss, _, _ = ops.gpu_preference_loss(x, tokens, offsets, refs, None, 0.5, 0.3)
    assert float(loss) == INF


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_policy_loss_of_far_ratios(dtype):
    """Ratios and KL terms whose exponential passes fp32: a row without an advantage has no gradient by its ratio, one
    past the clip none either, and nothing turns into NaN where entries have probability 0."""
    x, tokens, old, adv, ref = make(6, 300, dtype, seed=13)
    tokens %= 200
    x[:, 250:] = -INF
    logp = ops.gpu_token_logprobs(x, tokens)
    old = logp + torch.tensor([-100.0, -300.0, -0.1, -100.0, -95.0, 0.2], device=DEV)
    adv = torch.tensor([0.0, 0.0, 0.5, 2.0, -1.0, -0.3], device=DEV)
    _, grad = check_policy(x[:4], tokens[:4], old[:4], adv[:4], None, None, kl=0.0)
    assert not grad[0].any() and not grad[1].any() and grad[2].any() and not grad[3].any()
    _, _, grad = ops.gpu_policy_loss(x, tokens, old, adv)
    assert torch.isfinite(grad).all() and not grad[:, 250:].any() and grad[4].abs().max() > 1e37
    ref = logp + torch.tensor([0.1, 0.1, 0.1, 100.0, 0.1, 0.1], device=DEV)
    _, _, grad = ops.gpu_policy_loss(x, tokens, old, adv, ref, None, 0.2, 0.2, 0.05)
    assert torch.isfinite(grad).all() and not grad[:, 250:].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [7, 333, 2051])
def test_logits_and_gradient_beside_each_other(vocab, dtype):
    """Two column ranges of one table share no element; ranges that do are refused, around a row's end too."""
    rows = 5
    x, tokens, old, adv, ref = make(rows, vocab, dtype, seed=14)
    offsets, refs = torch.tensor([0, 2, 5], device=DEV), torch.tensor([-3.0, -4.0], device=DEV)
    want = ops.gpu_policy_loss(x, tokens, old, adv, ref), ops.gpu_preference_loss(x, tokens, offsets, refs)
    for first, second, width in ((0, vocab, 2 * vocab), (vocab + 3, 1, 2 * vocab + 5), (2, vocab + 9, 2 * vocab + 11)):
        table = torch.full((rows, width), 5.0, dtype=dtype, device=DEV)
        a, b = table[:, first:first + vocab], table[:, second:second + vocab]
        a.copy_(x)
        assert all(torch.equal(p, q) for p, q in zip(ops.gpu_policy_loss(a, tokens, old, adv, ref, out=b), want[0]))
        assert all(torch.equal(p, q) for p, q in zip(ops.gpu_preference_loss(a, tokens, offsets, refs, out=b), want[1]))
        assert torch.equal(a, x)
        table[:, first:first + vocab], table[:, second:second + vocab] = 5.0, 5.0
        assert bool((table == 5).all())
    flat = torch.zeros(rows * 3 * vocab, dtype=dtype, device=DEV)
    for stride, at in ((2 * vocab, vocab - 1), (2 * vocab, vocab + 1), (2 * vocab - 1, vocab), (2 * vocab, 2 * vocab - 1)):
        a, b = (flat.as_strided((rows, vocab), (stride, 1), o) for o in (0, at))
        for p, q in ((a, b), (b, a)):
            with pytest.raises(volta_amd.VoltaHipError):
                ops.gpu_policy_loss(p, tokens, old, adv, out=q)


@pytest.mark.parametrize("vocab", [3, 1000, 16389, 70001, 140001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_policy_loss_alone(vocab, dtype):
    """Without a gradient: the same loss and log-probabilities, bit for bit."""
    x, tokens, old, adv, ref = make(5, vocab, dtype, seed=15)
    mask = torch.tensor([1, 0, 1, 1, 1], dtype=torch.bool, device=DEV)
    for m in (None, mask):
        want = ops.gpu_policy_loss(x, tokens, old, adv, ref, m, 0.2, 0.3, 0.1, 0.8, 2.0)
        loss, logp, grad = ops.gpu_policy_loss(x, tokens, old, adv, ref, m, 0.2, 0.3, 0.1, 0.8, 2.0, grad=False)
        assert grad is None and torch.equal(loss, want[0]) and torch.equal(logp, want[1])
        l64, p64 = ref_policy(x, tokens, old, adv, ref, m, 0.2, 0.3, 0.1, 0.8)[:2]
        assert torch.allclose(logp.double(), p64, rtol=0, atol=8e-6) and abs(float(loss) - float(l64)) <= 2e-5 * max(1.0, abs(float(l64)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [50, 3001, 70001])
def test_preference_loss_temperature_and_scale(vocab, dtype):
    """logits / temperature as logits; the gradient by 1 / temperature and by the loss's own."""
    lens, smooth, beta, temperature, scale = [3, 5, 4, 1], 0.1, 0.3, 1.6, -2.5
    offsets = torch.tensor([0] + lens, device=DEV).cumsum(0)
    x, tokens, *_ = make(sum(lens), vocab, dtype, seed=16)
    cold = x.double() / temperature
    _, total, _ = ref_preference(cold, tokens, offsets, torch.zeros(4, device=DEV), None, 1.0, 0.0)
    refs = (total + torch.tensor([1.0, -2.0, 0.5, 0.0], device=DEV)).float()
    loss, seq, grad = ops.gpu_preference_loss(x, tokens, offsets, refs, None, beta, smooth, temperature, scale)
    l64, s64, g64 = ref_preference(cold, tokens, offsets, refs, None, beta, smooth)
    g64 = g64 * (scale / temperature)
    assert torch.allclose(seq.double(), s64, rtol=1e-6, atol=2e-4) and abs(float(loss) - float(l64)) <= 1e-4
    tol = 1e-4 * g64.abs().amax(1, keepdim=True) + (2.0 ** -8 * g64.abs() if dtype == torch.bfloat16 else 0)
    assert float(((grad.double() - g64).abs() - tol).max()) <= 1e-37


def test_preference_loss_is_nan_where_the_formula_is():
    """A NaN, an infinity or a token outside the vocabulary makes its pair's gradients NaN, and the mean; the other
    pair's, and what a mask leaves out, stay what they are.  Banned entries (-inf) have probability and gradient 0."""
    clean, tokens, *_ = make(8, 90, torch.float32, seed=17)
    tokens %= 60
    clean[:, 80:] = -INF
    offsets, refs = torch.tensor([0, 2, 4, 6, 8], device=DEV), torch.tensor([-9.0, -8.0, -9.0, -7.0], device=DEV)
    want = ops.gpu_preference_loss(clean, tokens, offsets, refs)
    l64, _, g64 = ref_preference(clean, tokens, offsets, refs, None, 0.1, 0.0)
    assert abs(float(want[0]) - float(l64)) <= 1e-4 and not want[2][:, 80:].any()
    assert float((want[2].double() - g64).abs().max()) <= 1e-4 * float(g64.abs().max())
    for value, token in ((float("nan"), None), (INF, None), (None, 90), (None, -1), (None, 1 << 40)):
        x, tok = clean.clone(), tokens.clone()
        if token is None:
            x[1, 5] = value
        else:
            tok[1] = token
        loss, seq, grad = ops.gpu_preference_loss(x, tok, offsets, refs)  # row 1: sequence 0, of pair 0 with sequence 2
        assert torch.isnan(loss).all() and torch.isnan(seq).tolist() == [True, False, False, False]
        assert all(bool(torch.isnan(grad[r]).any()) for r in (0, 1, 4, 5))
        assert torch.equal(grad[[2, 3, 6, 7]], want[2][[2, 3, 6, 7]])
        mask = torch.ones(8, dtype=torch.bool, device=DEV)
        mask[1] = False
        got = ops.gpu_preference_loss(x, tok, offsets, refs, mask)
        assert all(torch.equal(a, b) for a, b in zip(got, ops.gpu_preference_loss(clean, tokens, offsets, refs, mask)))
        assert not got[2][1].any()
