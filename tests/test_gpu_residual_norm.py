"""GPU: the norms around a block with its gate and residual scale, forward and backward,
against a plain implementation in 64 bits.

Tolerances: an output row's entries go through two sums of d terms (each off by some
2^-24 of its terms' absolute sum) and about ten roundings: 3e-6 of the largest, over the
row, of the sum of the entry's terms' sizes (they may cancel: one element's norm has
no gradient); a column sum over T rows: of that sum over the rows.  bf16 outputs add
one rounding, 2^-8 of the value at most."""
import pytest
import torch

import volta_amd
from volta_amd import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
REL = 3e-6


def make(rows, d, dtype, gate_rows, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    t = lambda *s, std=1.0, mean=0.0: (torch.randn(s, generator=g, device=DEV) * std + mean).to(dtype)  # noqa: E731
    return dict(x=t(rows, d, std=2.0), b=t(rows, d), gate=t(gate_rows, d, mean=0.5) if gate_rows else None,
                wp=t(d, std=0.3, mean=1.0), wn=t(d, std=0.3, mean=1.0), dy=t(rows, d), dn=t(rows, d))


def reference(t, scale, eps):
    """(outputs, sizes): each output in 64 bits and the size that its error is measured by."""
    v = {k: None if a is None else a.double() for k, a in t.items()}
    x, b, gate, wp, wn, dy, dn = (v[k] for k in ("x", "b", "gate", "wp", "wn", "dy", "dn"))
    rows, d = x.shape
    mean = lambda u: u.mean(1, keepdim=True)  # noqa: E731
    full = torch.ones_like(x) if gate is None else gate.repeat_interleave(rows // gate.shape[0], 0)
    rb = (mean(b.square()) + eps).rsqrt() if wp is not None else torch.ones((rows, 1), dtype=x.dtype, device=DEV)
    w1 = wp if wp is not None else torch.ones(d, dtype=x.dtype, device=DEV)
    bh = b * rb
    y = x + scale * full * bh * w1
    size_y = x.abs() + (scale * full * bh * w1).abs()
    out, size = dict(y=y), dict(y=size_y)
    total, size_t = (torch.zeros_like(x),) * 2 if dy is None else (dy, dy.abs())
    if wn is not None:
        ry = (mean(y.square()) + eps).rsqrt()
        yh, size_yh = y * ry, size_y * ry
        out["n"], size["n"] = yh * wn, size_yh * wn.abs()
        h = dn * wn
        total = total + ry * (h - yh * mean(h * yh))
        size_t = size_t + ry * (h.abs() + size_yh * mean(h.abs() * size_yh))
        out["dwn"], size["dwn"] = dn * yh, dn.abs() * size_yh
    out["dx"], size["dx"] = total, size_t
    size_t = size_t.amax(1, keepdim=True)
    k, size_k = scale * full * total * w1, abs(scale) * full.abs() * size_t * w1.abs()
    if wp is not None:
        out["db"], size["db"] = rb * (k - bh * mean(k * bh)), rb * (size_k + bh.abs() * mean(size_k * bh.abs()))
        out["dwp"], size["dwp"] = scale * full * total * bh, abs(scale) * full.abs() * size_t * bh.abs()
    else:
        out["db"], size["db"] = k, size_k
    if gate is not None:
        out["dgate"], size["dgate"] = scale * total * bh * w1, abs(scale) * size_t * (bh * w1).abs()
    for name in out:
        size[name] = size[name].amax(1, keepdim=True).expand_as(out[name])
        if name in ("dwn", "dwp", "dgate"):
            groups = gate.shape[0] if name == "dgate" else 1
            out[name], size[name] = (u.reshape(groups, rows // groups, d).sum(1) for u in (out[name], size[name]))
    return out, size


def check(t, scale=0.5, eps=1e-6, lead=None):
    dt = t["x"].dtype
    args = {k: (a.reshape(*lead, -1) if lead and a is not None and k in ("x", "b", "dy", "dn") else a) for k, a in t.items()}
    y, n, rstd = ops.gpu_residual_norm(args["x"], args["b"], t["gate"], t["wp"], t["wn"], scale, eps)
    got = dict(zip(("dx", "db", "dgate", "dwp", "dwn"), ops.gpu_residual_norm_backward(
        args["dy"], args["dn"] if t["wn"] is not None else None, args["x"], args["b"], rstd, t["gate"], t["wp"], t["wn"], scale)))
    got.update(y=y, n=n)
    want, size = reference(t, scale, eps)
    for name, a in got.items():
        if name not in want:
            assert a is None, name
            continue
        assert a.dtype == dt, name
        w = want[name].reshape(a.shape)
        tol = REL * size[name].reshape(a.shape) + (2.0 ** -8 * w.abs() if dt == torch.bfloat16 else 0)
        off = float(((a.double() - w).abs() - tol).max())
        assert off <= 1e-37, f"{name} off by {off:.3g} over its tolerance"
    return got


# every threads-per-row variant, its edges and odd widths
@pytest.mark.parametrize("d", [1, 7, 64, 1000, 1025, 1531, 4096, 4099, 8192, 9001, 16384])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_widths(d, dtype):
    check(make(6, d, dtype, 1))
    check(make(5, d, dtype, 5, seed=1))


# rows: one, fewer and more than the blocks; gates of one row, one for each run, one each
@pytest.mark.parametrize("rows,gate_rows", [(1, 1), (1, 0), (2, 1), (1000, 1), (4099, 1), (1536, 3), (1021 * 3, 3), (2600, 1300),
                                            (2049, 2049), (5000, 2500), (35, 7), (4096, 512), (1030, 515)])
@pytest.mark.parametrize("d", [72, 1100])
def test_rows_and_gates(rows, gate_rows, d):
    check(make(rows, d, torch.float32, gate_rows, seed=rows))
    check(make(rows, d, torch.bfloat16, gate_rows, seed=rows))


@pytest.mark.parametrize("d", [77, 300, 1531, 4096, 12001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_in_place(d, dtype):
    """The C entries with y = x and n = block, grad_x = grad_y and grad_block = grad_n, then grad_block = block."""
    rows = 530
    t = make(rows, d, dtype, 1)
    dt, st = ops.dtype_code(t["x"]), ops.stream_ptr(t["x"].device)
    gate, wp, wn = (t[k].data_ptr() for k in ("gate", "wp", "wn"))
    y, n, rstd = ops.gpu_residual_norm(t["x"], t["b"], t["gate"], t["wp"], t["wn"], 0.5, 1e-6)
    dx, db, dgate, dwp, dwn = ops.gpu_residual_norm_backward(t["dy"], t["dn"], t["x"], t["b"], rstd, t["gate"], t["wp"], t["wn"], 0.5)
    u = {k: t[k].clone() for k in ("x", "b", "dy", "dn")}
    r2, sums = torch.empty_like(rstd), [torch.empty_like(t[k]) for k in ("gate", "wp", "wn")]
    ops._call("vh_residual_norm", dt, u["x"].data_ptr(), u["b"].data_ptr(), gate, wp, wn, u["x"].data_ptr(), u["b"].data_ptr(),
              r2.data_ptr(), rows, d, 1, 0.5, 1e-6, st)
    assert torch.equal(u["x"], y) and torch.equal(u["b"], n) and torch.equal(r2, rstd)
    for over in ("dn", "b"):
        u = {k: t[k].clone() for k in ("x", "b", "dy", "dn")}
        ops._call("vh_residual_norm_backward", dt, u["dy"].data_ptr(), u["dn"].data_ptr(), u["x"].data_ptr(), u["b"].data_ptr(),
                  rstd.data_ptr(), gate, wp, wn, u["dy"].data_ptr(), u[over].data_ptr(), *(v.data_ptr() for v in sums), rows, d, 1,
                  0.5, st)
        assert torch.equal(u["dy"], dx) and torch.equal(u[over], db)
        for got, want in zip(sums, (dgate, dwp, dwn)):
            assert torch.equal(got, want)


# a block with several rows at once: as many as it holds, fewer, some of a gate row's left over
@pytest.mark.parametrize("d", [300, 513, 1531, 2049, 4096, 6200, 9001, 12000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_side_by_side(d, dtype):
    for rows, gate_rows in ((3, 1), (35, 5), (777, 1), (1300, 2), (1302, 434), (901, 901)):
        check(make(rows, d, dtype, gate_rows, seed=rows))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [96, 2500])
def test_parts_left_out(dtype, d):
    full = make(301, d, dtype, 7)
    for missing in (("wp",), ("wn",), ("gate",), ("dy",), ("gate", "wp"), ("gate", "wn"), ("wp", "wn"), ("gate", "wp", "wn"), ("gate", "wp", "dy")):
        t = dict(full)
        for k in missing:
            t[k] = None
        check(t)


def test_leading_dimensions_and_scale():
    t = make(24, 130, torch.bfloat16, 4)
    got = check(t, scale=-1.25, eps=1e-3, lead=(4, 6))
    assert got["y"].shape == (4, 6, 130) and got["dgate"].shape == (4, 130)


def test_zero_rows_of_a_block():
    """A block that puts out zeros has rms sqrt(eps): finite gradients; and an all-zero stream."""
    t = make(4, 200, torch.float32, 1)
    t["b"][1], t["b"][2], t["x"][2] = 0.0, 0.0, 0.0
    got = check(t)
    assert all(torch.isfinite(a).all() for a in got.values())


def test_no_rows():
    t = make(0, 64, torch.float32, 0)
    y, n, rstd = ops.gpu_residual_norm(t["x"], t["b"], None, t["wp"], t["wn"])
    assert y.shape == n.shape == (0, 64) and rstd.shape == (2, 0)
    dx, db, dg, dwp, dwn = ops.gpu_residual_norm_backward(t["dy"], t["dn"], t["x"], t["b"], rstd, None, t["wp"], t["wn"])
    assert dx.shape == (0, 64) and dg is None and not dwp.any() and not dwn.any()


def test_gradients_against_differences():
    """<gradient, direction> against central differences of sum(y gy + n gn), in 32 bits: h = 1e-2
    leaves h^2 of third derivatives and 1e-6 / h of the sums' rounding."""
    t = make(6, 400, torch.float32, 2)
    g = torch.Generator(device=DEV).manual_seed(3)
    grads = dict(zip(("x", "b", "gate", "wp", "wn"), ops.gpu_residual_norm_backward(
        t["dy"], t["dn"], t["x"], t["b"], ops.gpu_residual_norm(t["x"], t["b"], t["gate"], t["wp"], t["wn"], 0.5)[2],
        t["gate"], t["wp"], t["wn"], 0.5)))

    def total(u):
        y, n, _ = ops.gpu_residual_norm(u["x"], u["b"], u["gate"], u["wp"], u["wn"], 0.5)
        return float((y.double() * t["dy"].double()).sum() + (n.double() * t["dn"].double()).sum())

    h = 1e-2
    for k, grad in grads.items():
        v = torch.randn(t[k].shape, generator=g, device=DEV)
        slope = float((grad.double() * v.double()).sum())
        diff = (total(dict(t, **{k: t[k] + h * v})) - total(dict(t, **{k: t[k] - h * v}))) / (2 * h)
        assert abs(slope - diff) <= 5e-3 + 2e-3 * abs(slope), k


def test_runs_the_same_twice_and_on_another_stream():
    t = make(3000, 1531, torch.bfloat16, 3)
    one, s = check(t), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        y, n, rstd = ops.gpu_residual_norm(t["x"], t["b"], t["gate"], t["wp"], t["wn"], 0.5)
        back = ops.gpu_residual_norm_backward(t["dy"], t["dn"], t["x"], t["b"], rstd, t["gate"], t["wp"], t["wn"], 0.5)
    s.synchronize()
    for name, a in zip(("y", "n", "dx", "db", "dgate", "dwp", "dwn"), (y, n) + back):
        assert torch.equal(a, one[name]), name


def test_graph_replays():
    t = make(200, 512, torch.bfloat16, 1)
    call = lambda: ops.gpu_residual_norm_backward(t["dy"], t["dn"], t["x"], t["b"], ops.gpu_residual_norm(  # noqa: E731
        t["x"], t["b"], t["gate"], t["wp"], t["wn"])[2], t["gate"], t["wp"], t["wn"])
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        call()
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got = call()
    for seed in range(3):
        t["x"].copy_(make(200, 512, torch.bfloat16, 1, seed=seed)["x"])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, call()))


def test_refusals():
    t = make(6, 40, torch.float32, 2)
    x, b, gate, wp, wn = (t[k] for k in ("x", "b", "gate", "wp", "wn"))
    E = volta_amd.VoltaHipError
    for call, kind in ((lambda: ops.gpu_residual_norm(x, b[:5]), E), (lambda: ops.gpu_residual_norm(x, b, gate[:, :39].contiguous()), E),
                       (lambda: ops.gpu_residual_norm(x, b, make(4, 40, torch.float32, 4)["gate"]), E),  # 4 does not divide 6
                       (lambda: ops.gpu_residual_norm(x, b, gate, wp[:39].contiguous()), E),
                       (lambda: ops.gpu_residual_norm(x, b.bfloat16()), TypeError), (lambda: ops.gpu_residual_norm(x.half(), b.half()), TypeError),
                       (lambda: ops.gpu_residual_norm(x.t(), b.t()), ValueError), (lambda: ops.gpu_residual_norm(x, b, eps=-1.0), E),
                       (lambda: ops.gpu_residual_norm(torch.zeros((1, 16385), device=DEV), torch.zeros((1, 16385), device=DEV)), E)):
        with pytest.raises(kind):
            call()
    rstd = torch.ones((2, 6), device=DEV)
    for call, kind in ((lambda: ops.gpu_residual_norm_backward(None, None, x, b, rstd), E),  # no gradient at all
                       (lambda: ops.gpu_residual_norm_backward(t["dy"], None, x, b, rstd, None, None, wn), E),
                       (lambda: ops.gpu_residual_norm_backward(t["dy"], t["dn"], x, b, rstd), ValueError),
                       (lambda: ops.gpu_residual_norm_backward(t["dy"][:3], None, x, b, rstd), E),
                       (lambda: ops.gpu_residual_norm_backward(t["dy"], None, x, b, rstd[:1].contiguous()), E),
                       (lambda: ops.gpu_residual_norm_backward(t["dy"], None, x, b, rstd.double()), TypeError)):
        with pytest.raises(kind):
            call()
    assert ops.gpu_residual_norm(x.cpu(), b.cpu()) is None
    assert _lib.lib().vh_residual_norm(0, x.data_ptr(), None, None, None, None, x.data_ptr(), None, rstd.data_ptr(), 6, 40, 0, 1.0,
                                       1e-6, ops.stream_ptr(x.device)) == _lib.VH_ERR_BAD_ARG


def test_refuses_more_rows_than_a_launch_has_threads():
    t = make(6, 40, torch.float32, 2)
    x, r, s = t["x"].data_ptr(), torch.ones((2, 6), device=DEV), ops.stream_ptr(t["x"].device)
    rows = (1 << 26) - 15
    assert _lib.lib().vh_residual_norm(0, x, x, None, None, None, x, None, r.data_ptr(), rows, 8, 0, 1.0, 1e-6, s) == _lib.VH_ERR_UNSUPPORTED
    assert _lib.lib().vh_residual_norm_backward(0, x, None, x, x, r.data_ptr(), None, None, None, x, x, None, None, None, rows, 8, 0, 1.0,
                                                s) == _lib.VH_ERR_UNSUPPORTED


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_no_rows_leave_the_gate_no_gradient(dtype):
    """The sum over no rows is 0, whatever the buffer held: for weights and gates alike."""
    lib, s, dt = _lib.lib(), ops.stream_ptr(torch.device(DEV)), ops.dtype_code(torch.empty(0, dtype=dtype))
    E, width = _lib, 72
    one = torch.ones(width, dtype=dtype, device=DEV).data_ptr()

    def call(gate_rows, grad_gate):
        gate = torch.ones((max(gate_rows, 1), width), dtype=dtype, device=DEV)
        sums = [torch.full((width,), 7.0, dtype=dtype, device=DEV) for _ in range(2)]
        status = lib.vh_residual_norm_backward(dt, None, None, None, None, None, gate.data_ptr(), one, one, None, None,
                                               grad_gate, sums[0].data_ptr(), sums[1].data_ptr(), 0, width, gate_rows, 1.0, s)
        return status, sums

    for gate_rows in (1, 5):
        held = torch.full((gate_rows + 1, width), 7.0, dtype=dtype, device=DEV)
        status, sums = call(gate_rows, held.data_ptr())
        assert status == E.VH_OK and not held[:gate_rows].any() and bool((held[gate_rows:] == 7).all())
        assert not sums[0].any() and not sums[1].any()
    assert call(1, None)[0] == E.VH_ERR_BAD_ARG
    assert call(-1, one)[0] == E.VH_ERR_BAD_SHAPE
    assert call(0, None)[0] == E.VH_OK  # a gate row for each of no rows
    t = make(0, width, dtype, 1)
    y, n, rstd = ops.gpu_residual_norm(t["x"], t["b"], t["gate"], t["wp"], t["wn"])
    del one
    junk = torch.full((1, width), 7.0, dtype=dtype, device=DEV)
    del junk  # the next allocation of this size
    dgate = ops.gpu_residual_norm_backward(t["dy"], t["dn"], t["x"], t["b"], rstd, t["gate"], t["wp"], t["wn"])[2]
    assert dgate.shape == (1, width) and not dgate.any()


def test_refuses_outputs_that_overlap_in_part():
    """By the addresses alone.  An output may lie on an input of its size as a whole, or apart from all of them."""
    lib, s = _lib.lib(), ops.stream_ptr(torch.device(DEV))
    rows, width = 6, 40
    n = rows * width * 4
    buf = torch.ones(40 * n, dtype=torch.uint8, device=DEV)
    at = lambda i, off=0: buf.data_ptr() + i * 2 * n + off  # noqa: E731
    x, b, gate, wp, wn, y, out, rstd, dy, dn, dx, db, dgate, dwp, dwn = (at(i) for i in range(15))

    def forward(y=y, out=out, rstd=rstd):
        return lib.vh_residual_norm(0, x, b, gate, wp, wn, y, out, rstd, rows, width, 2, 1.0, 1e-6, s)

    def backward(dx=dx, db=db, dgate=dgate, dwp=dwp, dwn=dwn):
        return lib.vh_residual_norm_backward(0, dy, dn, x, b, rstd, gate, wp, wn, dx, db, dgate, dwp, dwn, rows, width, 2, 1.0, s)

    row = width * 4
    for call, wrong in ((forward, dict(y=x + row)), (forward, dict(y=b - row)), (forward, dict(out=b + 4)), (forward, dict(out=x + n - 4)),
                        (forward, dict(y=gate)), (forward, dict(out=wn)), (forward, dict(out=y)), (forward, dict(out=y + row)),
                        (forward, dict(rstd=x)), (forward, dict(rstd=y + 8)), (forward, dict(rstd=wp)),
                        (backward, dict(dx=dy + row)), (backward, dict(db=dn - 4)), (backward, dict(db=b + row)), (backward, dict(dx=x + 4)),
                        (backward, dict(dx=rstd)), (backward, dict(dgate=gate + row)), (backward, dict(dgate=dn)),
                        (backward, dict(dwp=wp + 4)), (backward, dict(dwn=dwp)), (backward, dict(db=dx)), (backward, dict(dwp=dgate + row)),
                        (backward, dict(dwn=rstd + 8))):
        assert call(**wrong) == _lib.VH_ERR_BAD_ARG, wrong
    for call, right in ((forward, {}), (forward, dict(y=x, out=b)), (forward, dict(y=x + n, out=b + n)), (backward, {}),
                        (backward, dict(dx=dy, db=dn)), (backward, dict(dx=dy, db=b)), (backward, dict(dwp=wp, dwn=wn, dgate=gate))):
        assert call(**right) == _lib.VH_OK, right
    torch.cuda.synchronize()


def test_backward_refuses_other_shapes_of_as_many_elements():
    """A transposed gradient or rstd would be misread; leading dimensions may be flattened."""
    t = make(6, 40, torch.float32, 1)
    y, n, rstd = ops.gpu_residual_norm(t["x"], t["b"], t["gate"], t["wp"], t["wn"])
    call = lambda dy, dn, r: ops.gpu_residual_norm_backward(dy, dn, t["x"], t["b"], r, t["gate"], t["wp"], t["wn"])  # noqa: E731
    want = call(t["dy"], t["dn"], rstd)
    for wrong in ((t["dy"].reshape(40, 6), t["dn"], rstd), (t["dy"], t["dn"].reshape(40, 6), rstd), (t["dy"].reshape(-1), t["dn"], rstd),
                  (t["dy"], t["dn"], rstd.reshape(6, 2)), (t["dy"], t["dn"], rstd.t().contiguous())):
        with pytest.raises(volta_amd.VoltaHipError):
            call(*wrong)
    got = call(t["dy"].reshape(2, 3, 40), t["dn"].reshape(1, 6, 40), rstd)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("d", [40, 1531, 4096, 9001])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_what_is_not_finite_stays_in_its_row(d, value):
    """A NaN or an infinity in a row's block, stream or gradient spoils that row and the sums over rows, no other row."""
    t = make(37, d, torch.float32, 37, seed=4)  # a gate row for each row
    forward = lambda u: ops.gpu_residual_norm(u["x"], u["b"], u["gate"], u["wp"], u["wn"], 0.5)  # noqa: E731
    backward = lambda u, r: ops.gpu_residual_norm_backward(u["dy"], u["dn"], u["x"], u["b"], r, u["gate"], u["wp"], u["wn"], 0.5)  # noqa: E731
    y, n, rstd = forward(t)
    dx, db, dgate, dwp, dwn = backward(t, rstd)
    others = torch.arange(37, device=DEV) != 20
    for name in ("x", "b", "dy", "dn"):
        u = dict(t, **{name: t[name].clone()})
        u[name][20, d // 2] = value
        y2, n2, rstd2 = forward(u)
        got = backward(u, rstd2)
        for a, b in zip((y2, n2) + got[:3], (y, n, dx, db, dgate)):
            assert torch.equal(a[others], b[others]), name
        if name in ("x", "b"):
            assert not torch.isfinite(n2[20]).all()
        assert not torch.isfinite(got[0][20]).all() and not torch.isfinite(got[1][20]).all()
        assert not torch.isfinite(got[3]).all()
