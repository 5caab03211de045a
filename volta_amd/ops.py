"""Python mirror of Volta's device-dispatch boundary (src/ops/gpu_ops.rs).

Each ``gpu_*`` function keeps the reference's name and argument order
(``gpu_ops.rs:151-861``) and calls the matching C-ABI entry of
libvolta_hip.so on torch device tensors.  Like the reference, the ``gpu_*``
functions return ``None`` instead of raising when the device path cannot run
(no GPU / CPU tensor), so a caller can keep a CPU fallback; shape errors
raise (the reference panics there).  Outputs are allocated by the callee, as
``GpuBuffer::zeros`` does in the reference.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _lib
from ._lib import BF16, F32, VoltaHipError, check, lib

_DTYPES = {torch.float32: F32, torch.bfloat16: BF16}


def dtype_code(t: torch.Tensor) -> int:
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise TypeError(f"unsupported dtype {t.dtype}; libvolta_hip takes float32 or bfloat16") from None


def stream_ptr(device=None) -> int:
    """The current stream's handle.  For a tensor's device without building a torch
    Stream object: 0.4 instead of 1.9 us, on a call that launches in 4 to 10."""
    if isinstance(device, torch.device) and device.type == "cuda" and device.index is not None and torch.cuda.is_initialized():
        return torch._C._cuda_getCurrentRawStream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


def ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("libvolta_hip takes device tensors")
    if not t.is_contiguous():
        raise ValueError("libvolta_hip takes contiguous tensors")
    return t.data_ptr()


def _same_dtype(*ts: torch.Tensor) -> int:
    code = dtype_code(ts[0])
    for t in ts[1:]:
        if t is not None and t.dtype != ts[0].dtype:
            raise TypeError("all tensor arguments of one call must share a dtype")
    return code


def _call(name: str, *args) -> None:
    check(getattr(lib(), name)(*args))


def expect_numel(t: Optional[torch.Tensor], n: int, what: str) -> None:
    """The C ABI carries no tensor sizes: a tensor smaller than its dimensions
    say would be read or written out of bounds.  Raises VH_ERR_BAD_SHAPE (the
    reference's assert_eq! panic, kernels.rs:1129-1130) before any launch.  An
    empty problem (n == 0, e.g. batch 0) touches no memory and is not checked."""
    if t is not None and n > 0 and t.numel() != n:
        raise VoltaHipError(_lib.VH_ERR_BAD_SHAPE,
                            f"{what}: tensor holds {t.numel()} elements, the dimensions give {n}")


def _optional(fn):
    """Reference semantics: Option::None when the device path is unavailable."""

    def wrapper(*args, **kwargs):
        for a in args:
            if isinstance(a, torch.Tensor) and not a.is_cuda:
                return None
        try:
            return fn(*args, **kwargs)
        except VoltaHipError as e:
            if e.status in (_lib.VH_ERR_NO_DEVICE, _lib.VH_ERR_OOM):
                return None
            raise

    wrapper.__name__ = fn.__name__
    wrapper.__doc__ = fn.__doc__
    return wrapper


# ---------------------------------------------------------------- matmul
@_optional
def gpu_matmul(a: torch.Tensor, b: torch.Tensor, m: int, k: int, n: int):
    """gpu_ops.rs:151 -- c[m,n] = a[m,k] . b[k,n]."""
    dt = _same_dtype(a, b)
    expect_numel(a, m * k, "gpu_matmul a")
    expect_numel(b, k * n, "gpu_matmul b")
    c = torch.empty((m, n), dtype=a.dtype, device=a.device)
    _call("vh_matmul", dt, ptr(a), ptr(b), ptr(c), m, k, n, stream_ptr(a.device))
    return c


@_optional
def gpu_matmul_backward_a(grad: torch.Tensor, b: torch.Tensor, m: int, k: int, n: int):
    """gpu_ops.rs:408 -- grad_a[m,k] = grad[m,n] . b[k,n]^T."""
    dt = _same_dtype(grad, b)
    expect_numel(grad, m * n, "gpu_matmul_backward_a grad")
    expect_numel(b, k * n, "gpu_matmul_backward_a b")
    out = torch.empty((m, k), dtype=grad.dtype, device=grad.device)
    _call("vh_matmul_backward_a", dt, ptr(grad), ptr(b), ptr(out), m, k, n, stream_ptr(grad.device))
    return out


@_optional
def gpu_matmul_backward_b(a: torch.Tensor, grad: torch.Tensor, m: int, k: int, n: int):
    """gpu_ops.rs:430 -- grad_b[k,n] = a[m,k]^T . grad[m,n]."""
    dt = _same_dtype(a, grad)
    expect_numel(a, m * k, "gpu_matmul_backward_b a")
    expect_numel(grad, m * n, "gpu_matmul_backward_b grad")
    out = torch.empty((k, n), dtype=a.dtype, device=a.device)
    _call("vh_matmul_backward_b", dt, ptr(a), ptr(grad), ptr(out), m, k, n, stream_ptr(a.device))
    return out


# ---------------------------------------------------------------- im2col / col2im
@_optional
def gpu_im2col(input, batch_size, channels, height, width, kernel_h, kernel_w, stride_h, stride_w, h_out, w_out):
    """gpu_ops.rs:515 -- (B,C,H,W) (already padded) -> (B*h_out*w_out, C*kh*kw)."""
    dt = dtype_code(input)
    expect_numel(input, batch_size * channels * height * width, "gpu_im2col input")
    col = torch.empty((batch_size * h_out * w_out, channels * kernel_h * kernel_w), dtype=input.dtype,
                      device=input.device)
    _call("vh_im2col", dt, ptr(input), ptr(col), batch_size, channels, height, width, kernel_h, kernel_w,
          stride_h, stride_w, h_out, w_out, stream_ptr(input.device))
    return col


@_optional
def gpu_col2im(col, batch_size, channels, height, width, kernel_h, kernel_w, stride_h, stride_w, h_out, w_out):
    """gpu_ops.rs:546 -- adjoint of gpu_im2col."""
    dt = dtype_code(col)
    expect_numel(col, batch_size * h_out * w_out * channels * kernel_h * kernel_w, "gpu_col2im col")
    out = torch.empty((batch_size, channels, height, width), dtype=col.dtype, device=col.device)
    _call("vh_col2im", dt, ptr(col), ptr(out), batch_size, channels, height, width, kernel_h, kernel_w,
          stride_h, stride_w, h_out, w_out, stream_ptr(col.device))
    return out


# ---------------------------------------------------------------- conv kernels
_CONV_OPERANDS = {  # which tensors each conv entry takes: x (input), w (weight), y (out_grad)
    "vh_direct_conv": "xw", "vh_igemm": "xw", "vh_conv_backward_input": "yw", "vh_igemm_backward_input": "yw",
    "vh_conv_backward_weight": "yx", "vh_igemm_backward_weight": "yx"}


def _conv_call(name, t0, t1, out_shape, dims):
    dt = _same_dtype(t0, t1)
    B, C, O, H, W, KH, KW = dims[:7]
    HO, WO = dims[11:13]
    sizes = {"x": B * C * H * W, "w": O * C * KH * KW, "y": B * O * HO * WO}
    for t, role in zip((t0, t1), _CONV_OPERANDS[name]):
        expect_numel(t, sizes[role], f"{name} {dict(x='input', w='weight', y='out_grad')[role]}")
    out = torch.empty(out_shape, dtype=t0.dtype, device=t0.device)
    _call(name, dt, ptr(t0), ptr(t1), ptr(out), *dims, stream_ptr(t0.device))
    return out


@_optional
def gpu_direct_conv(input, weight, batch_size, in_channels, out_channels, height, width, kernel_h, kernel_w,
                    stride_h, stride_w, pad_h, pad_w, h_out, w_out):
    """gpu_ops.rs:574 (stride before pad)."""
    dims = (batch_size, in_channels, out_channels, height, width, kernel_h, kernel_w, stride_h, stride_w,
            pad_h, pad_w, h_out, w_out)
    return _conv_call("vh_direct_conv", input, weight, (batch_size, out_channels, h_out, w_out), dims)


@_optional
def gpu_igemm(input, weight, batch_size, in_channels, out_channels, height, width, kernel_h, kernel_w,
              stride_h, stride_w, pad_h, pad_w, h_out, w_out):
    """gpu_ops.rs:622."""
    dims = (batch_size, in_channels, out_channels, height, width, kernel_h, kernel_w, stride_h, stride_w,
            pad_h, pad_w, h_out, w_out)
    return _conv_call("vh_igemm", input, weight, (batch_size, out_channels, h_out, w_out), dims)


@_optional
def gpu_conv_backward_input(out_grad, weight, batch_size, in_channels, out_channels, height, width, kernel_h,
                            kernel_w, stride_h, stride_w, pad_h, pad_w, h_out, w_out):
    """gpu_ops.rs:670."""
    dims = (batch_size, in_channels, out_channels, height, width, kernel_h, kernel_w, stride_h, stride_w,
            pad_h, pad_w, h_out, w_out)
    return _conv_call("vh_conv_backward_input", out_grad, weight, (batch_size, in_channels, height, width), dims)


@_optional
def gpu_conv_backward_weight(out_grad, input, batch_size, in_channels, out_channels, height, width, kernel_h,
                             kernel_w, stride_h, stride_w, pad_h, pad_w, h_out, w_out):
    """gpu_ops.rs:718 -- note (out_grad, input)."""
    dims = (batch_size, in_channels, out_channels, height, width, kernel_h, kernel_w, stride_h, stride_w,
            pad_h, pad_w, h_out, w_out)
    return _conv_call("vh_conv_backward_weight", out_grad, input, (out_channels, in_channels, kernel_h, kernel_w),
                      dims)


@_optional
def gpu_igemm_backward_input(out_grad, weight, batch_size, in_channels, out_channels, height, width, kernel_h,
                             kernel_w, stride_h, stride_w, pad_h, pad_w, h_out, w_out):
    """gpu_ops.rs:766."""
    dims = (batch_size, in_channels, out_channels, height, width, kernel_h, kernel_w, stride_h, stride_w,
            pad_h, pad_w, h_out, w_out)
    return _conv_call("vh_igemm_backward_input", out_grad, weight, (batch_size, in_channels, height, width), dims)


@_optional
def gpu_igemm_backward_weight(out_grad, input, batch_size, in_channels, out_channels, height, width, kernel_h,
                              kernel_w, stride_h, stride_w, pad_h, pad_w, h_out, w_out):
    """gpu_ops.rs:814."""
    dims = (batch_size, in_channels, out_channels, height, width, kernel_h, kernel_w, stride_h, stride_w,
            pad_h, pad_w, h_out, w_out)
    return _conv_call("vh_igemm_backward_weight", out_grad, input,
                      (out_channels, in_channels, kernel_h, kernel_w), dims)


# ---------------------------------------------------------------- glue: ReLU, sum loss
_UNARY_OPS = {"relu": _lib.UNARY_RELU}


def _unary_code(op: str) -> int:
    try:
        return _UNARY_OPS[op]
    except KeyError:
        raise ValueError(f"unary op {op!r}: only 'relu' is on this path") from None


@_optional
def gpu_unary(input: torch.Tensor, op: str):
    """gpu_ops.rs:171 -- elementwise op (ReLU: max(x, 0), unary.rs:272)."""
    code = _unary_code(op)
    x = input.contiguous()
    y = torch.empty_like(x)
    _call("vh_unary", dtype_code(x), code, ptr(x), ptr(y), x.numel(), stream_ptr(x.device))
    return y


@_optional
def gpu_unary_backward(out_grad: torch.Tensor, x: torch.Tensor, op: str):
    """gpu_ops.rs:186 -- ReLU: out_grad where x > 0, else 0 (unary.rs:150-155)."""
    code = _unary_code(op)
    dt = _same_dtype(out_grad, x)
    if out_grad.numel() != x.numel():
        raise ValueError("gpu_unary_backward: out_grad and x differ in size")
    dx = torch.empty_like(x)
    _call("vh_unary_backward", dt, code, ptr(out_grad), ptr(x), ptr(dx), x.numel(), stream_ptr(x.device))
    return dx


@_optional
def gpu_sum_reduce(data: torch.Tensor):
    """gpu_ops.rs:118 -- the fp32 sum of every element, returned to the host."""
    out = torch.empty((1,), dtype=torch.float32, device=data.device)
    _call("vh_sum_reduce", dtype_code(data), ptr(data), data.numel(), ptr(out), stream_ptr(data.device))
    return float(out.item())


def gpu_sum_backward(grad: float, input_size: int, dtype=torch.float32, device="cuda:0"):
    """gpu_ops.rs:452 -- a buffer of `input_size` elements equal to `grad`
    (SumGradFn; the autograd seed when grad = 1).  None without a device."""
    if not torch.cuda.is_available():
        return None
    out = torch.empty((input_size,), dtype=dtype, device=device)
    try:
        _call("vh_sum_backward", _DTYPES[dtype], float(grad), ptr(out), input_size, stream_ptr(out.device))
    except VoltaHipError as e:
        if e.status in (_lib.VH_ERR_NO_DEVICE, _lib.VH_ERR_OOM):
            return None
        raise
    return out


# ---------------------------------------------------------------- the step after dW
@_optional
def gpu_add(a: torch.Tensor, b: torch.Tensor):
    """gpu_ops.rs:17 as used by accumulate_grad (autograd.rs:158-184): a + b."""
    dt = _same_dtype(a, b)
    if a.numel() != b.numel():
        raise ValueError("gpu_add: size mismatch")
    out = a.clone()
    _call("vh_grad_accumulate", dt, ptr(out), ptr(b), out.numel(), stream_ptr(a.device))
    return out


@_optional
def gpu_optimizer_step(params: torch.Tensor, grads: torch.Tensor, state1: torch.Tensor, state2: torch.Tensor,
                       op: int, lr: float, beta1: float = 0.0, beta2: float = 0.0, t: float = 0.0, eps: float = 0.0,
                       weight_decay: float = 0.0):
    """gpu_ops.rs:496 -- updates params (and the states) in place; f32 tensors."""
    for x in (params, grads, state1, state2):
        if x.dtype != torch.float32:
            raise TypeError("gpu_optimizer_step takes float32 tensors")
    _call("vh_optimizer_step", op, lr, beta1, beta2, t, eps, weight_decay, ptr(params), ptr(grads), ptr(state1),
          ptr(state2), params.numel(), stream_ptr(params.device))
    return ()


# ---------------------------------------------------------------- losses over a vocabulary
def _logits(logits: torch.Tensor, what: str):
    """(dtype code, address, row stride, rows, vocabulary) of [rows, vocab] logits whose rows are contiguous."""
    if logits.dim() != 2:
        raise VoltaHipError(_lib.VH_ERR_BAD_SHAPE, f"{what}: logits are [rows, vocab], got {tuple(logits.shape)}")
    rows, vocab = logits.shape
    if vocab > 1 and logits.stride(1) != 1:
        raise ValueError(f"{what}: the entries of a row of logits must lie side by side")
    if not logits.is_cuda:
        raise ValueError("libvolta_hip takes device tensors")
    stride = logits.stride(0) if rows > 1 else max(vocab, 1)
    if stride < vocab:
        raise ValueError(f"{what}: rows of logits overlap")
    return dtype_code(logits), logits.data_ptr(), stride, rows, vocab


def _vector(t: Optional[torch.Tensor], n: int, dtypes, device, what: str, name: str) -> Optional[int]:
    """Address of a contiguous [n] tensor of one of `dtypes` (None passes)."""
    if t is None:
        return None
    if t.dtype in dtypes and t.numel() == n and t.device == device and t.is_contiguous():
        return t.data_ptr()
    if t.dtype not in dtypes:
        raise TypeError(f"{what} {name}: {t.dtype}, expected {' or '.join(str(d) for d in dtypes)}")
    if t.numel() != n:
        raise VoltaHipError(_lib.VH_ERR_BAD_SHAPE, f"{what} {name}: tensor holds {t.numel()} elements, the dimensions give {n}")
    if t.device != device:
        raise ValueError(f"{what} {name}: on {t.device}, the logits are on {device}")
    return ptr(t)


def _grad_logits(logits: torch.Tensor, grad: bool, out: Optional[torch.Tensor], what: str):
    """(tensor or None, address, stride) of the logits' gradient: a new tensor, or `out` (which may be the logits)."""
    rows, vocab = logits.shape
    if not grad:
        return None, None, vocab
    if out is None:
        out = torch.empty(rows, vocab, dtype=logits.dtype, device=logits.device)
        return out, out.data_ptr(), max(vocab, 1)
    if out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device:
        raise VoltaHipError(_lib.VH_ERR_BAD_SHAPE, f"{what}: out does not match the logits")
    _, address, stride, _, _ = _logits(out, what)
    return out, address, stride


_F32, _I64, _MASKS = (torch.float32,), (torch.int64,), (torch.bool, torch.uint8)


@_optional
def gpu_token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, temperature: float = 1.0):
    """log softmax(logits / temperature) of each row's token, fp32 [rows]: what old_logp and
    ref_logp of the losses below are made with.  tokens: int64 [rows]."""
    what = "gpu_token_logprobs"
    dt, x, stride, rows, vocab = _logits(logits, what)
    tok = _vector(tokens, rows, _I64, logits.device, what, "tokens")
    logp = torch.empty(rows, dtype=torch.float32, device=logits.device)
    _call("vh_token_logprobs", dt, x, stride, tok, ptr(logp), rows, vocab, temperature, stream_ptr(logits.device))
    return logp


@_optional
def gpu_policy_loss(logits: torch.Tensor, tokens: torch.Tensor, old_logp: torch.Tensor, advantages: torch.Tensor,
                    ref_logp: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None, clip_low: float = 0.2,
                    clip_high: float = 0.2, kl_coef: float = 0.0, temperature: float = 1.0, grad_scale: float = 1.0,
                    grad: bool = True, out: Optional[torch.Tensor] = None):
    """The clipped policy loss with its KL term, and its gradient in the same pass:
    (loss [1], logp [rows], grad_logits or None).

    With r = exp(logp - old_logp), A the row's advantage and d = ref_logp - logp the loss is the mean over the
    rows that ``mask`` keeps of -min(r A, clamp(r, 1 - clip_low, 1 + clip_high) A) + kl_coef (e^d - d - 1).
    Masked rows are not read; their logp is 0 and their gradient zeros.  ``grad_scale`` multiplies the
    gradient (the loss's own upstream gradient); ``out`` receives it and may be the logits themselves."""
    what = "gpu_policy_loss"
    dt, x, stride, rows, vocab = _logits(logits, what)
    dev = logits.device
    tok = _vector(tokens, rows, _I64, dev, what, "tokens")
    old = _vector(old_logp, rows, _F32, dev, what, "old_logp")
    adv = _vector(advantages, rows, _F32, dev, what, "advantages")
    ref = _vector(ref_logp, rows, _F32, dev, what, "ref_logp")
    keep = _vector(mask, rows, _MASKS, dev, what, "mask")
    g, address, g_stride = _grad_logits(logits, grad, out, what)
    logp, loss = old_logp.new_empty(rows), old_logp.new_empty(1)
    _call("vh_policy_loss", dt, x, stride, tok, old, adv, ref, keep, loss.data_ptr(), logp.data_ptr(), address,
          g_stride, rows, vocab, clip_low, clip_high, kl_coef, temperature, grad_scale, stream_ptr(dev))
    return loss, logp, g


@_optional
def gpu_preference_loss(logits: torch.Tensor, tokens: torch.Tensor, offsets: torch.Tensor, ref_logp: torch.Tensor,
                        mask: Optional[torch.Tensor] = None, beta: float = 0.1, label_smoothing: float = 0.0,
                        temperature: float = 1.0, grad_scale: float = 1.0, grad: bool = True,
                        out: Optional[torch.Tensor] = None):
    """The preference loss over pairs of sequences, and its gradient: (loss [1], seq_logp [2 pairs],
    grad_logits or None).

    Sequence s is rows offsets[s] .. offsets[s + 1] (offsets: int64 [2 pairs + 1]); pair i's preferred sequence
    is i, its rejected one pairs + i; ref_logp [2 pairs]: the reference model's sums of their log-probabilities.
    z = beta ((S_i - ref_i) - (S_(pairs+i) - ref_(pairs+i))); the loss is the mean over the pairs of
    -(1 - label_smoothing) log sigmoid(z) - label_smoothing log sigmoid(-z)."""
    what = "gpu_preference_loss"
    dt, x, stride, rows, vocab = _logits(logits, what)
    dev = logits.device
    if offsets.dim() != 1 or offsets.numel() < 3 or offsets.numel() % 2 == 0:
        raise VoltaHipError(_lib.VH_ERR_BAD_SHAPE, f"{what}: offsets hold 2 pairs + 1 values, got {tuple(offsets.shape)}")
    pairs = (offsets.numel() - 1) // 2
    tok = _vector(tokens, rows, _I64, dev, what, "tokens")
    off = _vector(offsets, 2 * pairs + 1, _I64, dev, what, "offsets")
    ref = _vector(ref_logp, 2 * pairs, _F32, dev, what, "ref_logp")
    keep = _vector(mask, rows, _MASKS, dev, what, "mask")
    g, address, g_stride = _grad_logits(logits, grad, out, what)
    seq, loss = ref_logp.new_empty(2 * pairs), ref_logp.new_empty(1)
    _call("vh_preference_loss", dt, x, stride, tok, off, ref, keep, loss.data_ptr(), seq.data_ptr(), address, g_stride,
          rows, vocab, pairs, beta, label_smoothing, temperature, grad_scale, stream_ptr(dev))
    return loss, seq, g


# ---------------------------------------------------------------- gated residual norms
def _norm_args(x, block, gate, post_weight, next_weight, what):
    """(dtype code, rows, width, gate rows) of the tensors of a residual norm; x may have any leading dimensions."""
    dt = _same_dtype(x, block, gate, post_weight, next_weight)
    if x.dim() < 1 or block.shape != x.shape:
        raise VoltaHipError(_lib.VH_ERR_BAD_SHAPE, f"{what}: x is {tuple(x.shape)}, block {tuple(block.shape)}")
    width = x.shape[-1]
    rows = x.numel() // width if width else 0
    if post_weight is not None and post_weight.numel() != width:
        raise VoltaHipError(_lib.VH_ERR_BAD_SHAPE, f"{what} post_weight: {post_weight.numel()} elements, rows have {width}")
    if next_weight is not None and next_weight.numel() != width:
        raise VoltaHipError(_lib.VH_ERR_BAD_SHAPE, f"{what} next_weight: {next_weight.numel()} elements, rows have {width}")
    gate_rows = 0
    if gate is not None:
        if gate.dim() < 1 or gate.shape[-1] != width:
            raise VoltaHipError(_lib.VH_ERR_BAD_SHAPE, f"{what}: gate rows of {tuple(gate.shape)}, rows have {width}")
        gate_rows = gate.numel() // width if width else 0
    return dt, rows, width, gate_rows


@_optional
def gpu_residual_norm(x: torch.Tensor, block: torch.Tensor, gate: Optional[torch.Tensor] = None,
                      post_weight: Optional[torch.Tensor] = None, next_weight: Optional[torch.Tensor] = None,
                      scale: float = 1.0, eps: float = 1e-6):
    """The norms around a block, fused with its gate and residual scale: (y, n or None, rstd [2, rows]).

    u = block / rms(block) * post_weight, y = x + scale * gate * u, n = y / rms(y) * next_weight, row by row of
    the last dimension.  Without post_weight u = block; without next_weight n is None.  gate [.., width]: one row
    for all rows, one for each run of rows / gate_rows consecutive rows, or one for each row."""
    dt, rows, width, gate_rows = _norm_args(x, block, gate, post_weight, next_weight, "gpu_residual_norm")
    y = torch.empty_like(x)
    n = torch.empty_like(x) if next_weight is not None else None
    rstd = torch.empty(2, rows, dtype=torch.float32, device=x.device)
    _call("vh_residual_norm", dt, ptr(x), ptr(block), ptr(gate), ptr(post_weight), ptr(next_weight), ptr(y), ptr(n),
          ptr(rstd), rows, width, gate_rows, scale, eps, stream_ptr(x.device))
    return y, n, rstd


def gpu_residual_norm_backward(grad_y: Optional[torch.Tensor], grad_n: Optional[torch.Tensor], x: torch.Tensor,
                               block: torch.Tensor, rstd: torch.Tensor, gate: Optional[torch.Tensor] = None,
                               post_weight: Optional[torch.Tensor] = None,
                               next_weight: Optional[torch.Tensor] = None, scale: float = 1.0):
    """Backward of :func:`gpu_residual_norm` with the same x, block, gate, weights and scale: (grad_x, grad_block,
    grad_gate, grad_post_weight, grad_next_weight), None for what was not given.  grad_y: the gradient of y by its
    other uses (None: it has none); grad_n: that of n."""
    return _residual_norm_backward(x, block, rstd, grad_y, grad_n, gate, post_weight, next_weight, scale)


@_optional
def _residual_norm_backward(x, block, rstd, grad_y, grad_n, gate, post_weight, next_weight, scale):
    what = "gpu_residual_norm_backward"
    dt, rows, width, gate_rows = _norm_args(x, block, gate, post_weight, next_weight, what)
    _same_dtype(x, grad_y, grad_n)
    for name, g in (("grad_y", grad_y), ("grad_n", grad_n)):
        # leading dimensions may be flattened, rows not
        if g is not None and (g.numel() != x.numel() or g.dim() < 1 or g.shape[-1] != width):
            raise VoltaHipError(_lib.VH_ERR_BAD_SHAPE, f"{what} {name}: {tuple(g.shape)}, x is {tuple(x.shape)}")
    if rstd.dtype != torch.float32:
        raise TypeError(f"{what}: rstd is float32")
    if tuple(rstd.shape) != (2, rows):
        raise VoltaHipError(_lib.VH_ERR_BAD_SHAPE, f"{what} rstd: {tuple(rstd.shape)}, the forward's is {(2, rows)}")
    if next_weight is None and grad_n is not None:
        raise ValueError(f"{what}: grad_n without next_weight")
    new = [torch.empty_like(t) if t is not None else None for t in (x, block, gate, post_weight, next_weight)]
    _call("vh_residual_norm_backward", dt, ptr(grad_y), ptr(grad_n), ptr(x), ptr(block), ptr(rstd), ptr(gate),
          ptr(post_weight), ptr(next_weight), *(ptr(t) for t in new), rows, width, gate_rows, scale,
          stream_ptr(x.device))
    return tuple(new)


# ---------------------------------------------------------------- orthogonalised updates
def _matrices(t: torch.Tensor, what: str):
    """(batch, rows, cols) of a matrix or a batch of them."""
    if t.dim() not in (2, 3):
        raise VoltaHipError(_lib.VH_ERR_BAD_SHAPE, f"{what}: [rows, cols] or [batch, rows, cols], got {tuple(t.shape)}")
    return (t.shape[0] if t.dim() == 3 else 1, t.shape[-2], t.shape[-1])


def _same_shape(t: torch.Tensor, like: torch.Tensor, what: str) -> None:
    if t.shape != like.shape:
        raise VoltaHipError(_lib.VH_ERR_BAD_SHAPE, f"{what}: {tuple(t.shape)}, the matrices are {tuple(like.shape)}")


@_optional
def gpu_orthogonalize(grad: torch.Tensor, steps: int = 5, eps: float = 1e-7, out: Optional[torch.Tensor] = None):
    """The Newton-Schulz orthogonalisation of a matrix, or of each of a batch: singular values to about 1,
    singular vectors kept.  ``out`` may be ``grad``.

    float32 matrices are computed to float32's accuracy; bfloat16 ones with fp16 products and fp32 sums, which over up
    to 5 steps is off by about the result's own rounding (what is to be more exact goes in as float32)."""
    what = "gpu_orthogonalize"
    batch, rows, cols = _matrices(grad, what)
    if out is None:
        out = torch.empty_like(grad)
    dt = _same_dtype(grad, out)
    _same_shape(out, grad, f"{what} out")
    _call("vh_orthogonalize", dt, ptr(grad), ptr(out), batch, rows, cols, steps, eps, stream_ptr(grad.device))
    return out


@_optional
def gpu_muon_step(params: torch.Tensor, grads: torch.Tensor, momentum: torch.Tensor, lr: float, beta: float = 0.95,
                  weight_decay: float = 0.0, nesterov: bool = True, steps: int = 5, eps: float = 1e-7,
                  in_first: bool = False):
    """One step of the orthogonalised-momentum optimiser on a matrix, or on each of a batch; params and momentum
    (float32) are updated in place:

    momentum = beta momentum + grads; u = grads + beta momentum (nesterov) or momentum;
    params = (1 - lr weight_decay) params - lr sqrt(max(1, outputs / inputs)) orthogonalize(u),

    with rows for outputs and cols for inputs, or, ``in_first``, as Linear's weights lie, the other way round.
    bfloat16 params and grads: products as in :func:`gpu_orthogonalize`; the momentum is float32 either way."""
    what = "gpu_muon_step"
    batch, rows, cols = _matrices(params, what)
    if in_first and rows != cols and rows and cols:
        # the entry's factor is that of [out, in]: what it is to be over what it will be, in lr, and out of the decay
        ratio = math.sqrt(cols / rows)
        lr, weight_decay = lr * ratio, weight_decay / ratio
    dt = _same_dtype(params, grads)
    if momentum.dtype != torch.float32:
        raise TypeError(f"{what}: momentum is float32")
    _same_shape(grads, params, f"{what} grads")
    _same_shape(momentum, params, f"{what} momentum")
    _call("vh_muon_step", dt, ptr(params), ptr(grads), ptr(momentum), batch, rows, cols, lr, beta, weight_decay,
          int(bool(nesterov)), steps, eps, stream_ptr(params.device))
    return ()


# ---------------------------------------------------------------- device storage: dtype and layout
def to_dtype(x: torch.Tensor, dtype) -> torch.Tensor:
    """Device cast f32 <-> bf16 (RNE), the library's conversion."""
    out = torch.empty(x.shape, dtype=dtype, device=x.device)
    _call("vh_cast", dtype_code(x), _DTYPES[dtype], ptr(x), ptr(out), x.numel(), stream_ptr(x.device))
    return out


def nchw_to_nhwc(x: torch.Tensor) -> torch.Tensor:
    B, C, H, W = x.shape
    out = torch.empty((B, H, W, C), dtype=x.dtype, device=x.device)
    _call("vh_nchw_to_nhwc", dtype_code(x), ptr(x), ptr(out), B, C, H, W, stream_ptr(x.device))
    return out


def nhwc_to_nchw(x: torch.Tensor) -> torch.Tensor:
    B, H, W, C = x.shape
    out = torch.empty((B, C, H, W), dtype=x.dtype, device=x.device)
    _call("vh_nhwc_to_nchw", dtype_code(x), ptr(x), ptr(out), B, C, H, W, stream_ptr(x.device))
    return out
