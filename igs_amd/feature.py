"""Operators in front of the Gaussian head: embedding lookup, layer norm and dropout on the HIP library.

The reference's module takes its `feature` [B, F, D] as given (src/igs/gs2d.py:611-635).  These are the
operators that make such a feature out of token ids or of a trunk's output, forward and backward:

  embedding_lookup(tokens, weight, scale, padding_idx)      scale * weight[tokens], dense gradient
  layer_norm(x, weight, bias, eps, dropout_p, seed, offset) norm over the last axis, dropout of its result
  dropout(x, p, seed, offset)                               counter-based mask, never stored

`GaussianSplatting2D` calls them when it is built with `num_embeddings=`, `feature_norm=` or
`feature_dropout=`.  fp32, fp16 and bf16; sums and norms are held in fp32 and every result is rounded
once; gradients of weights are summed in a fixed order (bit-reproducible).  Eager callers go through
`torch.autograd.Function`s; under `torch.compile` the same library calls are registered operators
(`igs_amd::embedding_fwd` and its like).  There is no CPU path: tensors must live on the GPU.  The
`naive_*` functions are the plain torch expressions (any device), what the module's `fused=False`
debug path uses.
"""
from __future__ import annotations

import math
from typing import List, Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._splat import _on, _stream

Tensor = torch.Tensor

_DTYPES = {torch.float32: _lib.IGS_F32, torch.float16: _lib.IGS_F16, torch.bfloat16: _lib.IGS_BF16}
_TOKENS = {torch.int64: 8, torch.int32: 4}


# --------------------------------------------------------------------------------------
# arguments
# --------------------------------------------------------------------------------------
def _dtype_of(t: Tensor, what: str) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{what} must be float32, float16 or bfloat16; got {t.dtype}")
    return code


def _on_gpu(first: Tensor, *others: Optional[Tensor]) -> None:
    """Every tensor whose address goes to a kernel lives on one GPU: a host pointer handed to a launch
    would be a memory fault, not an exception."""
    if first.device.type != "cuda":
        raise RuntimeError("the feature operators run on the GPU only (HIP kernels); got a tensor on "
                           f"{first.device}. The naive_* functions are the plain-torch expressions.")
    for t in others:
        if t is not None and t.device != first.device:
            raise RuntimeError(f"Expected all tensors to be on the same device, but got {first.device} and {t.device}")


def dropout_threshold(p: float) -> int:
    """The 16-bit limit of dropout probability p: an element is dropped if its 16-bit number is below
    it, so p acts in steps of 2^-16."""
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability must be in [0, 1]; got {p}")
    return math.floor(p * 65536 + 0.5)


def _seed(seed, offset, like: Tensor) -> Tuple[int, Optional[Tensor], int]:
    """(number, device tensor or None, offset): a seed is an int in [0, 2^63), or an int64 tensor of one
    element on the device, which the kernels read when they run (so a replayed graph sees its value of
    then)."""
    if type(offset) is not int and not isinstance(offset, (int, torch.SymInt)):
        raise TypeError(f"offset must be an int; got {type(offset).__name__}")
    if isinstance(seed, Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1:
            raise TypeError("a seed tensor holds one int64 element")
        if seed.device != like.device:
            raise RuntimeError(f"Expected all tensors to be on the same device, but got {like.device} and {seed.device} "
                               "(the seed)")
        return 0, seed.detach(), offset
    if seed is None:
        raise ValueError("dropout needs a seed (an int, or an int64 tensor of one element on the device)")
    if not isinstance(seed, (int, torch.SymInt)) or isinstance(seed, bool):
        raise TypeError(f"seed must be an int or an int64 tensor; got {type(seed).__name__}")
    if not torch.compiler.is_compiling() and not (0 <= seed < 1 << 63 and 0 <= offset < 1 << 63):
        raise ValueError("seed and offset must be in [0, 2^63)")
    return seed, None, offset


def _rows(x: Tensor) -> Tuple[Tensor, int]:
    """(x or a contiguous copy, distance of its rows in elements): rows of the last axis are taken where
    they are if they are dense and evenly spaced (slices of the last axis, expanded batches)."""
    if x.is_contiguous():
        return x, x.shape[-1]
    sizes, strides = x.shape, x.stride()
    if sizes[-1] != 1 and strides[-1] != 1:
        return x.contiguous(), sizes[-1]
    step = span = None
    for n, s in zip(reversed(sizes[:-1]), reversed(strides[:-1])):
        if n == 1:
            continue
        if span is None:
            step = s
        elif s != span:
            return x.contiguous(), sizes[-1]
        span = s * n
    return x, sizes[-1] if step is None else step


def _once(backward):
    """`once_differentiable` without its bookkeeping where no graph of the backward is being recorded (grad
    mode is off then): a training step of a small problem is bound by the host."""
    recorded = once_differentiable(backward)

    def run(ctx, grad):
        return recorded(ctx, grad) if torch.is_grad_enabled() else backward(ctx, grad)

    return run


# --------------------------------------------------------------------------------------
# embedding lookup
# --------------------------------------------------------------------------------------
def _embedding_fwd(tokens: Tensor, weight: Tensor, scale: float) -> Tensor:
    vocab, D = weight.shape
    if not tokens.is_contiguous():
        tokens = tokens.contiguous()
    step, column = weight.stride()
    if column != 1 and D > 1:
        weight, step = weight.contiguous(), D
    dev, dtype = weight.device, weight.dtype
    with _on(dev):
        out = torch.empty((*tokens.shape, D), dtype=dtype, device=dev)
        rc = _lib.load().igs_embedding_forward(weight.data_ptr(), step, _DTYPES[dtype], vocab, D, tokens.data_ptr(),
                                               _TOKENS[tokens.dtype], tokens.numel(), scale, out.data_ptr(), _stream(dev))
    if rc:
        _lib.check(rc, "igs_embedding_forward")
    return out


def _embedding_bwd(grad: Tensor, tokens: Tensor, vocab: int, scale: float, padding_idx: int) -> Tensor:
    if not grad.is_contiguous():
        grad = grad.contiguous()
    if not tokens.is_contiguous():
        tokens = tokens.contiguous()
    D, n, dtype, dev = grad.shape[-1], tokens.numel(), grad.dtype, grad.device
    code = _DTYPES[dtype]
    nbytes = _lib.embedding_workspace_bytes(vocab, D, code, n)
    with _on(dev):
        out = torch.empty((vocab, D), dtype=dtype, device=dev)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
        rc = _lib.load().igs_embedding_backward(grad.data_ptr(), code, tokens.data_ptr(), _TOKENS[tokens.dtype], n, vocab,
                                                D, scale, padding_idx, out.data_ptr(), ws.data_ptr() if nbytes else None,
                                                nbytes, _stream(dev))
    if rc:
        _lib.check(rc, "igs_embedding_backward")
    return out


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, weight, scale, padding_idx):
        ctx.save_for_backward(tokens)
        ctx.args = (weight.shape[0], scale, padding_idx)
        return _embedding_fwd(tokens, weight, scale)

    @staticmethod
    @_once
    def backward(ctx, grad):
        return None, _embedding_bwd(grad, ctx.saved_tensors[0], *ctx.args), None, None


@torch.library.custom_op("igs_amd::embedding_fwd", mutates_args=(), device_types="cuda")
def embedding_fwd(tokens: Tensor, weight: Tensor, scale: float, padding_idx: int) -> Tensor:
    return _embedding_fwd(tokens, weight, scale)


@embedding_fwd.register_fake
def _(tokens, weight, scale, padding_idx):
    return weight.new_empty((*tokens.shape, weight.shape[1]))


@torch.library.custom_op("igs_amd::embedding_bwd", mutates_args=(), device_types="cuda")
def embedding_bwd(grad: Tensor, tokens: Tensor, vocab: int, scale: float, padding_idx: int) -> Tensor:
    return _embedding_bwd(grad, tokens, vocab, scale, padding_idx)


@embedding_bwd.register_fake
def _(grad, tokens, vocab, scale, padding_idx):
    return grad.new_empty((vocab, grad.shape[-1]))


def _embedding_setup(ctx, inputs, output):
    tokens, weight, scale, padding_idx = inputs
    ctx.save_for_backward(tokens)
    ctx.args = (weight.shape[0], scale, padding_idx)


def _embedding_backward(ctx, grad):
    return None, torch.ops.igs_amd.embedding_bwd(grad, ctx.saved_tensors[0], *ctx.args), None, None


embedding_fwd.register_autograd(_embedding_backward, setup_context=_embedding_setup)


def embedding_lookup(tokens: Tensor, weight: Tensor, scale: float = 1.0, padding_idx: Optional[int] = None) -> Tensor:
    """scale * weight[tokens]: tokens (int32 or int64, any shape) and weight [V, D] -> [*tokens.shape, D]
    in weight's type.

    The gradient of weight is dense, [V, D]: each token's gradients are summed in fp32 in a fixed order
    and rounded once; the row `padding_idx` (negative counts from the end) gets none.  A token outside
    [0, V) gives a row of NaN and reaches no gradient: nothing here waits for the device, so it cannot
    raise."""
    if weight.dim() != 2 or weight.shape[0] == 0 or weight.shape[1] == 0:
        raise ValueError(f"weight must be [V, D] with V, D >= 1; got {tuple(weight.shape)}")
    if tokens.dtype not in _TOKENS:
        raise TypeError(f"tokens must be int32 or int64; got {tokens.dtype}")
    if weight.dtype not in _DTYPES:
        _dtype_of(weight, "weight")
    scale = float(scale)
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    V = weight.shape[0]
    if padding_idx is None:
        padding_idx = -1
    else:
        if not -V <= padding_idx < V:
            raise ValueError(f"padding_idx {padding_idx} is outside the table of {V} rows")
        padding_idx %= V
    if torch.compiler.is_compiling():
        return torch.ops.igs_amd.embedding_fwd(tokens, weight, scale, padding_idx)
    _on_gpu(weight, tokens)
    if weight.requires_grad and torch.is_grad_enabled():
        return _Embedding.apply(tokens, weight, scale, padding_idx)
    return _embedding_fwd(tokens, weight.detach(), scale)


def naive_embedding_lookup(tokens: Tensor, weight: Tensor, scale: float = 1.0, padding_idx: Optional[int] = None) -> Tensor:
    """Plain torch expression of `embedding_lookup` (any device, differentiable through autograd)."""
    rows = weight[tokens]
    if padding_idx is not None:
        pad = (tokens == padding_idx % weight.shape[0])[..., None]
        rows = torch.where(pad, rows.detach(), rows)
    return rows * scale


# --------------------------------------------------------------------------------------
# layer norm (with dropout of its result)
# --------------------------------------------------------------------------------------
def _norm_fwd(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], eps: float, threshold: int, seed: int,
              seed_tensor: Optional[Tensor], offset: int, want_stats: bool) -> Tuple[Tensor, Optional[Tensor]]:
    shape, dtype, dev = x.shape, x.dtype, x.device
    step = D = shape[-1]
    rows = x.numel() // D
    if not x.is_contiguous():
        x, step = _rows(x)
    wdtype, pw, pb = dtype, None, None
    if bias is not None:
        if not bias.is_contiguous():
            bias = bias.contiguous()
        wdtype, pb = bias.dtype, bias.data_ptr()
    if weight is not None:
        if not weight.is_contiguous():
            weight = weight.contiguous()
        wdtype, pw = weight.dtype, weight.data_ptr()
    with _on(dev):
        y = torch.empty(shape, dtype=dtype, device=dev)
        stats = torch.empty((rows, 2), dtype=torch.float32, device=dev) if want_stats else None
        rc = _lib.load().igs_layer_norm_forward(
            x.data_ptr(), step, _DTYPES[dtype], pw, pb, _DTYPES[wdtype], rows, D, eps, threshold, seed,
            None if seed_tensor is None else seed_tensor.data_ptr(), offset, y.data_ptr(),
            stats.data_ptr() if want_stats else None, _stream(dev))
    if rc:
        _lib.check(rc, "igs_layer_norm_forward")
    return y, stats


def _norm_bwd(grad: Tensor, x: Tensor, weight: Optional[Tensor], wdtype: torch.dtype, stats: Tensor, threshold: int,
              seed: int, seed_tensor: Optional[Tensor], offset: int, want_x: bool, want_w: bool, want_b: bool):
    shape, dtype, dev = x.shape, x.dtype, x.device
    step = D = shape[-1]
    rows = stats.shape[0]
    if not grad.is_contiguous():
        grad = grad.contiguous()
    if not x.is_contiguous():
        x, step = _rows(x)
    pw = None
    if weight is not None:
        if not weight.is_contiguous():
            weight = weight.contiguous()
        pw = weight.data_ptr()
    code, wcode = _DTYPES[dtype], _DTYPES[wdtype]
    nbytes = _lib.layer_norm_workspace_bytes(rows, D, code, wcode) if want_w or want_b else 0
    with _on(dev):
        gx = torch.empty(shape, dtype=dtype, device=dev) if want_x else None
        gw = torch.empty(D, dtype=wdtype, device=dev) if want_w else None
        gb = torch.empty(D, dtype=wdtype, device=dev) if want_b else None
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
        rc = _lib.load().igs_layer_norm_backward(
            grad.data_ptr(), x.data_ptr(), step, code, pw, wcode, stats.data_ptr(), rows, D, threshold, seed,
            None if seed_tensor is None else seed_tensor.data_ptr(), offset, gx.data_ptr() if want_x else None,
            gw.data_ptr() if want_w else None, gb.data_ptr() if want_b else None, ws.data_ptr() if nbytes else None,
            nbytes, _stream(dev))
    if rc:
        _lib.check(rc, "igs_layer_norm_backward")
    return gx, gw, gb


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, threshold, seed, seed_tensor, offset):
        y, stats = _norm_fwd(x, weight, bias, eps, threshold, seed, seed_tensor, offset, True)
        ctx.save_for_backward(x, weight, stats, seed_tensor)
        ctx.args = (threshold, seed, offset)
        ctx.wdtype = weight.dtype if weight is not None else bias.dtype if bias is not None else x.dtype
        return y

    @staticmethod
    @_once
    def backward(ctx, grad):
        x, weight, stats, seed_tensor = ctx.saved_tensors
        threshold, seed, offset = ctx.args
        need = ctx.needs_input_grad
        gx, gw, gb = _norm_bwd(grad, x, weight, ctx.wdtype, stats, threshold, seed, seed_tensor, offset, need[0],
                               need[1], need[2])
        return gx, gw, gb, None, None, None, None, None


@torch.library.custom_op("igs_amd::layer_norm_fwd", mutates_args=(), device_types="cuda")
def layer_norm_fwd(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], eps: float, threshold: int, seed: int,
                   seed_tensor: Optional[Tensor], offset: int) -> List[Tensor]:
    """[y, stats [rows, 2] (mean, 1 / standard deviation)]"""
    return list(_norm_fwd(x, weight, bias, eps, threshold, seed, seed_tensor, offset, True))


@layer_norm_fwd.register_fake
def _(x, weight, bias, eps, threshold, seed, seed_tensor, offset):
    return [x.new_empty(x.shape), x.new_empty((math.prod(x.shape[:-1]), 2), dtype=torch.float32)]


@torch.library.custom_op("igs_amd::layer_norm_bwd", mutates_args=(), device_types="cuda")
def layer_norm_bwd(grad: Tensor, x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], stats: Tensor,
                   threshold: int, seed: int, seed_tensor: Optional[Tensor], offset: int) -> List[Tensor]:
    """[grad_x, grad_weight (if weight), grad_bias (if bias)]"""
    wdtype = weight.dtype if weight is not None else bias.dtype if bias is not None else x.dtype
    g = _norm_bwd(grad, x, weight, wdtype, stats, threshold, seed, seed_tensor, offset, True, weight is not None,
                  bias is not None)
    return [t for t in g if t is not None]


@layer_norm_bwd.register_fake
def _(grad, x, weight, bias, stats, threshold, seed, seed_tensor, offset):
    return [x.new_empty(x.shape)] + [t.new_empty(t.shape) for t in (weight, bias) if t is not None]


def _norm_setup(ctx, inputs, output):
    x, weight, bias, eps, threshold, seed, seed_tensor, offset = inputs
    ctx.save_for_backward(x, weight, bias, output[1], seed_tensor)
    ctx.args = (threshold, seed, offset)


def _norm_backward(ctx, grads):
    if grads[0] is None:
        return (None,) * 8
    x, weight, bias, stats, seed_tensor = ctx.saved_tensors
    threshold, seed, offset = ctx.args
    g = iter(torch.ops.igs_amd.layer_norm_bwd(grads[0], x, weight, bias, stats, threshold, seed, seed_tensor, offset))
    gx = next(g)
    gw = next(g) if weight is not None else None
    gb = next(g) if bias is not None else None
    return gx, gw, gb, None, None, None, None, None


layer_norm_fwd.register_autograd(_norm_backward, setup_context=_norm_setup)


def layer_norm(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, eps: float = 1e-5,
               dropout_p: float = 0.0, seed=None, offset: int = 0) -> Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis, in x's type; with dropout_p > 0 the
    result of `dropout(layer_norm(x, ...), dropout_p, seed, offset)` without the pass over memory (and
    with one rounding).

    weight, bias [D] (either may be None) in x's type or fp32; other types are converted to fp32.  Rows
    that are dense and evenly spaced are read where they are."""
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"x must have a last axis of one element or more; got {tuple(x.shape)}")
    if x.dtype not in _DTYPES:
        _dtype_of(x, "x")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            if t.dim() != 1 or t.shape[0] != x.shape[-1]:
                raise ValueError(f"{name} must be [{x.shape[-1]}]; got {tuple(t.shape)}")
            if not t.is_floating_point():
                raise TypeError(f"{name} must be a floating-point tensor; got {t.dtype}")
    if (weight is not None and weight.dtype != x.dtype) or (bias is not None and bias.dtype != x.dtype):
        weight = weight if weight is None else weight.to(torch.float32)
        bias = bias if bias is None else bias.to(torch.float32)
    eps = float(eps)
    if not 0.0 <= eps < math.inf:
        raise ValueError(f"eps must be finite and not negative; got {eps}")
    threshold = dropout_threshold(dropout_p) if dropout_p else 0
    number, seed_tensor = 0, None
    if threshold:
        number, seed_tensor, offset = _seed(seed, offset, x)
    else:
        offset = 0
    if torch.compiler.is_compiling():
        return torch.ops.igs_amd.layer_norm_fwd(x, weight, bias, eps, threshold, number, seed_tensor, offset)[0]
    _on_gpu(x, weight, bias)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, eps, threshold, number, seed_tensor, offset)
    return _norm_fwd(x, weight, bias, eps, threshold, number, seed_tensor, offset, False)[0]


def naive_layer_norm(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, eps: float = 1e-5,
                     dropout_p: float = 0.0, seed=None, offset: int = 0) -> Tensor:
    """Plain torch expression of `layer_norm` (any device, differentiable through autograd)."""
    c = x - x.mean(-1, keepdim=True)
    y = c / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight
    if bias is not None:
        y = y + bias
    return naive_dropout(y, dropout_p, seed, offset) if dropout_p else y


# --------------------------------------------------------------------------------------
# dropout
# --------------------------------------------------------------------------------------
def _dropout(x: Tensor, threshold: int, seed: int, seed_tensor: Optional[Tensor], offset: int) -> Tensor:
    if not x.is_contiguous():
        x = x.contiguous()
    dtype, dev = x.dtype, x.device
    with _on(dev):
        y = torch.empty(x.shape, dtype=dtype, device=dev)
        rc = _lib.load().igs_dropout(x.data_ptr(), _DTYPES[dtype], x.numel(), threshold, seed,
                                     None if seed_tensor is None else seed_tensor.data_ptr(), offset, y.data_ptr(),
                                     _stream(dev))
    if rc:
        _lib.check(rc, "igs_dropout")
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, threshold, seed, seed_tensor, offset):
        ctx.save_for_backward(seed_tensor)
        ctx.args = (threshold, seed, offset)
        return _dropout(x, threshold, seed, seed_tensor, offset)

    @staticmethod
    @_once
    def backward(ctx, grad):
        threshold, seed, offset = ctx.args
        return _dropout(grad, threshold, seed, ctx.saved_tensors[0], offset), None, None, None, None


@torch.library.custom_op("igs_amd::dropout", mutates_args=(), device_types="cuda")
def dropout_op(x: Tensor, threshold: int, seed: int, seed_tensor: Optional[Tensor], offset: int) -> Tensor:
    return _dropout(x, threshold, seed, seed_tensor, offset)


@dropout_op.register_fake
def _(x, threshold, seed, seed_tensor, offset):
    return x.new_empty(x.shape)


def _dropout_setup(ctx, inputs, output):
    _, threshold, seed, seed_tensor, offset = inputs
    ctx.save_for_backward(seed_tensor)
    ctx.args = (threshold, seed, offset)


def _dropout_backward(ctx, grad):
    threshold, seed, offset = ctx.args
    return torch.ops.igs_amd.dropout(grad, threshold, seed, ctx.saved_tensors[0], offset), None, None, None, None


dropout_op.register_autograd(_dropout_backward, setup_context=_dropout_setup)


def dropout(x: Tensor, p: float, seed, offset: int = 0) -> Tensor:
    """Each element is 0 with probability p and x / (1 - p) otherwise (p in steps of 2^-16).

    The mask is a function of (seed, offset, linear index) alone: it is computed where it is used, in the
    forward and again in the backward, and never stored.  seed: an int in [0, 2^63), or an int64 tensor of
    one element on the device, read when the kernel runs: change it between replays of a captured graph
    (and not between a forward and its backward).  Calls of one step that must differ take different
    offsets.  A dropped element is 0 also where x is NaN or infinite."""
    if x.dtype not in _DTYPES:
        _dtype_of(x, "x")
    threshold = dropout_threshold(p)
    if threshold == 0:
        return x
    number, seed_tensor, offset = _seed(seed, offset, x)
    if torch.compiler.is_compiling():
        return torch.ops.igs_amd.dropout(x, threshold, number, seed_tensor, offset)
    _on_gpu(x)
    if x.requires_grad and torch.is_grad_enabled():
        return _Dropout.apply(x, threshold, number, seed_tensor, offset)
    return _dropout(x, threshold, number, seed_tensor, offset)


def _mul32(a: int, b: Tensor) -> Tuple[Tensor, Tensor]:
    """(high, low) 32 bits of the product of a 32-bit constant and 32-bit numbers held in int64."""
    low = a * (b & 0xFFFF)
    mid = a * (b >> 16) + (low >> 16)
    return mid >> 16, ((mid & 0xFFFF) << 16) | (low & 0xFFFF)


def dropout_keep_mask(shape, p: float, seed, offset: int = 0, device=None) -> Tensor:
    """The mask `dropout` uses (True: kept), from plain integer arithmetic on any device."""
    threshold = dropout_threshold(p)
    if isinstance(seed, Tensor):
        device = seed.device if device is None else device
        seed = seed.reshape(()).to(device)
    count = math.prod(shape)
    block = torch.arange((count + 7) // 8, dtype=torch.int64, device=device)
    c = [block & 0xFFFFFFFF, block >> 32, torch.full_like(block, offset & 0xFFFFFFFF),
         torch.full_like(block, offset >> 32)]
    k0, k1 = seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF
    for _ in range(7):
        (h0, l0), (h1, l1) = _mul32(0xD2511F53, c[0]), _mul32(0xCD9E8D57, c[2])
        c = [h1 ^ c[1] ^ k0, l1, h0 ^ c[3] ^ k1, l0]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    halves = torch.stack([h for w in c for h in (w & 0xFFFF, w >> 16)], dim=1)
    return (halves >= threshold).reshape(-1)[:count].reshape(shape)


def naive_dropout(x: Tensor, p: float, seed, offset: int = 0) -> Tensor:
    """Plain torch expression of `dropout` (any device, differentiable through autograd)."""
    threshold = dropout_threshold(p)
    if threshold == 0:
        return x
    keep = dropout_keep_mask(x.shape, p, seed, offset, x.device)
    return torch.where(keep, x * (65536 / (65536 - threshold) if threshold < 65536 else 0.0), torch.zeros_like(x))
