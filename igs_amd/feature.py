"""Operators in front of the Gaussian head: embedding lookup, layer norm and dropout on the HIP library.

The reference's module takes its `feature` [B, F, D] as given (src/igs/gs2d.py:611-635).  These are the
operators that make such a feature out of token ids or of a trunk's output, forward and backward:

  embedding_lookup(tokens, weight, scale, padding_idx)      scale * weight[tokens], dense gradient
  layer_norm(x, weight, bias, eps, dropout_p, seed, offset) norm over the last axis, dropout of its result
  dropout(x, p, seed, offset)                               counter-based mask, never stored

`GaussianSplatting2D` calls them when it is built with `num_embeddings=`, `feature_norm=` or
`feature_dropout=`.  fp32, fp16 and bf16; sums and norms are held in fp32 and every result is rounded
once; gradients of weights are summed in a fixed order (bit-reproducible).  Eager callers go through
native autograd nodes (csrc/igs_torch.cpp) around the C ABI; under `torch.compile`, `torch.export`,
`torch.jit.trace`, `make_fx` and other dispatch modes the same library calls are registered operators
(`igs_amd::embedding_fwd` and its like).  There is no CPU path: tensors must live on the GPU.  The
`naive_*` functions are the plain torch expressions (any device), what the module's `fused=False`
debug path uses.
"""
from __future__ import annotations

import math
from typing import List, Optional, Tuple

import torch

from . import _lib

Tensor = torch.Tensor

_SEED_END = 1 << 63


# --------------------------------------------------------------------------------------
# arguments
# --------------------------------------------------------------------------------------
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
    if type(seed) is int and type(offset) is int:
        if not (0 <= seed < _SEED_END and 0 <= offset < _SEED_END):
            raise ValueError("seed and offset must be in [0, 2^63)")
        return seed, None, offset
    if not isinstance(offset, (int, torch.SymInt)) or isinstance(offset, bool):
        raise TypeError(f"offset must be an int; got {type(offset).__name__}")
    if type(offset) is int and not 0 <= offset < _SEED_END:
        raise ValueError("seed and offset must be in [0, 2^63)")
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
    return seed, None, offset


_torch_binding = None


def _native():
    """The binding's module, on the library that _lib has loaded; raises if either is missing."""
    global _torch_binding
    if _torch_binding is None:
        lib = _lib.load()
        try:
            from . import _igs_torch
        except ImportError as e:
            raise _lib.IGSLibraryError(f"igs_amd/_igs_torch.so cannot be loaded ({e}): build it first "
                                       "(python -m igs_amd.build)") from e
        _igs_torch.bind(lib._handle)
        _torch_binding = _igs_torch
    return _torch_binding


# --------------------------------------------------------------------------------------
# embedding lookup
# --------------------------------------------------------------------------------------
@torch.library.custom_op("igs_amd::embedding_fwd", mutates_args=(), device_types="cuda")
def embedding_fwd(tokens: Tensor, weight: Tensor, scale: float, padding_idx: int) -> Tensor:
    return _native().embedding_fwd(tokens, weight, scale)


@embedding_fwd.register_fake
def _(tokens, weight, scale, padding_idx):
    return weight.new_empty((*tokens.shape, weight.shape[1]))


@torch.library.custom_op("igs_amd::embedding_bwd", mutates_args=(), device_types="cuda")
def embedding_bwd(grad: Tensor, tokens: Tensor, vocab: int, scale: float, padding_idx: int) -> Tensor:
    return _native().embedding_bwd(grad, tokens, vocab, scale, padding_idx)


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
    if torch.compiler.is_compiling():
        V = weight.shape[0]
        if padding_idx is not None and not -V <= padding_idx < V:
            raise ValueError(f"padding_idx {padding_idx} is outside the table of {V} rows")
        return torch.ops.igs_amd.embedding_fwd(tokens, weight, float(scale), -1 if padding_idx is None else padding_idx % V)
    native = _torch_binding or _native()
    y = native.embedding(tokens, weight, scale, padding_idx)
    if y is None:   # something records the operators
        y = torch.ops.igs_amd.embedding_fwd(tokens, weight, float(scale), native.padding_row(weight, padding_idx))
    return y


def naive_embedding_lookup(tokens: Tensor, weight: Tensor, scale: float = 1.0, padding_idx: Optional[int] = None) -> Tensor:
    """Plain torch expression of `embedding_lookup` (any device, differentiable through autograd)."""
    V = weight.shape[0]
    inside = (tokens >= 0) & (tokens < V)
    rows = weight[torch.where(inside, tokens, 0)]
    if padding_idx is not None:
        rows = torch.where((tokens == padding_idx % V)[..., None], rows.detach(), rows)
    return torch.where(inside[..., None], rows * scale, math.nan)


# --------------------------------------------------------------------------------------
# layer norm (with dropout of its result)
# --------------------------------------------------------------------------------------
@torch.library.custom_op("igs_amd::layer_norm_fwd", mutates_args=(), device_types="cuda")
def layer_norm_fwd(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], eps: float, threshold: int, seed: int,
                   seed_tensor: Optional[Tensor], offset: int) -> List[Tensor]:
    """[y, stats [rows, 2] (mean, 1 / standard deviation)]"""
    return list(_native().layer_norm_fwd(x, weight, bias, eps, threshold, seed, seed_tensor, offset))


@layer_norm_fwd.register_fake
def _(x, weight, bias, eps, threshold, seed, seed_tensor, offset):
    return [x.new_empty(x.shape), x.new_empty((math.prod(x.shape[:-1]), 2), dtype=torch.float32)]


@torch.library.custom_op("igs_amd::layer_norm_bwd", mutates_args=(), device_types="cuda")
def layer_norm_bwd(grad: Tensor, x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], stats: Tensor,
                   threshold: int, seed: int, seed_tensor: Optional[Tensor], offset: int) -> List[Tensor]:
    """[grad_x, grad_weight (if weight), grad_bias (if bias)]"""
    return _native().layer_norm_bwd(grad, x, weight, bias, stats, threshold, seed, seed_tensor, offset)


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
    threshold, number, seed_tensor = 0, 0, None
    if dropout_p:
        threshold = dropout_threshold(dropout_p)
        if threshold:
            number, seed_tensor, offset = _seed(seed, offset, x)
    if not threshold:
        offset = 0
    if not torch.compiler.is_compiling():
        y = (_torch_binding or _native()).layer_norm(x, weight, bias, eps, threshold, number, seed_tensor, offset)
        if y is not None:   # else something records the operators
            return y
    if any(t is not None and t.dtype != x.dtype for t in (weight, bias)):
        weight = weight if weight is None else weight.to(torch.float32)
        bias = bias if bias is None else bias.to(torch.float32)
    return torch.ops.igs_amd.layer_norm_fwd(x, weight, bias, float(eps), threshold, number, seed_tensor, offset)[0]


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
@torch.library.custom_op("igs_amd::dropout", mutates_args=(), device_types="cuda")
def dropout_op(x: Tensor, threshold: int, seed: int, seed_tensor: Optional[Tensor], offset: int) -> Tensor:
    return _native().dropout_plain(x, threshold, seed, seed_tensor, offset)


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
    offsets.  A dropped element is 0 also where x is NaN or infinite.  Where nothing can be dropped
    (p < 2^-17) the result is x itself, as with torch's dropout, and not a copy."""
    threshold = dropout_threshold(p)
    if threshold == 0:
        return x
    number, seed_tensor, offset = _seed(seed, offset, x)
    if not torch.compiler.is_compiling():
        y = (_torch_binding or _native()).dropout(x, threshold, number, seed_tensor, offset)
        if y is not None:   # else something records the operators
            return y
    return torch.ops.igs_amd.dropout(x, threshold, number, seed_tensor, offset)


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
