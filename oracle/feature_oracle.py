"""CPU restatement of the feature operators in 64 bits (TEST INFRASTRUCTURE ONLY): embedding lookup and
its dense gradient, layer norm forward and backward, dropout from the counter-based generator.  Never
imported by the product package.

Pins (tests/test_oracle_feature.py): Philox4x32 against its authors' published known answers (seven
and ten rounds), the gradients against differences, the mask's rate.
"""
from __future__ import annotations

import math

import numpy as np
import torch

F64 = torch.float64


def philox4x32(counter, key, rounds):
    """One block with Python integers: counter (4 words), key (2 words) -> 4 words.  Salmon, Moraes,
    Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3" (2011)."""
    c, k = list(counter), list(key)
    for _ in range(rounds):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def dropout_numbers(count, seed, offset, first=0):
    """16-bit numbers of the elements first .. first + count - 1 (first a multiple of 8)."""
    assert first % 8 == 0
    blocks = np.arange(first // 8, first // 8 + -(-count // 8), dtype=np.uint64)
    m, h = np.uint64(0xFFFFFFFF), np.uint64(32)
    c = [blocks & m, blocks >> h, np.full_like(blocks, offset % 2 ** 32), np.full_like(blocks, offset // 2 ** 32)]
    k = [seed % 2 ** 32, seed // 2 ** 32]
    for _ in range(7):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> h) ^ c[1] ^ np.uint64(k[0]), b & m, (a >> h) ^ c[3] ^ np.uint64(k[1]), a & m]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    out = np.empty((len(blocks), 8), dtype=np.int64)
    for j in range(8):
        out[:, j] = (c[j // 2] >> np.uint64(16 * (j % 2))) & np.uint64(0xFFFF)
    return torch.from_numpy(out.reshape(-1)[:count])


def dropout_factors(shape, p, seed, offset=0):
    """What each element is multiplied by: 0 or 65536 / (65536 - t), t = round(65536 p)."""
    t = math.floor(p * 65536 + 0.5)
    keep = dropout_numbers(math.prod(shape), seed, offset).reshape(shape) >= t
    return keep.to(F64) * (65536.0 / (65536 - t) if t < 65536 else 0.0)


def embedding(tokens, weight, scale=1.0):
    """scale * weight[t]; NaN rows for tokens outside the table."""
    w = weight.to(F64)
    ok = (tokens >= 0) & (tokens < w.shape[0])
    out = w[torch.where(ok, tokens, torch.zeros_like(tokens)).long()] * scale
    return torch.where(ok[..., None], out, torch.full_like(out, float("nan")))


def embedding_grad(tokens, grad, vocab, scale=1.0, padding_idx=None):
    """(gradient [V, D], sum of magnitudes of the terms of each element)."""
    D = grad.shape[-1]
    t, g = tokens.reshape(-1).long(), grad.reshape(-1, D).to(F64)
    ok = (t >= 0) & (t < vocab)
    if padding_idx is not None:
        ok &= t != padding_idx % vocab
    out, mag = torch.zeros(vocab, D, dtype=F64), torch.zeros(vocab, D, dtype=F64)
    out.index_add_(0, t[ok], g[ok])
    mag.index_add_(0, t[ok], g[ok].abs())
    return out * scale, mag * abs(scale)


def layer_norm(x, weight=None, bias=None, eps=1e-5, factors=None):
    """(y, mean, rstd)"""
    x = x.to(F64)
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    y = (x - mean) * rstd
    if weight is not None:
        y = y * weight.to(F64)
    if bias is not None:
        y = y + bias.to(F64)
    return (y if factors is None else torch.where(factors == 0, torch.zeros_like(y), y * factors)), mean, rstd


def layer_norm_grad(grad, x, weight=None, eps=1e-5, factors=None):
    """(dx, dweight, dbias) by the closed form."""
    x, d = x.to(F64), grad.to(F64)
    if factors is not None:
        d = torch.where(factors == 0, torch.zeros_like(d), d * factors)
    _, mean, rstd = layer_norm(x, eps=eps)
    h = (x - mean) * rstd
    g = d if weight is None else d * weight.to(F64)
    dx = rstd * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    D = x.shape[-1]
    return dx, (d * h).reshape(-1, D).sum(0), d.reshape(-1, D).sum(0)
