"""Pins of the feature operators' oracle (oracle/feature_oracle.py) and of the plain torch expressions, on the CPU."""
import math

import pytest
import torch

from oracle import feature_oracle as F

F64 = torch.float64


def test_philox_known_answers():
    """The authors' published known answers of Philox4x32 (ten rounds) and of its seven-round form."""
    ones = 0xFFFFFFFF
    assert F.philox4x32([0] * 4, [0] * 2, 10) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert F.philox4x32([ones] * 4, [ones] * 2, 10) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert F.philox4x32([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0], 10) == \
        [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]
    assert F.philox4x32([0] * 4, [0] * 2, 7) == [0x5F6FB709, 0x0D893F64, 0x4F121F81, 0x4F730A48]
    assert F.philox4x32([ones] * 4, [ones] * 2, 7) == [0x5207DDC2, 0x45165E59, 0x4D8EE751, 0x8C52F662]


@pytest.mark.parametrize("seed,offset,first", [(0, 0, 0), (123456789012345, 77, 40), (2 ** 63 - 1, 2 ** 40 + 5, 2 ** 36)])
def test_numbers_are_the_blocks_halves(seed, offset, first):
    """Vectorised numbers = halves of the scalar blocks, low half first, eight per block."""
    u = F.dropout_numbers(21, seed, offset, first)
    for i in range(21):
        b = first // 8 + i // 8
        w = F.philox4x32([b % 2 ** 32, b >> 32, offset % 2 ** 32, offset >> 32], [seed % 2 ** 32, seed >> 32], 7)
        assert int(u[i]) == (w[(i % 8) // 2] >> (16 * (i % 2))) & 0xFFFF


@pytest.mark.parametrize("p", [0.0, 1e-6, 0.1, 0.5, 0.999, 1.0])
def test_mask_rate_and_plain_mask(p):
    """The plain expression's mask is the oracle's, and its rate is p within five standard deviations."""
    import igs_amd

    n = 100003
    keep = igs_amd.dropout_keep_mask((n,), p, 4242, 9)
    f = F.dropout_factors((n,), p, 4242, 9)
    q = round(p * 65536) / 65536
    if q < 1:
        assert torch.equal(keep, f != 0)
        assert bool((f[f != 0] == 1 / (1 - q)).all())
    else:
        assert not keep.any() and not f.any()
    assert abs(float((~keep).double().mean()) - q) <= 5 * math.sqrt(q * (1 - q) / n) + 1e-12
    # a seed tensor is the same number
    assert torch.equal(keep, igs_amd.dropout_keep_mask((n,), p, torch.tensor([4242]), 9))


def test_layer_norm_gradient_against_differences_and_autograd():
    import igs_amd

    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 11, generator=g, dtype=F64)
    w, b, up = torch.randn(11, generator=g, dtype=F64), torch.randn(11, generator=g, dtype=F64), torch.randn(5, 11, generator=g, dtype=F64)
    fac = F.dropout_factors((5, 11), 0.3, 5, 2)
    dx, dw, db = F.layer_norm_grad(up, x, w, 1e-5, fac)
    loss = lambda x_, w_, b_: float((F.layer_norm(x_, w_, b_, 1e-5, fac)[0] * up).sum())
    h = 1e-5
    for grad, t, at in ((dx, x, 0), (dw, w, 1), (db, b, 2)):
        for i in range(0, t.numel(), 3):
            args = []
            for s in (h, -h):
                a = [x.clone(), w.clone(), b.clone()]
                a[at].view(-1)[i] += s
                args.append(loss(*a))
            # rounding 1e-15 |loss| / h and truncation h^2 x third derivative: both below 1e-8 here
            assert abs((args[0] - args[1]) / (2 * h) - float(grad.reshape(-1)[i])) < 1e-7
    lv = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = igs_amd.naive_layer_norm(*lv, 1e-5, 0.3, 5, 2)
    assert torch.allclose(y, F.layer_norm(x, w, b, 1e-5, fac)[0], rtol=1e-12, atol=1e-12)
    for got, want in zip(torch.autograd.grad(y, lv, up), (dx, dw, db)):
        assert torch.allclose(got, want, rtol=1e-10, atol=1e-12)


def test_embedding_gradient_against_autograd_of_the_plain_expression():
    import igs_amd

    g = torch.Generator().manual_seed(2)
    w = torch.randn(7, 3, generator=g, dtype=F64, requires_grad=True)
    t = torch.tensor([[0, 6, 6], [2, 0, 6]])
    up = torch.randn(2, 3, 3, generator=g, dtype=F64)
    for pad in (None, 6, -7):
        y = igs_amd.naive_embedding_lookup(t, w, 2.5, pad)
        assert torch.equal(y.detach(), F.embedding(t, w.detach(), 2.5))
        (got,) = torch.autograd.grad(y, w, up)
        want, mag = F.embedding_grad(t, up, 7, 2.5, pad)
        assert torch.allclose(got, want, rtol=1e-13, atol=1e-13) and bool((mag >= want.abs() - 1e-12).all())
    assert bool(F.embedding(torch.tensor([7, -1, 1]), w.detach()).isnan().any(-1).tolist() == [True, True, False])
