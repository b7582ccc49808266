"""Feature operators on the GPU (through the C ABI) against the fp64 oracle.

Tolerances are bounds of the arithmetic, per element.  u = 2^-24 is half a step of fp32, uT half a step of the tensor's
type (finfo.eps / 2), sub half of the type's least subnormal.  A kernel's sum of n terms per row adds at most n / 64 + 16
of them in one chain of additions (64 lanes or more share a row of more than 512 elements; narrower rows have 8 elements
or fewer per lane; the rest is a tree), so its error is at most gamma * sum |terms| with gamma = (n / 64 + 16) u.  The
sums over rows and over equal tokens are taken with the crudest bound, n u, whatever their order."""
import math

import pytest
import torch

from oracle import feature_oracle as F

pytestmark = pytest.mark.gpu
F64 = torch.float64
U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
ids = lambda v: str(v).replace("torch.", "")


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


@pytest.fixture(scope="module")
def igs():
    import igs_amd

    return igs_amd


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def sub(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def rounded(ref, dtype):
    """Bound of the final rounding of a value near ref."""
    return ref.abs() * half_step(dtype) * 1.01 + sub(dtype)


def check(got, ref, tol, what):
    got = got.detach().to(F64).cpu()
    assert got.shape == ref.shape, what
    bad = ~((got - ref).abs() <= tol) & ~(got.isnan() & ref.isnan())
    assert not bool(bad.any()), (what, int(bad.sum()), float(((got - ref).abs() / tol).nan_to_num(0).max()))


def normal(shape, seed, dtype, mean=0.0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g, dtype=F64) * std + mean).to(dtype)


def some_tokens(n, vocab, seed, kind, dtype=torch.int64):
    g = torch.Generator().manual_seed(seed)
    u = torch.rand(n, generator=g, dtype=F64)
    if kind == "skew":
        t = torch.exp(u * math.log(vocab + 1)) - 1
    elif kind == "one":
        t = torch.full_like(u, vocab // 2)
    elif kind == "ends":
        t = torch.where(u < 0.5, torch.zeros_like(u), torch.full_like(u, vocab - 1))
    elif kind == "sorted":
        t = (torch.arange(n, dtype=F64) * vocab / max(n, 1))
    else:
        t = u * vocab
    return t.long().clamp_(0, vocab - 1).to(dtype)


# ---------------------------------------------------------------------------------- embedding lookup
def lookup_tolerance(ref, dtype):
    return ref.abs() * 2 * U + rounded(ref, dtype)       # the scale's and the product's roundings


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("n,vocab,D", [(1, 1, 1), (1, 8192, 1024), (3, 7, 5), (77, 50, 8), (64, 5, 64), (130, 1000, 333),
                                       (1000, 300, 72), (9, 11, 4100), (5, 3, 2049), (257, 2, 16), (4099, 999, 12)])
def test_lookup(igs, dev, dtype, n, vocab, D):
    w, t = normal((vocab, D), n + D, dtype), some_tokens(n, vocab, n, "uniform")
    for scale in (1.0, math.sqrt(D) + 0.1):
        got = igs.embedding_lookup(t.to(dev), w.to(dev), scale)
        assert got.dtype == dtype
        ref = F.embedding(t, w, scale)
        check(got, ref, lookup_tolerance(ref, dtype), "lookup")
    assert torch.equal(igs.embedding_lookup(t.to(dev), w.to(dev)).cpu(), w[t])            # scale 1 is exact
    assert torch.equal(igs.embedding_lookup(t.to(dev, torch.int32), w.to(dev)).cpu(), w[t])


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
def test_lookup_of_views(igs, dev, dtype):
    """Tables and tokens as strided or misaligned views; tokens of several axes; none at all."""
    base = normal((40, 50), 1, dtype).to(dev)
    t = some_tokens(60, 20, 2, "uniform").view(3, 20).to(dev)
    flat = normal((40 * 50 + 3,), 3, dtype).to(dev)
    for w in (base[:20], base[10:30, :48], base[::2, 1:34], base[:, :20].t()[:20], flat[1:1001].view(20, 50), flat[3:803].view(20, 40),
              base[:1].expand(20, 50)):
        for tok in (t, t.t(), t[:, ::3], t[1], t[:, :0]):
            got = igs.embedding_lookup(tok, w, 1.0)
            assert torch.equal(got, w[tok]) and got.is_contiguous()
    tok = torch.cat([t.view(-1).int(), t.view(-1).int()])[1:8]     # 4-byte aligned only
    assert torch.equal(igs.embedding_lookup(tok, base[:20]), base[:20][tok.long()])


def test_lookup_out_of_range_tokens(igs, dev):
    w = normal((6, 10), 1, torch.float32)
    t = torch.tensor([0, 6, -1, 5, 2 ** 40, -2 ** 63, 3])
    wd = w.to(dev).requires_grad_(True)
    y = igs.embedding_lookup(t.to(dev), wd)
    check(y, F.embedding(t, w), 1e-30, "NaN rows")
    up = normal((7, 10), 2, torch.float32)
    (g,) = torch.autograd.grad(y, wd, up.to(dev))
    want, _ = F.embedding_grad(t, up, 6)
    assert torch.equal(g.cpu().double(), want)


GRADS = [(1, 1, 1), (1, 9, 7), (2, 3, 64), (63, 40, 8), (64, 4, 1024), (65, 100, 33), (300, 2, 16), (1024, 8192, 40), (1025, 33, 520),
         (2048, 5, 9), (4097, 70000, 8), (4096, 300, 100), (20000, 257, 24), (8193, 1, 65), (16385, 200003, 4), (70001, 1000, 3),
         (5000, 64, 2056)]


def gradient_tolerance(ref, mag, counts, dtype):
    # the sum's additions, the scale's and the product's roundings
    return mag * U * (counts[:, None] + 3) * 1.01 + rounded(ref, dtype)


@pytest.mark.parametrize("kind", ["uniform", "skew", "one", "ends", "sorted"])
@pytest.mark.parametrize("n,vocab,D", GRADS)
def test_lookup_gradient(igs, dev, n, vocab, D, kind):
    for dtype in DTYPES if (n + D) % 2 or n < 100 else DTYPES[:1]:
        t, up = some_tokens(n, vocab, n + 1, kind), normal((n, D), D, dtype)
        counts = torch.bincount(t, minlength=vocab).to(F64)
        w = torch.zeros(vocab, D, dtype=dtype, device=dev, requires_grad=True)
        for scale, pad in ((1.0, None), (0.37, vocab // 2)):
            y = igs.embedding_lookup(t.to(dev), w, scale, pad)
            (g,) = torch.autograd.grad(y, w, up.to(dev))
            assert g.dtype == dtype
            ref, mag = F.embedding_grad(t, up, vocab, scale, pad)
            check(g, ref, gradient_tolerance(ref, mag, counts, dtype), ("gradient", dtype, scale, pad))
        y = igs.embedding_lookup(t.to(dev, torch.int32), w, scale, pad)
        (again,) = torch.autograd.grad(y, w, up.to(dev))
        assert torch.equal(g, again)                    # bit for bit, whatever the width of the ids


def test_lookup_gradient_many_tokens(igs, dev):
    """More tokens than one pass of any part of the sort holds; a run of equal tokens longer than that."""
    n, vocab, D = 1 << 20, 100000, 2
    g = torch.Generator().manual_seed(5)
    t = torch.randint(0, vocab, (n,), generator=g)
    t[::3] = 77777
    up = torch.randint(-3, 4, (n, D), generator=g).float()       # whole numbers: the fp32 sums are exact below 2^24
    w = torch.zeros(vocab, D, device=dev, requires_grad=True)
    (got,) = torch.autograd.grad(igs.embedding_lookup(t.to(dev), w), w, up.to(dev))
    want, _ = F.embedding_grad(t, up, vocab)
    assert torch.equal(got.cpu().double(), want)


def test_lookup_gradient_of_no_tokens_and_of_an_expanded_upstream(igs, dev):
    w = torch.randn(9, 12, device=dev, requires_grad=True)
    y = igs.embedding_lookup(torch.empty(0, 4, dtype=torch.int64, device=dev), w)
    assert y.shape == (0, 4, 12)
    assert not torch.autograd.grad(y.sum(), w)[0].any()
    t = torch.tensor([1, 1, 8], device=dev)
    (g,) = torch.autograd.grad(igs.embedding_lookup(t, w, 2.0).sum(), w)      # stride-0 upstream gradient
    assert g[:, 0].tolist() == [0, 4, 0, 0, 0, 0, 0, 0, 2] and bool((g == g[:, :1]).all())


# ---------------------------------------------------------------------------------- layer norm
def gamma(n):
    return (n / 64 + 16) * U


def norm_bounds(x, eps):
    """(h, its error bound, rstd, relative bound of rstd) from rounding alone: the mean is off by at most
    gamma mean|x| =: m, which shifts every deviation by m and the variance by m^2 (a shift is orthogonal to the
    deviations); the variance's own sum is off by gamma, and a handful of single roundings follow."""
    x = x.to(F64)
    D = x.shape[-1]
    _, mean, rstd = F.layer_norm(x, eps=eps)
    h = (x - mean) * rstd
    m = (gamma(D) + 2 * U) * x.abs().mean(-1, keepdim=True)
    rel = 0.5 * (gamma(D) + 4 * U + (m * rstd) ** 2) + 4 * U
    return h, m * rstd * (1 + rel) + h.abs() * (rel + 3 * U), rstd, rel


def norm_tolerance(x, w, b, eps, factors, ref, dtype):
    h, eh, _, _ = norm_bounds(x, eps)
    w = torch.ones(x.shape[-1], dtype=F64) if w is None else w.to(F64)
    t = w.abs() * eh + 2 * U * ((h * w).abs() + (0 if b is None else b.to(F64).abs()))
    if factors is not None:
        t = t * factors + ref.abs() * 2 * U
    return t * 1.01 + rounded(ref, dtype)


def norm_grad_tolerances(up, x, w, eps, factors, refs, dtypes):
    h, eh, rstd, rel = norm_bounds(x, eps)
    D = x.shape[-1]
    d = up.to(F64) if factors is None else torch.where(factors == 0, torch.zeros_like(factors), up.to(F64) * factors)
    g = (d if w is None else d * w.to(F64)).abs()
    mean = lambda v: v.mean(-1, keepdim=True)
    s0, s1 = mean(g), mean(g * h.abs())
    e0 = (gamma(D) + 5 * U) * s0
    e1 = (gamma(D) + 6 * U) * s1 + mean(g * eh)
    tx = rstd * (4 * U * g + e0 + h.abs() * e1 + eh * (s1 + e1) + 5 * U * (g + s0 + h.abs() * s1))
    tx = (tx + (rel + 2 * U) * refs[0].abs()) * 1.01 + rounded(refs[0], dtypes[0])
    R = x.numel() // D
    flat = lambda v: v.reshape(-1, D).sum(0)
    chain = (R + 8) * U
    tw = (flat(d.abs() * eh) * (1 + chain) + chain * flat((d * h).abs())) * 1.01 + rounded(refs[1], dtypes[1])
    tb = chain * flat(d.abs()) * 1.01 + rounded(refs[2], dtypes[1])
    return tx, tw, tb


NORMS = [(1, 1), (5, 2), (3, 7), (2, 8), (33, 9), (9, 64), (70, 65), (17, 100), (4, 256), (257, 333), (3, 512), (5, 513), (1, 1024), (300, 1024),
         (6, 1032), (7, 2047), (2, 2048), (3, 4104), (2, 5001), (3, 8192), (2, 8205), (2, 16384), (2, 16390), (1, 33000), (1, 70001)]


@pytest.mark.parametrize("p", [0.0, 0.3])
@pytest.mark.parametrize("dtype,wdtype", [(torch.float32,) * 2, (torch.bfloat16,) * 2, (torch.float16,) * 2, (torch.bfloat16, torch.float32),
                                          (torch.float16, torch.float32)], ids=ids)
@pytest.mark.parametrize("R,D", NORMS)
def test_layer_norm(igs, dev, dtype, wdtype, R, D, p):
    x, up = normal((R, D), R + D, dtype, 0.4, 1.7), normal((R, D), D, dtype)
    w, b = normal((D,), 3, wdtype, 1.0, 0.3), normal((D,), 4, wdtype)
    factors = F.dropout_factors((R, D), p, 11, 3) if p else None
    kw = dict(eps=1e-5, dropout_p=p, seed=11, offset=3) if p else dict(eps=1e-5)
    ref, _, _ = F.layer_norm(x, w, b, 1e-5, factors)
    lv = [v.to(dev).requires_grad_(True) for v in (x, w, b)]
    y = igs.layer_norm(*lv, **kw)
    assert y.dtype == dtype
    check(y, ref, norm_tolerance(x, w, b, 1e-5, factors, ref, dtype), "y")
    with torch.no_grad():
        assert torch.equal(igs.layer_norm(*lv, **kw), y)
    grads = torch.autograd.grad(y, lv, up.to(dev), retain_graph=True)
    assert [v.dtype for v in grads] == [dtype, wdtype, wdtype]
    refs = F.layer_norm_grad(up, x, w, 1e-5, factors)
    for name, got, r, tol in zip(("dx", "dw", "db"), grads, refs, norm_grad_tolerances(up, x, w, 1e-5, factors, refs, (dtype, wdtype))):
        check(got, r, tol, name)
    again = torch.autograd.grad(y, lv, up.to(dev))
    assert all(torch.equal(a, c) for a, c in zip(grads, again))          # bit-reproducible
    # any subset of the gradients alone is the same
    for k in range(3):
        part = [v.detach().requires_grad_(i == k) for i, v in enumerate(lv)]
        (one,) = torch.autograd.grad(igs.layer_norm(*part, **kw), part[k], up.to(dev))
        assert torch.equal(one, grads[k])


@pytest.mark.parametrize("R,D", [(5000, 24), (3001, 130), (2053, 1024), (20000, 8), (701, 1500), (1100, 2050), (1030, 5000), (150, 20003)])
def test_layer_norm_weight_gradient_over_many_rows(igs, dev, R, D):
    for dtype in DTYPES:
        x, up = normal((R, D), R, dtype, 0.4, 1.7), normal((R, D), D, dtype)
        w, b = normal((D,), 3, torch.float32, 1.0, 0.3), normal((D,), 4, torch.float32)
        lv = [v.to(dev).requires_grad_(True) for v in (x, w, b)]
        grads = torch.autograd.grad(igs.layer_norm(*lv), lv, up.to(dev))
        refs = F.layer_norm_grad(up, x, w)
        for name, got, r, tol in zip(("dx", "dw", "db"), grads, refs, norm_grad_tolerances(up, x, w, 1e-5, None, refs, (dtype, torch.float32))):
            check(got, r, tol, name)


def test_layer_norm_optional_weights_and_types(igs, dev):
    x, up = normal((7, 40), 1, torch.float32), normal((7, 40), 2, torch.float32)
    w, b = normal((40,), 3, torch.float32, 1.0, 0.3), normal((40,), 4, torch.float32)
    for ww, bb in ((None, None), (w, None), (None, b)):
        lv = [x.to(dev).requires_grad_(True)] + [None if v is None else v.to(dev).requires_grad_(True) for v in (ww, bb)]
        y = igs.layer_norm(*lv)
        ref = F.layer_norm(x, ww, bb)[0]
        check(y, ref, norm_tolerance(x, ww, bb, 1e-5, None, ref, torch.float32), "y")
        refs = F.layer_norm_grad(up, x, ww)
        tols = norm_grad_tolerances(up, x, ww, 1e-5, None, refs, (torch.float32,) * 2)
        got = torch.autograd.grad(y, [v for v in lv if v is not None], up.to(dev))
        keep = [i for i, v in enumerate(lv) if v is not None]
        for i, v in zip(keep, got):
            check(v, refs[i], tols[i], i)
    # weights of a third type are converted to fp32, and their gradients back
    w16 = w.to(torch.bfloat16).to(dev).requires_grad_(True)
    y = igs.layer_norm(x.to(dev), w16)
    ref = F.layer_norm(x, w16.detach().cpu())[0]
    check(y, ref, norm_tolerance(x, w16.detach().cpu(), None, 1e-5, None, ref, torch.float32), "converted")
    assert torch.autograd.grad(y, w16, up.to(dev))[0].dtype == torch.bfloat16
    wt = w.to(dev)[None].expand(2, 40).t().reshape(-1)[::2]             # a strided weight
    assert torch.equal(igs.layer_norm(x.to(dev), wt), igs.layer_norm(x.to(dev), w.to(dev)))


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
def test_layer_norm_of_views(igs, dev, dtype):
    """Rows read in place, copied, broadcast or misaligned give what a contiguous copy gives."""
    base = normal((6, 10, 48), 1, dtype).to(dev)
    flat = normal((6 * 48 + 5,), 2, dtype).to(dev)
    views = (base[..., :40], base[:, ::2], base[..., 3:36], base.transpose(0, 1), base[..., ::2], flat[1:289].view(6, 48),
             flat[5:].view(6, 48), base[:1].expand(4, 10, 48), base[:, :1].expand(6, 3, 48), base[2, 3], base[:, :0])
    for v in views:
        D = v.shape[-1]
        w, b = normal((D,), 3, dtype, 1.0, 0.3).to(dev), normal((D,), 4, dtype).to(dev)
        up = normal(tuple(v.shape), 5, dtype).to(dev)
        res = []
        for x in (v, v.clone(memory_format=torch.contiguous_format)):
            x = x.detach().requires_grad_(True)
            ws = [w.clone().requires_grad_(True), b.clone().requires_grad_(True)]
            y = igs.layer_norm(x, *ws, dropout_p=0.2, seed=5)
            res.append((y, *torch.autograd.grad(y, [x, *ws], up)))
        for a, c in zip(*res):
            assert a.shape == c.shape
            if v.data_ptr() % 16 == 0 and v.stride(-1) == 1 and all(s % 8 == 0 for s in v.stride()[:-1]):
                assert torch.equal(a, c)
            else:   # another variant (other order of the sums): two results within the bound of a handful of steps of fp32
                assert torch.allclose(a.float(), c.float(), rtol=2.1 * half_step(dtype) + 1e-5, atol=1e-5)


def test_layer_norm_far_mean_and_constant_rows(igs, dev):
    """A mean far above the deviation, rows without any (0 / sqrt(eps)), and eps = 0."""
    x = torch.cat([normal((4, 777), 1, torch.float32, 3000.0, 1.0), torch.full((2, 777), 5.0)])
    ref = F.layer_norm(x)[0]
    check(igs.layer_norm(x.to(dev)), ref, norm_tolerance(x, None, None, 1e-5, None, ref, torch.float32), "far mean")
    ref = F.layer_norm(x[:4], eps=0.0)[0]
    check(igs.layer_norm(x[:4].to(dev), eps=0.0), ref, norm_tolerance(x[:4], None, None, 0.0, None, ref, torch.float32), "eps 0")


def test_layer_norm_non_finite_rows_stay_alone(igs, dev):
    for D in (24, 1024, 3000):
        x = normal((9, D), 1, torch.float32)
        x[2, 3], x[5, D - 1] = float("nan"), float("inf")
        xd = x.to(dev).requires_grad_(True)
        y = igs.layer_norm(xd)
        (g,) = torch.autograd.grad(y, xd, torch.ones_like(y))
        clean = x.clone()
        clean[2, 3], clean[5, D - 1] = 0.0, 0.0
        cd = clean.to(dev).requires_grad_(True)
        yc = igs.layer_norm(cd)
        (gc,) = torch.autograd.grad(yc, cd, torch.ones_like(yc))
        rows = [r for r in range(9) if r not in (2, 5)]
        assert torch.equal(y[rows], yc[rows]) and torch.equal(g[rows], gc[rows])
        assert bool(y[2].isnan().all()) and bool(y[5].isnan().all()) and bool(g[2].isnan().all())


def test_layer_norm_gradient_against_differences(igs, dev):
    """The GPU's gradient along a direction against the difference quotient of the fp64 definition; the quotient's own
    truncation is what it changes by when the step doubles."""
    x, up, v = normal((20, 96), 1, torch.float32), normal((20, 96), 2, torch.float32), normal((20, 96), 3, torch.float32)
    w, b = normal((96,), 4, torch.float32, 1.0, 0.3), normal((96,), 5, torch.float32)
    fac = F.dropout_factors((20, 96), 0.25, 8)
    xd = x.to(dev).requires_grad_(True)
    y = igs.layer_norm(xd, w.to(dev), b.to(dev), dropout_p=0.25, seed=8)
    (g,) = torch.autograd.grad(y, xd, up.to(dev))
    loss = lambda t: float((F.layer_norm(x.to(F64) + t * v.to(F64), w, b, 1e-5, fac)[0] * up.to(F64)).sum())
    q = lambda h: (loss(h) - loss(-h)) / (2 * h)
    refs = F.layer_norm_grad(up, x, w, 1e-5, fac)
    tol = float((norm_grad_tolerances(up, x, w, 1e-5, fac, refs, (torch.float32,) * 2)[0] * v.to(F64).abs()).sum())
    assert abs(float((g.cpu().to(F64) * v.to(F64)).sum()) - q(1e-4)) <= tol + abs(q(1e-4) - q(2e-4)) + 1e-9


# ---------------------------------------------------------------------------------- dropout
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (3, 5), (128, 512), (1000, 333), (1 << 20,)], ids=str)
def test_dropout_is_the_defined_mask(igs, dev, dtype, shape):
    x, up = normal(shape, 1, dtype), normal(shape, 2, dtype)
    for p, seed, offset in ((0.1, 0, 0), (0.5, 2 ** 62 + 12345, 2 ** 33 + 1), (0.99, 7, 5), (1.0, 3, 0)):
        f = F.dropout_factors(shape, p, seed, offset).float()
        xd = x.to(dev).requires_grad_(True)
        y = igs.dropout(xd, p, seed, offset)
        # one fp32 product and one rounding: the same on any machine
        assert torch.equal(y.cpu(), torch.where(f == 0, torch.zeros(()), x.float() * f).to(dtype))
        (g,) = torch.autograd.grad(y, xd, up.to(dev))
        assert torch.equal(g.cpu(), torch.where(f == 0, torch.zeros(()), up.float() * f).to(dtype))
        s = torch.tensor([seed], device=dev)
        assert torch.equal(igs.dropout(xd, p, s, offset), y)
        assert torch.equal(igs.naive_dropout(xd.float(), p, s, offset).to(dtype), y) or dtype != torch.float32


def test_dropout_views_and_non_finite_values(igs, dev):
    base = normal((40, 50), 1, torch.float16).to(dev)
    flat = normal((1003,), 2, torch.float16).to(dev)
    for v in (base.t(), base[:, 3:], base[::3], flat[1:], flat[3:900].view(3, 299), base[:1].expand(9, 50), base[:, :0], base[0, 0]):
        assert torch.equal(igs.dropout(v, 0.4, 9), igs.dropout(v.clone(memory_format=torch.contiguous_format), 0.4, 9))
    x = torch.full((4096,), float("nan"), device=dev)
    x[::2] = float("inf")
    y = igs.dropout(x, 0.5, 3)
    keep = igs.dropout_keep_mask((4096,), 0.5, 3, device=dev)
    assert not y[~keep].any() and not bool(y[keep].isfinite().any())
    w = torch.ones(64, device=dev)
    w[5] = float("inf")
    r = normal((64, 64), 3, torch.float32).to(dev)
    y = igs.layer_norm(r, w, dropout_p=0.5, seed=3)
    keep = igs.dropout_keep_mask((64, 64), 0.5, 3, device=dev)
    assert not y[~keep].any() and not bool(y[:, 5][keep[:, 5]].isfinite().any())


def test_fused_dropout_is_the_operator_s_mask(igs, dev):
    for R, D, dtype in ((33, 1024, torch.bfloat16), (40, 77, torch.float32), (9, 4104, torch.float16), (3, 20000, torch.float32)):
        x = normal((R, D), 1, dtype).to(dev)
        w, b = normal((D,), 2, torch.float32, 1.0, 0.2).to(dev), normal((D,), 3, torch.float32, 5.0).to(dev)
        y = igs.layer_norm(x, w, b, dropout_p=0.3, seed=21, offset=4)
        keep = igs.dropout_keep_mask((R, D), 0.3, 21, 4, dev)
        assert torch.equal(y == 0, ~keep)          # the bias keeps what stays away from zero


# ---------------------------------------------------------------------------------- large offsets
def test_offsets_beyond_32_bits(igs, dev):
    """Element indices above 2^32: the last rows of a long gather, a long norm and a long dropout."""
    D, n = 65536, 65536 + 9
    w = torch.randn(11, D, device=dev, dtype=torch.float16)
    t = torch.randint(0, 11, (n,), device=dev)
    y = igs.embedding_lookup(t, w)                              # 4.3e9 elements
    for i in (0, n // 2, n - 1):
        assert torch.equal(y[i], w[t[i]])
    d = igs.dropout(y, 0.3, 5)
    first = (n - 1) * D
    u = F.dropout_numbers(D, 5, 0, first)
    f = (u >= round(0.3 * 65536)).float() * (65536 / (65536 - round(0.3 * 65536)))
    assert torch.equal(d[-1].cpu(), (w[t[-1]].cpu().float() * f).half())
    del d
    z = igs.layer_norm(y)
    one = igs.layer_norm(y[-1:].clone())
    assert torch.equal(z[-1:], one)
    del z, y
    # a table of more than 2^32 elements: its last row, and the gradient's
    V = 65536 + 5
    big = torch.zeros(V, D, device=dev, dtype=torch.float16)
    big[-1] = w[3]
    big[V // 2] = w[4]
    leaf = big.requires_grad_(True)
    y = igs.embedding_lookup(torch.tensor([V - 1, V // 2, V - 1], device=dev), leaf)
    assert torch.equal(y, torch.stack([w[3], w[4], w[3]]))
    (g,) = torch.autograd.grad(y, leaf, torch.ones_like(y))
    assert bool((g[-1] == 2).all()) and bool((g[V // 2] == 1).all()) and float(g[:: 4096].float().sum()) == (D if (V // 2) % 4096 == 0 else 0) + (2 * D if (V - 1) % 4096 == 0 else 0)


def test_tensors_larger_than_the_caches(igs, dev):
    """Tensors that are read and written past the caches give what the cached ones give: the lookup's gradient of whole
    numbers is exact, and a norm's rows do not depend on how many there are."""
    n, V, D = 100003, 700, 1024
    g = torch.Generator(dev).manual_seed(1)
    t = torch.randint(0, V, (n,), generator=g, device=dev)
    up = torch.randint(-1, 2, (n, D), generator=g, device=dev, dtype=torch.int8).to(torch.bfloat16)
    w = torch.randn(V, D, generator=g, device=dev).to(torch.bfloat16).requires_grad_(True)
    y = igs.embedding_lookup(t, w)
    assert torch.equal(y, w.detach()[t])
    (got,) = torch.autograd.grad(y, w, up)
    want = torch.zeros(V, D, device=dev).index_add_(0, t, up.float())     # whole numbers below 2^24: exact in any order
    assert torch.equal(got, want.to(torch.bfloat16))
    x = y.detach().requires_grad_(True)
    z = igs.layer_norm(x, dropout_p=0.25, seed=3)
    (gx,) = torch.autograd.grad(z, x, up)
    for r in (0, 50000, n - 9):
        part = x.detach()[r:r + 9].clone().requires_grad_(True)
        f = igs.layer_norm(part)
        keep = igs.dropout_keep_mask((n * D,), 0.25, 3, device=dev).view(n, D)[r:r + 9]
        # (the masked gradient of the slice is rounded to bf16, 2^-9 of each of the three terms of its rows)
        masked = torch.where(keep, up[r:r + 9].float() * (65536 / (65536 - 16384)), 0.0)
        (gp,) = torch.autograd.grad(f, part, masked.to(torch.bfloat16))
        assert torch.equal(z[r:r + 9] == 0, ~keep | (z[r:r + 9] == 0))
        assert torch.allclose(gx[r:r + 9].float(), gp.float(), rtol=2 ** -7, atol=1e-2 * float(gp.float().abs().max()))
        whole = igs.layer_norm(x.detach())[r:r + 9]
        assert torch.equal(whole, f.detach())


# ---------------------------------------------------------------------------------- together, streams, graphs
def chain(igs, t, w, gw, gb, seed):
    f = igs.embedding_lookup(t, w, 1.5, 0)
    return igs.layer_norm(f, gw, gb, dropout_p=0.2, seed=seed, offset=1)


def test_lookup_norm_dropout_together(igs, dev):
    """Tokens to normalised features and back to the table's gradient, against the composed oracle in fp64; the
    tolerance of the table's gradient is the norm's bound carried through the (linear) sum over tokens."""
    V, D, n = 60, 136, 500
    t = some_tokens(n, V, 1, "skew")
    w, gw, gb = normal((V, D), 1, torch.float32), normal((D,), 2, torch.float32, 1.0, 0.3), normal((D,), 3, torch.float32)
    up = normal((n, D), 4, torch.float32)
    lv = [v.to(dev).requires_grad_(True) for v in (w, gw, gb)]
    y = chain(igs, t.to(dev), *lv, 77)
    f = F.embedding(t, w, 1.5)
    f32 = f.float()                                            # the lookup's own rounding is an input of the norm
    fac = F.dropout_factors((n, D), 0.2, 77, 1)
    ref = F.layer_norm(f32, gw, gb, 1e-5, fac)[0]
    check(y, ref, norm_tolerance(f32, gw, gb, 1e-5, fac, ref, torch.float32), "y")
    got = torch.autograd.grad(y, lv, up.to(dev))
    refs = F.layer_norm_grad(up, f32, gw, 1e-5, fac)
    tols = norm_grad_tolerances(up, f32, gw, 1e-5, fac, refs, (torch.float32,) * 2)
    check(got[1], refs[1], tols[1], "dw")
    check(got[2], refs[2], tols[2], "db")
    want, mag = F.embedding_grad(t, refs[0], V, 1.5, 0)
    carried, _ = F.embedding_grad(t, tols[0], V, 1.5, 0)
    counts = torch.bincount(t, minlength=V).to(F64)
    check(got[0], want, carried + gradient_tolerance(want, mag, counts, torch.float32), "table")


def test_two_streams_at_once(igs, dev):
    """Calls interleaved on two streams do not share workspaces."""
    V, D, n = 3000, 264, 9000
    data = []
    for s in range(2):
        t = some_tokens(n, V, s, "skew").to(dev)
        data.append((t, *[normal(sh, s, torch.float32, m).to(dev) for sh, m in (((V, D), 0.0), ((D,), 1.0), ((D,), 0.0))], normal((n, D), 9 + s, torch.float32).to(dev)))

    def step(t, w, gw, gb, up, seed):
        lv = [v.detach().requires_grad_(True) for v in (w, gw, gb)]
        y = chain(igs, t, *lv, seed)
        return (y.detach(), *torch.autograd.grad(y, lv, up))

    want = [step(*data[s], s) for s in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(3):
        for s in range(2):
            with torch.cuda.stream(streams[s]):
                got[s].append(step(*data[s], s))
    torch.cuda.synchronize()
    for s in range(2):
        for r in got[s]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[s]))


def test_training_step_is_graph_capturable(igs, dev):
    """Forward and backward of the three in one captured graph; each replay reads the seed of its time, and eager work
    runs between the replays."""
    V, D, n = 3000, 264, 5000
    t = some_tokens(n, V, 3, "skew").to(dev)
    w, gw, gb = normal((V, D), 1, torch.float32).to(dev), normal((D,), 2, torch.float32, 1.0).to(dev), normal((D,), 3, torch.float32).to(dev)
    up, seed = normal((n, D), 4, torch.float32).to(dev), torch.zeros(1, dtype=torch.int64, device=dev)

    def step():
        lv = [v.detach().requires_grad_(True) for v in (w, gw, gb)]
        y = igs.dropout(chain(igs, t, *lv, seed), 0.1, seed, 5)
        return (y.detach(), *torch.autograd.grad(y, lv, up))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.cuda.graph(other):                        # a second one: neither may work in the other's buffers
        out2 = step()
    for k in (5, 6, 5, 2 ** 60):
        seed.fill_(k)
        up.add_(0.25)
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        assert all(torch.equal(a, b) for a, b in zip(out2, want))
    assert not torch.equal(igs.dropout(w, 0.5, 1), igs.dropout(w, 0.5, 2))
    assert not torch.equal(igs.dropout(w, 0.5, 1, 0), igs.dropout(w, 0.5, 1, 1))


def test_a_seed_changed_before_the_backward_is_refused(igs, dev):
    seed = torch.tensor([4], device=dev)
    x = torch.randn(100, device=dev, requires_grad=True)
    y = igs.dropout(x, 0.5, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_backward_twice_and_second_derivatives(igs, dev):
    """A second backward without retain_graph and a derivative of the gradient raise; a graph recorded for something else
    does not."""
    x, w, t = torch.randn(5, 8, device=dev), torch.randn(8, device=dev), torch.tensor([1, 2, 2], device=dev)
    table = torch.randn(4, 8, device=dev)
    for f, leaf in ((lambda v: igs.embedding_lookup(t, v), table), (lambda v: igs.layer_norm(v, w), x),
                    (lambda v: igs.layer_norm(x, v, dropout_p=0.2, seed=1), w), (lambda v: igs.dropout(v, 0.5, 1), x)):
        v = leaf.clone().requires_grad_(True)
        y = f(v)
        up = torch.randn_like(y).requires_grad_(True)
        (g,) = torch.autograd.grad(y, v, up, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiate twice"):
            g.sum().backward()
        y = f(v)
        (h,) = torch.autograd.grad(y, v, up.detach())
        assert torch.equal(g.detach(), h)
    y = igs.layer_norm(x.clone().requires_grad_(True), w)
    y.sum().backward()
    with pytest.raises(RuntimeError, match="second time"):
        y.sum().backward()
    with torch.inference_mode():
        assert torch.equal(igs.layer_norm(x, w), igs.layer_norm(x.clone(), w))
    import torch.autograd.forward_ad as fwAD

    with fwAD.dual_level():                              # a tangent would be lost without a word
        dual = fwAD.make_dual(x, torch.ones_like(x))
        for f in (lambda: igs.layer_norm(dual), lambda: igs.dropout(dual, 0.5, 1),
                  lambda: igs.embedding_lookup(t, fwAD.make_dual(table, table))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f()


def test_function_transforms_and_fake_tensors_raise(igs, dev):
    """torch.func's wrappers and fake tensors hold no memory that a kernel could read: refused, never a wrong result."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    x, t, table = torch.randn(5, 8, device=dev), torch.tensor([1, 2, 2], device=dev), torch.randn(4, 8, device=dev)
    for f, leaf in ((lambda v: igs.embedding_lookup(t, v), table), (igs.layer_norm, x), (lambda v: igs.dropout(v, 0.5, 1), x)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.grad(lambda v: f(v).sum())(leaf)
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.vmap(f)(leaf.expand(3, *leaf.shape))
        with FakeTensorMode(allow_non_fake_inputs=True), pytest.raises((RuntimeError, NotImplementedError)):
            f(torch.empty(4, 8, device=dev))
    assert torch.equal(igs.embedding_lookup(t, table), table[t])


def test_checkpointed_module_draws_the_same_mask_again(igs, dev):
    """The module draws its dropout seed on the device from torch's generator, whose state a checkpoint restores for the
    recomputation (of the devices of its tensor arguments): gradients are bit-equal to those of the plain step from the
    same generator state."""
    from torch.utils.checkpoint import checkpoint

    torch.manual_seed(4)
    m = igs.GaussianSplatting2D(8, 64, num_embeddings=30, feature_norm=True, feature_dropout=0.4).to(dev)
    t = torch.randint(0, 30, (2, 16), device=dev)
    res = []
    for run in (lambda: m(t, size=(12, 16))[0], lambda: checkpoint(lambda a: m(a, size=(12, 16))[0], t, use_reentrant=False)):
        m.zero_grad()
        torch.manual_seed(7)
        img = run()
        img.square().sum().backward()
        res.append([img.detach()] + [p.grad.clone() for p in m.parameters()])
    assert len(res[0]) == len(res[1]) and all(torch.equal(a, b) for a, b in zip(*res))


def test_mixed_devices_raise(igs, dev):
    w, t, x = torch.randn(5, 4, device=dev), torch.tensor([1]), torch.randn(3, 4, device=dev)
    with pytest.raises(RuntimeError, match="same device"):
        igs.embedding_lookup(t, w)
    with pytest.raises(RuntimeError, match="GPU only"):
        igs.embedding_lookup(t.to(dev), w.cpu())
    with pytest.raises(RuntimeError, match="same device"):
        igs.layer_norm(x, torch.ones(4))
    with pytest.raises(RuntimeError, match="same device"):
        igs.dropout(x, 0.5, torch.tensor([1]))
    ops = torch.ops.igs_amd                             # the registered operators, called directly
    for call in (lambda: ops.embedding_fwd(t, w, 1.0, -1), lambda: ops.embedding_fwd(x[0], w, 1.0, -1),
                 lambda: ops.embedding_fwd(t.to(dev), w[0], 1.0, -1), lambda: ops.embedding_bwd(x, t.to(dev), 5, 1.0, -1),
                 lambda: ops.embedding_bwd(x[:1], t, 5, 1.0, -1), lambda: ops.layer_norm_fwd(x, w[0, :3], None, 1e-5, 0, 0, None, 0),
                 lambda: ops.layer_norm_fwd(x, w[0], w[0].half(), 1e-5, 0, 0, None, 0),
                 lambda: ops.layer_norm_fwd(x, torch.ones(4), None, 1e-5, 0, 0, None, 0),
                 lambda: ops.layer_norm_bwd(x[:2], x, None, None, torch.zeros(3, 2, device=dev), 0, 0, None, 0),
                 lambda: ops.layer_norm_bwd(x.half(), x, None, None, torch.zeros(3, 2, device=dev), 0, 0, None, 0),
                 lambda: ops.layer_norm_bwd(x, x, None, None, torch.zeros(2, 2, device=dev), 0, 0, None, 0),
                 lambda: ops.dropout(x, 9, 0, torch.zeros(2, device=dev, dtype=torch.int64), 0),
                 lambda: ops.dropout(x.double(), 9, 0, None, 0), lambda: ops.dropout(x, 70000, 0, None, 0)):
        with pytest.raises(RuntimeError):
            call()
    # an upstream gradient of another type is converted, as torch does
    leaf = x.half().requires_grad_(True)
    (g,) = torch.autograd.grad(igs.dropout(leaf, 0.5, 1), leaf, torch.ones(3, 4, device=dev))
    assert g.dtype == torch.float16 and torch.equal(g, igs.dropout(torch.ones(3, 4, device=dev).half(), 0.5, 1))


# ---------------------------------------------------------------------------------- the module
def test_module_with_tokens_norm_and_dropout(igs, dev):
    """GaussianSplatting2D with its front against the same module's plain torch path (fp32 both): the splat's own bounds
    (1e-6 + 1e-5 |ref| forward, 1e-4 of the largest gradient), with the head's features alike to fp32 rounding."""
    torch.manual_seed(1)
    m = igs.GaussianSplatting2D(8, 128, num_embeddings=50, emb_scale=1.5, padding_idx=0, feature_norm=True, feature_dropout=0.2).to(dev)
    m.dropout_seed = 1234
    t = torch.randint(0, 50, (2, 24), device=dev)
    up = torch.randn(2, 3, 20, 28, device=dev)
    res = []
    for fused in (True, False):
        m.zero_grad()
        img, feat = m(t, size=(20, 28), fused=fused)
        img.backward(up)
        res.append((img.detach(), feat.detach(), {k: v.grad.clone() for k, v in m.named_parameters()}))
    (a, fa, ga), (b, fb, gb) = res
    assert torch.allclose(fa, fb, rtol=1e-5, atol=1e-5)
    assert torch.allclose(a, b, rtol=1e-4, atol=1e-5)
    assert sorted(ga) == ["embedding.weight", "norm.bias", "norm.weight", "proj.bias", "proj.weight"]
    for k in ga:
        assert float((ga[k] - gb[k]).abs().max()) <= 1e-3 * float(gb[k].abs().max()) + 1e-7, k
    assert not ga["embedding.weight"][0].any()
    # a device seed drawn per call from torch's generator
    m.dropout_seed = None
    torch.manual_seed(7)
    one = m(t, size=(20, 28))[1]
    two = m(t, size=(20, 28))[1]
    torch.manual_seed(7)
    assert torch.equal(m(t, size=(20, 28))[1], one) and not torch.equal(one, two)
    m.eval()
    assert torch.equal(m(t, size=(20, 28))[1], m(t, size=(20, 28))[1])
    # dropout without the norm, features instead of tokens
    m2 = igs.GaussianSplatting2D(8, 128, feature_dropout=0.5).to(dev)
    m2.dropout_seed = 3
    f = torch.randn(2, 24, 128, device=dev)
    plain = igs.GaussianSplatting2D(8, 128).to(dev)
    plain.load_state_dict(m2.state_dict())
    assert torch.equal(m2(f, size=(20, 28))[0], plain(igs.dropout(f, 0.5, 3), size=(20, 28))[0])


def test_compiled_operators(igs, dev):
    """Under torch.compile the three are graph nodes (fullgraph) with the eager results, forward and backward."""
    V, D, n = 70, 72, 90
    t = some_tokens(n, V, 1, "skew").to(dev)
    w, gw, gb = normal((V, D), 1, torch.float32).to(dev), normal((D,), 2, torch.float32, 1.0).to(dev), normal((D,), 3, torch.float32).to(dev)
    up, seed = normal((n, D), 4, torch.float32).to(dev), torch.tensor([31], device=dev)

    def fn(t, w, gw, gb, seed):
        return igs.dropout(chain(igs, t, w, gw, gb, seed), 0.3, seed, 2)

    torch._dynamo.reset()
    comp = torch.compile(fn, fullgraph=True)
    res = []
    for f in (fn, comp):
        lv = [v.detach().requires_grad_(True) for v in (w, gw, gb)]
        y = f(t, *lv, seed)
        res.append((y.detach(), *torch.autograd.grad(y, lv, up)))
    for a, b in zip(*res):
        assert torch.equal(a, b)
    m = igs.GaussianSplatting2D(4, 72, num_embeddings=70, feature_norm=True, feature_dropout=0.2).to(dev)
    m.dropout_seed = seed
    ids = t[:24].view(2, 12)
    torch._dynamo.reset()
    want, got = m(ids, size=(9, 11)), torch.compile(lambda v: m(v, size=(9, 11)), fullgraph=True)(ids)
    assert torch.allclose(got[1], want[1], rtol=1e-5, atol=1e-6) and torch.allclose(got[0], want[0], rtol=1e-4, atol=1e-5)
    m.dropout_seed = None                                # a seed drawn on the device inside the graph
    torch.compile(lambda v: m(v, size=(9, 11)), fullgraph=True)(ids)[0].sum().backward()
    assert bool(m.embedding.weight.grad.isfinite().all()) and bool(m.embedding.weight.grad.any())


# ---------------------------------------------------------------------------------- tracers and dispatch modes
def traced_chain(igs, t, seed):
    """tokens and weights -> features, with every operator and with weights of another type than the rows'."""
    def fn(w, gw, gb):
        f = igs.layer_norm(igs.embedding_lookup(t, w, 1.5, -2), gw, gb, dropout_p=0.2, seed=seed, offset=1)
        return igs.dropout(igs.layer_norm(f, gw.bfloat16()), 0.1, seed, 5)
    return fn


def traced_inputs(dev, first):
    V, D = 40, 72
    return [normal(s, first + i, torch.float32, m).to(dev) for i, (s, m) in enumerate((((V, D), 0.0), ((D,), 1.0), ((D,), 0.0)))]


@pytest.mark.parametrize("tensor_seed", [False, True])
@pytest.mark.parametrize("how", ["jit", "fx"])
def test_traced_functions_compute_the_operators(igs, dev, how, tensor_seed):
    """A trace records the registered operators: on other inputs than it was made with it gives the eager results, forward
    and (a traced graph being differentiable) backward."""
    from torch.fx.experimental.proxy_tensor import make_fx

    t = some_tokens(50, 40, 1, "skew").to(dev)
    fn = traced_chain(igs, t, torch.tensor([31], device=dev) if tensor_seed else 31)
    trace = make_fx(fn) if how == "fx" else None
    traced = trace(*traced_inputs(dev, 1)) if how == "fx" else torch.jit.trace(fn, tuple(traced_inputs(dev, 1)))
    up = normal((50, 72), 9, torch.float32).to(dev)
    res = []
    for f in (fn, traced):
        lv = [v.requires_grad_(True) for v in traced_inputs(dev, 20)]
        y = f(*lv)
        res.append((y.detach(), *torch.autograd.grad(y, lv, up)))
    for a, b in zip(*res):
        assert torch.equal(a, b)


def test_traced_gradients_compute_the_operators(igs, dev):
    """make_fx of a gradient: of a function traced whole, and of one that was called before the trace began."""
    from torch.fx.experimental.proxy_tensor import make_fx

    t = some_tokens(50, 40, 1, "skew").to(dev)
    fn = traced_chain(igs, t, 31)
    lv = [v.requires_grad_(True) for v in traced_inputs(dev, 1)]
    first, up = normal((50, 72), 8, torch.float32).to(dev), normal((50, 72), 9, torch.float32).to(dev)
    whole = lambda w, gw, gb, g: torch.autograd.grad(fn(w, gw, gb), (w, gw, gb), g)
    other = [v.requires_grad_(True) for v in traced_inputs(dev, 20)]
    for a, b in zip(make_fx(whole)(*lv, first)(*other, up), whole(*other, up)):
        assert torch.equal(a, b)
    y = fn(*lv)
    want = torch.autograd.grad(y, lv, up, retain_graph=True)
    later = make_fx(lambda g: torch.autograd.grad(y, lv, g, retain_graph=True))(first)
    for a, b in zip(later(up), want):
        assert torch.equal(a, b)
    example = first.clone()                              # (a trace replaces its example wherever it meets it: not the norm's x)
    for which in range(3):                               # a part of the inputs alone
        w = igs.layer_norm(first, lv[1], lv[2]) if which else igs.embedding_lookup(t, lv[0])
        (want,) = torch.autograd.grad(w, lv[which], up, retain_graph=True)
        (got,) = make_fx(lambda g: torch.autograd.grad(w, lv[which], g, retain_graph=True))(example)(up)
        assert torch.equal(got, want)
    b = igs.layer_norm(first, None, lv[2])               # a bias without a weight
    (got,) = make_fx(lambda g: torch.autograd.grad(b, lv[2], g, retain_graph=True))(example)(up)
    assert torch.equal(got, torch.autograd.grad(b, lv[2], up)[0])


def test_dispatch_modes_see_the_operators(igs, dev):
    """A mode that counts what is dispatched sees one operator per call, forward and backward, and the results stay."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Count(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.seen = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.seen.append(func.name())
            return func(*args, **(kwargs or {}))

    t = some_tokens(50, 40, 1, "skew").to(dev)
    fn = traced_chain(igs, t, 31)
    lv, up = [v.requires_grad_(True) for v in traced_inputs(dev, 1)], normal((50, 72), 9, torch.float32).to(dev)
    y = fn(*lv)
    want = torch.autograd.grad(y, lv, up, retain_graph=True)
    with Count() as c:
        assert torch.equal(fn(*lv).detach(), y.detach())
    ours = [n for n in c.seen if n.startswith("igs_amd::")]
    assert ours == ["igs_amd::embedding_fwd", "igs_amd::layer_norm_fwd", "igs_amd::layer_norm_fwd", "igs_amd::dropout"], ours
    with Count() as c:
        got = torch.autograd.grad(y, lv, up)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    ours = [n for n in c.seen if n.startswith("igs_amd::")]
    assert ours == ["igs_amd::dropout", "igs_amd::layer_norm_bwd", "igs_amd::layer_norm_bwd", "igs_amd::embedding_bwd"], ours


def test_lazily_negated_tensors(igs, dev):
    """Tensors whose negation is yet to be done (the imaginary part of a conjugate), as every argument of every operator and
    as the upstream gradient, give what the negated copies give."""
    z = torch.view_as_complex(normal((9, 1, 2), 1, torch.float32).to(dev))
    t = torch.tensor([3, 8, 3, 0], device=dev)
    neg = torch._neg_view
    x, w, b, table, up = [normal(s, i, torch.float32, 1.0).to(dev) for i, s in enumerate(((6, 24), (24,), (24,), (9, 24), (6, 24)))]
    for lazy in (z.conj().imag, neg(table), neg(table)[:, :7], neg(table).t()):
        assert lazy.is_neg()
        assert torch.equal(igs.embedding_lookup(t, lazy), lazy.clone().resolve_neg()[t])
    assert torch.equal(igs.embedding_lookup(neg(-t), table), table[t])
    for lazy in (z.conj().imag, z.conj().imag[:1], neg(x), neg(x)[:, 3:], neg(x).t()):
        done = lazy.resolve_neg()
        assert lazy.is_neg() and not done.is_neg()
        assert torch.equal(igs.dropout(lazy, 0.3, 5), igs.dropout(done, 0.3, 5))
        assert torch.equal(igs.layer_norm(lazy), igs.layer_norm(done))
    res = []
    for f in (neg, torch.neg):
        lv = [f(v).detach().requires_grad_(True) for v in (x, w, b, table)]
        assert lv[0].is_neg() == (f is neg)
        y = igs.dropout(igs.layer_norm(lv[0], lv[1], lv[2]), 0.3, 5)
        e = igs.embedding_lookup(t, lv[3], 2.0)
        res.append((y.detach(), e.detach(), *torch.autograd.grad(y, lv[:3], f(up)), *torch.autograd.grad(e, lv[3], f(up)[:4])))
    for a, c in zip(*res):
        assert torch.equal(a, c)
    for node in (lambda v: igs.dropout(v, 0.3, 5), igs.layer_norm, lambda v: igs.embedding_lookup(t[:1], v)):
        leaf = z.real.clone().requires_grad_(True)       # one element: contiguous whatever its strides
        y = node(leaf)
        g = z.conj().imag[:y.shape[0]]
        assert g.is_neg() and torch.equal(*[torch.autograd.grad(y, leaf, v, retain_graph=True)[0] for v in (g, g.resolve_neg())])
    with pytest.raises(RuntimeError, match="seed"):
        igs.dropout(x, 0.3, neg(torch.tensor([5], device=dev)))


# ---------------------------------------------------------------------------------- tensors past the caches
def check_here(got, ref, tol, what):
    """`check` without the copy to the host."""
    assert got.shape == ref.shape, what
    err = (got.detach().to(F64) - ref).abs()
    assert bool((err <= tol).all()), (what, float((err / tol).max()))


def big_normal(shape, seed, dtype, dev, shift, mean=0.0, std=1.0):
    """Normal numbers made on the device, `shift` elements behind an aligned address."""
    g = torch.Generator(dev).manual_seed(seed)
    n = math.prod(shape)
    flat = torch.empty(n + shift, device=dev, dtype=dtype)
    flat[shift:] = (torch.randn(n, generator=g, device=dev) * std + mean).to(dtype)
    return flat[shift:].view(shape)


# (rows, D): rows that are and are not whole packs, narrow ones, ones of more than 4096 elements, ones shorter than a pack;
# 192 MB or more each, from which on tensors go past the caches
PAST_CACHES = [(torch.bfloat16, torch.float32, 98611, 1021, 0), (torch.float32, torch.float32, 49311, 1021, 1),
               (torch.float16, torch.float16, 98611, 1021, 3), (torch.float32, torch.float32, 49157, 1024, 0),
               (torch.bfloat16, torch.bfloat16, 4194307, 25, 1), (torch.float16, torch.float32, 24571, 4101, 0),
               (torch.float32, torch.float32, 6133, 8207, 1), (torch.float32, torch.float32, 16777219, 3, 0)]


@pytest.mark.parametrize("p", [0.0, 0.25])
@pytest.mark.parametrize("dtype,wdtype,R,D,shift", PAST_CACHES, ids=str)
def test_norm_past_the_caches(igs, dev, dtype, wdtype, R, D, shift, p):
    """Every value of the forward that a backward follows, of the forward alone and of the three gradients against the
    64-bit definition, by the bounds of the other sizes; the two forwards bit for bit."""
    assert R * D * dtype.itemsize >= 192 << 20
    x, up = big_normal((R, D), 1, dtype, dev, shift, 0.4, 1.7), big_normal((R, D), 2, dtype, dev, shift)
    assert shift == 0 or x.data_ptr() % 16
    w, b = normal((D,), 3, wdtype, 1.0, 0.3).to(dev), normal((D,), 4, wdtype).to(dev)
    factors = None
    if p:
        t = round(p * 65536)
        factors = igs.dropout_keep_mask((R, D), p, 11, 3, dev).to(F64) * (65536 / (65536 - t))
    kw = dict(dropout_p=p, seed=11, offset=3) if p else {}
    lv = [v.requires_grad_(True) for v in (x, w, b)]
    y = igs.layer_norm(*lv, **kw)
    with torch.no_grad():
        assert torch.equal(igs.layer_norm(*lv, **kw), y)
    grads = torch.autograd.grad(y, lv, up)
    x, w, b = [v.detach() for v in lv]
    ref = F.layer_norm(x, w, b, 1e-5, factors)[0]
    check_here(y, ref, norm_tolerance(x, w, b, 1e-5, factors, ref, dtype), "y")
    refs = F.layer_norm_grad(up, x, w, 1e-5, factors)
    tols = norm_grad_tolerances(up, x, w, 1e-5, factors, refs, (dtype, wdtype))
    for name, got, r, tol in zip(("dx", "dw", "db"), grads, refs, tols):
        check_here(got, r, tol, name)


@pytest.mark.parametrize("dtype,n,D,shift", [(torch.bfloat16, 98611, 1021, 1), (torch.float32, 49311, 1021, 1), (torch.float16, 98611, 1021, 0),
                                             (torch.float32, 16777219, 3, 0), (torch.bfloat16, 4194307, 25, 3)], ids=str)
def test_lookup_past_the_caches(igs, dev, dtype, n, D, shift):
    """Rows of a misaligned table, some tokens outside it, come bit for bit; the gradient of a misaligned upstream of whole
    numbers, whose sums are exact in any order, does too."""
    assert n * D * dtype.itemsize >= 192 << 20
    V = 7001
    w = big_normal((V, D), 1, dtype, dev, shift).requires_grad_(True)
    g = torch.Generator(dev).manual_seed(2)
    t = torch.randint(0, V, (n,), generator=g, device=dev)
    t[::1000], t[1::1000] = -1, V
    t[5::7] = 13                                             # a frequent one: an exact sum of 2^23 ones at most
    inside = (t >= 0) & (t < V)
    y = igs.embedding_lookup(t, w)
    assert torch.equal(y[inside], w.detach()[t[inside]]) and bool(y[~inside].isnan().all())
    flat = torch.empty(n * D + shift, device=dev, dtype=dtype)
    flat[shift:] = torch.randint(-1, 2, (n * D,), generator=g, device=dev, dtype=torch.int8).to(dtype)
    up = flat[shift:].view(n, D)
    (got,) = torch.autograd.grad(y, w, up)
    want = torch.zeros(V, D, device=dev).index_add_(0, t[inside], up[inside].float())
    assert torch.equal(got, want.to(dtype))


# ---------------------------------------------------------------------------------- bit equality of views and of the module
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
def test_views_give_the_bits_of_their_copies(igs, dev, dtype):
    """The arrangement of a row over threads is a function of its length and type alone, whatever its address and stride."""
    base, flat = normal((6, 10, 48), 1, dtype).to(dev), normal((6 * 48 + 5,), 2, dtype).to(dev)
    views = (base[..., :40], base[:, ::2], base[..., 3:36], base.transpose(0, 1), base[..., ::2], flat[1:289].view(6, 48), flat[5:].view(6, 48),
             flat[3:261].view(2, 129), base[:1].expand(4, 10, 48), base[:, :1].expand(6, 3, 48), base[2, 3], base[..., 7:8], base[:, :0])
    for v in views:
        D = v.shape[-1]
        w, b = normal((D + 1,), 3, dtype, 1.0, 0.3).to(dev)[1:], normal((D,), 4, dtype).to(dev)
        up = normal(tuple(v.shape), 5, dtype).to(dev)
        res = []
        for x in (v, v.clone(memory_format=torch.contiguous_format)):
            x = x.detach().requires_grad_(True)
            ws = [w.detach().requires_grad_(True), b.detach().requires_grad_(True)]
            y = igs.layer_norm(x, *ws, dropout_p=0.2, seed=5)
            res.append((y, *torch.autograd.grad(y, [x, *ws], up)))
        for a, c in zip(*res):
            assert a.shape == c.shape and torch.equal(a, c)


def test_module_is_its_operators_and_the_plain_module(igs, dev):
    """The module with its front against the operators called one by one in front of the module without: image, features and
    every gradient bit for bit (the same kernels on the same numbers)."""
    torch.manual_seed(1)
    m = igs.GaussianSplatting2D(8, 128, num_embeddings=50, emb_scale=1.5, padding_idx=0, feature_norm=True, feature_dropout=0.2).to(dev)
    m.dropout_seed = 1234
    plain = igs.GaussianSplatting2D(8, 128).to(dev)
    plain.load_state_dict({k: v for k, v in m.state_dict().items() if k.startswith("proj")})
    t, up = torch.randint(0, 50, (2, 24), device=dev), torch.randn(2, 3, 20, 28, device=dev)
    img, feat = m(t, size=(20, 28))
    img.backward(up)
    lv = [v.detach().clone().requires_grad_(True) for v in (m.embedding.weight, m.norm.weight, m.norm.bias)]
    f = igs.layer_norm(igs.embedding_lookup(t, lv[0], 1.5, 0), lv[1], lv[2], m.norm.eps, 0.2, 1234)
    want, want_feat = plain(f, size=(20, 28))
    want.backward(up)
    assert torch.equal(img, want) and torch.equal(feat, want_feat)
    assert all(torch.equal(a.grad, b.grad) for a, b in zip((m.embedding.weight, m.norm.weight, m.norm.bias, *m.proj.parameters()),
                                                           (*lv, *plain.proj.parameters())))
    assert bool(m.embedding.weight.grad.any()) and not m.embedding.weight.grad[0].any()


def test_direct_calls_that_would_read_beside_a_tensor_are_refused(igs, dev):
    """The registered operators with what the public functions never pass: refused on the host."""
    ops = torch.ops.igs_amd
    x, stats = torch.randn(3, 16, device=dev).bfloat16(), torch.zeros(3, 2, device=dev)
    for wtype in (torch.int8, torch.uint8, torch.float64, torch.float16):
        w = torch.ones(16, device=dev, dtype=wtype)
        for weight, bias in ((w, None), (None, w), (w, w)):
            with pytest.raises(RuntimeError):
                ops.layer_norm_fwd(x, weight, bias, 1e-5, 0, 0, None, 0)
            with pytest.raises(RuntimeError):
                ops.layer_norm_bwd(x, x, weight, bias, stats, 0, 0, None, 0)
    for threshold in (2 ** 32, -1, 65537):
        for call in (lambda: ops.dropout(x, threshold, 0, None, 0), lambda: ops.layer_norm_fwd(x, None, None, 1e-5, threshold, 0, None, 0),
                     lambda: ops.layer_norm_bwd(x, x, None, None, stats, threshold, 0, None, 0)):
            with pytest.raises(RuntimeError, match="threshold"):
                call()


class Front(torch.nn.Module):
    """Tokens -> (image, Gaussians, diversity loss of the normalised tokens) through the module and what stands around it."""

    def __init__(self, igs, dev, size):
        super().__init__()
        self.size = size
        torch.manual_seed(1)
        self.m = igs.GaussianSplatting2D(4, 32, num_embeddings=30, emb_scale=1.5, feature_norm=True).to(dev)
        self.koleo = igs.koleo_diversity_loss

    def forward(self, t):
        img, feat = self.m(t, size=self.size)
        return img, feat, self.koleo(self.m.embedding.weight[None])


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("how", ["jit", "fx", "export"])
def test_traced_module_from_tokens_to_the_image(igs, dev, how, grad):
    """A trace of the whole module, its first use at this image size, computes the image for other tokens; the module itself
    works afterwards."""
    from torch.fx.experimental.proxy_tensor import make_fx

    f = Front(igs, dev, (9, 11 + 2 * ["jit", "fx", "export"].index(how) + grad))
    a, b = [torch.randint(0, 30, (2, 6), device=dev, generator=torch.Generator(dev).manual_seed(k)) for k in (1, 2)]
    with torch.set_grad_enabled(grad):
        if how == "jit":
            traced = torch.jit.trace(f, (a,), check_trace=False)
        elif how == "fx":
            traced = make_fx(f)(a)
        else:
            traced = torch.export.export(f, (a,), strict=False).module()
    want, other = f(b), f(a)
    assert bool(want[0].isfinite().all()) and not torch.equal(want[0], other[0])
    for x, y in zip(traced(b), want):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
def test_registered_operators_by_opcheck_and_with_dynamic_sizes(igs, dev, dtype):
    """torch's own checks of the five operators (schema, autograd registration, fake tensors, AOT dispatch with static and
    dynamic sizes), and the chain compiled for changing sizes against the eager one, forward and backward."""
    ops, check = torch.ops.igs_amd, torch.library.opcheck
    t, seed = torch.randint(0, 9, (2, 5), device=dev), torch.tensor([5], device=dev)
    w, x = torch.randn(9, 16, device=dev).to(dtype).requires_grad_(), torch.randn(2, 5, 16, device=dev).to(dtype).requires_grad_()
    lw, lb = torch.randn(16, device=dev, requires_grad=True), torch.randn(16, device=dev, requires_grad=True)
    d = lambda v: v.detach()
    stats = ops.layer_norm_fwd(d(x), d(lw), None, 1e-5, 0, 0, None, 0)[1]
    turned = d(x).transpose(0, 1).requires_grad_()
    for op, args in ((ops.embedding_fwd, (t, w, 2.0, -1)), (ops.embedding_bwd, (d(x), t, 9, 2.0, 3)), (ops.layer_norm_fwd, (x, lw, lb, 1e-5, 100, 7, None, 0)),
                     (ops.layer_norm_fwd, (turned, lw, None, 1e-5, 100, 7, seed, 0)), (ops.layer_norm_bwd, (d(x), d(x), d(lw), d(lb), stats, 100, 7, None, 0)),
                     (ops.dropout, (x, 30000, 7, seed, 3)), (ops.dropout, (turned, 30000, 7, None, 3))):
        check(op.default, args)

    def fn(t, w, a, b, seed):
        f = igs.layer_norm(igs.embedding_lookup(t, w, 1.5, -1), a, b, dropout_p=0.3, seed=seed, offset=2)
        return igs.dropout(f, 0.2, seed, 9)

    torch._dynamo.reset()
    compiled = torch.compile(fn, fullgraph=True, dynamic=True)
    for n, D in ((7, 24), (130, 33), (1, 40)):
        leaves = [torch.randn(9, D, device=dev).to(dtype), torch.randn(D, device=dev), torch.randn(D, device=dev).to(dtype)]
        tokens, s, up = torch.randint(0, 9, (n,), device=dev), torch.tensor([n], device=dev), torch.randn(n, D, device=dev).to(dtype)
        res = []
        for f in (fn, compiled):
            lv = [v.detach().requires_grad_(True) for v in leaves]
            y = f(tokens, *lv, s)
            res.append((y.detach(), *torch.autograd.grad(y, lv, up)))
        for a, c in zip(*res):
            assert torch.equal(a, c)
