"""Host side of the feature operators: refusals, plan arithmetic and status codes of the C ABI, shape functions, the
module's options.  No kernel is launched, no GPU needed."""
import ctypes

import pytest
import torch

import igs_amd
from igs_amd import _lib, feature


@pytest.fixture(scope="module")
def lib():
    from igs_amd import build

    if build.is_stale():
        build.build(verbose=False)
    return _lib.load()


def test_embedding_refusals():
    w, t = torch.randn(5, 4), torch.tensor([1, 2])
    with pytest.raises(RuntimeError, match="GPU only"):
        igs_amd.embedding_lookup(t, w)
    for bad in (torch.randn(5), torch.randn(0, 4), torch.randn(5, 0), torch.randn(2, 3, 4)):
        with pytest.raises(ValueError, match=r"\[V, D\]"):
            igs_amd.embedding_lookup(t, bad)
    for bad in (t.float(), t.bool(), t.to(torch.int16), t.to(torch.uint8)):
        with pytest.raises(TypeError, match="tokens"):
            igs_amd.embedding_lookup(bad, w)
    with pytest.raises(TypeError, match="weight"):
        igs_amd.embedding_lookup(t, w.double())
    for bad in (float("nan"), float("inf")):
        with pytest.raises(ValueError, match="scale"):
            igs_amd.embedding_lookup(t, w, bad)
    for bad in (5, -6):
        with pytest.raises(ValueError, match="padding_idx"):
            igs_amd.embedding_lookup(t, w, padding_idx=bad)


def test_layer_norm_refusals():
    x = torch.randn(3, 4)
    with pytest.raises(RuntimeError, match="GPU only"):
        igs_amd.layer_norm(x)
    for bad in (torch.tensor(1.0), torch.randn(3, 0)):
        with pytest.raises(ValueError, match="last axis"):
            igs_amd.layer_norm(bad)
    with pytest.raises(TypeError, match="x must be"):
        igs_amd.layer_norm(x.double())
    for bad in (torch.randn(3), torch.randn(4, 1), torch.randn(4, 4)):
        with pytest.raises(ValueError, match="weight"):
            igs_amd.layer_norm(x, bad)
        with pytest.raises(ValueError, match="bias"):
            igs_amd.layer_norm(x, None, bad)
    with pytest.raises(TypeError, match="weight"):
        igs_amd.layer_norm(x, torch.ones(4, dtype=torch.int64))
    for bad in (-1e-5, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="eps"):
            igs_amd.layer_norm(x, eps=bad)
    with pytest.raises(ValueError, match="seed"):
        igs_amd.layer_norm(x, dropout_p=0.5)


def test_dropout_refusals():
    x = torch.randn(3, 4)
    with pytest.raises(RuntimeError, match="GPU only"):
        igs_amd.dropout(x, 0.5, 1)
    for bad in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="probability"):
            igs_amd.dropout(x, bad, 1)
    with pytest.raises(TypeError, match="x must be"):
        igs_amd.dropout(x.double(), 0.5, 1)
    for bad in (-1, 1 << 63):
        with pytest.raises(ValueError, match=r"2\^63"):
            igs_amd.dropout(x, 0.5, bad)
        with pytest.raises(ValueError, match=r"2\^63"):
            igs_amd.dropout(x, 0.5, 1, offset=bad)
        with pytest.raises(ValueError, match=r"2\^63"):
            igs_amd.dropout(x, 0.5, torch.tensor([1]), offset=bad)
    for bad in (1.5, True, "1"):
        with pytest.raises(TypeError, match="seed"):
            igs_amd.dropout(x, 0.5, bad)
    with pytest.raises(TypeError, match="offset"):
        igs_amd.dropout(x, 0.5, 1, offset=1.0)
    for bad in (torch.tensor([1, 2]), torch.tensor([1], dtype=torch.int32)):
        with pytest.raises(TypeError, match="seed tensor"):
            igs_amd.dropout(x, 0.5, bad)
    with pytest.raises(RuntimeError, match="same device"):
        igs_amd.dropout(torch.empty(3, device="meta"), 0.5, torch.tensor([1]))
    assert igs_amd.dropout(x, 0.0, None) is x and igs_amd.dropout(x, 2.0 ** -18, 1) is x   # nothing is dropped
    assert feature.dropout_threshold(1.0) == 65536 and feature.dropout_threshold(0.1) == 6554


def test_status_codes(lib):
    """Arguments are rejected before anything is launched (4096 is never read)."""
    p, E, N = ctypes.c_void_p(4096), _lib.EmbeddingPlan(), _lib.LayerNormPlan()
    odd = ctypes.c_void_p(4097)
    assert lib.igs_embedding_plan(10, 8, 0, 5, ctypes.byref(E)) == 0 and (E.vocab, E.D, E.count) == (10, 8, 5)
    assert lib.igs_embedding_plan(10, 8, 0, 5, None) == -1
    assert lib.igs_embedding_plan(10, 8, 3, 5, ctypes.byref(E)) == -11
    for v, d, n in ((0, 8, 5), (10, 0, 5), (10, (1 << 20) + 1, 5), (10, 8, -1), (1 << 31, 8, 5), (10, 8, 1 << 31)):
        assert lib.igs_embedding_plan(v, d, 0, n, ctypes.byref(E)) == -2
    fwd = lib.igs_embedding_forward
    assert fwd(p, 8, 0, 10, 8, p, 2, 5, 1.0, p, None) == -11
    assert fwd(p, 8, 7, 10, 8, p, 4, 5, 1.0, p, None) == -11
    assert fwd(p, -1, 0, 10, 8, p, 4, 5, 1.0, p, None) == -12
    assert fwd(p, 8, 0, 10, 8, p, 4, 5, float("nan"), p, None) == -12
    assert fwd(None, 8, 0, 10, 8, p, 4, 5, 1.0, p, None) == -1
    assert fwd(odd, 8, 0, 10, 8, p, 4, 5, 1.0, p, None) == -7
    assert fwd(None, 8, 0, 10, 8, None, 4, 0, 1.0, None, None) == 0         # no tokens: no work
    bwd = lib.igs_embedding_backward
    big = 1 << 40
    assert bwd(p, 0, p, 8, 5, 10, 8, 1.0, 10, p, p, big, None) == -12
    assert bwd(p, 0, p, 8, 5, 10, 8, 1.0, -2, p, p, big, None) == -12
    assert bwd(p, 0, p, 8, 5, 10, 8, 1.0, -1, None, p, big, None) == -1
    assert bwd(p, 0, None, 8, 5, 10, 8, 1.0, -1, p, p, big, None) == -1
    assert bwd(p, 0, odd, 8, 5, 10, 8, 1.0, -1, p, p, big, None) == -7
    assert bwd(p, 0, p, 8, 5, 10, 8, 1.0, -1, p, ctypes.c_void_p(4100), big, None) == -7
    lib.igs_embedding_plan(10, 8, 0, 5, ctypes.byref(E))
    if E.ws_bytes:
        assert bwd(p, 0, p, 8, 5, 10, 8, 1.0, -1, p, p, E.ws_bytes - 1, None) == -4
        assert bwd(p, 0, p, 8, 5, 10, 8, 1.0, -1, p, None, big, None) == -1
    d = lib.igs_dropout
    assert d(p, 5, 8, 100, 0, None, 0, p, None) == -11 and d(p, 0, -1, 100, 0, None, 0, p, None) == -2
    assert d(p, 0, 8, -1, 0, None, 0, p, None) == -12 and d(p, 0, 8, 65537, 0, None, 0, p, None) == -12
    assert d(p, 0, 8, 100, 0, ctypes.c_void_p(4100), 0, p, None) == -7 and d(None, 0, 8, 100, 0, None, 0, p, None) == -1
    assert d(odd, 1, 8, 100, 0, None, 0, p, None) == -7 and d(None, 0, 0, 100, 0, None, 0, None, None) == 0
    assert lib.igs_layer_norm_plan(10, 8, 0, 0, ctypes.byref(N)) == 0 and (N.rows, N.D) == (10, 8)
    assert lib.igs_layer_norm_plan(10, 8, 0, 0, None) == -1
    assert lib.igs_layer_norm_plan(10, 8, 0, 1, ctypes.byref(N)) == -11     # fp32 rows with fp16 weights
    assert lib.igs_layer_norm_plan(10, 8, 1, 2, ctypes.byref(N)) == -11
    for r, D in ((-1, 8), (10, 0), (10, (1 << 20) + 1), (1 << 31, 8)):
        assert lib.igs_layer_norm_plan(r, D, 0, 0, ctypes.byref(N)) == -2
    f = lib.igs_layer_norm_forward
    assert f(p, 8, 0, p, p, 0, 10, 8, -1.0, 0, 0, None, 0, p, p, None) == -12
    assert f(p, -8, 0, p, p, 0, 10, 8, 1e-5, 0, 0, None, 0, p, p, None) == -12
    assert f(p, 8, 0, p, p, 0, 10, 8, 1e-5, 70000, 0, None, 0, p, p, None) == -12
    assert f(None, 8, 0, p, p, 0, 10, 8, 1e-5, 0, 0, None, 0, p, p, None) == -1
    assert f(p, 8, 0, p, odd, 0, 10, 8, 1e-5, 0, 0, None, 0, p, p, None) == -7
    assert f(p, 8, 0, p, p, 0, 10, 8, 1e-5, 0, 0, None, 0, p, ctypes.c_void_p(4100), None) == -7
    assert f(None, 8, 0, p, p, 0, 0, 8, 1e-5, 0, 0, None, 0, None, None, None) == 0
    b = lib.igs_layer_norm_backward
    assert b(p, p, 8, 0, p, 0, None, 10, 8, 0, 0, None, 0, p, p, p, p, big, None) == -1
    assert b(p, p, 8, 0, p, 0, p, 10, 8, -3, 0, None, 0, p, p, p, p, big, None) == -12
    assert b(p, p, 8, 1, p, 2, p, 10, 8, 0, 0, None, 0, p, p, p, p, big, None) == -11
    assert b(odd, p, 8, 0, p, 0, p, 10, 8, 0, 0, None, 0, p, p, p, p, big, None) == -7
    lib.igs_layer_norm_plan(10, 8, 0, 0, ctypes.byref(N))
    if N.ws_bytes:
        assert b(p, p, 8, 0, p, 0, p, 10, 8, 0, 0, None, 0, p, p, p, p, N.ws_bytes - 1, None) == -4
        assert b(p, p, 8, 0, p, 0, p, 10, 8, 0, 0, None, 0, p, p, p, None, big, None) == -1
    assert b"element type" in lib.igs_status_string(-11) and b"range" in lib.igs_status_string(-12)


def test_plan_structs_match_the_header():
    import os
    import re

    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "igs_hip.h")).read()
    for name, mirror in (("igs_embedding_plan_t", _lib.EmbeddingPlan), ("igs_layer_norm_plan_t", _lib.LayerNormPlan)):
        body = re.sub(r"/\*.*?\*/", "", text[text.index(f"typedef struct {name} {{"):text.index(f"}} {name};")], flags=re.S)
        fields = []
        for decl in body.split("{", 1)[1].split(";"):
            if decl.strip():
                typ, rest = decl.strip().split(None, 1)
                fields += [(f.strip(), typ) for f in rest.split(",")]
        want = {"int32_t": ctypes.c_int32, "int64_t": ctypes.c_int64, "uint64_t": ctypes.c_uint64}
        assert [(n, want[t]) for n, t in fields] == list(mirror._fields_)


def test_shape_functions():
    """What torch.compile is told about the operators (meta tensors)."""
    m = lambda *s, dtype=torch.bfloat16: torch.empty(*s, device="meta", dtype=dtype)
    ops = torch.ops.igs_amd
    t = m(2, 5, dtype=torch.int64)
    y = ops.embedding_fwd(t, m(9, 16), 2.0, -1)
    assert y.shape == (2, 5, 16) and y.dtype == torch.bfloat16
    assert ops.embedding_bwd(y, t, 9, 2.0, -1).shape == (9, 16)
    w = m(16, dtype=torch.float32)
    y, stats = ops.layer_norm_fwd(m(2, 5, 16), w, None, 1e-5, 0, 0, None, 0)
    assert y.shape == (2, 5, 16) and y.dtype == torch.bfloat16 and stats.shape == (10, 2) and stats.dtype == torch.float32
    g = ops.layer_norm_bwd(y, m(2, 5, 16), w, None, stats, 0, 0, None, 0)
    assert [(tuple(v.shape), v.dtype) for v in g] == [((2, 5, 16), torch.bfloat16), ((16,), torch.float32)]
    assert ops.dropout(m(3, 7), 100, 1, None, 0).shape == (3, 7)


@pytest.mark.parametrize("make,step", [
    (lambda b: b, 24), (lambda b: b[..., :10], 24), (lambda b: b[:, ::2], 48), (lambda b: b[:, :1], 96),
    (lambda b: b[:1, :1], 24), (lambda b: b.transpose(1, 2), None), (lambda b: b[..., ::2], None),
    (lambda b: b[:1, :1].expand(7, 5, 24), 0), (lambda b: b[:, :1].expand(2, 4, 24), None), (lambda b: b[..., :1], 24),
    (lambda b: b[:, :2], None)])
def test_rows_taken_in_place(make, step):
    """Rows that are dense and evenly spaced keep their memory; everything else is copied."""
    v = make(torch.arange(2 * 4 * 24, dtype=torch.float32).view(2, 4, 24))
    got, s = feature._native().rows_of(v)
    if step is None:
        assert got.is_contiguous() and s == v.shape[-1] and torch.equal(got, v)
    else:
        assert got.data_ptr() == v.data_ptr() and got.stride() == v.stride()
        rows, D = v.numel() // v.shape[-1], v.shape[-1]
        if rows > 1:
            assert s == step
        assert torch.equal(torch.as_strided(v, (rows, D), (s, 1)), v.reshape(rows, D))


def test_module_defaults_are_unchanged_and_options_add_parameters():
    torch.manual_seed(0)
    a = igs_amd.GaussianSplatting2D(4, 32)
    after = torch.rand(1)
    assert sorted(a.state_dict()) == ["proj.bias", "proj.weight"]
    torch.manual_seed(0)
    b = igs_amd.GaussianSplatting2D(4, 32, num_embeddings=11, emb_scale=2.0, padding_idx=3, feature_norm=True,
                                    feature_dropout=0.25)
    assert sorted(b.state_dict()) == ["embedding.weight", "norm.bias", "norm.weight", "proj.bias", "proj.weight"]
    assert torch.equal(a.proj.weight, b.proj.weight) and torch.equal(a.proj.bias, b.proj.bias)
    torch.manual_seed(0)
    igs_amd.GaussianSplatting2D(4, 32, feature_norm=True, feature_dropout=0.5)
    assert torch.equal(torch.rand(1), after)           # no draw of its own without a table
    with pytest.raises(ValueError, match="probability"):
        igs_amd.GaussianSplatting2D(4, 32, feature_dropout=1.5)
    with pytest.raises(TypeError, match="no embedding table"):
        a(torch.zeros(2, 3, dtype=torch.int64), size=(4, 4))


def test_modules_copied_and_pickled_whole():
    """Copies keep the front; a module pickled before there was one still runs."""
    import copy
    import pickle

    m = igs_amd.GaussianSplatting2D(4, 16, num_embeddings=11, feature_norm=True)
    t = torch.randint(0, 11, (2, 5))
    want = m(t, size=(6, 7), fused=False)[0]
    for c in (copy.deepcopy(m), pickle.loads(pickle.dumps(m))):
        assert torch.equal(c(t, size=(6, 7), fused=False)[0], want)
    plain = igs_amd.GaussianSplatting2D(4, 16)
    state = plain.__getstate__() if hasattr(plain, "__getstate__") else plain.__dict__
    state = {k: v for k, v in dict(state or plain.__dict__).items()
             if k not in ("emb_scale", "feature_dropout", "dropout_seed", "embedding", "norm")}
    old = igs_amd.GaussianSplatting2D.__new__(igs_amd.GaussianSplatting2D)
    old.__setstate__(state)
    x = torch.randn(2, 5, 16)
    assert torch.equal(old(x, size=(6, 7), fused=False)[0], plain(x, size=(6, 7), fused=False)[0])


def test_module_debug_path_on_the_cpu():
    """fused=False: lookup, norm and dropout as plain torch, then the plain splat; the mask is the operator's."""
    torch.manual_seed(3)
    m = igs_amd.GaussianSplatting2D(4, 16, num_embeddings=11, emb_scale=2.0, feature_norm=True, feature_dropout=0.25)
    m.dropout_seed = 99
    t = torch.randint(0, 11, (2, 5))
    img, feat = m(t, size=(6, 7), fused=False)
    f = m.embedding.weight[t] * 2.0
    f = torch.nn.functional.layer_norm(f, (16,), m.norm.weight, m.norm.bias, m.norm.eps)
    keep = igs_amd.dropout_keep_mask(f.shape, 0.25, 99)
    plain = igs_amd.GaussianSplatting2D(4, 16)
    plain.load_state_dict({k: v for k, v in m.state_dict().items() if k.startswith("proj")})
    want_img, want_feat = plain(torch.where(keep, f / 0.75, torch.zeros_like(f)), size=(6, 7), fused=False)
    assert torch.allclose(feat, want_feat, rtol=1e-5, atol=1e-6) and torch.allclose(img, want_img, rtol=1e-5, atol=1e-6)
    img.sum().backward()
    assert m.embedding.weight.grad is not None and m.norm.weight.grad is not None
    m.eval()
    a, b = m(t, size=(6, 7), fused=False)[0], m(t, size=(6, 7), fused=False)[0]
    assert torch.equal(a, b)                             # no dropout in evaluation
    m.train()
    m.dropout_seed = None
    assert not torch.equal(m(t, size=(6, 7), fused=False)[1], m(t, size=(6, 7), fused=False)[1])   # a new seed per call
    torch.manual_seed(5)
    a = m(t, size=(6, 7), fused=False)[1]
    torch.manual_seed(5)
    assert torch.equal(a, m(t, size=(6, 7), fused=False)[1])                                        # torch's generator governs it
    m(torch.randn(2, 5, 16), size=(6, 7), fused=False)   # features still pass


# ---------------------------------------------------------------------------------- direct calls below the public functions
def norm_bwd_arguments(dtype=torch.bfloat16, D=16, rows=3):
    x = torch.randn(rows, D).to(dtype)
    return torch.randn(rows, D).to(dtype), x, torch.zeros(rows, 2)


@pytest.mark.parametrize("wtype", [torch.int8, torch.uint8, torch.bool, torch.int64, torch.float64, torch.float16], ids=str)
def test_norm_backward_refuses_weights_of_other_types(wtype):
    """Weight or bias alone, of a type that the kernels would read and write as another: refused by the library's own check,
    before anything is launched (so without a GPU too)."""
    grad, x, stats = norm_bwd_arguments()
    w = torch.ones(16).to(wtype)
    bwd = feature._native().layer_norm_bwd
    for weight, bias in ((w, None), (None, w), (w, w)):
        with pytest.raises(RuntimeError, match="element type"):
            bwd(grad, x, weight, bias, stats, 0, 0, None, 0)


def test_norm_backward_refuses_a_bias_that_does_not_fit():
    """A bias of another type or length than the weight's beside a good weight (its gradient would be the weight's)."""
    grad, x, stats = norm_bwd_arguments()
    w = torch.ones(16)
    bwd = feature._native().layer_norm_bwd
    with pytest.raises(RuntimeError, match="one type"):
        bwd(grad, x, w, w.bfloat16(), stats, 0, 0, None, 0)
    with pytest.raises(RuntimeError, match="must be"):
        bwd(grad, x, w, torch.ones(15), stats, 0, 0, None, 0)


@pytest.mark.parametrize("threshold", [-1, 65537, 1 << 32, (1 << 32) + 100, -(1 << 32)])
def test_thresholds_are_checked_in_64_bits(threshold):
    """One whose lower 32 bits are a good threshold (2^32: no dropout) is refused like any other outside 0..65536."""
    native, x = feature._native(), torch.randn(3, 16)
    grad, xb, stats = norm_bwd_arguments()
    for call in (lambda: native.dropout_plain(x, threshold, 1, None, 0),
                 lambda: native.layer_norm_fwd(x, None, None, 1e-5, threshold, 1, None, 0),
                 lambda: native.layer_norm_bwd(grad, xb, None, None, stats, threshold, 1, None, 0)):
        with pytest.raises(RuntimeError, match="threshold is in 0..65536"):
            call()


def test_rows_of_a_negative_view():
    """A lazily negated tensor (the imaginary part of a conjugate) has the other sign in memory: it is copied."""
    x = torch.randn(5, 6)
    rows, step = feature._native().rows_of(torch._neg_view(x))
    assert not rows.is_neg() and step == 6 and torch.equal(rows, -x)
    z = torch.randn(5, 1, dtype=torch.complex64)
    rows, step = feature._native().rows_of(z.conj().imag)
    assert not rows.is_neg() and step == 1 and torch.equal(rows, -z.imag)


def test_subclasses_with_a_norm_of_their_own():
    """A subclass that has submodules called `norm` and `feature_dropout` and applies them itself, written when the module
    had none: the module's forward leaves them alone, built, copied and unpickled."""
    import copy

    class Own(igs_amd.GaussianSplatting2D):
        def __init__(self):
            super().__init__(4, 16)
            self.norm, self.feature_dropout, self.feature_norm = torch.nn.Tanh(), torch.nn.Dropout(0.0), torch.nn.Identity()

        def forward(self, feature, **kw):
            return super().forward(self.feature_dropout(self.feature_norm(self.norm(feature))), **kw)

    torch.manual_seed(2)
    m, plain, x = Own(), igs_amd.GaussianSplatting2D(4, 16), torch.randn(2, 5, 16)
    plain.load_state_dict(m.state_dict())
    want = plain(torch.tanh(x), size=(6, 7), fused=False)
    state = {k: v for k, v in m.__dict__.items() if k not in ("emb_scale", "feature_dropout", "dropout_seed", "_feature_norm")}
    state["_modules"] = {k: v for k, v in m._modules.items() if k != "embedding"}
    before = Own.__new__(Own)                            # pickled before the module had a front
    before.__setstate__(state)
    for c in (m, copy.deepcopy(m), before):
        got = c(x, size=(6, 7), fused=False)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_modules_pickled_with_a_norm_and_no_flag_keep_it():
    """State as it was when the presence of `norm` alone said that the module normalises."""
    m, x = igs_amd.GaussianSplatting2D(4, 16, feature_norm=True), torch.randn(2, 5, 16)
    state = {k: v for k, v in m.__dict__.items() if k != "_feature_norm"}
    old = igs_amd.GaussianSplatting2D.__new__(igs_amd.GaussianSplatting2D)
    old.__setstate__(state)
    assert torch.equal(old(x, size=(6, 7), fused=False)[1], m(x, size=(6, 7), fused=False)[1])


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32], ids=str)
def test_plain_lookup_of_tokens_outside_the_table(dtype):
    """The plain expression says what the operator says of them: a row of NaN, no gradient (a negative one is not taken from
    the table's end), so that the module's debug path and the fused one agree."""
    from oracle import feature_oracle as F

    w, up = torch.randn(6, 10), torch.randn(8, 10)
    t = torch.tensor([0, 6, -1, 5, 2 ** 31 - 1, -2 ** 31, 3, 5]).to(dtype)
    for pad in (None, 3, -6):
        leaf = w.clone().requires_grad_(True)
        y = igs_amd.naive_embedding_lookup(t, leaf, 2.0, pad)
        assert torch.equal(y.detach().nan_to_num(7.0), F.embedding(t, w, 2.0).float().nan_to_num(7.0))
        assert y.isnan().all(-1).tolist() == [False, True, True, False, True, True, False, False]
        (g,) = torch.autograd.grad(y, leaf, up)
        # sums of two terms and a factor of two: exact but for one rounding of fp32
        assert torch.allclose(g.double(), F.embedding_grad(t, up, 6, 2.0, pad)[0], rtol=2.0 ** -23, atol=0)
    m = igs_amd.GaussianSplatting2D(4, 16, num_embeddings=11)
    feat = m(torch.tensor([[1, -1], [11, 2]]), size=(6, 7), fused=False)[1].view(2, 2, -1)
    assert feat.isnan().all(-1).tolist() == [[False, True], [True, False]]


def test_feature_kernels_have_no_build_switches():
    """Sizes of shared arrays and the limits that keep calls within them are one constant each: nothing on a compiler's
    command line can move a limit past its array."""
    import os

    csrc = os.path.join(os.path.dirname(feature.__file__), "csrc")
    for name in ("igs_feature.hip", "igs_feature_common.h", "igs_feature_host.h", "igs_embedding.h", "igs_dropout.h", "igs_norm.hip",
                 "igs_layer_norm.h"):
        text = open(os.path.join(csrc, name)).read()
        assert "#ifndef" not in text and "#ifdef" not in text, name


@pytest.mark.parametrize("n", [1025, 8192, 8193, 100000])
def test_workspace_refusals_of_the_lookup_gradient(lib, n):
    """More tokens than one launch takes need a workspace: one byte less than the plan's, or none at all, is refused before
    anything is launched."""
    p, E, big = ctypes.c_void_p(4096), _lib.EmbeddingPlan(), 1 << 40
    for vocab, D, dtype in ((10, 8, 0), (50021, 333, 1), (1 << 20, 1024, 2)):
        assert lib.igs_embedding_plan(vocab, D, dtype, n, ctypes.byref(E)) == 0
        assert E.ws_bytes >= 8 * n                       # sorted keys and their places
        for width in (4, 8):
            bwd = lambda ws, size: lib.igs_embedding_backward(p, dtype, p, width, n, vocab, D, 1.0, -1, p, ws, size, None)
            assert bwd(p, E.ws_bytes - 1) == -4 and bwd(p, 0) == -4
            assert bwd(None, E.ws_bytes) == -1 and bwd(None, big) == -1
            assert bwd(ctypes.c_void_p(4100), big) == -7


@pytest.mark.parametrize("rows,D", [(1, 8), (10, 8), (1000, 1024), (10, 5000), (3, 100000)])
def test_workspace_refusals_of_the_norm_gradient(lib, rows, D):
    p, N, big = ctypes.c_void_p(4096), _lib.LayerNormPlan(), 1 << 40
    for dtype in (0, 1, 2):
        assert lib.igs_layer_norm_plan(rows, D, dtype, 0, ctypes.byref(N)) == 0
        assert N.ws_bytes >= 8 * D and N.partials >= 1   # a partial row of two sums at least
        bwd = lambda ws, size: lib.igs_layer_norm_backward(p, p, D, dtype, p, 0, p, rows, D, 0, 0, None, 0, p, p, p, ws, size, None)
        assert bwd(p, N.ws_bytes - 1) == -4 and bwd(p, 0) == -4
        assert bwd(None, N.ws_bytes) == -1 and bwd(None, big) == -1
        assert bwd(ctypes.c_void_p(4104), big) == -7
