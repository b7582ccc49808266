"""Timed cases of the feature operators that stand in front of the Gaussian head: the embedding lookup with its
gradient, layer norm (optionally followed by dropout) forward and backward, and dropout from a counter-based
generator.

Definitions (t: tokens, W: table, s: scale):
  embedding   y_i = s W[t_i];  dW[v] = s sum over i with t_i = v of dy_i, zero for the padding token
  layer norm  h = (x - mean) / sqrt(var + eps), y = h w + b;  dx = r (g - mean g - h mean(g h)) with g = dy w,
              dw = sum over rows of dy h, db = sum over rows of dy
  dropout     element i is dropped if its 16-bit number u_i is below round(65536 p), and scaled by
              65536 / (65536 - round(65536 p)) otherwise.  u_i is half i % 2 of word (i % 8) / 2 of the Philox4x32
              block i / 8 (seven rounds; Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as
              1, 2, 3", 2011) with the counter (block, offset) and the seed as its key.
"""
import math

import torch

own = False

EPS = 1e-5
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one token of a codebook looked up while an image is decoded token by token: latency
        {"name": "embed_one_token", "op": "embedding", "n": 1, "vocab": 8192, "dim": 1024, "dtype": "f32",
         "skew": False, "padded": False, "scale": 1.0, "train": False},
        # the benchmarked module's feature block [8, 128, 1024] as tokens of a codebook, training
        {"name": "embed_module_batch", "op": "embedding", "n": 1024, "vocab": 8192, "dim": 1024, "dtype": "f32",
         "skew": False, "padded": False, "scale": 1.0, "train": True},
        # a long training batch over a large vocabulary with a few very frequent tokens and padding
        {"name": "embed_long_skewed", "op": "embedding", "n": 131072, "vocab": 65536, "dim": 1024, "dtype": "bf16",
         "skew": True, "padded": True, "scale": 1.0, "train": True},
        # sizes that divide by nothing: rows that start at odd addresses, scaled by sqrt(dim)
        {"name": "embed_odd", "op": "embedding", "n": 4099, "vocab": 50021, "dim": 333, "dtype": "f16",
         "skew": True, "padded": False, "scale": 18.25, "train": True},
        # one feature normalised in front of the head while decoding: latency
        {"name": "norm_one_row", "op": "norm", "rows": 1, "dim": 1024, "dtype": "bf16", "wdtype": "bf16", "p": 0.0,
         "train": False},
        # the benchmarked module's feature block [8, 128, 1024], training
        {"name": "norm_module_batch", "op": "norm", "rows": 1024, "dim": 1024, "dtype": "f32", "wdtype": "f32",
         "p": 0.0, "train": True},
        # a long batch under autocast: 16-bit activations, 32-bit weights
        {"name": "norm_long", "op": "norm", "rows": 131072, "dim": 1024, "dtype": "bf16", "wdtype": "f32", "p": 0.0,
         "train": True},
        # few wide rows of an odd length
        {"name": "norm_wide_odd", "op": "norm", "rows": 2053, "dim": 8205, "dtype": "f16", "wdtype": "f16", "p": 0.0,
         "train": True},
        # norm and dropout in front of the head as one operator, training
        {"name": "norm_dropout", "op": "norm", "rows": 32768, "dim": 1024, "dtype": "bf16", "wdtype": "f32", "p": 0.1,
         "train": True},
        # the feature block that the diversity loss takes, [1, 128, 512]: latency
        {"name": "dropout_small", "op": "dropout", "rows": 128, "dim": 512, "dtype": "f32", "p": 0.1, "train": False},
        # dropout of a long batch's activations, training
        {"name": "dropout_long", "op": "dropout", "rows": 65536, "dim": 1024, "dtype": "bf16", "p": 0.1,
         "train": True},
        # the three together as the module calls them: tokens, features, norm with dropout, gradients of all weights
        {"name": "token_features", "op": "chain", "n": 8192, "vocab": 8192, "dim": 1024, "dtype": "f32",
         "skew": True, "padded": False, "scale": 1.0, "p": 0.1, "train": True},
    ]


MOST_VALUES = 1 << 26  # values of one drawn array at most


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["embedding", "embedding", "norm", "norm", "dropout", "chain"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    train = op == "chain" or rng.random() < 0.75
    p = round(rng.uniform(0.02, 0.6), 3)
    if op == "norm":
        dim = _log_int(rng, 8, 24000)
        rows = _log_int(rng, 1, min(131072, MOST_VALUES // dim))
        return {"op": op, "rows": rows, "dim": dim, "dtype": dtype, "wdtype": rng.choice(["f32", dtype]),
                "p": p if rng.random() < 0.4 else 0.0, "train": train}
    if op == "dropout":
        dim = _log_int(rng, 8, 8192)
        return {"op": op, "rows": _log_int(rng, 1, min(131072, (MOST_VALUES >> 1) // dim)), "dim": dim, "dtype": dtype,
                "p": p, "train": train}
    dim = _log_int(rng, 8, 4096)
    n = _log_int(rng, 1, min(131072, (MOST_VALUES >> 1) // dim))
    vocab = _log_int(rng, 16, min(131072, (MOST_VALUES >> 1) // dim))
    case = {"op": op, "n": n, "vocab": vocab, "dim": dim, "dtype": "f32" if op == "chain" else dtype,
            "skew": rng.random() < 0.5, "padded": rng.random() < 0.3, "scale": round(math.sqrt(dim), 3)
            if rng.random() < 0.5 else 1.0, "train": train}
    if op == "chain":
        case["p"] = p
    return case


def _tokens(case, gen):
    """Uniform ids, or ids whose frequency falls like 1 / rank; the last eighth is padding where asked for."""
    n, vocab = case["n"], case["vocab"]
    u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
    t = torch.exp(u * math.log(vocab + 1)) - 1 if case["skew"] else u * vocab
    t = t.to(torch.int64).clamp_(0, vocab - 1)
    if case["padded"]:
        t[n - n // 8:] = vocab - 1
    return t


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(int(seed) * 7919 + 17)
    dtype, dim, train = DTYPES[case["dtype"]], case["dim"], case["train"]

    def normal(*shape, mean=0.0, std=1.0, to=dtype):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(std).add_(mean).to(to)

    state = {"op": case["op"], "train": train, "p": case.get("p", 0.0), "seed": (int(seed) * 0x9E3779B97F4A7C15) % (1 << 63),
             "offset": int(seed) % 1000}
    if case["op"] in ("embedding", "chain"):
        state["tokens"] = _tokens(case, gen)
        state["weight"] = normal(case["vocab"], dim, std=0.5 if case["op"] == "chain" else 0.02).requires_grad_(train)
        state["scale"] = case["scale"]
        state["padding_idx"] = case["vocab"] - 1 if case["padded"] else None
        rows = case["n"]
    else:
        rows = case["rows"]
        state["x"] = normal(rows, dim, mean=0.3, std=1.5).requires_grad_(train)
    if case["op"] in ("norm", "chain"):
        to = DTYPES[case.get("wdtype", "f32")]
        state["w"] = normal(dim, mean=1.0, std=0.1, to=to).requires_grad_(train)
        state["b"] = normal(dim, std=0.1, to=to).requires_grad_(train)
    if train:
        state["grad"] = normal(rows, dim)
    return state


# ---------------------------------------------------------------------------------- plain forms
def _mul32(a, b):
    """(high, low) 32 bits of the product of a 32-bit constant and 32-bit numbers held in int64."""
    low = a * (b & 0xFFFF)
    mid = a * (b >> 16) + (low >> 16)
    return mid >> 16, ((mid & 0xFFFF) << 16) | (low & 0xFFFF)


def _keep(shape, p, seed, offset, device):
    """(truth values of the elements that stay, their factor)."""
    count = math.prod(shape)
    block = torch.arange((count + 7) // 8, dtype=torch.int64, device=device)
    c0, c1 = block & 0xFFFFFFFF, block >> 32
    c2, c3 = torch.full_like(block, offset & 0xFFFFFFFF), torch.full_like(block, offset >> 32)
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(7):
        h0, l0 = _mul32(0xD2511F53, c0)
        h1, l1 = _mul32(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    words = torch.stack([c0, c1, c2, c3], dim=1)
    u = torch.stack([words & 0xFFFF, words >> 16], dim=2).reshape(-1)[:count].reshape(shape)
    t = math.floor(p * 65536 + 0.5)
    return u >= t, 65536 / (65536 - t) if t < 65536 else 0.0


def _drop(v, kept):
    """`kept` is what _keep says, or None for no dropout."""
    return v if kept is None else torch.where(kept[0], v * kept[1], torch.zeros_like(v))


def _embedding_plain(tokens, weight, scale):
    return (weight[tokens].float() * scale).to(weight.dtype)


def _embedding_grad_plain(tokens, weight, scale, padding_idx, grad):
    g = torch.zeros(weight.shape, dtype=torch.float32, device=weight.device).index_add_(0, tokens, grad.float())
    if padding_idx is not None:
        g[padding_idx] = 0
    return (g * scale).to(weight.dtype)


def _norm_plain(x, w, b, kept):
    """(y, normalised rows, 1 / standard deviation); the last two in 32 bits."""
    v = x.float()
    c = v - v.mean(-1, keepdim=True)
    r = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + EPS)
    h = c * r
    return _drop(h * w.float() + b.float(), kept).to(x.dtype), h, r


def _norm_grad_plain(h, r, x, w, b, kept, grad):
    dy = _drop(grad.float(), kept)
    g = dy * w.float()
    dx = r * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    return dx.to(x.dtype), (dy * h).sum(0).to(w.dtype), dy.sum(0).to(b.dtype)


def _run_plain(s):
    op, train = s["op"], s["train"]
    if op == "embedding":
        out = {"y": _embedding_plain(s["tokens"], s["weight"], s["scale"])}
        if train:
            out["dweight"] = _embedding_grad_plain(s["tokens"], s["weight"], s["scale"], s["padding_idx"], s["grad"])
        return out
    x = s["x"] if op != "chain" else _embedding_plain(s["tokens"], s["weight"], s["scale"])
    kept = _keep(x.shape, s["p"], s["seed"], s["offset"], x.device) if s["p"] else None
    if op == "dropout":
        out = {"y": _drop(x.float(), kept).to(x.dtype)}
        if train:
            out["dx"] = _drop(s["grad"].float(), kept).to(x.dtype)
        return out
    y, h, r = _norm_plain(x, s["w"], s["b"], kept)
    out = {"y": y}
    if train:
        dx, out["dw"], out["db"] = _norm_grad_plain(h, r, x, s["w"], s["b"], kept, s["grad"])
        if op == "norm":
            out["dx"] = dx
        else:
            out["dweight"] = _embedding_grad_plain(s["tokens"], s["weight"], s["scale"], s["padding_idx"], dx)
    return out


# ---------------------------------------------------------------------------------- the framework's operators
def _run_own(s):
    import igs_amd

    op, train = s["op"], s["train"]
    if op == "embedding":
        y = igs_amd.embedding_lookup(s["tokens"], s["weight"], scale=s["scale"], padding_idx=s["padding_idx"])
        names, leaves = ["dweight"], [s["weight"]]
    elif op == "norm":
        y = igs_amd.layer_norm(s["x"], s["w"], s["b"], eps=EPS, dropout_p=s["p"], seed=s["seed"], offset=s["offset"])
        names, leaves = ["dx", "dw", "db"], [s["x"], s["w"], s["b"]]
    elif op == "dropout":
        y = igs_amd.dropout(s["x"], s["p"], s["seed"], offset=s["offset"])
        names, leaves = ["dx"], [s["x"]]
    else:
        f = igs_amd.embedding_lookup(s["tokens"], s["weight"], scale=s["scale"], padding_idx=s["padding_idx"])
        y = igs_amd.layer_norm(f, s["w"], s["b"], eps=EPS, dropout_p=s["p"], seed=s["seed"], offset=s["offset"])
        names, leaves = ["dw", "db", "dweight"], [s["w"], s["b"], s["weight"]]
    out = {"y": y.detach()}
    if train:
        out.update(zip(names, torch.autograd.grad(y, leaves, s["grad"])))
    return out


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _run_plain(state)


def _distinct(case):
    """Expected number of different tokens in a case."""
    n, vocab = case["n"], case["vocab"]
    if case["skew"]:
        i = torch.arange(vocab, dtype=torch.float64)
        q = torch.log((i + 2) / (i + 1)) / math.log(vocab + 1)
    else:
        q = torch.full((vocab,), 1.0 / vocab, dtype=torch.float64)
    drawn = n - n // 8 if case["padded"] else n
    return float((1 - (1 - q) ** drawn).sum())


def work(case):
    dim, e, train = case["dim"], BYTES[case["dtype"]], case["train"]
    if case["op"] in ("embedding", "chain"):
        n, vocab = case["n"], case["vocab"]
        moved, flops = n * 8 + _distinct(case) * dim * e + n * dim * e, n * dim
        if train:  # the upstream gradient read, the dense gradient written
            moved, flops = moved + (n + vocab) * dim * e, flops + 2 * n * dim
        if case["op"] == "chain":
            moved, flops = moved + 4 * dim * 4, flops + 25 * n * dim
        return {"bytes": moved, "flops": flops}
    values = case["rows"] * dim
    moved = 2 * values * e * (2 if train else 1)
    if case["op"] == "dropout":
        return {"bytes": moved, "flops": values * (2 if train else 1)}
    moved += 2 * dim * BYTES[case["wdtype"]] * (2 if train else 1)
    return {"bytes": moved, "flops": values * (21 if train else 8)}


# ---------------------------------------------------------------------------------- the definitions in 64 bits
def _exact_keep(shape, p, seed, offset):
    import numpy as np

    count = math.prod(shape)
    mask, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    word = np.zeros((4, -(-count // 8)), dtype=np.uint64)
    word[0] = np.arange(word.shape[1], dtype=np.uint64)
    word[1] = word[0] >> half
    word[0] &= mask
    word[2], word[3] = offset % (1 << 32), offset // (1 << 32)
    key = [seed % (1 << 32), seed // (1 << 32)]
    for _ in range(7):
        a, b = word[0] * np.uint64(0xD2511F53), word[2] * np.uint64(0xCD9E8D57)
        word = np.stack([(b >> half) ^ word[1] ^ np.uint64(key[0]), b & mask,
                         (a >> half) ^ word[3] ^ np.uint64(key[1]), a & mask])
        key = [(key[0] + 0x9E3779B9) % (1 << 32), (key[1] + 0xBB67AE85) % (1 << 32)]
    u = np.ascontiguousarray(word.T.astype("<u4")).view("<u2").reshape(-1)[:count]
    t = int(p * 65536 + 0.5)
    keep = torch.from_numpy((u >= t).astype(np.float64)).reshape(shape).cuda()
    return keep * (65536.0 / (65536 - t))


def exact(case, seed):
    s = prepare(case, seed)
    s = {k: v.detach() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    up = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    out = {}
    op, train = case["op"], case["train"]
    if op in ("embedding", "chain"):
        x = torch.index_select(up["weight"], 0, s["tokens"]) * s["scale"]
    else:
        x = up["x"]
    keep = _exact_keep(x.shape, s["p"], s["seed"], s["offset"]) if s["p"] else None
    dy = up.get("grad")
    if op in ("norm", "chain"):
        var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
        h = (x - mean) * torch.rsqrt(var + EPS)
        y = torch.addcmul(up["b"], h, up["w"])
        if keep is not None:
            y = y * keep
        out["y"] = y
        if train:
            dy = dy * keep if keep is not None else dy
            out["dw"], out["db"] = torch.linalg.vecdot(dy, h, dim=0), torch.sum(dy, 0)
            # the Jacobian of the normalisation, applied by projecting dy w off the constant and off h
            g = dy * up["w"]
            g = g - torch.mean(g, -1, keepdim=True)
            dx = (g - h * (torch.linalg.vecdot(g, h) / x.shape[-1])[:, None]) * torch.rsqrt(var + EPS)
            if op == "norm":
                out["dx"] = dx
            dy = dx
    elif op == "dropout":
        out["y"] = x * keep
        if train:
            out["dx"] = dy * keep
    else:
        out["y"] = x
    if op in ("embedding", "chain") and train:
        order = torch.argsort(s["tokens"], stable=True)
        ids, counts = torch.unique_consecutive(s["tokens"][order], return_counts=True)
        dweight = torch.zeros_like(up["weight"])
        dweight[ids] = torch.segment_reduce(dy[order], "sum", lengths=counts, axis=0) * s["scale"]
        if s["padding_idx"] is not None:
            dweight[s["padding_idx"]] = 0
        out["dweight"] = dweight
    return out
