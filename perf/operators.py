"""The operators of ``igs_b200.features`` as measurable cases: what stands between an image's
tokens and the feature vectors that ``GaussianSplatting2D`` turns into gaussians.

* ``embed``: rows of a shared codebook by token, times a scale; its gradient adds up the
  upstream rows of every token.
* ``layer_norm``: every feature vector normalised to mean 0 and variance 1, times a weight, plus
  a bias; its gradient with the two column sums.
* ``dropout``: a share of the values set to zero by a counter-based generator; the mask is a
  function of (seed, offset, place) and is never stored.

``run`` computes a case in plain torch operations (``own = False``) or with the package's own
entry points (``own = True``).
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # One image decoded from its tokens: the module's own configuration (128 features of 1024
        # numbers), a codebook of 8192 rows, no gradient.  Latency.
        {"name": "embed_image", "op": "embed", "both": False, "type": "fp32", "batch": 1, "length": 128, "dim": 1024,
         "rows": 8192, "law": "uniform", "ragged": False, "index": "int64"},
        # A training batch of 64 images of 1024 tokens; some tokens (flat background) are far
        # commoner than others, so that one row's gradient has thousands of terms.
        {"name": "embed_batch", "op": "embed", "both": True, "type": "bf16", "batch": 64, "length": 1024, "dim": 1024,
         "rows": 16384, "law": "zipf", "ragged": False, "index": "int64"},
        # Images of different token counts in one padded batch, odd sizes throughout, 32-bit tokens.
        {"name": "embed_ragged", "op": "embed", "both": True, "type": "fp32", "batch": 48, "length": 577, "dim": 771,
         "rows": 5003, "law": "uniform", "ragged": True, "index": "int32"},
        # Few tokens against a large codebook: writing the gradient's zero rows is the work.
        {"name": "embed_table", "op": "embed", "both": True, "type": "bf16", "batch": 4, "length": 256, "dim": 1024,
         "rows": 131072, "law": "uniform", "ragged": False, "index": "int64"},
        # A single feature vector.  Latency.
        {"name": "norm_token", "op": "norm", "both": False, "type": "bf16", "weights": "bf16", "batch": 1, "length": 1,
         "dim": 1024},
        # The features of one image (the module's own configuration), no gradient.  Latency.
        {"name": "norm_image", "op": "norm", "both": False, "type": "fp32", "weights": "fp32", "batch": 1,
         "length": 128, "dim": 1024},
        # The same training batch as above, 16-bit features with 32-bit weights.
        {"name": "norm_train", "op": "norm", "both": True, "type": "bf16", "weights": "fp32", "batch": 64,
         "length": 1024, "dim": 1024},
        # A width that is a multiple of nothing.
        {"name": "norm_odd", "op": "norm", "both": True, "type": "fp32", "weights": "fp32", "batch": 9, "length": 777,
         "dim": 1111},
        # Wide feature vectors.
        {"name": "norm_wide", "op": "norm", "both": True, "type": "fp16", "weights": "fp16", "batch": 16,
         "length": 128, "dim": 8192},
        # The features of one image during a fit: forward and gradient.  Latency.
        {"name": "dropout_image", "op": "dropout", "both": True, "type": "fp32", "batch": 1, "length": 128,
         "dim": 1024, "p": 0.1},
        # The training batch.
        {"name": "dropout_train", "op": "dropout", "both": True, "type": "bf16", "batch": 64, "length": 1024,
         "dim": 1024, "p": 0.1},
        # Odd sizes, every other value dropped.
        {"name": "dropout_odd", "op": "dropout", "both": True, "type": "fp16", "batch": 13, "length": 1009,
         "dim": 517, "p": 0.5},
    ]


MOST_BYTES = 1 << 27  # of one [batch, length, dim] tensor: the largest listed ones


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: lengths from a single token to the training batch, widths from 16 to 8192."""
    op = rng.choice(["embed", "norm", "dropout"])
    case = {"op": op, "both": rng.random() < (0.75 if op != "dropout" else 1.0),
            "type": rng.choice(["fp32", "bf16", "fp16"])}
    dim = _spread(rng, 16, 8192)
    if rng.random() < 0.5:  # half of the widths are the round ones that models have
        dim = max(16, dim // 64 * 64)
    most = MOST_BYTES // (dim * SIZE[case["type"]])
    batch = _spread(rng, 1, min(64, most))
    case.update(batch=batch, length=_spread(rng, 1, min(2048, max(1, most // batch))), dim=dim)
    if op == "embed":
        rows = _spread(rng, 16, 131072)
        case.update(rows=max(1, min(rows, (1 << 28) // (dim * SIZE[case["type"]]))),
                    law=rng.choice(["uniform", "zipf"]), ragged=rng.random() < 0.5,
                    index=rng.choice(["int64", "int32"]))
    elif op == "norm":
        case.update(weights=rng.choice(["fp32", case["type"]]))
    else:
        case.update(p=rng.choice([0.05, 0.1, 0.25, 0.5]))
    return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
EMPTY = -1  # the token of a place behind an image's last one
EPS = 1e-5


def _shares(case):
    """The probability of every codebook row."""
    v = np.arange(1, case["rows"] + 1, dtype=np.float64)
    p = 1.0 / v if case["law"] == "zipf" else np.ones_like(v)
    return p / p.sum()


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    dtype = DTYPES[case["type"]]
    shape = (case["batch"], case["length"], case["dim"])

    def normal(*size, std=1.0, mean=0.0, dtype=dtype):
        return torch.randn(*size, generator=gen, device=dev).mul_(std).add_(mean).to(dtype)

    s = {"case": dict(case)}
    if case["op"] == "embed":
        # (the running sum of the shares is taken on the host: on the GPU its last bits change from one
        # call to the next, and with them a few of the tokens)
        upto = torch.from_numpy(np.cumsum(_shares(case))).to(dev)
        n = case["batch"] * case["length"]
        at = torch.rand(n, generator=gen, device=dev, dtype=torch.float64)
        rank = torch.searchsorted(upto, at, right=True).clamp_(max=case["rows"] - 1)
        place = torch.randperm(case["rows"], generator=gen, device=dev)  # common tokens lie anywhere in the table
        tokens = place[rank].view(case["batch"], case["length"])
        if case["ragged"]:
            lengths = torch.randint(0, case["length"] + 1, (case["batch"], 1), generator=gen, device=dev)
            tokens = torch.where(torch.arange(case["length"], device=dev) < lengths, tokens, EMPTY)
        s["tokens"] = tokens.to(torch.int32 if case["index"] == "int32" else torch.int64)
        s["empty"] = EMPTY if case["ragged"] else None
        s["scale"] = math.sqrt(case["dim"])
        s["table"] = normal(case["rows"], case["dim"], std=case["dim"] ** -0.5).requires_grad_(case["both"])
    elif case["op"] == "norm":
        wtype = DTYPES[case["weights"]]
        spread = torch.rand(shape[0], shape[1], 1, generator=gen, device=dev).mul_(2.75).add_(0.25)  # 0.25 to 3
        centre = torch.randn(shape[0], shape[1], 1, generator=gen, device=dev)
        x = torch.randn(shape, generator=gen, device=dev).mul_(spread).add_(centre).to(dtype)
        s["x"] = x.requires_grad_(case["both"])
        s["weight"] = normal(case["dim"], std=0.1, mean=1.0, dtype=wtype).requires_grad_(case["both"])
        s["bias"] = normal(case["dim"], std=0.1, dtype=wtype).requires_grad_(case["both"])
    else:
        s["x"] = normal(*shape).requires_grad_(case["both"])
        # (seed, offset): one generator state, as a training loop keeps it on the device
        s["state"] = torch.randint(0, 1 << 62, (2,), generator=gen, device=dev)
    if case["both"]:
        s["dy"] = normal(*shape, std=0.05)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return _OWN[case["op"]](state, case["both"])
    with torch.no_grad():
        return _PLAIN[case["op"]](state, case["both"])


def _own_embed(s, both):
    from igs_b200 import features

    y = features.embed(s["tokens"], s["table"], scale=s["scale"], empty=s["empty"])
    if not both:
        return {"y": y}
    (g,) = torch.autograd.grad(y, (s["table"],), s["dy"])
    return {"y": y.detach(), "d_table": g}


def _own_norm(s, both):
    from igs_b200 import features

    y = features.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS)
    if not both:
        return {"y": y}
    gx, gw, gb = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])
    return {"y": y.detach(), "d_x": gx, "d_weight": gw, "d_bias": gb}


def _own_dropout(s, both):
    from igs_b200 import features

    y = features.dropout(s["x"], s["case"]["p"], s["state"])
    if not both:
        return {"y": y}
    (g,) = torch.autograd.grad(y, (s["x"],), s["dy"])
    return {"y": y.detach(), "d_x": g}


def _plain_embed(s, both):
    tokens, table, scale = s["tokens"].long(), s["table"], s["scale"]
    rows, dim = table.shape
    if s["empty"] is None:
        y = (table[tokens].float() * scale).to(table.dtype)
        there = None
    else:
        there = tokens != s["empty"]
        y = table[torch.where(there, tokens, 0)].float() * scale
        y = torch.where(there[..., None], y, 0.0).to(table.dtype)
    if not both:
        return {"y": y}
    # places without a token add to a row behind the table's last
    keys = tokens if there is None else torch.where(there, tokens, rows)
    g = torch.zeros(rows + 1, dim, device=table.device)
    g.index_add_(0, keys.reshape(-1), s["dy"].float().reshape(-1, dim))
    return {"y": y, "d_table": (g[:rows] * scale).to(table.dtype)}


def _plain_norm(s, both):
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    xc = x - x.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((xc * xc).mean(-1, keepdim=True) + EPS)
    xhat = xc * rstd
    y = (xhat * w + b).to(s["x"].dtype)
    if not both:
        return {"y": y}
    dy = s["dy"].float()
    g = dy * w
    gx = (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True)) * rstd
    gw, gb = (dy * xhat).sum((0, 1)), dy.sum((0, 1))
    return {"y": y, "d_x": gx.to(s["x"].dtype), "d_weight": gw.to(s["weight"].dtype), "d_bias": gb.to(s["bias"].dtype)}


# Philox4x32 with 7 rounds (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2,
# 3", 2011).  Value i of the tensor takes word i % 4 of the block whose counter is (i // 4, offset),
# both as 64-bit numbers, and whose key is the seed; it is kept when the word is at least p * 2^32.
PHILOX_M = (0xD2511F53, 0xCD9E8D57)
PHILOX_W = (0x9E3779B9, 0xBB67AE85)
PHILOX_ROUNDS = 7
M32 = 0xFFFFFFFF


def _philox_words(blocks, state):
    """[blocks, 4] random words as int64; products of two 32-bit numbers wrap in 64 bits, their
    upper half is masked out again."""
    q = torch.arange(blocks, device=state.device)
    seed, offset = state[0], state[1]
    c0, c1 = q & M32, q >> 32
    c2, c3 = (offset & M32).expand(blocks), ((offset >> 32) & M32).expand(blocks)
    k0, k1 = seed & M32, (seed >> 32) & M32
    for _ in range(PHILOX_ROUNDS):
        a, b = c0 * PHILOX_M[0], c2 * PHILOX_M[1]
        c0, c1, c2, c3 = ((b >> 32) & M32) ^ c1 ^ k0, b & M32, ((a >> 32) & M32) ^ c3 ^ k1, a & M32
        k0, k1 = (k0 + PHILOX_W[0]) & M32, (k1 + PHILOX_W[1]) & M32
    return torch.stack([c0, c1, c2, c3], -1)


def _plain_dropout(s, both):
    x, p = s["x"], s["case"]["p"]
    n = x.numel()
    words = _philox_words((n + 3) // 4, s["state"]).reshape(-1)[:n].view(x.shape)
    keep = words >= int(p * 2.0 ** 32)
    scale = 1.0 / (1.0 - p)
    y = torch.where(keep, x.float() * scale, 0.0).to(x.dtype)
    if not both:
        return {"y": y}
    return {"y": y, "d_x": torch.where(keep, s["dy"].float() * scale, 0.0).to(x.dtype)}


_OWN = {"embed": _own_embed, "norm": _own_norm, "dropout": _own_dropout}
_PLAIN = {"embed": _plain_embed, "norm": _plain_norm, "dropout": _plain_dropout}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    n = case["batch"] * case["length"]
    size = SIZE[case["type"]]
    one = n * case["dim"] * size  # one pass over a [batch, length, dim] tensor
    values = n * case["dim"]
    if case["op"] == "embed":
        index = n * (4 if case["index"] == "int32" else 8)
        # half of a ragged batch's places hold a token, on average; the others' upstream rows are not needed
        held = n * (0.5 if case["ragged"] else 1.0)
        touched = float((1.0 - (1.0 - _shares(case)) ** held).sum()) * case["dim"] * size
        if not case["both"]:
            return {"bytes": int(index + touched + one), "flops": int(values)}
        table = case["rows"] * case["dim"] * size
        return {"bytes": int(index + touched + one + one * held / n + table), "flops": int(values + held * case["dim"])}
    if case["op"] == "norm":
        weights = 2 * case["dim"] * SIZE[case["weights"]]
        if not case["both"]:
            return {"bytes": 2 * one + weights, "flops": 8 * values}
        return {"bytes": 4 * one + 2 * weights, "flops": 20 * values}
    return {"bytes": (4 if case["both"] else 2) * one, "flops": (4 if case["both"] else 2) * values}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _EXACT[case["op"]](s, case["both"])


def _exact_embed(s, both):
    table = s["table"].double() * s["scale"]
    rows, dim = table.shape
    table = torch.cat([table, table.new_zeros(1, dim)])  # the row of places without a token
    at = s["tokens"].long().reshape(-1)
    if s["empty"] is not None:
        at = at.masked_fill(at == s["empty"], rows)
    res = {"y": table.index_select(0, at).view(*s["tokens"].shape, dim)}
    if both:
        # upstream rows in the order of their tokens, then differences of running sums at the borders
        order = torch.argsort(at, stable=True)
        ends = torch.searchsorted(at[order], torch.arange(rows, device=at.device), right=True)
        out = []
        for cols in s["dy"].reshape(-1, dim).split(256, dim=1):
            run_sum = torch.cat([table.new_zeros(1, cols.shape[1]), cols.double()[order].cumsum(0)])
            upto = run_sum[ends]
            out.append(torch.diff(upto, dim=0, prepend=table.new_zeros(1, cols.shape[1])) * s["scale"])
        res["d_table"] = torch.cat(out, 1)
    return res


def _exact_norm(s, both):
    x, w, b = (s[k].double() for k in ("x", "weight", "bias"))
    var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
    sd = (var + EPS).sqrt()
    z = (x - mean) / sd
    res = {"y": torch.addcmul(b, z, w)}
    if both:
        dy, d = s["dy"].double(), x.shape[-1]
        g = dy * w
        along = torch.einsum("bld,bld->bl", g, z)[..., None]
        res["d_x"] = (d * g - g.sum(-1, keepdim=True) - z * along) / (d * sd)
        res["d_weight"] = torch.einsum("bld,bld->d", dy, z)
        res["d_bias"] = torch.einsum("bld->d", dy)
    return res


def _exact_dropout(s, both):
    x, p = s["x"], s["case"]["p"]
    seed, offset = (int(v) for v in s["state"].tolist())
    n = x.numel()
    blocks = (n + 3) // 4
    lo = np.uint64(M32)
    half = np.uint64(32)
    ctr = np.zeros((4, blocks), np.uint64)
    ctr[0] = np.arange(blocks, dtype=np.uint64) & lo
    ctr[1] = np.arange(blocks, dtype=np.uint64) >> half
    ctr[2], ctr[3] = offset & M32, offset >> 32
    key = [seed & M32, seed >> 32]
    for _ in range(PHILOX_ROUNDS):
        prod = [ctr[0] * np.uint64(PHILOX_M[0]), ctr[2] * np.uint64(PHILOX_M[1])]
        ctr = np.stack([(prod[1] >> half) ^ ctr[1] ^ np.uint64(key[0]), prod[1] & lo,
                        (prod[0] >> half) ^ ctr[3] ^ np.uint64(key[1]), prod[0] & lo])
        key = [(k + w) & M32 for k, w in zip(key, PHILOX_W)]
    words = torch.from_numpy(ctr.T.reshape(-1)[:n].astype(np.int64)).to(x.device).view(x.shape)
    factor = (words >= int(p * 2.0 ** 32)).double() / (1.0 - p)
    res = {"y": x.double() * factor}
    if both:
        res["d_x"] = s["dy"].double() * factor
    return res


_EXACT = {"embed": _exact_embed, "norm": _exact_norm, "dropout": _exact_dropout}
