"""The feature operators (igs_b200.features) on the GPU against their 64-bit forms, within the
bounds of tests/_features_ref.py, at the sizes, layouts and values where they can go wrong."""
import gc

import numpy as np
import pytest
import torch

from tests import _features_ref as ref

pytestmark = pytest.mark.gpu
TYPES = ["fp32", "bf16", "fp16"]


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def _normal(gen, *shape, dtype=torch.float32, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=gen, device=gen.device) * std + mean).to(dtype)


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


# ---------------------------------------------------------------------------
# embedding
# ---------------------------------------------------------------------------
def _check_embed(tokens, table, dy, scale=1.0, empty=None, what=""):
    from igs_b200 import features

    leaf = table.detach().requires_grad_()
    y = features.embed(tokens, leaf, scale=scale, empty=empty)
    assert y.shape == (*tokens.shape, table.shape[1]) and y.dtype == table.dtype and y.is_contiguous()
    tok = tokens.cpu().numpy().astype(np.int64)
    want, err = ref.embed(tok, ref.f64(table), scale, empty)
    ref.assert_within(y, want, err, what + " y")
    with torch.no_grad():
        # (compared as integers: NaN rows count as equal when their bits are)
        bits = torch.int32 if y.dtype == torch.float32 else torch.int16
        assert torch.equal(features.embed(tokens, table, scale=scale, empty=empty).view(bits), y.detach().view(bits))
    (g,) = torch.autograd.grad(y, leaf, dy)
    assert g.shape == table.shape and g.dtype == table.dtype
    want, err = ref.embed_grad(tok, ref.f64(dy), table.shape[0], scale, empty)
    ref.assert_within(g, want, err, what + " d_table")
    return y, g


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,rows,D", [
    (1, 1, 1), (1, 7, 1024), (2, 3, 5), (31, 2, 33), (33, 1000, 64), (257, 16, 129), (500, 501, 8), (1024, 300, 96),
    (2047, 5, 40), (2049, 1030, 72), (4097, 70000, 24), (9001, 1 << 20, 3), (20011, 257, 17),
    (9001, 16384, 9), (9500, 16385, 7), (8193, 1024, 6), (8193, 1025, 6), (151552, 1025, 4), (151553, 2048, 4)])
def test_embed_sizes(dev, dtype, n, rows, D):
    gen = _gen(dev, n * 31 + D)
    t = ref.DTYPES[dtype]
    tokens = torch.randint(0, rows, (n,), generator=gen, device=dev)
    _check_embed(tokens, _normal(gen, rows, D, dtype=t), _normal(gen, n, D, dtype=t), scale=1.7)


@pytest.mark.parametrize("n,rows,D", [(70000, 300, 240), (17001, 5000, 1000), (33000, (1 << 20) + 9, 520)])
def test_embed_many_places_of_wide_rows(dev, n, rows, D):
    """The sort of many places in one, two and three passes, over wide rows; some places empty."""
    gen = _gen(dev, n)
    tokens = torch.randint(-1, rows, (n,), generator=gen, device=dev)
    tokens[: n // 3] = tokens[0].clamp(min=0)  # a run over many chunks
    from igs_b200 import features

    table = torch.zeros(rows, D, device=dev, requires_grad=True)
    dy = _normal(gen, n, D)
    (g,) = torch.autograd.grad(features.embed(tokens, table, empty=-1), table, dy)
    # the rows that have a token, in 64 bits on the device; all others are zero
    held = tokens >= 0
    uniq, at, times = torch.unique(tokens[held], return_inverse=True, return_counts=True)
    want = torch.zeros(len(uniq), D, dtype=torch.float64, device=dev).index_add_(0, at, dy[held].double())
    size = torch.zeros_like(want).index_add_(0, at, dy[held].double().abs())
    assert ((g[uniq].double() - want).abs() <= 1.01 * ref.U * times[:, None] * size + 1e-40).all()
    g[uniq] = 0
    assert not g.any()


@pytest.mark.parametrize("n", [40, 3000, 12000, 70000])
@pytest.mark.parametrize("kind", ["one_token", "two_tokens", "first_and_last", "sorted", "reversed", "common"])
def test_embed_token_patterns(dev, kind, n):
    """Runs of every length across the borders of the chunks that the sums are cut into."""
    rows, D = 1500, 20
    gen = _gen(dev, n)
    i = torch.arange(n, device=dev)
    tokens = {"one_token": torch.full_like(i, 77), "two_tokens": torch.where(i % 3 == 0, 5, 1499),
              "first_and_last": torch.where(i < n // 2, 0, rows - 1), "sorted": i * rows // n,
              "reversed": (n - 1 - i) * rows // n,
              "common": torch.where(torch.rand(n, generator=gen, device=dev) < 0.7, 700,
                                    torch.randint(0, rows, (n,), generator=gen, device=dev))}[kind]
    _check_embed(tokens, _normal(gen, rows, D), _normal(gen, n, D), what=kind)


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("empty", [-1, 3, 10 ** 6])
def test_embed_padded_batch(dev, index, empty):
    """Ragged lengths, zero among them; the empty token may lie inside or outside the table."""
    gen = _gen(dev, 5)
    tokens = torch.randint(0, 60, (6, 50), generator=gen, device=dev)
    lengths = torch.tensor([50, 0, 1, 17, 49, 32], device=dev)
    tokens = torch.where(torch.arange(50, device=dev) < lengths[:, None], tokens, empty).to(index)
    table, dy = _normal(gen, 60, 36), _normal(gen, 6, 50, 36)
    dy[tokens == empty] = float("nan")  # what comes back for empty places does not matter
    y, g = _check_embed(tokens, table, dy, empty=empty)
    assert (y[tokens == empty] == 0).all() and torch.isfinite(g).all()
    if empty == 3:
        assert (g[3] == 0).all()


def test_embed_nothing_held(dev):
    """No tokens at all, and only empty places: zeros everywhere."""
    gen = _gen(dev, 6)
    table = _normal(gen, 9, 12)
    y, g = _check_embed(torch.zeros(0, dtype=torch.int64, device=dev), table, _normal(gen, 0, 12))
    assert (g == 0).all()
    for n in (1, 100, 20000):
        y, g = _check_embed(torch.full((n,), -1, device=dev), table, _normal(gen, n, 12), empty=-1)
        assert (y == 0).all() and (g == 0).all()


@pytest.mark.parametrize("n", [64, 20000])
def test_embed_tokens_outside_the_table(dev, n):
    """A row of NaN and no gradient, for every kind of outside; neighbours stay what they are."""
    gen = _gen(dev, 8)
    tokens = torch.randint(0, 11, (n,), generator=gen, device=dev)
    for k, bad in enumerate((11, -1, -(1 << 62), (1 << 62), (1 << 32) + 2, -(1 << 32))):
        tokens[k * 9] = bad
    y, g = _check_embed(tokens, _normal(gen, 11, 16, dtype=torch.bfloat16), _normal(gen, n, 16, dtype=torch.bfloat16))
    assert y[0].isnan().all() and torch.isfinite(g.float()).all()


def test_embed_strides_and_shapes(dev):
    gen = _gen(dev, 9)
    wide = _normal(gen, 40, 50)
    tokens = torch.randint(0, 40, (4, 6, 8), generator=gen, device=dev)
    dy = _normal(gen, 4, 6, 8, 19)
    for table in (wide[:, 3:22], wide[:, ::2][:, :19], wide.t()[:40, :19], wide[::2, :19].repeat(2, 1)[:40]):
        _check_embed(tokens, table, dy)
    # rows on 16-byte boundaries, and one element behind them
    for first in (0, 1, 4):
        table = wide[:, first:first + 32]
        _check_embed(tokens, table, _normal(gen, 4, 6, 8, 32))
    _check_embed(tokens[:, ::2, 1:5], wide, _normal(gen, 4, 3, 4, 50))           # strided tokens
    _check_embed(tokens[0, 0, 0], wide, _normal(gen, 50))                        # a single token without a batch
    _check_embed(tokens[..., 0], wide, _normal(gen, 1, 1, 50).expand(4, 6, 50))  # an upstream gradient of stride 0
    shared = _normal(gen, 1, 50).expand(40, 50)                                  # all rows the same memory
    _check_embed(tokens[0], shared, _normal(gen, 6, 8, 50))


def test_embed_offsets_beyond_32_bits(dev):
    """A table of more than 2^31 numbers, places in its last rows."""
    from igs_b200 import features

    rows, D = (1 << 21) + 5, 1030
    assert rows * D > 1 << 31
    table = torch.zeros(rows, D, dtype=torch.bfloat16, device=dev)
    at = torch.tensor([0, rows - 1, rows // 2, rows - 1], device=dev)
    vals = _normal(_gen(dev, 1), 4, D, dtype=torch.bfloat16)
    vals[3] = vals[1]
    table[at] = vals
    table.requires_grad_()
    y = features.embed(at, table)
    assert torch.equal(y, vals)
    (g,) = torch.autograd.grad(y, table, torch.ones_like(vals))
    assert (g[0] == 1).all() and (g[rows // 2] == 1).all() and (g[rows - 1] == 2).all()
    assert int((g != 0).any(1).sum()) == 3
    del y, g, table
    torch.cuda.empty_cache()


# ---------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------
def _check_norm(x, w, b, dy, eps=1e-5, what=""):
    from igs_b200 import features

    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b)]
    y = features.layer_norm(*leaves, eps=eps)
    assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous()
    with torch.no_grad():
        assert torch.equal(features.layer_norm(x, w, b, eps=eps), y.detach())
    D = x.shape[-1]
    f = ref.layer_norm(ref.f64(x).reshape(-1, D), None if w is None else ref.f64(w), None if b is None else ref.f64(b), eps)
    ref.assert_within(y.reshape(-1, D), f["y"], f["e_y"], what + " y")
    g = ref.layer_norm_grad(f, ref.f64(dy).reshape(-1, D))
    got = torch.autograd.grad(y, [t for t in leaves if t is not None], dy)
    assert got[0].shape == x.shape and got[0].dtype == x.dtype
    ref.assert_within(got[0].reshape(-1, D), g["dx"], g["e_dx"], what + " dx")
    rest = list(got[1:])
    for t, name in ((w, "dw"), (b, "db")):
        if t is not None:
            r = rest.pop(0)
            assert r.dtype == t.dtype
            ref.assert_within(r, g[name], g["e_" + name], what + " " + name)
    return y, got


@pytest.mark.parametrize("dtype,wtype", [("fp32", "fp32"), ("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp16"),
                                         ("fp16", "fp32")])
@pytest.mark.parametrize("rows,D", [
    (1, 1), (1, 1024), (3, 2), (2, 31), (5, 33), (70, 64), (33, 100), (17, 127), (9, 256), (130, 257), (8, 512), (65, 520),
    (40, 1000), (128, 1024), (7, 1111), (6, 1536), (5, 2047), (12, 2048), (3, 4100), (4, 8192), (2, 16384), (3, 16392),
    (2, 20001), (2500, 16), (700, 48)])
def test_layer_norm_sizes(dev, dtype, wtype, rows, D):
    gen = _gen(dev, rows * 131 + D)
    t, wt = ref.DTYPES[dtype], ref.DTYPES[wtype]
    x = _normal(gen, rows, D, dtype=t, std=2.0, mean=0.3)
    _check_norm(x, _normal(gen, D, dtype=wt, std=0.5, mean=1.0), _normal(gen, D, dtype=wt), _normal(gen, rows, D, dtype=t))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [24, 1000, 5000, 17001])
def test_layer_norm_optional_parts(dev, dtype, D):
    gen = _gen(dev, D)
    t = ref.DTYPES[dtype]
    x, dy = _normal(gen, 2, 3, D, dtype=t), _normal(gen, 2, 3, D, dtype=t)
    w, b = _normal(gen, D, dtype=t), _normal(gen, D, dtype=t)
    for ws in ((None, None), (w, None), (None, b)):
        _check_norm(x, *ws, dy)


def test_layer_norm_only_what_is_asked_for(dev):
    """Gradients of some inputs alone are the same bits as of all."""
    from igs_b200 import features

    gen = _gen(dev, 2)
    x, w, b, dy = _normal(gen, 30, 96), _normal(gen, 96), _normal(gen, 96), _normal(gen, 30, 96)
    _, (gx, gw, gb) = _check_norm(x, w, b, dy)
    for k, want in enumerate((gx, gw, gb)):
        leaves = [x.clone(), w.clone(), b.clone()]
        leaves[k].requires_grad_()
        (g,) = torch.autograd.grad(features.layer_norm(*leaves), leaves[k], dy)
        assert torch.equal(g, want)


@pytest.mark.parametrize("D", [64, 1024, 3001, 9000, 20000])
def test_layer_norm_hard_rows(dev, D):
    """Constant rows (variance 0: exactly the bias), rows far from zero, tiny and huge rows."""
    gen = _gen(dev, D)
    x = _normal(gen, 8, D)
    x[0], x[1] = 0.0, 1234.567
    x[2] = x[2] * 0.01 + 300.0
    x[3] *= 1e-6
    x[4] *= 1e12
    x[5, 1:] = 0.0
    w, b, dy = _normal(gen, D), _normal(gen, D), _normal(gen, 8, D)
    y, (gx, _, _) = _check_norm(x, w, b, dy)
    assert torch.equal(y[0], b) and torch.equal(y[1], b)
    _check_norm(x[2:], w, b, dy[2:], eps=0.0)


@pytest.mark.parametrize("D", [40, 1024, 9000, 17000])
def test_layer_norm_not_finite(dev, D):
    """A row with an infinity or NaN is NaN throughout; the other rows do not notice."""
    from igs_b200 import features

    gen = _gen(dev, D)
    x, w, b, dy = _normal(gen, 9, D), _normal(gen, D), _normal(gen, D), _normal(gen, 9, D)
    clean, (gclean, _, _) = _check_norm(x, w, b, dy)
    bad = x.clone()
    bad[2, D // 3], bad[5, 0], bad[7, D - 1] = float("inf"), float("nan"), float("-inf")
    bad.requires_grad_()
    y = features.layer_norm(bad, w, b)
    (g,) = torch.autograd.grad(y, bad, dy)
    for r in range(9):
        if r in (2, 5, 7):
            assert y[r].isnan().all() and g[r].isnan().all()
        else:
            assert torch.equal(y[r], clean[r]) and torch.equal(g[r], gclean[r])


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_layer_norm_strides(dev, dtype):
    gen, t = _gen(dev, 4), ref.DTYPES[dtype]
    wide = _normal(gen, 30, 4, 200, dtype=t)
    w, b = _normal(gen, 400, dtype=t)[::2], _normal(gen, 200, dtype=t)
    for x in (wide[:, 1], wide[::2, 2], wide.transpose(0, 1), wide[..., 1:], wide[0, 0], wide[:1, :3], wide[:, 0, 8:136],
              wide[:, 0, 3:131], wide[:, 0].t().contiguous().t(), wide[:1, 0].expand(7, 200), wide[:, :, ::2]):
        D = x.shape[-1]
        _check_norm(x, w[:D], b[:D], _normal(gen, *x.shape, dtype=t))
    x = wide[:, 0]
    _check_norm(x, w, b, _normal(gen, 1, 200, dtype=t).expand(30, 200))
    one_behind = b.new_empty(201)[1:].copy_(b)  # weights off their 16-byte boundary
    _check_norm(x, one_behind, one_behind, _normal(gen, 30, 200, dtype=t))


def test_layer_norm_no_rows(dev):
    gen = _gen(dev, 4)
    for shape in ((0, 32), (3, 0, 32)):
        y, (gx, gw, gb) = _check_norm(_normal(gen, *shape), _normal(gen, 32), _normal(gen, 32), _normal(gen, *shape))
        assert (gw == 0).all() and (gb == 0).all()


@pytest.mark.parametrize("rows,D", [(5000, 1024), (3001, 520), (40000, 64), (601, 8192)])
def test_layer_norm_many_rows(dev, rows, D):
    gen = _gen(dev, rows)
    x, dy = _normal(gen, rows, D, dtype=torch.bfloat16), _normal(gen, rows, D, dtype=torch.bfloat16)
    _check_norm(x, _normal(gen, D), _normal(gen, D), dy)


def test_layer_norm_offsets_beyond_32_bits(dev):
    """More than 2^31 values: the last rows are the same bits as in a call of their own, and a
    constant upstream gradient of one in the last row alone is found by the column sums."""
    from igs_b200 import features

    rows, D = (1 << 21) + 3, 1032
    x = torch.zeros(rows, D, dtype=torch.bfloat16, device=dev)
    tail = _normal(_gen(dev, 3), 5, D, dtype=torch.bfloat16)
    x[-5:] = tail
    w, b = _normal(_gen(dev, 4), D), _normal(_gen(dev, 5), D)
    x.requires_grad_()
    b.requires_grad_()
    y = features.layer_norm(x, w, b)
    with torch.no_grad():
        assert torch.equal(y[-5:], features.layer_norm(tail, w, b))
    dy = torch.zeros_like(y)
    dy[-1] = 1
    gx, gb = torch.autograd.grad(y, (x, b), dy)
    del y, dy
    assert (gb == 1).all()
    leaf = tail.clone().requires_grad_()
    dt = torch.zeros_like(tail)
    dt[-1] = 1
    (gt,) = torch.autograd.grad(features.layer_norm(leaf, w, b.detach()), leaf, dt)
    assert torch.equal(gx[-5:], gt) and not gx[:-5].any()
    del x, gx
    torch.cuda.empty_cache()


# ---------------------------------------------------------------------------
# dropout
# ---------------------------------------------------------------------------
def _check_dropout(x, p, seed, offset, dy, use_state, what=""):
    from igs_b200 import features

    leaf = x.detach().requires_grad_()
    signed = lambda v: v - (1 << 64) if v >= 1 << 63 else v
    # the tensor form: its offset and the argument add up
    args = (torch.tensor([signed(seed), signed((offset - 3) % (1 << 64))], device=x.device), 3) if use_state else (seed, offset)
    y = features.dropout(leaf, p, *args)
    assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous()
    want, err = ref.dropout(ref.f64(x).reshape(-1), p, seed, offset)
    ref.assert_within(y.reshape(-1), want, err, what + " y")
    (g,) = torch.autograd.grad(y, leaf, dy)
    want, err = ref.dropout(ref.f64(dy).reshape(-1), p, seed, offset)
    ref.assert_within(g.reshape(-1), want, err, what + " dx")
    return y, g


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1,), (3,), (4,), (5,), (7, 9), (2, 3, 8), (1023,), (16, 64), (33, 129), (4, 2048), (70001,),
                                   (1, 128, 1024)])
def test_dropout_sizes(dev, dtype, shape):
    gen, t = _gen(dev, 11), ref.DTYPES[dtype]
    x, dy = _normal(gen, *shape, dtype=t), _normal(gen, *shape, dtype=t)
    _check_dropout(x, 0.3, 0x1234567890ABCDEF, 17, dy, False)
    _check_dropout(x, 0.3, 0xF234567890ABCDEF, (1 << 64) - 1, dy, True)


@pytest.mark.parametrize("p", [0.0, 1e-9, 2.0 ** -32, 0.1, 0.5, 0.999, 1.0 - 2.0 ** -32, 1.0])
def test_dropout_shares(dev, p):
    gen = _gen(dev, 12)
    x, dy = _normal(gen, 9999), _normal(gen, 9999)
    y, _ = _check_dropout(x, p, 5, 6, dy, False)
    if p == 0.0:
        assert torch.equal(y, x)


def test_dropout_not_finite(dev):
    """A dropped value is zero whatever was there; a kept one keeps its infinity or NaN."""
    from igs_b200 import features

    keep = torch.from_numpy(ref.words(0, 400, 9, 0) >= np.uint64(1 << 31)).to(dev)
    for v in (float("inf"), float("-inf"), float("nan"), torch.finfo(torch.float32).min):
        y = features.dropout(torch.full((400,), v, device=dev), 0.5, 9)
        assert (y[~keep] == 0).all() and not torch.isfinite(y[keep]).any()
    assert (features.dropout(torch.full((400,), float("nan"), device=dev), 1.0, 9) == 0).all()


def test_dropout_strides_and_empty(dev):
    gen = _gen(dev, 13)
    wide = _normal(gen, 12, 30)
    for x in (wide.t(), wide[:, 1:], wide[::2], wide[:, :1].expand(12, 30), wide[0, 0], wide.reshape(-1)[1:]):
        _check_dropout(x, 0.25, 3, 4, _normal(gen, *x.shape), False)
    off = torch.empty(1001, dtype=torch.bfloat16, device=dev)[1:].normal_(generator=gen)  # off its 16-byte boundary
    _check_dropout(off, 0.25, 3, 4, _normal(gen, 1000, dtype=torch.bfloat16), True)
    assert wide[:0].numel() == 0
    _check_dropout(wide[:0], 0.25, 3, 4, wide[:0], False)


def test_dropout_offsets_beyond_32_bits(dev):
    from igs_b200 import features

    n, look = (1 << 31) + 4096 + 3, 4099
    x = torch.ones(n, dtype=torch.bfloat16, device=dev)
    y = features.dropout(x, 0.5, 77, 2)
    for first in (0, (1 << 31) - 2048, n - look):
        first -= first % 4
        want, err = ref.dropout(np.ones(min(look, n - first)), 0.5, 77, 2, first)
        ref.assert_within(y[first:first + want.size], want, err, f"from {first}")
    del x, y
    torch.cuda.empty_cache()


# ---------------------------------------------------------------------------
# all three: refusals, repeatability, streams, graphs, differences
# ---------------------------------------------------------------------------
def test_refusals(dev):
    from igs_b200 import features

    x = torch.zeros(3, 4, device=dev)
    tok = torch.zeros(2, dtype=torch.int64, device=dev)
    for call, exc in [
        (lambda: features.embed(tok, x.double()), TypeError), (lambda: features.embed(tok.float(), x), TypeError),
        (lambda: features.embed(tok.to(torch.int16), x), TypeError), (lambda: features.embed([0, 1], x), TypeError),
        (lambda: features.embed(tok.cpu(), x), RuntimeError), (lambda: features.embed(tok, x[0]), ValueError),
        (lambda: features.embed(tok, x[:0]), ValueError), (lambda: features.embed(tok, x[:, :0]), ValueError),
        (lambda: features.embed(tok, x, scale=float("nan")), ValueError),
        (lambda: features.embed(tok, x, scale=1e39), ValueError), (lambda: features.embed(tok, x, empty=1.5), TypeError),
        (lambda: features.embed(tok, x, empty=1 << 63), ValueError),
        (lambda: features.layer_norm(x.long()), TypeError), (lambda: features.layer_norm(x[0, 0]), ValueError),
        (lambda: features.layer_norm(x[:, :0]), ValueError), (lambda: features.layer_norm(x, x[0, :3]), ValueError),
        (lambda: features.layer_norm(x, x), ValueError), (lambda: features.layer_norm(x, x[0].half()), TypeError),
        (lambda: features.layer_norm(x.half(), x[0], x[0].half()), TypeError),
        (lambda: features.layer_norm(x.half(), x[0].bfloat16()), TypeError),
        (lambda: features.layer_norm(x, x[0].cpu()), RuntimeError), (lambda: features.layer_norm(x, eps=-1e-5), ValueError),
        (lambda: features.layer_norm(x, eps=float("inf")), ValueError),
        (lambda: features.dropout(x, -0.1, 0), ValueError), (lambda: features.dropout(x, 1.1, 0), ValueError),
        (lambda: features.dropout(x, float("nan"), 0), ValueError), (lambda: features.dropout(x, 0.5, -1), ValueError),
        (lambda: features.dropout(x, 0.5, 1 << 64), ValueError), (lambda: features.dropout(x, 0.5, 0, -1), ValueError),
        (lambda: features.dropout(x, 0.5, 0.5), TypeError), (lambda: features.dropout(x, 0.5, tok.int()), ValueError),
        (lambda: features.dropout(x, 0.5, tok[:1]), ValueError), (lambda: features.dropout(x, 0.5, tok.cpu()), RuntimeError),
        (lambda: features.dropout(x.to(torch.uint8), 0.5, 0), TypeError),
    ]:
        with pytest.raises(exc):
            call()
    # the state must not change between forward and backward
    state = torch.tensor([1, 2], device=dev)
    leaf = x.clone().requires_grad_()
    y = features.dropout(leaf, 0.5, state)
    state[1] += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def _passes(dev, seed, n=3000, rows=400, D=136, dtype=torch.bfloat16):
    """(inputs, function of them that runs all three forward and backward and returns every output)"""
    from igs_b200 import features

    gen = _gen(dev, seed)
    ins = {"tokens": torch.randint(-1, rows, (n,), generator=gen, device=dev), "table": _normal(gen, rows, D, dtype=dtype),
           "w": _normal(gen, D), "b": _normal(gen, D), "dy": _normal(gen, n, D, dtype=dtype),
           "state": torch.tensor([seed, 5], device=dev)}

    def run(i):
        table, w, b = (i[k].detach().requires_grad_() for k in ("table", "w", "b"))
        f = features.embed(i["tokens"], table, scale=2.0, empty=-1)
        y = features.layer_norm(f, w, b)
        z = features.dropout(y, 0.2, i["state"])
        return [t.detach() for t in (f, y, z, *torch.autograd.grad(z, (table, w, b), i["dy"]))]

    return ins, run


def test_differentiable_once(dev):
    """A second derivative raises instead of passing for zero; so does a second backward pass."""
    from igs_b200 import features

    x = torch.randn(6, 16, device=dev, requires_grad=True)
    w = torch.randn(16, device=dev, requires_grad=True)
    tok = torch.tensor([0, 3, 3], device=dev)
    for y, leaf in ((features.embed(tok, x), x), (features.layer_norm(x, w), w), (features.dropout(x, 0.5, 1), x)):
        (g,) = torch.autograd.grad((y * y).sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            g.sum().backward()
    y = features.layer_norm(x, w)
    y.sum().backward()
    with pytest.raises(RuntimeError, match="second time"):
        y.sum().backward()
    y = features.layer_norm(x, w)
    with torch.no_grad():
        x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.parametrize("dtype", TYPES)
def test_upstream_gradients_off_their_boundary(dev, dtype):
    """Contiguous upstream gradients that start one value behind a 16-byte boundary."""
    gen, t = _gen(dev, 31), ref.DTYPES[dtype]
    shifted = lambda *shape: _normal(gen, int(np.prod(shape)) + 1, dtype=t)[1:].view(*shape)
    _check_embed(torch.randint(0, 30, (90,), generator=gen, device=dev), _normal(gen, 30, 64, dtype=t), shifted(90, 64))
    _check_norm(_normal(gen, 90, 64, dtype=t), _normal(gen, 64, dtype=t), _normal(gen, 64, dtype=t), shifted(90, 64))
    _check_norm(shifted(1500, 64), _normal(gen, 64, dtype=t), _normal(gen, 64, dtype=t), _normal(gen, 1500, 64, dtype=t))
    _check_dropout(_normal(gen, 90, 64, dtype=t), 0.3, 8, 9, shifted(90, 64), False)


def test_first_calls_inside_a_capture():
    """In a process of its own: nothing has to run before a capture (no call allocates, synchronises
    or sets up in a way that a capture forbids)."""
    import subprocess
    import sys

    code = """
import torch
from igs_b200 import features
dev = torch.device("cuda", 0)
gen = torch.Generator(device=dev).manual_seed(0)
tok = torch.randint(0, 500, (9000,), generator=gen, device=dev)
table = torch.randn(500, 264, generator=gen, device=dev, requires_grad=True)
w = torch.randn(264, generator=gen, device=dev, requires_grad=True)
state = torch.tensor([1, 2], device=dev)
def run():
    f = features.layer_norm(features.embed(tok, table), w)
    y = features.dropout(f, 0.5, state)
    return (y, *torch.autograd.grad(y, (table, w), torch.ones_like(y)))
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    outs = run()
g.replay()
for a, b in zip(outs, run()):
    assert torch.equal(a, b)
print("same")
"""
    res = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=240,
                         cwd=str(__import__("pathlib").Path(__file__).resolve().parents[1]))
    assert res.returncode == 0 and "same" in res.stdout, res.stderr[-2000:]


def test_same_bits_every_time(dev):
    ins, run = _passes(dev, 1, n=40000, rows=300)
    first = run(ins)
    for _ in range(4):
        for a, b in zip(first, run(ins)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("n,rows", [(3000, 400), (12000, 400), (12000, 5000)])
def test_two_streams_at_once(dev, n, rows):
    """Two calls in flight on two streams, none of them the default one: each as on its own.  (Every
    kind of sort; blocks of two sorts that wait for their like fit the device together.)"""
    ins1, run = _passes(dev, 2, n=n, rows=rows)
    ins2, _ = _passes(dev, 3, n=n, rows=rows)
    want1, want2 = run(ins1), run(ins2)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got1 = got2 = None
    for _ in range(10):
        with torch.cuda.stream(s1):
            got1 = run(ins1)
        with torch.cuda.stream(s2):
            got2 = run(ins2)
    torch.cuda.synchronize()
    for a, b in zip(want1 + want2, got1 + got2):
        assert torch.equal(a, b)


def test_captured_and_replayed(dev):
    """Two graphs of the whole run, replayed in turn on new inputs, agree with eager calls bit for
    bit; the generator's state is read at replay."""
    cases = [_passes(dev, 4), _passes(dev, 5, n=20000, rows=70, D=64)]
    fresh = [_passes(dev, 6)[0], _passes(dev, 7, n=20000, rows=70, D=64)[0]]
    want = []
    for (ins, run), new in zip(cases, fresh):
        want.append([[t.clone() for t in run(ins)], [t.clone() for t in run(new)]])
    gc.collect()  # (no eager autograd graph of the captured leaves is alive)
    graphs = []
    side = torch.cuda.Stream()
    for ins, run in cases:
        static = {k: v.clone() for k, v in ins.items()}
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(static)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = run(static)
        graphs.append((g, static, outs))
    for which in (0, 1, 0):
        for (g, static, _), (ins, _), new in zip(graphs, cases, fresh):
            for k, v in (ins if which == 0 else new).items():
                static[k].copy_(v)
            g.replay()
        for (_, _, outs), w in zip(graphs, want):
            for a, b in zip(outs, w[which]):
                assert torch.equal(a, b)


def test_gradients_against_differences_of_the_kernels(dev):
    """(L(v + h d) - L(v - h d)) / 2h of the kernels' own outputs, summed in 64 bits, against their
    gradient.  The outputs' bounds allow sum |dy| e_y / h; what h itself costs is taken from the
    64-bit form at the same points."""
    from igs_b200 import features

    gen = _gen(dev, 21)
    rows, D, h = 6, 48, 2.0 ** -5
    x, w, b, dy = (_normal(gen, *s) for s in ((rows, D), (D,), (D,), (rows, D)))
    dirs = [_normal(gen, *t.shape) for t in (x, w, b)]
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(features.layer_norm(*leaves), leaves, dy)
    f = ref.layer_norm(ref.f64(x), ref.f64(w), ref.f64(b), 1e-5)
    g64 = ref.layer_norm_grad(f, ref.f64(dy))
    for k, (grad, key) in enumerate(zip(grads, ("dx", "dw", "db"))):
        vals, exact, slack = [], [], 0.0
        for sign in (1, -1):
            at = [t + sign * h * d if i == k else t for i, (t, d) in enumerate(zip((x, w, b), dirs))]
            y = features.layer_norm(*at)
            fe = ref.layer_norm(*(ref.f64(t) for t in at), 1e-5)
            vals.append(float((ref.f64(y) * ref.f64(dy)).sum()))
            exact.append(float((fe["y"] * ref.f64(dy)).sum()))
            slack += float((np.abs(ref.f64(dy)) * 1.01 * fe["e_y"]).sum()) / (2 * h)
        d64 = ref.f64(dirs[k])
        step = abs((exact[0] - exact[1]) / (2 * h) - float((g64[key] * d64).sum()))
        slack += float((1.01 * g64["e_" + key] * np.abs(d64)).sum())
        diff, analytic = (vals[0] - vals[1]) / (2 * h), float((ref.f64(grad) * d64).sum())
        assert abs(diff - analytic) <= step + slack, (key, diff, analytic, step, slack)


# ---------------------------------------------------------------------------
# the three together, as the model uses them
# ---------------------------------------------------------------------------
def _feature_chain(model, k, state):
    """The model's features in 64 bits with autograd, from plain operations."""
    table = model.codebook.detach().double().requires_grad_()
    w, b = model.norm_weight.detach().double().requires_grad_(), model.norm_bias.detach().double().requires_grad_()
    f = table[model.tokens[:, :k]] * model.scale
    c = f - f.mean(-1, keepdim=True)
    f = c / torch.sqrt((c * c).mean(-1, keepdim=True) + 1e-5) * w + b
    keep = ref.words(0, f.numel(), *state) >= np.uint64(int(model.dropout * 2.0 ** 32))
    keep = torch.from_numpy(keep).to(f.device).view(f.shape)
    return torch.where(keep, f / (1 - model.dropout), 0.0), (table, w, b)


def test_splatter_with_tokens_norm_and_dropout(dev):
    """Two images of shared codebook rows: the rendered features and the gradients of codebook,
    weight and bias under the gradient that the renderer itself hands back.  Bounds: chains of
    fewer than 100 roundings of 2^-24 on sums of at most 64 terms of like size: 1e-5 of the
    largest value."""
    from igs_b200 import fit

    torch.manual_seed(3)
    gen = torch.Generator().manual_seed(4)
    tokens = torch.randint(0, 10, (2, 24), generator=gen)
    model = fit.ProgressiveSplatter(24, 40, 6, tokens=tokens, rows=10, scale=0.5, norm=True, dropout=0.25, seed=9).to(dev)
    for k, step in ((24, 0), (7, 1)):
        f = model.features(k)
        assert f.shape == (2, k, 40) and model.dropout_state.tolist() == [9, step + 1]
        f.retain_grad()
        image, _ = model.gs(f, (32, 40))
        model.zero_grad()
        (image - 0.5).square().mean().backward()
        want, leaves = _feature_chain(model, k, (9, step))
        err = lambda a, b: float((a.double() - b).abs().max() / b.abs().max())
        assert err(f.detach(), want.detach()) <= 1e-5
        grads = torch.autograd.grad(want, leaves, f.grad.double())
        for p, g in zip((model.codebook, model.norm_weight, model.norm_bias), grads):
            assert err(p.grad, g) <= 1e-5
    model.eval()
    assert torch.equal(model.features(5), model.features(5)) and model.dropout_state.tolist() == [9, 2]


def test_fit_progressive_with_tokens(dev):
    """The training loop runs on the options and moves every parameter; a model without them
    renders what it always did."""
    from igs_b200 import fit

    torch.manual_seed(0)
    target = torch.rand(3, 3, 24, 24, device=dev)
    tokens = torch.randint(0, 12, (3, 16))
    model = fit.ProgressiveSplatter(16, 32, 4, tokens=tokens, rows=12, norm=True, dropout=0.1).to(dev)
    before = {n: p.detach().clone() for n, p in model.named_parameters()}
    hist, ks = fit.fit_progressive(model, target, steps=6, lr=1e-3)
    assert hist.shape == (6,) and torch.isfinite(hist).all() and len(ks) == 6
    for n, p in model.named_parameters():
        assert torch.isfinite(p).all() and not torch.equal(p.detach(), before[n]), n
    assert model.dropout_state.tolist() == [0, 6]
    plain = fit.ProgressiveSplatter(8, 32, 4).to(dev)
    a, _ = plain(num_active_features=4, size=(16, 16))
    b, _ = plain.gs(plain.feature[:, :4], (16, 16))
    assert torch.equal(a, b)


def test_splatter_step_in_a_graph_draws_new_masks(dev):
    from igs_b200 import fit

    torch.manual_seed(1)
    model = fit.ProgressiveSplatter(8, 16, 2, dropout=0.5, seed=3).to(dev)
    with torch.no_grad():
        model.features()
    g = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(g):
        f = model.features()
    seen = []
    for _ in range(3):
        step = int(model.dropout_state[1])
        g.replay()
        want, err = ref.dropout(ref.f64(model.feature).reshape(-1), 0.5, 3, step)
        ref.assert_within(f.reshape(-1), want, err, f"replay at {step}")
        seen.append(f.clone())
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])
