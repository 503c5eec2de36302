"""The feature operators' sums on whole numbers, which 32 bits add up exactly in any order as long as they
stay below 2^24: a place or row that is lost, doubled or added to the wrong sum shows as itself.  And the
layer norm's rows at widths that give them to every kind of group of threads."""
import numpy as np
import pytest
import torch

from tests import _features_ref as ref
from tests.test_layer_norm_rows_gpu import _layer_norm

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def _whole(gen, most, *shape):
    return torch.randint(-most, most + 1, shape, generator=gen, device=gen.device)


# ---------------------------------------------------------------------------
# the embedding's gradient
# ---------------------------------------------------------------------------
def _tokens(kind, n, rows, gen):
    i = torch.arange(n, device=gen.device)
    rand = torch.randint(0, rows, (n,), generator=gen, device=gen.device)
    if kind == "zipf":  # row r about 1 / r as often as the first, the rows in any order
        upto = torch.from_numpy(np.cumsum(1.0 / np.arange(1, rows + 1))).to(gen.device)
        at = torch.rand(n, generator=gen, device=gen.device, dtype=torch.float64) * upto[-1]
        rank = torch.searchsorted(upto, at, right=True).clamp_(max=rows - 1)
        return torch.randperm(rows, generator=gen, device=gen.device)[rank]
    return {"one_token": torch.full_like(i, rows // 2), "two_tokens": torch.where(i % 3 == 0, 5, rows - 1),
            "first_and_last": torch.where(i < n // 2, 0, rows - 1), "sorted": i * rows // n,
            "reversed": (n - 1 - i) * rows // n, "uniform": rand, "padded": torch.where(rand % 5 == 0, -1, rand),
            "common": torch.where(torch.rand(n, generator=gen, device=gen.device) < 0.7, rows // 3, rand)}[kind]


def _check_embed(dev, dtype, kind, n, rows, D):
    from igs_b200 import features

    gen, t = torch.Generator(device=dev).manual_seed(n + rows + D), ref.DTYPES[dtype]
    tokens = _tokens(kind, n, rows, gen)
    table = _whole(gen, 8, rows, D).to(t).requires_grad_()
    dy = _whole(gen, 8, n, D)  # |sums| <= 8 n < 2^24
    assert 8 * n < 1 << 24
    y = features.embed(tokens, table, empty=-1)
    held = tokens >= 0
    assert torch.equal(y, torch.where(held[:, None], table.detach()[tokens.clamp(min=0)], 0.0))
    (g,) = torch.autograd.grad(y, table, dy.to(t))
    want = torch.zeros(rows, D, dtype=torch.float64, device=dev).index_add_(0, tokens[held], dy[held].double())
    assert torch.equal(g, want.float().to(t))  # (whole numbers below 2^24; one rounding)


@pytest.mark.parametrize("n", [40, 3000, 8192, 8193, 12000, 70000, 152000])
@pytest.mark.parametrize("kind", ["one_token", "two_tokens", "first_and_last", "sorted", "reversed", "uniform", "padded", "common"])
@pytest.mark.parametrize("rows", [1000, 1500])
def test_embed_patterns(dev, kind, n, rows):
    """One digit, the whole row as the digit, and more places than one tile a block."""
    _check_embed(dev, "fp32", kind, n, rows, 20)


@pytest.mark.parametrize("dtype,D", [("fp32", 771), ("fp32", 2600), ("fp32", 2601), ("bf16", 517), ("bf16", 1033), ("bf16", 1542),
                                     ("fp16", 2600), ("fp16", 5003), ("bf16", 4104)])
@pytest.mark.parametrize("kind,n,rows", [("one_token", 9000, 300), ("common", 20000, 5003), ("zipf", 12000, 70000), ("sorted", 30000, 1200),
                                         ("padded", 4000, 77)])
def test_embed_wide_rows(dev, dtype, D, kind, n, rows):
    """Rows of every access width that take several slabs of columns, with runs over many chunks."""
    _check_embed(dev, dtype, kind, n, rows, D)


@pytest.mark.parametrize("kind", ["zipf", "uniform"])
def test_embed_training_batch(dev, kind):
    """64 images of 1024 tokens from a codebook of 16384 rows of 1024 bf16 values."""
    _check_embed(dev, "bf16", kind, 65536, 16384, 1024)


# ---------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------
# (type, D): groups of 8 to 512 threads, rows moved 16, 4 and 2 bytes at a time
WIDTHS = [("fp32", 24), ("fp32", 64), ("fp32", 65), ("fp32", 1000), ("fp32", 1024), ("fp32", 1111), ("fp32", 3001), ("fp32", 4096),
          ("fp32", 8192), ("bf16", 32), ("bf16", 33), ("fp16", 256), ("bf16", 1024), ("fp16", 1542), ("bf16", 1111), ("fp16", 2048),
          ("bf16", 3001), ("bf16", 3002), ("fp16", 4096), ("bf16", 5002), ("fp16", 7001), ("bf16", 8192)]


@pytest.mark.parametrize("dtype,D", WIDTHS)
def test_layer_norm_groups(dev, dtype, D):
    """Enough rows that every block takes several, forward and gradient."""
    from igs_b200 import features

    rows = 12000 if D < 100 else 2500 if D < 4000 else 1500
    gen, t = torch.Generator(device=dev).manual_seed(D), ref.DTYPES[dtype]
    x, dy = (torch.randn(rows, D, generator=gen, device=dev).to(t) for _ in range(2))
    x[:, 0] += 3.0
    w, b = (torch.randn(D, generator=gen, device=dev) for _ in range(2))
    leaves = [v.requires_grad_() for v in (x, w, b)]
    y = features.layer_norm(*leaves)
    f = _layer_norm(ref.f64(x), ref.f64(w), ref.f64(b), 1e-5)
    ref.assert_within(y, f["y"], f["e_y"], "y")
    g = ref.layer_norm_grad(f, ref.f64(dy))
    for got, name in zip(torch.autograd.grad(y, leaves, dy), ("dx", "dw", "db")):
        ref.assert_within(got, g[name], g["e_" + name], name)


@pytest.mark.parametrize("rows", [1, 700, 3001, 40000])
@pytest.mark.parametrize("dtype,D", WIDTHS + [("fp32", 9000), ("bf16", 20001)])
def test_layer_norm_column_sums(dev, dtype, D, rows):
    """Rows of the numbers -2 to 2 that begin with 0 and sum to 0: the mean and every distance from it are
    exact, and the variance, below 4, is lost in the rounding of 2^26 + variance, whose step is 8 (4 below):
    rstd = 2^-13.  Then dbias and 2^13 dweight are whole numbers of at most 8 and 16 rows."""
    from igs_b200 import features

    if rows * D > 1 << 28:
        rows //= 10
    assert 16 * rows < 1 << 24
    gen, t = torch.Generator(device=dev).manual_seed(D * 3 + rows), ref.DTYPES[dtype]
    x = torch.zeros(rows, D, device=dev, dtype=torch.int64)
    half = (D - 1) // 2
    x[:, 1:1 + half] = _whole(gen, 2, rows, half)
    x[:, 1 + half:1 + 2 * half] = -x[:, 1:1 + half].flip(1)
    dy = _whole(gen, 8, rows, D)
    w, b = torch.ones(D, device=dev, requires_grad=True), torch.zeros(D, device=dev, requires_grad=True)
    leaf = x.to(t).requires_grad_()
    y = features.layer_norm(leaf, w, b, eps=2.0 ** 26)
    assert torch.equal(y, (x.double() * 2.0 ** -13).to(t))
    gx, gw, gb = torch.autograd.grad(y, (leaf, w, b), dy.to(t))
    assert torch.equal(gb, dy.sum(0).float())
    assert torch.equal(gw * 2.0 ** 13, (dy * x).sum(0).float())
    w, b = w.detach().requires_grad_(), b.detach().requires_grad_()
    gw2, gb2 = torch.autograd.grad(features.layer_norm(leaf.detach(), w, b, eps=2.0 ** 26), (w, b), dy.to(t))  # without dx
    assert torch.equal(gw2, gw) and torch.equal(gb2, gb)
