"""Layer norm on rows with one value far from the others, wherever it stands, within bounds that do
not grow with its distance from the row's first value."""
import numpy as np
import pytest
import torch

from tests import _features_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def _layer_norm(x, w, b, eps):
    """ref.layer_norm with the bounds of: a pivot p at a distance of at most delta from the mean; c = x - p,
    one rounding of |c| <= |x - mean| + delta; the mean of c, sums of at most H additions in a chain;
    sum c^2 / D less the squared mean of c; xhat = c rstd - (mean of c) rstd; the affine map.  delta itself
    is known from the first pass over x - x[0].  First order, 1.05 for the higher ones."""
    u = ref.U
    f = ref.layer_norm(x, w, b, eps)
    mean = x.mean(1, keepdims=True)
    xc, H, sd = np.abs(x - mean), f["H"], f["sd"]
    delta = u * np.abs(mean) + u * (H + 4) * np.abs(x - x[:, :1]).mean(1, keepdims=True)
    away = xc.mean(1, keepdims=True) + delta
    e_c = u * 2 * (xc + delta) + u * (H + 5) * away
    square = (xc * xc).mean(1, keepdims=True) + delta * delta
    f["r"] = (u * (H + 6) * square + 2 * u * (H + 5) * delta * away) / (2 * sd * sd) + 3 * u
    f["e_xhat"] = 1.05 * (e_c / sd + np.abs(f["xhat"]) * (f["r"] + 2 * u))
    f["e_y"] = np.abs(f["w"]) * f["e_xhat"] + u * np.abs(f["y"])
    return f


@pytest.mark.parametrize("rows", [9, 1600])
@pytest.mark.parametrize("D", [24, 64, 257, 1024, 1111, 3001, 4096, 8192, 17001])
def test_rows_with_one_far_value(dev, rows, D):
    from igs_b200 import features

    gen = torch.Generator(device=dev).manual_seed(D + rows)
    x = torch.randn(rows, D, generator=gen, device=dev)
    far = torch.tensor([1e3, -1e4, 1e6, 30.0], device=dev)
    for k in range(rows):  # the first value of most rows, another one of the others
        x[k, 0 if k % 3 else (7 * k) % D] = far[k % 4]
    dy = torch.randn(rows, D, generator=gen, device=dev)
    w, b = torch.randn(D, generator=gen, device=dev), torch.randn(D, generator=gen, device=dev)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = features.layer_norm(*leaves)
    f = _layer_norm(ref.f64(x), ref.f64(w), ref.f64(b), 1e-5)
    ref.assert_within(y, f["y"], f["e_y"], "y")
    with torch.no_grad():
        bare = features.layer_norm(x)
    ref.assert_within(bare, f["xhat"], f["e_xhat"], "xhat")
    g = ref.layer_norm_grad(f, ref.f64(dy))
    for got, name in zip(torch.autograd.grad(y, leaves, dy), ("dx", "dw", "db")):
        ref.assert_within(got, g[name], g["e_" + name], name)


@pytest.mark.parametrize("D", [64, 1000, 1024, 8192, 17001])
def test_rows_of_two_neighbouring_numbers(dev, D):
    """Rows that differ from a constant in the last bit of a few values, the first one among them or
    not: the variance is that of a few steps.  Everything before the sums' rounding is exact: distances
    are 0 or 1 step whatever the pivot, so sums are whole numbers of steps."""
    from igs_b200 import features

    x = torch.full((1400, D), 1234.567, device=dev)
    up = torch.nextafter(x[0, 0], x.new_tensor(2000.0))
    gen = torch.Generator(device=dev).manual_seed(D)
    few = torch.rand(1400, D, generator=gen, device=dev) < 0.01
    few[::2, 0] = True
    few[:, 5], few[:, 6] = True, False
    x[few] = up
    for rows in (slice(0, 8), slice(0, 1400)):
        y = features.layer_norm(x[rows], eps=0.0)
        f = ref.layer_norm(ref.f64(x[rows]), None, None, 0.0)
        # D, the mean of c, its square and var: a handful of roundings each, at most doubled by the subtraction
        ref.assert_within(y, f["xhat"], 16 * ref.U * (np.abs(f["xhat"]) + 1 / f["sd"] * np.abs(np.diff(ref.f64(x[0, 5:7])))), "xhat")
