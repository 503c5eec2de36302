"""The feature operators without a GPU: refusals at both levels, and the 64-bit forms that the GPU
tests compare with (their gradients against differences, their generator against published words)."""
import ctypes

import numpy as np
import pytest
import torch

from tests import _features_ref as ref


def test_cpu_tensors_and_wrong_types_are_refused():
    from igs_b200 import features

    x = torch.zeros(3, 4)
    with pytest.raises(RuntimeError, match="no CPU path"):
        features.embed(torch.zeros(2, dtype=torch.int64), x)
    with pytest.raises(RuntimeError, match="no CPU path"):
        features.layer_norm(x)
    with pytest.raises(RuntimeError, match="no CPU path"):
        features.dropout(x, 0.5, 0)
    with pytest.raises(TypeError, match="torch.Tensor"):
        features.layer_norm([1.0])


def test_c_abi_refuses_bad_arguments_before_any_cuda_call():
    from igs_b200 import _lib

    lib = _lib.load()
    one = ctypes.c_void_p(256)  # never dereferenced: every call below fails its checks first

    def embed(tok=one, tb=8, n=4, table=one, dt=0, rows=5, D=8, stride=8, scale=1.0, out=one):
        return lib.igs_embed(tok, tb, n, table, dt, rows, D, stride, scale, 0, 0, out, 0, None)

    for bad in (dict(tok=None), dict(table=None), dict(out=None), dict(tb=2), dict(n=-1), dict(dt=3), dict(rows=0),
                dict(D=0), dict(stride=-1), dict(scale=float("inf")), dict(scale=float("nan"))):
        assert embed(**bad) == -1, bad
    assert embed(n=1 << 31) == -3 and embed(rows=1 << 31) == -3 and embed(D=(1 << 22) + 1) == -3
    assert embed(n=0, tok=None, out=None) == 0

    size = ctypes.c_size_t(0)
    assert lib.igs_embed_grad_workspace_bytes(4, 5, 8, 0, 0, None) == -1
    assert lib.igs_embed_grad_workspace_bytes(4, 0, 8, 0, 0, ctypes.byref(size)) == -1
    assert lib.igs_embed_grad_workspace_bytes(1 << 31, 5, 8, 0, 0, ctypes.byref(size)) == -3

    def embed_grad(tok=one, n=4, dy=one, dt=0, rows=5, D=8, scale=1.0, out=one, ws=one, nb=1 << 30):
        return lib.igs_embed_grad(tok, 8, n, dy, dt, rows, D, scale, 0, 0, out, ws, nb, 0, None)

    for bad in (dict(tok=None), dict(dy=None), dict(out=None), dict(dt=-1), dict(rows=0), dict(scale=float("inf"))):
        assert embed_grad(**bad) == -1, bad
    assert embed_grad(ws=None) == -2 and embed_grad(nb=16) == -2 and embed_grad(ws=ctypes.c_void_p(264)) == -2

    def norm(x=one, dt=1, rows=4, D=8, stride=8, w=one, b=one, wdt=0, eps=1e-5, y=one, stats=one):
        return lib.igs_layer_norm(x, dt, rows, D, stride, w, b, wdt, eps, y, stats, 0, None)

    for bad in (dict(x=None), dict(y=None), dict(dt=9), dict(wdt=2), dict(rows=-1), dict(D=0), dict(stride=-8),
                dict(eps=-1.0), dict(eps=float("nan")), dict(stats=ctypes.c_void_p(260))):
        assert norm(**bad) == -1, bad
    assert norm(rows=0, x=None, y=None) == 0

    def norm_grad(dy=one, x=one, dt=1, rows=4, wdt=0, stats=one, dx=one, dw=one, db=one, ws=one, nb=1 << 30):
        return lib.igs_layer_norm_grad(dy, x, dt, rows, 8, 8, one, wdt, stats, dx, dw, db, ws, nb, 0, None)

    for bad in (dict(dy=None), dict(x=None), dict(stats=None), dict(stats=ctypes.c_void_p(260)), dict(wdt=2), dict(rows=-1)):
        assert norm_grad(**bad) == -1, bad
    assert norm_grad(ws=None) == -2 and norm_grad(nb=16) == -2 and norm_grad(ws=ctypes.c_void_p(264)) == -2

    def dropout(x=one, dt=0, n=4, p=0.5, y=one):
        return lib.igs_dropout(x, dt, n, p, 0, 0, None, y, 0, None)

    for bad in (dict(x=None), dict(y=None), dict(dt=3), dict(n=-1), dict(p=-0.1), dict(p=1.5), dict(p=float("nan"))):
        assert dropout(**bad) == -1, bad
    assert dropout(n=0, x=None, y=None) == 0


def test_generator_words():
    # published words of Philox4x32 at 7 and 10 rounds, counter and key zero; all ones at 10
    assert ref.philox([0] * 4, [0] * 2, 7) == [0x5F6FB709, 0x0D893F64, 0x4F121F81, 0x4F730A48]
    assert ref.philox([0] * 4, [0] * 2, 10) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert ref.philox([ref.LOW] * 4, [ref.LOW] * 2, 10) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    seed, offset, first = 0x123456789ABCDEF0, 0xFEDCBA9876543210, 4 * ((1 << 32) - 1)  # blocks across 2^32
    got = ref.words(first, 8, seed, offset)
    for j, block in enumerate(((1 << 32) - 1, 1 << 32)):
        want = ref.philox([block & ref.LOW, block >> 32, offset & ref.LOW, offset >> 32], [seed & ref.LOW, seed >> 32])
        assert got[4 * j:4 * j + 4].tolist() == want


def test_gradient_formulas_against_differences():
    """Central differences in 64 bits: their error is h^2 times a third derivative plus 2^-53 / h
    times the loss; with h = 2^-14 and values of order one both are below 1e-7."""
    rng = np.random.default_rng(0)
    h = 2.0 ** -14
    # layer norm, every input
    x, w, b = rng.normal(size=(3, 7)) + 0.5, rng.normal(size=7), rng.normal(size=7)
    dy = rng.normal(size=(3, 7))
    loss = lambda x, w, b: float((ref.layer_norm(x, w, b, 1e-5)["y"] * dy).sum())
    g = ref.layer_norm_grad(ref.layer_norm(x, w, b, 1e-5), dy)
    for name, at, arg in (("dx", 0, x), ("dw", 1, w), ("db", 2, b)):
        for idx in np.ndindex(arg.shape):
            args = [[x, w, b], [x, w, b]]
            for sign, a in ((1, args[0]), (-1, args[1])):
                moved = arg.copy()
                moved[idx] += sign * h
                a[at] = moved
            diff = (loss(*args[0]) - loss(*args[1])) / (2 * h)
            assert abs(diff - g[name][idx]) <= 1e-6 * (1 + abs(diff)), (name, idx)
    # embedding: linear, so differences are exact but for rounding
    tokens = np.array([[0, 2, 2], [-1, 4, 0]])
    table, dy = rng.normal(size=(5, 3)), rng.normal(size=(2, 3, 3))
    g, _ = ref.embed_grad(tokens, dy, 5, 1.5, -1)
    for idx in np.ndindex(table.shape):
        up, down = table.copy(), table.copy()
        up[idx] += h
        down[idx] -= h
        diff = ((ref.embed(tokens, up, 1.5, -1)[0] - ref.embed(tokens, down, 1.5, -1)[0]) * dy).sum() / (2 * h)
        assert abs(diff - g[idx]) <= 1e-9


def test_splatter_options_are_checked():
    from igs_b200 import fit

    make = lambda **kw: fit.ProgressiveSplatter(4, 8, 2, **kw)
    for bad in (dict(tokens=[0, 1, 2, 3]), dict(rows=5), dict(tokens=[0, 1, 2], rows=5), dict(tokens=[0, 1, 2, 5], rows=5),
                dict(tokens=[0, 1, 2, -1], rows=5), dict(tokens=[0.0, 1.0, 2.0, 3.0], rows=5), dict(scale=2.0),
                dict(dropout=1.0), dict(dropout=-0.1)):
        with pytest.raises(ValueError):
            make(**bad)
    plain = make()
    assert sorted(n for n, _ in plain.named_parameters()) == ["feature", "gs.proj.bias", "gs.proj.weight"]
    assert not list(plain.named_buffers())
    full = make(tokens=[[0, 1, 2, 3], [4, 4, 4, 4]], rows=5, norm=True, dropout=0.5, seed=7)
    assert sorted(n for n, _ in full.named_parameters()) == ["codebook", "gs.proj.bias", "gs.proj.weight", "norm_bias",
                                                             "norm_weight"]
    assert full.tokens.shape == (2, 4) and full.dropout_state.tolist() == [7, 0]
    assert full.diverse(2).shape == (1, 5, 8) and plain.diverse(2).shape == (1, 2, 8)
