"""What reaches the feature operators other than by a plain call: tensors that come back changed in
the backward pass, derivatives of other kinds, views whose values are not what lies in memory."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def _calls(dev):
    """{name: (leaves, function of them)}, the inputs strided, in several dimensions and in one"""
    from igs_b200 import features

    gen = torch.Generator(device=dev).manual_seed(3)
    normal = lambda *s: torch.randn(s, generator=gen, device=dev)
    wide, tokens = normal(30, 4, 200), torch.randint(-1, 30, (40, 3), generator=gen, device=dev)
    w, b, state = normal(400)[::2], normal(200), torch.tensor([[5, 6], [7, 8]], device=dev)
    leaf = lambda t: t.detach().requires_grad_()
    calls = {}
    for name, x in (("slice", wide[:, 1]), ("narrow", wide[:, 0, 8:136]), ("crossed", wide.transpose(0, 1)),
                    ("columns", wide[:, 0].t().contiguous().t()), ("shared", wide[:1, 0].expand(7, 200)),
                    ("one", wide[0, 0])):
        D = x.shape[-1]
        calls["norm " + name] = ([leaf(x), leaf(w[:D]), leaf(b[:D])], features.layer_norm)
        calls["bare norm " + name] = ([leaf(x)], features.layer_norm)
    calls["embed"] = ([leaf(wide[:, 2, 3:180])], lambda t: features.embed(tokens[:, 1:], t, empty=-1))
    calls["dropout"] = ([leaf(wide[:, 1])], lambda x: features.dropout(x, 0.5, state[:, 0]))
    calls["dropout by number"] = ([leaf(wide[:, 1])], lambda x: features.dropout(x, 0.5, 9))
    return calls


def _grads(leaves, fn):
    y = fn(*leaves)
    dy = torch.arange(y.numel(), device=y.device, dtype=y.dtype).view(y.shape).sin()
    return torch.autograd.grad(y, leaves, dy)


def _same(a, b):
    assert len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


LAYOUTS = {
    "contiguous": lambda t: t.clone(memory_format=torch.contiguous_format),
    # (none of them moves a row off its 16-byte boundary: the kernels add in the same order)
    "crossed": lambda t: t.permute(*reversed(range(t.dim()))).contiguous().permute(*reversed(range(t.dim()))),
    "spread": lambda t: torch.stack([t, t], -1)[..., 0],
    "wider rows": lambda t: torch.cat([t, t], -1)[..., :t.shape[-1]],
    "shifted": lambda t: torch.cat([t.new_zeros(4), t.reshape(-1)])[4:].view(t.shape),
}


@pytest.mark.parametrize("layout", LAYOUTS)
def test_saved_tensors_come_back_in_another_layout(dev, layout):
    """Gradients are the same bits wherever the saved tensors have been in between."""
    for name, (leaves, fn) in _calls(dev).items():
        want = _grads(leaves, fn)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, LAYOUTS[layout]):
            _same(_grads(leaves, fn), want)


def test_saved_tensors_kept_on_the_host(dev):
    for pin in (False, True):
        for name, (leaves, fn) in _calls(dev).items():
            want = _grads(leaves, fn)
            with torch.autograd.graph.save_on_cpu(pin_memory=pin):
                _same(_grads(leaves, fn), want)


def test_recomputed_forwards(dev):
    from torch.utils.checkpoint import checkpoint

    for name, (leaves, fn) in _calls(dev).items():
        want = _grads(leaves, fn)
        _same(_grads(leaves, lambda *a: checkpoint(fn, *a, use_reentrant=False)), want)


@pytest.mark.parametrize("what", ["fewer", "more", "type", "place"])
def test_other_tensors_that_come_back_are_refused(dev, what):
    """A shorter, longer, retyped or host tensor: an error before anything is read."""
    other = {"fewer": lambda t: t[:-1].clone(), "more": lambda t: torch.cat([t, t[:1]]),
             "type": lambda t: t.to(torch.int32 if t.dtype == torch.int64 else torch.float64),
             "place": lambda t: t.cpu()}[what]
    for name, (leaves, fn) in _calls(dev).items():
        if name == "dropout by number":
            continue  # (nothing is saved)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, other):
            y = fn(*leaves)
            with pytest.raises(RuntimeError, match="came back in the backward pass"):
                torch.autograd.grad(y, leaves, torch.ones_like(y))


def test_upstream_gradients_of_another_size_are_refused(dev):
    """Handed to the node itself, past the checks of the engine."""
    for name, (leaves, fn) in _calls(dev).items():
        y = fn(*leaves)
        for bad in (torch.ones(1, device=dev), torch.ones_like(y)[..., :-1], torch.ones_like(y).double(),
                    torch.ones_like(y).cpu()):
            with pytest.raises(RuntimeError, match="came back in the backward pass"):
                y.grad_fn(bad)
        got = y.grad_fn(torch.ones_like(y))  # (the right one, for the first time)
        got = [got] if isinstance(got, torch.Tensor) else [g for g in got if g is not None]
        _same(got, torch.autograd.grad(fn(*leaves).sum(), leaves))


def test_forward_mode_is_refused(dev):
    """No operator has a forward-mode formula: an error, not a result whose tangent is lost."""
    import torch.autograd.forward_ad as fwd

    for name, (leaves, fn) in _calls(dev).items():
        with fwd.dual_level():
            for i in range(len(leaves)):
                ins = [t.detach().clone() for t in leaves]  # (torch makes no dual of rows that share memory)
                ins[i] = fwd.make_dual(ins[i], torch.ones_like(ins[i]))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    fn(*ins)
            y = fn(*leaves)
            dy = fwd.make_dual(torch.ones_like(y), torch.ones_like(y))  # forward over reverse
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y, leaves, dy)
        _grads(leaves, fn)


def test_transforms_are_refused(dev):
    """Tracing would record the result as a constant; the others hand in tensors without memory."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    for name, (leaves, fn) in _calls(dev).items():
        ins = [t.detach() for t in leaves]
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(fn, tuple(ins), check_trace=False)
        with pytest.raises(RuntimeError):
            torch.func.vmap(fn)(*[t.expand(2, *t.shape) for t in ins])
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda *a: fn(*a).sum())(*ins)
        with pytest.raises(RuntimeError), FakeTensorMode(allow_non_fake_inputs=True) as mode:
            fn(*[mode.from_tensor(t) for t in ins])


def test_negated_views(dev):
    """Real tensors whose sign torch keeps beside the memory (imaginary parts of conjugates)."""
    from igs_b200 import features

    gen = torch.Generator(device=dev).manual_seed(8)
    z = torch.complex(*(torch.randn(40, 1, generator=gen, device=dev) for _ in range(2)))
    column, tokens = z.conj().imag, torch.randint(0, 40, (9,), generator=gen, device=dev)
    wide = torch._neg_view(torch.randn(40, 24, generator=gen, device=dev))
    dy = torch._neg_view(torch.randn(40, 24, generator=gen, device=dev))
    assert column.is_neg() and wide.is_neg() and dy.is_neg()
    vec, bias = torch._neg_view(wide[0].clone()), column[:1, 0]
    plain = lambda t: t.clone().resolve_neg()
    for fn, ins, up in ((lambda t: features.embed(tokens, t), [column], None), (lambda t: features.embed(tokens, t), [wide], None),
                        (lambda t: features.dropout(t, 0.5, 3), [column[0]], None),
                        (lambda t: features.dropout(t, 0.5, 3), [wide], dy),
                        (lambda *t: features.layer_norm(*t), [wide, vec, vec], dy),
                        (lambda *t: features.layer_norm(*t), [column, bias, bias], None)):
        want_y = fn(*[plain(t) for t in ins])
        assert torch.equal(fn(*ins), want_y)
        up = torch.ones_like(want_y) if up is None else up
        leaves, want_leaves = [t.detach().requires_grad_() for t in ins], [plain(t).requires_grad_() for t in ins]
        _same(torch.autograd.grad(fn(*leaves), leaves, up), torch.autograd.grad(fn(*want_leaves), want_leaves, plain(up)))
