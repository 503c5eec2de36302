"""fit_progressive on models other than a plain ProgressiveSplatter."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def test_a_model_of_ones_own(dev):
    """All that the loop asks of a model: num_features, feature [1,N,D], and a call with
    num_active_features and size."""
    from igs_b200 import fit

    class Own(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.num_features = 8
            self.feature = torch.nn.Parameter(torch.randn(1, 8, 12))
            self.out = torch.nn.Linear(12, 3 * 6 * 5)

        def forward(self, num_active_features=None, size=None):
            return self.out(self.feature[:, :num_active_features].mean(1)).view(1, 3, *size), None

    torch.manual_seed(0)
    model = Own().to(dev)
    before = model.feature.detach().clone()
    hist, ks = fit.fit_progressive(model, torch.rand(1, 3, 6, 5, device=dev), steps=3, lr=1e-3)
    assert torch.isfinite(hist).all() and len(ks) == 3 and not torch.equal(model.feature.detach(), before)


def test_large_codebooks_are_spread_over_what_a_step_uses(dev):
    """The term's matrix is quadratic in its rows: 36000 of them would take 5 GB a copy."""
    from igs_b200 import fit
    from igs_b200.reg import koleo_diversity_loss

    torch.manual_seed(1)
    rows = 36000
    tokens = torch.randint(0, rows, (6, 1500))
    model = fit.ProgressiveSplatter(1500, 8, 1, tokens=tokens, rows=rows).to(dev)
    used = torch.unique(tokens[:, :100]).to(dev)
    spread = model.diverse(100)
    assert torch.equal(spread[0], model.codebook[used])
    (g,) = torch.autograd.grad(koleo_diversity_loss(spread), model.codebook)
    assert g[used].abs().sum() > 0 and not g[torch.isin(torch.arange(rows, device=dev), used, invert=True)].any()
    many = model.diverse(1500)  # about 8000 distinct rows
    assert torch.unique(tokens).numel() > fit.DIVERSE_ROWS and many.shape == (1, fit.DIVERSE_ROWS, 8)
    where = {tuple(r): i for i, r in enumerate(model.codebook.tolist())}
    picked = [where[tuple(r)] for r in many[0].tolist()]
    assert len(set(picked)) == len(picked) and set(picked) <= set(tokens.flatten().tolist())

    target = torch.rand(6, 3, 16, 16, device=dev)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    hist, _ = fit.fit_progressive(model, target, steps=2, lr=1e-3, chunk=1500)
    assert torch.isfinite(hist).all() and torch.cuda.max_memory_allocated() - before < 1 << 30
    small = fit.ProgressiveSplatter(4, 8, 2, tokens=[0, 1, 2, 3], rows=fit.DIVERSE_ROWS)
    assert small.diverse(2).shape == (1, fit.DIVERSE_ROWS, 8)
