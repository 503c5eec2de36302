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
