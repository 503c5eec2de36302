"""The measurable cases of the feature operators (perf/operators.py): what a case is made of
follows from the case and its seed alone, so that two programs that prepare it compare the same."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _cases():
    from perf import operators

    return operators.listed()


@pytest.mark.parametrize("case", _cases(), ids=lambda c: c["name"])
def test_inputs_follow_from_the_seed_alone(case):
    from perf import operators

    first = operators.prepare(case, 7)
    for _ in range(6):
        again = operators.prepare(case, 7)
        assert again.keys() == first.keys()
        for k, v in first.items():
            assert torch.equal(again[k], v) if isinstance(v, torch.Tensor) else again[k] == v, k
    other = operators.prepare(case, 8)
    for k, v in first.items():
        if isinstance(v, torch.Tensor):
            assert not torch.equal(other[k], v), k


def test_tokens_have_their_case_s_shares():
    """How often each rank is drawn, against n p: n independent draws are off by more than six
    standard deviations sqrt(n p (1 - p)) with a chance below 1e-8, 20 of the commonest together
    below 1e-6; a place is 1 draw, hence the + 1."""
    from perf import operators

    (case,) = [c for c in operators.listed() if c.get("law") == "zipf"]
    s = operators.prepare(case, 3)
    counts = torch.bincount(s["tokens"].reshape(-1).long(), minlength=case["rows"]).sort(descending=True).values
    n = int(counts.sum())
    p = torch.from_numpy(operators._shares(case))[:20]
    off = (counts[:20].cpu().double() - n * p).abs()
    assert (off <= 6 * (n * p * (1 - p)).sqrt() + 1).all(), off
