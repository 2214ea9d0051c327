"""The losses' methods on an optimizer: which workspace and state a call gets. No kernel is launched here."""
import pytest

from cuda_transformer_b200 import losses


class Owner(losses.LossCalls):
    state, loss_workspace = "state", "the owner's"


@pytest.mark.parametrize("workspace,used", [(None, "the owner's"), ("another", "another")])
def test_a_call_may_bring_its_own_workspace(monkeypatch, workspace, used):
    seen = {}
    monkeypatch.setattr(losses, "distill_loss", lambda *a: seen.update(distill=a))
    monkeypatch.setattr(losses, "balance_loss", lambda *a: seen.update(balance=a))
    Owner().distill_loss("z", "dz", "y", "v", "i", "lse", "row", vocab=7, temperature=2.0, soft_weight=4.0, hard_weight=0.5, stream=3,
                         workspace=workspace)
    assert seen["distill"] == ("z", "dz", "y", "v", "i", "lse", "state", "row", used, 7, 2.0, 4.0, 0.5, 3)
    Owner().balance_loss("r", "dr", "c", "y", "counts", "loss", weight=0.1, accumulate=True, add_to_state=False, stream=4,
                         workspace=workspace)
    assert seen["balance"] == ("r", "dr", "c", "y", "state", "counts", "loss", used, 0.1, True, False, 4)
