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


@pytest.mark.parametrize("dtype,columns,k", [("F16", 1_700_000, 1), ("BF16", 1_300_000, 1024), ("F32", 900_000, 1), ("F32", 700_000, 1024),
                                             ("F16", 2 ** 31 - 1, 0), ("F32", 2 ** 31 - 1, 0)])
def test_rows_longer_than_sixteen_sms_hold_are_refused_before_any_cuda_call(dtype, columns, k):
    from cuda_transformer_b200 import _lib, build
    build.build()
    lib, A = _lib.load(), 1 << 20       # A stands for an aligned device pointer: never read
    t = getattr(_lib, dtype)
    assert lib.b200amp_distill_loss(A, columns, A + 64, columns, t, 4, columns, columns, A, A, t, A, A, k, 1.0, 1.0, 0.5, A, A, A,
                                    None) == _lib.ERR_LIMIT
    assert b"columns" in lib.b200amp_last_error()


@pytest.mark.parametrize("dtype,columns,k", [("F16", 1_800_000, 1), ("BF16", 1_500_000, 1024), ("F32", 900_000, 1), ("F32", 2 ** 31 - 1, 5)])
def test_top_logits_refuses_them_too(dtype, columns, k):
    from cuda_transformer_b200 import _lib, build
    build.build()
    lib, A = _lib.load(), 1 << 20
    assert lib.b200amp_top_logits(A, getattr(_lib, dtype), 4, columns, columns, k, 1.0, A, A, A, None) == _lib.ERR_LIMIT
    assert b"columns" in lib.b200amp_last_error()
