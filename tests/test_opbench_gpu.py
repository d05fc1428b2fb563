"""opbench times the operation alone: what its inputs need is made before."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("op", ["linear_int8_grouped", "gemm_grouped", "gemm_grouped_wgrad", "linear_train",
                                "linear_train_int8"])
def test_group_bounds_are_made_once(op, monkeypatch, capsys):
    from tensorcoreptx_b200 import opbench
    made = []
    plain = torch.tensor
    monkeypatch.setattr(torch, "tensor", lambda *a, **k: made.append(1) or plain(*a, **k))
    opbench.main([op, "--m", "96", "--n", "128", "--k", "256", "--groups", "3", "--iters", "5", "--warmup", "2"])
    assert "per call" in capsys.readouterr().out
    assert len(made) == 1
