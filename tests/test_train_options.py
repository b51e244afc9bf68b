"""Combinations of the driver's options that would train on lost digits are refused, and AdamW has a learning rate of its own
(no GPU needed)."""
import pytest
import torch

from cafe_amd import train

HIP = ["--dense-ops", "hip"]


@pytest.mark.parametrize("argv,word", [
    (HIP + ["--dense-dtype", "f16"], "float16"),
    (HIP + ["--dense-dtype", "f16", "--optimizer", "adamw"], "float16"),
    (HIP + ["--dense-dtype", "bf16"], "master weights"),
    (HIP + ["--dense-dtype", "bf16", "--optimizer", "sgd", "--dense-learning-rate", "0.1"], "master weights"),
])
def test_refused(argv, word, capsys):
    with pytest.raises(SystemExit):
        train.parse(argv)
    assert word in capsys.readouterr().err


def test_learning_rates():
    rate = lambda *argv: train.parse(HIP + list(argv)).dense_learning_rate             # noqa: E731
    assert rate() == 0.1 and rate("--learning-rate", "0.3") == 0.3
    assert rate("--optimizer", "adamw") == 1e-3 and rate("--optimizer", "adamw8bit", "--learning-rate", "0.3") == 1e-3
    assert rate("--optimizer", "adamw", "--dense-learning-rate", "0.02", "--dense-dtype", "bf16") == 0.02


@pytest.mark.gpu
def test_a_float16_head_is_not_trained():
    from cafe_amd.ctr_models import CafeCTRModel
    counts = [4000, 197, 25000]
    m = CafeCTRModel("dlrm", counts, 16, compress_rate=0.05, threshold=3, ln_bot=[13, 32, 16], ln_top=[0, 32, 1], dense_ops="hip",
                     dense_dtype=torch.float16)
    dense, ids = torch.rand(64, 13, device="cuda"), torch.stack([torch.arange(64, device="cuda") % n for n in counts])
    with torch.no_grad():
        assert m(dense, ids).isfinite().all()
    opt = torch.optim.SGD(m.dense_parameters(), lr=0.1)
    with pytest.raises(ValueError, match="float16"):
        m.train_step(dense, ids, torch.zeros(64, 1, device="cuda"), opt, 0.1)
