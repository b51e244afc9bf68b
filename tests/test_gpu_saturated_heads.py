"""Confident predictions through the heads with dense_ops="hip": the gradient of the loss in the logit is p - label, however
far out the logit and whatever the head's type.

The last layer's weights are 0 and its bias is the logit (halves, which 16 bits hold), so that every sample has it and the
bias's gradient is the mean of p - label over the batch.  Tolerance: p, its distance to the label and the batch's share of
it are a few float32 operations, 8 2^-24; dz rounded to the type (u), summed, rounded again (u); below the normal range half
a subnormal step of B values.  The probability's own path divides by the p that was rounded, off by half a step of at least
one: a factor of 1.5, and nothing at 0 and 1."""
import pytest
import torch
import torch.nn.functional as nnf

from cafe_amd import train
from cafe_amd.ctr_models import CafeCTRHead, CafeCTRModel

pytestmark = pytest.mark.gpu
B = 64
LOGITS = [0.0, 5.0, 6.0, 6.5, 7.0, 8.0, 9.0, 12.0, 16.0, 17.0, 17.5, 18.0, 20.0, 30.0]
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def with_logit(head, z):
    """Every sample's logit is z, and the layer whose bias's gradient is that of the logit."""
    with torch.no_grad():
        if head.kind == "wdl":                                  # sigmoid(0) + wide
            head.top_l[-2].weight.zero_()
            head.top_l[-2].bias.zero_()
            head.wide.weight.zero_()
            head.wide.bias.fill_(z - 0.5)
            return head.wide
        last = head.last_layer if head.kind == "dcn" else head.top_l[-2]
        last.weight.zero_()
        last.bias.fill_(z)
        return last


def build(kind, t):
    torch.manual_seed(0)
    head = CafeCTRHead(kind, 6, 16, 13, ln_bot=[13, 32, 16], ln_top=[0, 64, 32, 1], seed=5, dense_ops="hip", dense_dtype=t).cuda()
    return head, torch.rand(B, 13, device="cuda"), torch.randn(6, B, 16, device="cuda")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("kind", ["dlrm", "wdl", "dcn"])
def test_the_loss_of_the_logit(kind, t):
    head, dense, emb = build(kind, t)
    u, tiny = torch.finfo(t).eps / 2, torch.finfo(t).smallest_normal * torch.finfo(t).eps
    for z in LOGITS + [-z for z in LOGITS]:
        last = with_logit(head, z)
        for label in (0.0, 1.0):
            out = head.logits(dense, emb)
            assert out.dtype == torch.float32 and (out == z).all()
            loss = nnf.binary_cross_entropy_with_logits(out, torch.full((B, 1), label, device="cuda"))
            db, = torch.autograd.grad(loss, last.bias)
            far = torch.tensor(z if label == 0 else -z, dtype=torch.float64)
            want = float(torch.sigmoid(far)) * (1 if label == 0 else -1)
            off = 8 * 2.0 ** -24 * (abs(want) + label) + 2.02 * u * abs(want) + B * tiny
            assert abs(float(db) - want) <= off, (z, label, float(db), want)
            assert abs(float(loss.detach()) - float(nnf.softplus(far))) <= 8 * 2.0 ** -24 * (1 + abs(z)), (z, label)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("kind", ["dlrm", "wdl", "dcn"])
def test_the_loss_of_the_probability_does_not_blow_up(kind, t):
    """BCELoss on forward(): at most 1.5 times the gradient at label 0 and 1, and none where the probability is the label's
    opposite to the last bit."""
    head, dense, emb = build(kind, t)
    for z in LOGITS + [-z for z in LOGITS]:
        last = with_logit(head, z)
        for label in (0.0, 1.0):
            out = head(dense, emb)
            db, = torch.autograd.grad(nnf.binary_cross_entropy(out, torch.full((B, 1), label, device="cuda")), last.bias)
            want = float(torch.sigmoid(torch.tensor(z if label == 0 else -z, dtype=torch.float64)))
            assert abs(float(db)) <= 1.51 * want + 2.0 ** -20, (z, label, float(db))
            if kind != "wdl" and float(out[0].detach()) in (0.0, 1.0):
                assert float(db) == 0.0


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["dlrm", "wdl", "dcn"])
def test_a_training_step_from_a_confident_wrong_model(kind, t):
    """One step of SGD at lr 1 moves the bias by the mean of p - label, 1 - e^-9, and leaves everything finite."""
    torch.manual_seed(0)
    counts = [4000, 197, 25000, 800, 12000, 161]
    m = CafeCTRModel(kind, counts, 16, compress_rate=0.05, threshold=3, ln_bot=[13, 32, 16], ln_top=[0, 64, 32, 1], seed=5, dense_ops="hip",
                     dense_dtype=t)
    last = with_logit(m.head, 9.0)
    before = float(last.bias.detach())
    opt = torch.optim.SGD(m.dense_parameters(), lr=1.0)
    ids = torch.stack([torch.arange(B, device="cuda") % n for n in counts])
    batch = [(torch.rand(B, 13, device="cuda"), ids, torch.zeros(B, 1, device="cuda"))]
    test_loss, hits = train.evaluate(m, batch)
    assert abs(test_loss - 9.0) <= 1e-3 and hits == 0.0
    loss = m.train_step(torch.rand(B, 13, device="cuda"), ids, torch.zeros(B, 1, device="cuda"), opt, 0.1)
    assert abs(float(loss) - 9.0) <= 1e-3                       # 9 + ln(1 + e^-9)
    want = before - (1 - 1.234e-4)
    assert abs(float(last.bias.detach()) - want) <= 3 * torch.finfo(t).eps * 9
    assert all(p.isfinite().all() for p in m.parameters()) and m.embedding.weight_high.isfinite().all()
