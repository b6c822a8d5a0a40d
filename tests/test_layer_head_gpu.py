"""The networks with `projection_norm: layer`, and a train step of them with FusedMuon, against the float64 torch
restatement with its BatchNorm1d exchanged for a layer norm (oracle/torch_port.py, pinned to the reference's fixtures).

Tolerances are those of the BatchNorm1d head's own tests (embeddings 1e-5, loss 1e-4, gradients 2e-3 max|g| per tensor):
the trunk's rounding, which they bound, is the same, and the layer norm adds 64 float32 roundings of one embedding."""
import json
import logging
import os
import tempfile
from pathlib import Path

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from golden_util import bn_fed_bias
from oracle import torch_port as tp

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def layer_port(monkeypatch):
    """oracle/torch_port.py with a layer norm behind the projection."""
    bn, count = tp._bn, tp._count
    monkeypatch.setattr(tp, "_bn", lambda sd, name, y, train: F.layer_norm(
        y, y.shape[1:], sd[name + ".weight"], sd[name + ".bias"], 1e-5) if name == "projection.1" else bn(sd, name, y, train))
    monkeypatch.setattr(tp, "_count", lambda sd, names, train: count(sd, [n for n in names if n != "projection.1"], train))
    return tp


def doubles(sd):
    return {k: v.detach().cpu().clone().double() if v.is_floating_point() else v.cpu().clone() for k, v in sd.items()}


def build(kind, D, att, seed):
    from phoneme_contrast_amd.models import model_registry
    torch.manual_seed(seed)
    m = model_registry.create(kind, {"embedding_dim": D, "use_attention": att, "dropout_rate": 0.1,
                                     "projection_norm": "layer", "hidden_dims": [16, 32, 64, 128]})
    with torch.no_grad():  # weights and biases away from 1 and 0
        for p in m.projection[1].parameters():
            p.add_(0.2 * torch.randn(p.shape))
        m.projection[0].bias.add_(0.1 * torch.randn(D))
    return m


@pytest.mark.parametrize("kind,B,T,D,att", [("phoneme_cnn", 6, 100, 128, True), ("phoneme_cnn", 3, 57, 64, False),
                                            ("phoneme_cnn", 1, 64, 32, True), ("phoneme_cnn", 5, 41, 7, True),
                                            ("phoneme_cnn_deep", 4, 100, 128, True), ("phoneme_cnn_deep", 1, 80, 256, True)])
def test_forward_and_gradients(layer_port, kind, B, T, D, att):
    m = build(kind, D, att, B * 100 + T)
    sd = doubles(m.state_dict())
    assert "projection.1.running_mean" not in sd and "projection.1.weight" in sd
    m = m.cuda().train()
    x = torch.randn(B, 1, 40, T)
    ch = (32, 64, 128) if kind == "phoneme_cnn" else (16, 32, 64, 128)
    masks = [(torch.rand(B, c) >= 0.1).float() / 0.9 for c in ch]
    m.set_dropout_masks(masks)
    e = m(x.cuda())
    up = torch.randn(B, D)
    e.backward(up.cuda())
    names = tp.param_names(sd)
    for k in names:
        sd[k].requires_grad_(True)
    er = layer_port.forward(sd, x.double(), True, [k.double() for k in masks])
    er.backward(up.double())
    assert (e.detach().cpu().double() - er.detach()).abs().max() < 1e-5
    got = dict(m.named_parameters())
    for k in names:
        g, r = got[k].grad.cpu().double(), sd[k].grad
        if bn_fed_bias(k, None) and not k.startswith("projection"):
            assert g.abs().max() < 1e-4 and r.abs().max() < 1e-4, k
            continue
        assert (g - r).abs().max() <= 2e-3 * r.abs().max() + 1e-12, k
    m.eval()
    with torch.no_grad():
        ev = m(x.cuda()).cpu()
        ref = layer_port.forward(doubles(m.state_dict()), x.double(), False)
    assert (ev.double() - ref).abs().max() < 1e-5


def test_an_embedding_does_not_depend_on_its_batch():
    """In evaluation mode every sample is computed by itself with either norm; with the layer norm the projection head
    is so in training too: the same pooled features give the same bits whatever else the batch holds."""
    m = build("phoneme_cnn", 128, True, 5).cuda().eval()
    x = torch.randn(9, 1, 40, 100, device="cuda")
    with torch.no_grad():
        assert torch.allclose(m(x)[:4], m(x[:4]), atol=1e-6)


def test_unknown_norm_is_refused():
    from phoneme_contrast_amd.models import PhonemeNet
    with pytest.raises(ValueError, match="projection_norm"):
        PhonemeNet({"projection_norm": "group"})
    with pytest.raises(ValueError, match="more than 1 value"):
        PhonemeNet({}).cuda().train()(torch.randn(1, 1, 40, 64, device="cuda"))


def test_training_steps_with_orthogonalised_updates(layer_port):
    """Two steps of the whole train step: network with layer norm, SupCon, FusedMuon.  The gradients are checked against
    the float64 port at the step's own parameters, the update against its formula on the step's own gradients (the
    iteration magnifies a gradient's rounding in its smallest singular directions: the two are separate claims)."""
    from phoneme_contrast_amd.losses import SupervisedContrastiveLoss
    from phoneme_contrast_amd.optim import FusedMuon
    from test_muon_gpu import adam_reference, reference_step
    m = build("phoneme_cnn", 64, True, 11).cuda().train()
    opt = FusedMuon(m.parameters(), lr=3e-3, weight_decay=1e-2)
    x, labels = torch.randn(12, 1, 40, 100), torch.arange(12) // 3
    fn = SupervisedContrastiveLoss(temperature=0.15)
    zeros = {n: torch.zeros_like(p).cpu().double() for n, p in m.named_parameters()}
    mom, second = dict(zeros), dict(zeros)
    for step in (1, 2):
        sd = doubles(m.state_dict())
        masks = [(torch.rand(12, c) >= 0.1).float() / 0.9 for c in (32, 64, 128)]
        m.set_dropout_masks(masks)
        loss = fn(m(x.cuda()), labels.cuda())
        opt.zero_grad()
        loss.backward()
        grads = {n: p.grad.detach().cpu().double() for n, p in m.named_parameters()}
        opt.step()
        names = tp.param_names(sd)
        for k in names:
            sd[k].requires_grad_(True)
        ref = tp.supcon(layer_port.forward(sd, x.double(), True, [k.double() for k in masks]), labels, 0.15, 0.07)
        ref.backward()
        assert abs(loss.item() - ref.item()) < 1e-4
        for n, p in m.named_parameters():
            if not (bn_fed_bias(n, None) and not n.startswith("projection")):
                assert (grads[n] - sd[n].grad).abs().max() <= 2e-3 * sd[n].grad.abs().max() + 1e-12, n
            got, before = p.detach().cpu().double(), sd[n].detach()
            if p.dim() >= 2 and min(p.shape[0], p.numel() // p.shape[0]) > 1:
                want, mom[n], tol = reference_step(before, grads[n], mom[n], 3e-3, 0.95, True, 1e-2, "rms")
                assert (got - want).norm().item() <= tol, n
            else:
                want, mom[n], second[n] = adam_reference(before, grads[n], mom[n], second[n], step, 3e-3, 1e-2)
                # where the moments are rounding noise (a bias in front of a norm), Adam's quotient is noise too
                loud = grads[n].abs() > 1e-7
                assert ((got - want).abs() <= 16 * 2.0 ** -24 * (want.abs() + 4 * 3e-3))[loud].all(), n


def test_train_entry_with_layer_norm_and_orthogonalised_updates():
    """scripts/train.py with accel.optimizer=muon model.projection_norm=layer: clipping, schedule, checkpoints."""
    from test_trainer_gpu import _compose, _train_module
    out = Path(tempfile.mkdtemp())
    cfg = _compose(["accel.synthetic_data=true", "accel.synthetic.num_classes=48", "accel.synthetic.samples_per_class=3",
                    "data.contrastive.classes_per_batch=8", "training.epochs=2", "training.batch_size=32", "model=cnn_small",
                    "accel.optimizer=muon", "model.projection_norm=layer"], out)
    mod = _train_module()
    tr = mod.main(cfg)
    m = json.load(open(out / "metrics.json"))
    assert len(m["train_loss"]) == 2 and all(np.isfinite(m["train_loss"])) and m["train_lr"][1] < m["train_lr"][0]
    from phoneme_contrast_amd.optim import FusedMuon
    assert isinstance(tr.optimizer, FusedMuon)
    saved = torch.load(out / "checkpoints" / "checkpoint_final.pt", weights_only=True, map_location="cuda")
    state = saved["optimizer_state_dict"]["state"]
    assert any("momentum_buffer" in s for s in state.values()) and any("exp_avg" in s for s in state.values())
    tr.load_checkpoint(out / "checkpoints" / "checkpoint_final.pt")
    with pytest.raises(ValueError, match="accel.optimizer"):
        mod.setup_model(_compose(["accel.optimizer=sgd"], out), torch.device("cuda"))
    logging.getLogger("phoneme_contrast").handlers.clear()


def test_gradient_buckets_and_global_flat_steps():
    """flat_grad_views of FusedMuon is the backward's own buffer (no copy), and clipping acts on it."""
    from phoneme_contrast_amd import distributed as ddp
    from phoneme_contrast_amd.optim import FusedMuon
    m = build("phoneme_cnn", 128, True, 3).cuda().train()
    opt = FusedMuon(m.parameters(), lr=1e-3)
    assert ddp.covers(opt, m)
    e = m(torch.randn(4, 1, 40, 64, device="cuda"))
    e.backward(torch.randn_like(e))
    (flat,) = opt.flat_grad_views()
    first = next(m.parameters())
    assert flat.data_ptr() == first.grad.data_ptr() and flat.numel() == sum(p.numel() for p in m.parameters())
    norm = ddp.clip_flat_([flat], 1e-3)
    assert torch.linalg.vector_norm(flat).item() <= 1e-3 * 1.001 and norm.item() > 0
    opt.step(flat_grads=[flat])
    assert all(torch.isfinite(p).all() for p in m.parameters())


@pytest.mark.parametrize("att", [True, False])
def test_a_training_embedding_depends_on_no_other_sample(att):
    """In training the trunk's BatchNorm2d mixes samples; with weights of 0 they hand on their biases, whatever the batch, and
    the dropout masks tell the samples apart.  The head's embedding of a sample then has the same bits alone and in any
    batch with the layer norm, and does not with BatchNorm1d.  (The deep network's head is the same code; its last block
    has no mask behind its last norm.)"""
    def embed(model, masks, pick, x):
        for m in model.modules():
            if isinstance(m, torch.nn.BatchNorm2d):
                m.weight.data.zero_()
                m.bias.data.copy_(torch.linspace(0.5, 1.5, m.bias.numel()))
        model.set_dropout_masks([k[pick] for k in masks])
        with torch.no_grad():
            return model(x[pick].cuda())
    x = torch.randn(9, 1, 40, 100)
    masks = [(torch.rand(9, c) >= 0.3).float() / 0.7 for c in (32, 64, 128)]
    layer = build("phoneme_cnn", 128, att, 7).cuda().train()
    from phoneme_contrast_amd.models import model_registry
    batch = model_registry.create("phoneme_cnn", {**layer.config, "projection_norm": "batch"})
    batch.load_state_dict(layer.state_dict(), strict=False)
    batch = batch.cuda().train()
    whole, mixed = embed(layer, masks, torch.arange(9), x), embed(batch, masks, torch.arange(9), x)
    assert (whole[0] - whole[1]).abs().max() > 1e-3  # (the samples do differ)
    for pick in ([3], [0], [8, 3], [5, 1, 2, 3], [3, 3, 3, 0, 7, 6]):
        pick = torch.tensor(pick)
        assert torch.equal(embed(layer, masks, pick, x), whole[pick.cuda()])
        if len(pick) > 1:
            assert (embed(batch, masks, pick, x) - mixed[pick.cuda()]).abs().max() > 1e-3
