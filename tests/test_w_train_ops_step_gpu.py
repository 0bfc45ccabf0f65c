"""The Trainer's step with the fused optimizer and the layer norm kernel: against torch's on a small network, eagerly and
captured, and the synthetic CMR-style step with all of it together."""
import os
import sys

import pytest
import torch

from nnutils import train_utils

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "examples"))


class Small(train_utils.Trainer):
    """Two blocks with layer norms on random vectors."""
    graph_inputs = ("x", "y")

    def init_dataset(self):
        g = torch.Generator().manual_seed(1)
        data = [(torch.randn(40, generator=g), torch.randn(5, generator=g)) for _ in range(64)]
        self.dataloader = torch.utils.data.DataLoader(data, batch_size=self.opts.batch_size, shuffle=False, drop_last=True)

    def define_model(self):
        torch.manual_seed(2)
        nn = torch.nn
        self.model = nn.Sequential(nn.Linear(40, 160), nn.LayerNorm(160), nn.ReLU(), nn.Linear(160, 90), nn.LayerNorm(90),
                                   nn.ReLU(), nn.Linear(90, 5))

    def define_criterion(self):
        pass

    def set_input(self, batch):
        self.x, self.y = (t.to(self.device) for t in batch)

    def forward(self, total_steps=0):
        self.total_loss = (self.model(self.x).float() - self.y).square().mean()


def trained(tmp_path, *argv, steps=6, scale=None):
    parser = train_utils.add_training_flags()
    o = parser.parse_args(["--num_iter", str(steps), "--batch_size", "8", "--print_scalars", "0", "--learning_rate", "1e-3",
                           "--checkpoint_dir", str(tmp_path), "--epoch_fraction", "1.0", *argv])
    t = Small(o)
    t.init_training()
    if scale is not None:
        t._scaler = torch.amp.GradScaler("cuda", init_scale=scale)
    assert t.train() == steps
    return t


def weights(t):
    return [p.detach().clone() for p in t.model.parameters()]


def test_fused_step_and_layer_norm_follow_torchs(tmp_path):
    import sv3d
    a = trained(tmp_path, "--amp", "0")
    b = trained(tmp_path, "--amp", "0", "--optim", "adamw", "--hip_layer_norm", "1")
    assert type(a.optimizer) is torch.optim.Adam and type(a.model[1]) is torch.nn.LayerNorm
    assert type(b.optimizer) is sv3d.optim.AdamW and type(b.model[1]) is type(b.model[4]) is sv3d.LayerNorm
    # six float32 steps of 1e-3: a step is lr times a ratio of moments that roundings change by some 1e-6, more only
    # where a gradient is near eps, the size of the loss of digits in a sum
    for x, y in zip(weights(a), weights(b)):
        assert float((x - y).abs().max()) < 1e-4


def test_loss_scale_goes_through_the_fused_step(tmp_path):
    t = trained(tmp_path, "--optim", "adamw", "--hip_layer_norm", "1", scale=256.0)
    assert all(float(s["step"]) == 6.0 for s in t.optimizer.state.values())
    assert float(t.optimizer.total_norm) < 100.0       # of unscaled gradients: scaled ones are 256 times as large
    assert all(torch.isfinite(w).all() for w in weights(t))


@pytest.mark.parametrize("optim, room", [("adamw", 1e-4), ("adamw8", 1e-3)])
def test_whole_step_captured_follows_the_eager_one(tmp_path, optim, room):
    """--cuda_graph 2 with the fused optimizer: three eager steps, capture, replays.  Eight steps of 1e-3 move a weight by
    8e-3; last-bit differences of the library's products may turn a rounding of an 8-bit moment, an eighth of a step."""
    argv = ["--optim", optim, "--hip_layer_norm", "1", "--amp", "0", "--weight_decay", "0.01"]
    a, b = trained(tmp_path, *argv, steps=8), trained(tmp_path, *argv, "--cuda_graph", "2", steps=8)
    assert b._graph is not None and b._graph["whole"]
    for x, y in zip(weights(a), weights(b)):
        assert float((x - y).abs().max()) < room
    assert all(float(s["step"]) == 8.0 for s in b.optimizer.state.values())


def test_cmr_step_with_8_bit_moments_layer_norms_and_a_captured_step(tmp_path):
    import cmr_synthetic
    argv = ["--num_iter", "7", "--batch_size", "2", "--img_size", "64", "--subdivide", "2", "--tex_size", "4",
            "--num_parts", "3", "--seg_train", "1", "--checkpoint_dir", str(tmp_path), "--print_scalars", "0",
            "--dataset_size", "32", "--learning_rate", "1e-3", "--optim", "adamw8", "--fc_norm", "layer", "--cuda_graph", "2"]
    o = cmr_synthetic.parse(argv)
    o.epoch_fraction = 1.0
    t = cmr_synthetic.ShapeTrainer(o)
    t.init_training()
    t._scaler = torch.amp.GradScaler("cuda", init_scale=256.0)
    before = [p.detach().clone() for p in t.model.parameters()]
    part = t.part_basis_generator.w.detach().clone()
    assert t.train() == 7
    assert t._graph is not None and t._graph["whole"] and torch.isfinite(t.total_loss)
    states = list(t.optimizer.state.values()) + list(t.optimizer_2.state.values())
    assert states and all(float(s["step"]) == 7.0 for s in states)
    assert any(s["exp_avg"].dtype == torch.uint8 for s in states) and any(s["exp_avg"].dtype == torch.float32 for s in states)
    moved = [not torch.equal(p, q) for p, q in zip(t.model.parameters(), before)]
    assert all(torch.isfinite(p).all() for p in t.model.parameters()) and sum(moved) > 0.9 * len(moved)
    assert not torch.equal(part, t.part_basis_generator.w)
    norms = [m for m in t.model.modules() if type(m).__name__ == "LayerNorm"]
    assert len(norms) == 2 and all(m.weight.grad is not None and m.weight.grad.abs().max() > 0 for m in norms)
