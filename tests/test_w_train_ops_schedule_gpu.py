"""The captured step with the fused optimizer under a schedule: weights that get their first gradient on a branch that is
captured later."""
import pytest
import torch

from nnutils import train_utils
from test_w_train_ops_step_gpu import Small, weights

pytestmark = pytest.mark.gpu


class Scheduled(Small):
    """The last layer joins in at some steps only, the first of them after the other branch was captured."""

    def graph_key(self, total_steps):
        return total_steps >= 5 and total_steps % 2 == 1

    def forward(self, total_steps=0):
        h = self.model[:6](self.x).float()
        self.total_loss = h.square().mean()
        if self.graph_key(total_steps):
            self.total_loss = self.total_loss + (self.model[6](h) - self.y).square().mean()


def trained(tmp_path, *argv, steps=10):
    o = train_utils.add_training_flags().parse_args(
        ["--num_iter", str(steps), "--batch_size", "4", "--print_scalars", "0", "--learning_rate", "1e-3", "--amp", "0",
         "--checkpoint_dir", str(tmp_path), "--epoch_fraction", "1.0", *argv])
    t = Scheduled(o)
    t.init_training()
    assert t.train() == steps
    return t


@pytest.mark.parametrize("optim, room", [("adamw", 1e-4), ("adamw8", 1e-3)])
def test_weights_whose_first_gradient_comes_with_a_later_capture(tmp_path, optim, room):
    """Ten steps of 1e-3, the last layer's three (5, 7, 9); differences as in the captured step without a schedule."""
    a, b = trained(tmp_path, "--optim", optim), trained(tmp_path, "--optim", optim, "--cuda_graph", "2")
    assert len(b._graphs) == 2 and all(g["whole"] for g in b._graphs.values())
    for x, y in zip(weights(a), weights(b)):
        assert float((x - y).abs().max()) < room
    for t in (a, b):
        last = list(t.model[6].parameters())
        assert [float(t.optimizer.state[p]["step"]) for p in last] == [3.0] * len(last)
        assert all(float(s["step"]) == 10.0 for p, s in t.optimizer.state.items() if all(p is not q for q in last))
