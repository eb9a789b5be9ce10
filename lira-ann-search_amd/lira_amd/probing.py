"""The probing model that sits between partition ranking and the scan.

LIRA scores every partition with a two-tower MLP (model_probing.py:5-39):
sigmoid(fc([dist_tower(standardised centroid distances) || vec_tower(query)])).
It is *called* on the query path (search.cpp:430-445) but it is a handful of
small dense layers, so it runs as a PyTorch-ROCm module (hipBLASLt GEMMs) by
default; ``MX4Probe`` is its 4-bit form on the library's own kernels.  Parameter
names match MLP_2_Input, so a state_dict or a TorchScript file trained by the
reference loads unchanged.
"""
from __future__ import annotations

import torch
from torch import nn


def _tower(n_in: int, hidden: int, n_out: int) -> nn.Sequential:
    return nn.Sequential(nn.Linear(n_in, hidden), nn.ReLU(), nn.Linear(hidden, n_out), nn.ReLU())


class MLP_2_Input(nn.Module):  # noqa: N801 - reference class name, kept for drop-in loading
    """input_dim1 = n_bkt (distance features), input_dim2 = d, output_dim = n_bkt."""

    def __init__(self, input_dim1: int, input_dim2: int, output_dim: int):
        super().__init__()
        self.distance_net = _tower(input_dim1, 128, 64)
        self.vector_net = _tower(input_dim2, 128, 64)
        self.fc = nn.Sequential(nn.Linear(128, 128), nn.ReLU(), nn.Linear(128, output_dim), nn.Sigmoid())

    def forward(self, x_dist: torch.Tensor, x_vec: torch.Tensor) -> torch.Tensor:
        return self.fc(torch.cat((self.distance_net(x_dist), self.vector_net(x_vec)), dim=1))

    def logits(self, x_dist: torch.Tensor, x_vec: torch.Tensor) -> torch.Tensor:
        """The scores before the sigmoid: what a distillation loss takes."""
        return self.fc[:-1](torch.cat((self.distance_net(x_dist), self.vector_net(x_vec)), dim=1))


class MX4Linear(nn.Module):
    """A linear layer in 4 bits: packed weights and the bias as buffers, so that ``state_dict()``, ``to()`` and copies
    take them along.  Runs where they are on the GPU."""

    def __init__(self, weight: torch.Tensor, bias: torch.Tensor):
        super().__init__()
        from .mx4 import mx4_quantize
        with torch.no_grad():
            w = mx4_quantize(weight.float())
            self.register_buffer("codes", w.codes)
            self.register_buffer("scales", w.scales)
            self.register_buffer("bias", bias.float().clone())
        self.in_features, self.out_features = w.k, w.n
        self._packed = w

    def weight(self):
        """The MX4Tensor of the buffers as they are now (``to()`` and ``load_state_dict(assign=True)`` put others
        in their place)."""
        from .mx4 import MX4Tensor
        w, codes, scales = self._packed, self._buffers["codes"], self._buffers["scales"]
        if w.codes is not codes or w.scales is not scales:
            w = self._packed = MX4Tensor(codes, scales, self.in_features)
        return w

    def forward(self, x: torch.Tensor, activation: str | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
        from .mx4 import mx4_linear
        return mx4_linear(x, self.weight(), self._buffers["bias"], activation, out=out)


class MX4Probe(nn.Module):
    """A trained probing model in 4 bits: the layers of MLP_2_Input (model_probing.py:5-39) with
    packed weights, the activations packed on the way into each (lira_mx4_linear: bias and ReLU or
    sigmoid in the product's epilogue).  Takes the place of the fp32 model in ``ProbePipeline`` and
    ``SearchEngine``; inference alone.  ``model``: an MLP_2_Input, or any module with its state_dict
    (a TorchScript file of the reference), on the GPU.
    """

    _LAYERS = ("distance_net.0", "distance_net.2", "vector_net.0", "vector_net.2", "fc.0", "fc.2")

    def __init__(self, model: nn.Module):
        super().__init__()
        state = model.state_dict()
        names = [k + e for k in self._LAYERS for e in (".weight", ".bias")]
        missing, more = [k for k in names if k not in state], [k for k in state if k not in names]
        if missing or more:
            raise ValueError("MX4Probe needs an MLP_2_Input: the model has " +
                             (f"no {missing[0]}" if missing else f"{more[0]} as well"))
        # (the names of MLP_2_Input's layers)
        for net in ("distance_net", "vector_net", "fc"):
            self.add_module(net, nn.ModuleDict({
                i: MX4Linear(state[f"{net}.{i}.weight"], state[f"{net}.{i}.bias"]) for i in ("0", "2")}))

    @torch.no_grad()
    def forward(self, x_dist: torch.Tensor, x_vec: torch.Tensor) -> torch.Tensor:
        # (straight to the layers' code: nn.Module's own call takes as long on the host as a layer)
        d0, d2, v0, v2, f0, f2 = (layer.forward for net in self._modules.values() for layer in net._modules.values())
        nd = self.distance_net["2"].out_features
        both = torch.empty((x_dist.shape[0], nd + self.vector_net["2"].out_features), dtype=torch.float32,
                           device=x_dist.device)
        d2(d0(x_dist.float(), "relu"), "relu", out=both[:, :nd])
        v2(v0(x_vec.float(), "relu"), "relu", out=both[:, nd:])
        return f2(f0(both, "relu"), "sigmoid")


class NearestCentroidProbe(nn.Module):
    """Scores 1.0 for the nprobe smallest distance features, else 0.0.

    With scaler mean 0 / scale 1 and a threshold in (0, 1], the threshold probe
    of search.cpp:447-466 then selects exactly the IVF nprobe nearest centroids
    (the oracle's construction).  Ties at the boundary score 1.
    """

    def __init__(self, nprobe: int):
        super().__init__()
        self.nprobe = nprobe

    def forward(self, x_dist: torch.Tensor, x_vec: torch.Tensor) -> torch.Tensor:
        kth = torch.topk(x_dist, self.nprobe, dim=1, largest=False).values[:, -1:]
        return (x_dist <= kth).float()


@torch.no_grad()
def probe_scores(model, dist_scaled: torch.Tensor, q: torch.Tensor, batch: int = 65536) -> torch.Tensor:
    """Model scores (n, n_bkt) for a whole query batch (model_infer, model_probing.py:135-156)."""
    outs = [model(dist_scaled[s:s + batch], q[s:s + batch]) for s in range(0, q.shape[0], batch)]
    return torch.cat(outs).float() if outs else torch.zeros((0, dist_scaled.shape[1]), device=q.device)


def standard_scaler(dist: torch.Tensor):
    """sklearn StandardScaler.fit over (n, B) distances, as utils.py:139-142 /
    166-178 save it for search.cpp: per-bucket mean and population std, a zero
    std replaced by 1 (search.cpp:247 does the same at use)."""
    d = dist.double()
    mean = d.mean(0)
    std = d.std(0, unbiased=False)
    std = torch.where(std == 0, torch.ones_like(std), std)
    return mean.float(), std.float()


def fit_probe_to_nearest(model: nn.Module, dist_scaled_fn, nprobe: int, steps: int = 300, batch: int = 4096,
                         lr: float = 2e-3, seed: int = 0, distill_weight: float = 0.0,
                         temperature: float = 1.0) -> nn.Module:
    """Train MLP_2_Input to score each query's nprobe nearest centroids 1 and
    the rest 0 (BCE, Adam), from batches dist_scaled_fn(batch, step) ->
    (standardised distances (n, B), queries (n, d)).

    A synthetic stand-in for LIRA's training on kNN partition labels
    (model_probing.py:41-54, LIRA_smallscale.py:308-329; training is outside
    the query-time hot path), so that the MLP-probed pipeline selects a
    realistic number of partitions at threshold 0.5 instead of a random-init
    model's arbitrary ones.

    distill_weight > 0 adds that much of distill_topk_loss: the exact ranking is
    the teacher, the nprobe smallest distances (negated) its top logits, so the model
    also learns the ORDER of the near partitions, which the 0 / 1 targets leave out.
    """
    torch.manual_seed(seed)
    opt = torch.optim.Adam(model.parameters(), lr=lr)
    lossf = nn.BCELoss()
    model.train()
    for it in range(steps):
        xd, xq = dist_scaled_fn(batch, it)
        near = torch.topk(xd, nprobe, dim=1, largest=False)
        target = (xd <= near.values[:, -1:]).float()
        opt.zero_grad(set_to_none=True)
        if distill_weight > 0:
            from .distill import distill_topk_loss
            logits = model.logits(xd, xq)
            loss = lossf(torch.sigmoid(logits), target) + \
                distill_weight * distill_topk_loss(logits, near.indices, -near.values, temperature)
        else:
            loss = lossf(model(xd, xq), target)
        loss.backward()
        opt.step()
    model.eval()
    return model
