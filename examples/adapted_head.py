"""A head on the engine's descriptors, fine-tuned to several datasets at once and served for all of them together.

Every dataset stands for a level of theory, or a user, whose energies differ from the model's by a correction of its own.  The engine
evaluates the systems once; the scalars of its two layers (H1 and M1, 2 K numbers an atom) go through

    layer norm  ->  shared projection + low-rank adapter of the system's dataset  ->  SiLU  ->  readout

and the sum over a system's atoms is its correction.  The projection is fixed; the adapters, the layer norm's weight and bias and the
readout are trained by AdamW, on batches that hold systems of all datasets.  Data and weights are synthetic (random systems, a random-
initialised model, corrections made by a teacher of the same form).

    python examples/adapted_head.py [--steps 300] [--state-bits 8]
"""
import argparse
import os
import sys
import tempfile

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from symmetrix_amd import finetune, modelgen, neighbors, systems  # noqa: E402
from symmetrix_amd.mace import MACE  # noqa: E402


class AdaptedHead:
    """Corrections to energies from descriptors [atoms, d], one adapter a dataset."""

    def __init__(self, d, hidden, rank, datasets, seed, spread=0.0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        normal = lambda *s, scale: torch.randn(*s, generator=g, device="cuda") * scale          # noqa: E731
        self.projection = normal(hidden, d, scale=d ** -0.5)
        self.A = normal(datasets, rank, d, scale=d ** -0.5)
        self.B = normal(datasets, hidden, rank, scale=spread)          # (zeros: the shared projection alone at first)
        self.weight, self.bias = torch.ones(d, device="cuda"), torch.zeros(d, device="cuda")
        self.readout = normal(hidden, scale=hidden ** -0.5)

    def parameters(self):
        return [self.weight, self.bias, self.A, self.B, self.readout]

    def __call__(self, descriptors, dataset):
        """A number an atom; dataset: the adapter of every atom (int32, -1: none)."""
        x = finetune.layer_norm(descriptors, self.weight, self.bias)
        return torch.nn.functional.silu(finetune.adapted_linear(x, self.projection, self.A, self.B, None, dataset)) @ self.readout


def evaluate(model, path, count, atoms, seed):
    """Descriptors of `count` random systems [atoms, 2 K], and the system of every atom."""
    rows, system = [], []
    for i in range(count):
        pos, cell, species = systems.random_box(atoms, 0.1, [0.5, 0.3, 0.2], seed=seed + i)
        nl = neighbors.neighbor_list(pos, cell, model.r_cut)
        ea = neighbors.edge_arrays(nl, species)
        model.compute_node_energies_forces(ea["num_nodes"], ea["node_types"], ea["num_neigh"], ea["neigh_indices"], ea["neigh_types"], ea["xyz"], ea["r"])
        K = model.num_channels
        H1 = model.H1.reshape(atoms, -1, K)[:, 0]          # (the scalars among features of all orders)
        rows.append(np.concatenate([H1, model.M1.reshape(atoms, K)], axis=1))
        system += [i] * atoms
    return torch.tensor(np.concatenate(rows), dtype=torch.float32, device="cuda"), torch.tensor(system, device="cuda")


def per_system(numbers, system, count):
    return torch.zeros(count, device="cuda").index_add_(0, system, numbers)


def run(steps=300, datasets=4, per_dataset=6, atoms=40, channels=32, hidden=64, rank=4, state_bits=32, seed=0, quiet=False):
    """Trains a head and serves it; returns the loss before and after, and the corrections served."""
    handle, path = tempfile.mkstemp(suffix=".json")
    os.close(handle)
    try:
        modelgen.write_model(path, atomic_numbers=[1, 6, 8], num_channels=channels, L_max=1, r_cut=4.0, num_spline_points=64, seed=seed)
        model = MACE(path, "float32")
    finally:
        os.unlink(path)
    count = datasets * per_dataset
    descriptors, system = evaluate(model, path, count, atoms, seed)
    scale = descriptors.std(0, keepdim=True).clamp(min=1e-6)
    descriptors = descriptors / scale
    dataset = (system % datasets).to(torch.int32)          # systems of all datasets, in the order they came in
    teacher = AdaptedHead(descriptors.shape[1], hidden, rank, datasets, seed + 100, spread=0.5)
    wanted = per_system(teacher(descriptors, dataset), system, count) / atoms

    head = AdaptedHead(descriptors.shape[1], hidden, rank, datasets, seed + 200)
    head.projection, head.readout = teacher.projection, teacher.readout.clone()          # the shared projection is known
    params = [p.requires_grad_() for p in head.parameters()]
    optimizer = finetune.AdamW(params, lr=1e-2, weight_decay=1e-4, state_bits=state_bits)
    losses = []
    for step in range(steps):
        for p in params:
            p.grad = None
        loss = (per_system(head(descriptors, dataset), system, count) / atoms - wanted).square().mean()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
        if not quiet and step % 50 == 0:
            print(f"step {step}: loss {float(losses[-1]):.3e}", flush=True)
    # served: one call for the systems of all datasets
    with torch.no_grad():
        served = per_system(head(descriptors, dataset), system, count)
    if not quiet:
        print(f"loss {float(losses[0]):.3e} -> {float(losses[-1]):.3e} after {steps} steps, moments in {state_bits} bits")
    return float(losses[0]), float(losses[-1]), served, (head, descriptors, dataset, system, count)


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=300)
    ap.add_argument("--state-bits", type=int, default=32, choices=(8, 32))
    a = ap.parse_args()
    run(steps=a.steps, state_bits=a.state_bits)
