"""A head on the engine's descriptors with layers of every element's own, trained by clipped gradients.

The scalars of the engine's two layers (H1 and M1, 2 K numbers an atom) go through

    layer norm  +  the element's row of a table  ->  the element's layer  ->  SiLU  ->  the element's readout

and the sum over a system's atoms is its correction to the energy.  A batch's atoms are sorted by element once; both layers and all
gradients go by that.  AdamW takes the norm of all gradients and clips them in its own pass.  Data and weights are synthetic (random
systems, a random-initialised model, corrections made by a teacher of the same form).

    python examples/element_head.py [--steps 300] [--max-norm 1.0] [--dtype float32]
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

ELEMENTS = [1, 6, 8]


class ElementHead:
    """Corrections to energies from descriptors [atoms, d] and the atoms' elements."""

    def __init__(self, d, hidden, elements, seed, dtype=torch.float32):
        g = torch.Generator(device="cuda").manual_seed(seed)
        normal = lambda *s, scale: (torch.randn(*s, generator=g, device="cuda") * scale).to(dtype)          # noqa: E731
        self.elements = elements
        self.weight, self.bias = torch.ones(d, device="cuda", dtype=dtype), torch.zeros(d, device="cuda", dtype=dtype)
        self.table = normal(elements, d, scale=0.5)
        self.layer, self.layer_bias = normal(elements, hidden, d, scale=d ** -0.5), normal(elements, hidden, scale=0.1)
        self.readout, self.shift = normal(elements, 1, hidden, scale=hidden ** -0.5), normal(elements, 1, scale=0.1)

    def parameters(self):
        return [self.weight, self.bias, self.table, self.layer, self.layer_bias, self.readout, self.shift]

    def __call__(self, descriptors, element):
        """A number an atom; element: the element of every atom (int32), or its RowGroups."""
        x = finetune.layer_norm(descriptors, self.weight, self.bias) + finetune.embedding(self.table, element)
        h = torch.nn.functional.silu(finetune.grouped_linear(x, self.layer, self.layer_bias, element))
        return finetune.grouped_linear(h, self.readout, self.shift, element)[:, 0]


def evaluate(model, count, atoms, seed):
    """Descriptors of `count` random systems [atoms, 2 K], the element of every atom and its system."""
    rows, element, system = [], [], []
    for i in range(count):
        pos, cell, species = systems.random_box(atoms, 0.1, [0.5, 0.3, 0.2], seed=seed + i)
        nl = neighbors.neighbor_list(pos, cell, model.r_cut)
        ea = neighbors.edge_arrays(nl, species)
        model.compute_node_energies_forces(ea["num_nodes"], ea["node_types"], ea["num_neigh"], ea["neigh_indices"], ea["neigh_types"], ea["xyz"], ea["r"])
        K = model.num_channels
        H1 = model.H1.reshape(atoms, -1, K)[:, 0]          # (the scalars among features of all orders)
        rows.append(np.concatenate([H1, model.M1.reshape(atoms, K)], axis=1))
        element.append(np.asarray(ea["node_types"], dtype=np.int32))
        system += [i] * atoms
    return (torch.tensor(np.concatenate(rows), dtype=torch.float32, device="cuda"), torch.tensor(np.concatenate(element), device="cuda"),
            torch.tensor(system, device="cuda"))


def per_system(numbers, system, count):
    return torch.zeros(count, device="cuda").index_add_(0, system, numbers.float())


def run(steps=300, count=24, atoms=40, channels=32, hidden=64, max_norm=1.0, dtype=torch.float32, seed=0, quiet=False):
    """Trains a head; returns the loss before and after, the gradients' norm in every step, and the head with its batch."""
    handle, path = tempfile.mkstemp(suffix=".json")
    os.close(handle)
    try:
        modelgen.write_model(path, atomic_numbers=ELEMENTS, num_channels=channels, L_max=1, r_cut=4.0, num_spline_points=64, seed=seed)
        model = MACE(path, "float32")
    finally:
        os.unlink(path)
    descriptors, element, system = evaluate(model, count, atoms, seed)
    descriptors = (descriptors / descriptors.std(0, keepdim=True).clamp(min=1e-6)).to(dtype)
    d = descriptors.shape[1]
    element = finetune.group_rows(element, len(ELEMENTS))          # once for all calls of a batch
    with torch.no_grad():
        wanted = per_system(ElementHead(d, hidden, len(ELEMENTS), seed + 100, dtype)(descriptors, element), system, count) / atoms

    head = ElementHead(d, hidden, len(ELEMENTS), seed + 200, dtype)
    params = [p.requires_grad_() for p in head.parameters()]
    optimizer = finetune.AdamW(params, lr=3e-3, weight_decay=1e-4, masters=True if dtype != torch.float32 else None)
    losses, norms = [], []
    for step in range(steps):
        for p in params:
            p.grad = None
        loss = (per_system(head(descriptors, element), system, count) / atoms - wanted).square().mean()
        loss.backward()
        norms.append(optimizer.step(max_norm=max_norm))
        losses.append(loss.detach())
        if not quiet and step % 50 == 0:
            print(f"step {step}: loss {float(losses[-1]):.3e}, the gradients' norm {float(norms[-1]):.3e}", flush=True)
    if not quiet:
        print(f"loss {float(losses[0]):.3e} -> {float(losses[-1]):.3e} after {steps} steps")
    return float(losses[0]), float(losses[-1]), [float(n) for n in norms], (head, descriptors, element, system)


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=300)
    ap.add_argument("--max-norm", type=float, default=1.0)
    ap.add_argument("--dtype", default="float32", choices=("float32", "bfloat16", "float16"))
    a = ap.parse_args()
    run(steps=a.steps, max_norm=a.max_norm, dtype=getattr(torch, a.dtype))
