"""Fits per-species networks over NEP descriptors to energies, on the GPU from positions to updates:

    neighbour lists and descriptors of a batch   capi.nblist_build_batch, capi.nep_descriptors
    atoms sorted by species, and back            fitnet.route, dispatch, combine
    three layers, one set per species            fitnet.dense (tanh, residual)
    updates of the layers' matrices              fitnet.orthogonalize of their momentum (Muon); plain steps for the rest

    python examples/fit_species_network.py [--steps 300] [--dtype f32|bf16] [--width 128]

The targets are energies of a NEP model with random parameters over random crystals of three species, of different sizes: a padded batch, in which
padding has species -1. Prints the error per atom (in units of the targets' spread) as it goes."""
import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from ai2pot_b200 import capi, fitnet, synth  # noqa: E402

NTYPES, RCUT, UMAX = 3, 6.0, 64


def batch_of_crystals(frames, seed):
    """Neighbour tensors of `frames` perturbed crystals of 27 to 125 atoms, and their descriptors and energies by a random NEP model."""
    rng = np.random.default_rng(seed)
    structures = []
    for _ in range(frames):
        n = int(rng.integers(27, 126))
        cell, pos = synth.cubic_lattice(int(np.ceil(n ** (1 / 3) - 1e-9)), float(rng.uniform(2.8, 3.2)), 0.2, rng, np.float32, nocc=n)
        structures.append((cell, pos, rng.integers(0, NTYPES, n)))
    npad = max(len(s[1]) for s in structures)
    coords, types = np.zeros((frames, npad, 3), np.float32), np.full((frames, npad), -1, np.int32)
    for b, (_, pos, ty) in enumerate(structures):
        coords[b, :len(pos)], types[b, :len(ty)] = pos, ty
    binum = torch.tensor([len(s[1]) for s in structures], dtype=torch.int32, device="cuda")
    nb = capi.nblist_build_batch(np.stack([s[0] for s in structures]), binum, torch.from_numpy(coords).cuda(), RCUT, UMAX)
    types = torch.from_numpy(types).cuda()
    nb.update(btypes=types.clamp(min=0), ntypes=NTYPES, nghost=0)
    model = capi.to_device(synth.nep_model(NTYPES, rng, np.float32, sigma=0.5))
    energy = capi.nep_efv(model, nb, virial=False)[0]
    return types, capi.nep_descriptors(model, nb), energy / binum


class SpeciesNetwork(torch.nn.Module):
    """One network of two hidden layers for each species; every atom's energy comes from the network of its species."""

    def __init__(self, inputs, width, ntypes, dtype, generator):
        super().__init__()
        def stack(outer, inner):
            return torch.nn.Parameter((torch.randn(ntypes, outer, inner, generator=generator, device="cuda") * inner ** -0.5).to(dtype))
        def zeros(outer):
            return torch.nn.Parameter(torch.zeros(ntypes, outer, dtype=dtype, device="cuda"))
        self.w1, self.b1 = stack(width, inputs), zeros(width)
        self.w2, self.b2 = stack(width, width), zeros(width)
        self.w3, self.b3 = stack(1, width), zeros(1)

    def forward(self, types, descriptors):
        """types [atoms] (padding: negative), descriptors [atoms, inputs] -> energies [atoms] (padding: zero)."""
        route = fitnet.route(types, self.w1.shape[0])
        h = fitnet.dispatch(descriptors, route)
        h = fitnet.dense(h, self.w1, self.b1, activation="tanh", offsets=route.offsets)
        h = fitnet.dense(h, self.w2, self.b2, residual=h, activation="tanh", offsets=route.offsets)
        e = fitnet.dense(h, self.w3, self.b3, offsets=route.offsets)
        return fitnet.combine(e, torch.ones(types.shape[0], 1, device=types.device), route)[:, 0]


class Muon:
    """Momentum whose direction is orthogonalised, for stacks of matrices; plain momentum steps for everything else."""

    def __init__(self, matrices, others, lr, lr_others, momentum=0.9):
        self.groups = [(list(matrices), lr, True), (list(others), lr_others, False)]
        self.momentum = momentum
        self.buffers = {}

    @torch.no_grad()
    def step(self, scale=1.0):
        for params, lr, orthogonal in self.groups:
            for p in params:
                buf = self.buffers.setdefault(p, torch.zeros_like(p, dtype=torch.float32))
                buf.mul_(self.momentum).add_(p.grad)
                update = fitnet.orthogonalize(buf.to(p.dtype)) if orthogonal else buf
                p.add_(update.to(p.dtype), alpha=-lr * scale)
                p.grad = None


def fit(steps=300, dtype=torch.float32, width=128, frames=64, seed=0, report=None):
    """Returns the root mean square errors per atom, in units of the targets' spread, before the first and after the last step."""
    types, descriptors, target = batch_of_crystals(frames, seed)
    atoms = types.reshape(-1)
    present = (atoms >= 0)
    x = descriptors.reshape(atoms.shape[0], -1)
    mean, std = x[present].mean(0), x[present].std(0) + 1e-6
    x = (((x - mean) / std) * present[:, None]).to(dtype)
    target = (target - target.mean()) / target.std()
    count = present.view(types.shape).sum(1)
    net = SpeciesNetwork(x.shape[1], width, NTYPES, dtype, torch.Generator(device="cuda").manual_seed(seed))
    optimiser = Muon([net.w1, net.w2], [net.w3, net.b1, net.b2, net.b3], lr=0.02, lr_others=0.02)
    errors = []
    for step in range(steps + 1):
        energy = net(atoms, x).float().view(types.shape).sum(1) / count
        loss = ((energy - target) ** 2).mean()
        if step in (0, steps) or (report and step % 50 == 0):
            errors.append(float(loss.detach()) ** 0.5)
            if report:
                report(step, errors[-1])
        if step < steps:
            loss.backward()
            optimiser.step(1.0 - step / steps)
    fitnet.check()
    return errors[0], errors[-1]


if __name__ == "__main__":
    parser = argparse.ArgumentParser()
    parser.add_argument("--steps", type=int, default=300)
    parser.add_argument("--width", type=int, default=128)
    parser.add_argument("--dtype", choices=["f32", "bf16"], default="f32")
    a = parser.parse_args()
    fit(a.steps, {"f32": torch.float32, "bf16": torch.bfloat16}[a.dtype], a.width, report=lambda step, e: print(f"step {step:4d}  error per atom {e:.4f}"))
