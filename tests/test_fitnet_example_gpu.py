"""The fitting example runs the operators together, from positions to orthogonalised updates, and learns."""
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_fit_species_network(dtype):
    import fit_species_network as example
    before, after = example.fit(steps=150, dtype=dtype, width=96, frames=32)
    assert after < 0.5 * before and after < 0.5, (before, after)


def test_network_is_the_same_as_one_per_species():
    """Energies and gradients equal those of separate networks over masked atoms, in 64 bits."""
    import fit_species_network as example
    net = example.SpeciesNetwork(20, 48, 3, torch.float32, torch.Generator(device="cuda").manual_seed(1))
    g = torch.Generator(device="cuda").manual_seed(2)
    types = torch.randint(-1, 3, (700,), generator=g, device="cuda", dtype=torch.int32)
    x = torch.randn(700, 20, generator=g, device="cuda")
    e = net(types, x)
    e.sum().backward()
    p = {k: v.detach().double().requires_grad_() for k, v in net.named_parameters()}
    want = torch.zeros(700, dtype=torch.float64, device="cuda")
    for t in range(3):
        rows = (types == t).nonzero()[:, 0]
        h = torch.tanh(x[rows].double() @ p["w1"][t].T + p["b1"][t])
        h = h + torch.tanh(h @ p["w2"][t].T + p["b2"][t])
        want = want.index_put((rows,), (h @ p["w3"][t].T + p["b3"][t])[:, 0])
    want.sum().backward()
    assert float((e.double() - want).abs().max()) < 1e-5 * float(want.abs().max()) and not bool(e[types < 0].any())
    for k, v in net.named_parameters():
        err = (v.grad.double() - p[k].grad).abs().max()
        assert float(err) < 1e-5 * float(p[k].grad.abs().max()), k
