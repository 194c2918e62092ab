"""The fitting-network operators in 64 bits, and how far a result in fewer bits may be from them (test infrastructure).

Bounds are elementwise and hold for any order of summation: a float sum of n products has an error of at most (n + 2) 2^-24 times the sum
of the products' magnitudes; it is doubled here because a tensor core may cut instead of round. u is the type's unit roundoff (half the
distance of neighbouring numbers, relative)."""
import math

import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -24}     # absolute error of results that underflow
U32 = 2.0 ** -24


def act(z, name):
    """Activation and slope."""
    if name == "tanh":
        t = torch.tanh(z)
        return t, 1 - t * t
    if name == "silu":
        p = torch.sigmoid(z)
        return z * p, p + z * p * (1 - p)
    if name == "gelu":
        p = 0.5 * torch.erfc(-z / math.sqrt(2.0))
        return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return z, torch.ones_like(z)


def groups_of(offsets, rows):
    return [(0, rows)] if offsets is None else [(int(a), int(b)) for a, b in zip(offsets[:-1], offsets[1:])]


def dense(x, weight, bias, residual, name, offsets, gy=None):
    """{name: (value, bound)} of the layer and, if gy is given, of its gradients. Tensors of any type; computed in 64 bits."""
    dtype = x.dtype
    u, tiny = U[dtype], TINY[dtype]
    d = lambda t: None if t is None else t.detach().double()
    x, weight, bias, residual, gy = d(x), d(weight), d(bias), d(residual), d(gy)
    stacked = weight.dim() == 3
    w3 = weight if stacked else weight[None]
    b2 = None if bias is None else bias.reshape(w3.shape[0], w3.shape[1])
    rows, inner, outer = x.shape[0], x.shape[1], w3.shape[1]
    y, ey = torch.zeros(rows, outer, dtype=torch.float64, device=x.device), torch.zeros(rows, outer, dtype=torch.float64, device=x.device)
    gx, egx = torch.zeros_like(x), torch.zeros_like(x)
    gw, egw, gb, egb = torch.zeros_like(w3), torch.zeros_like(w3), torch.zeros_like(w3[:, :, 0]), torch.zeros_like(w3[:, :, 0])
    gr = torch.zeros_like(y)
    for e, (r0, r1) in enumerate(groups_of(offsets, rows)):
        s = slice(r0, r1)
        z, mag = x[s] @ w3[e].T, x[s].abs() @ w3[e].abs().T
        if b2 is not None:
            z, mag = z + b2[e], mag + b2[e].abs()
        ez = 2 * (inner + 2) * U32 * mag
        a, slope = act(z, name)
        # every activation's slope is below 1.13 in magnitude; its own evaluation is good to 16 roundings of the largest term
        ea = 1.13 * ez + (0 if name == "none" else 16 * U32 * (1 + a.abs()))
        y[s] = a if residual is None else a + residual[s]
        ey[s] = ea + (u + 2 * U32) * (y[s].abs() + ea) + tiny + (0 if residual is None else 2 * U32 * (a.abs() + residual[s].abs()))
        if gy is None:
            continue
        gz = gy[s] * slope
        # slopes change by at most 1 per unit of z; slope and gz are rounded to the type
        egz = torch.zeros_like(gz) if name == "none" else gy[s].abs() * (ez + 32 * U32 + u * slope.abs() + tiny) + u * gz.abs() + tiny
        gx[s] = gz @ w3[e]
        egx[s] = egz @ w3[e].abs() + 2 * (outer + 2) * U32 * ((gz.abs() + egz) @ w3[e].abs()) + u * gx[s].abs() + tiny
        gw[e] = gz.T @ x[s]
        n = r1 - r0
        egw[e] = egz.T @ x[s].abs() + 2 * (n + 2) * U32 * ((gz.abs() + egz).T @ x[s].abs()) + u * gw[e].abs() + tiny
        gb[e] = gz.sum(0)
        egb[e] = egz.sum(0) + 2 * (n + 2) * U32 * (gz.abs() + egz).sum(0) + u * gb[e].abs() + tiny
        gr[s] = gy[s]
    out = {"y": (y, ey)}
    if gy is not None:
        shape = (lambda t: t) if stacked else (lambda t: t[0])
        out.update(gx=(gx, egx * 1.1), gweight=(shape(gw), shape(egw) * 1.1), gbias=(shape(gb), shape(egb) * 1.1), gresidual=(gr, torch.zeros_like(gr)))
    return out


def orthogonalize(g, steps, coefficients, eps, dtype=torch.float64):
    x = g.to(dtype)
    x = x / (torch.linalg.vector_norm(x.double(), dim=(-2, -1), keepdim=True).to(dtype) + eps)
    a, b, c = coefficients
    for _ in range(steps):
        if x.shape[-2] <= x.shape[-1]:
            gram = x @ x.mT
            x = a * x + (b * gram + c * (gram @ gram)) @ x
        else:
            gram = x.mT @ x
            x = a * x + x @ (b * gram + c * (gram @ gram))
    return x


def route(index, experts):
    """order, position, offsets of a host list of slots."""
    bins = [[] for _ in range(experts + 1)]
    for s, e in enumerate(index):
        bins[e if 0 <= e < experts else experts].append(s)
    order, position, offsets = [], [-1] * len(index), [0]
    for e in range(experts):
        for s in bins[e]:
            position[s] = len(order)
            order.append(s)
        offsets.append(len(order))
    return order + [-1 - s for s in bins[experts]], position, offsets
