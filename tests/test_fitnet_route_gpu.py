"""Rows sorted by network and back (fitnet.route, dispatch, combine) against host lists and sums in 64 bits."""
import pytest
import torch

import fitnet_ref as ref

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from ai2pot_b200 import fitnet


def make_index(tokens, k, experts, dropped, seed, dtype=torch.int32):
    g = torch.Generator().manual_seed(seed)
    index = torch.randint(0, experts, (tokens, k), generator=g)
    index[torch.rand(tokens, k, generator=g) < dropped] = -1
    return index.to(dtype)


@pytest.mark.parametrize("tokens,k,experts,dropped", [
    (0, 1, 3, 0.0), (1, 1, 1, 0.0), (1, 8, 3, 0.5), (31, 1, 2, 0.0), (33, 3, 5, 0.3), (216, 1, 3, 0.0), (1000, 2, 128, 0.1), (1000, 1, 1024, 0.0), (500, 2, 7, 1.0),
    (16384, 1, 4, 0.0), (16385, 1, 4, 0.2), (9323, 2, 8, 0.33), (100003, 3, 16, 0.05), (70001, 1, 1024, 0.3), (1048576, 1, 4, 0.0)])
def test_route(tokens, k, experts, dropped):
    for dtype in (torch.int32, torch.int64):
        index = make_index(tokens, k, experts, dropped, tokens + experts, dtype)
        got = fitnet.route(index.cuda(), experts)
        order, position, offsets = ref.route(index.reshape(-1).tolist(), experts)
        assert got.order.tolist() == order
        assert got.position.reshape(-1).tolist() == position and got.position.shape == (tokens, k)
        assert got.offsets.tolist() == offsets


def test_route_drops_what_names_no_network():
    index = torch.tensor([0, 5, -7, 4, 2, 2 ** 31 - 1, -2 ** 31, 4])
    got = fitnet.route(index.cuda(), 5)
    assert got.offsets.tolist() == [0, 1, 1, 2, 2, 4] and got.order.tolist() == [0, 4, 3, 7, -2, -3, -6, -7]
    wide = fitnet.route(torch.tensor([2 ** 32, 1, -2 ** 40, 2 ** 32 + 1]).cuda(), 3)      # their low words would name networks
    assert wide.position.reshape(-1).tolist() == [-1, 0, -1, -1]


def run_all(index, experts, width, dtype, seed=0, x_view=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    tokens, k = index.shape
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x, ys, w = normal(tokens, width).to(dtype), normal(tokens * k, width).to(dtype), normal(tokens, k)
    gxs, gy = normal(tokens * k, width).to(dtype), normal(tokens, width).to(dtype)
    if x_view is not None:
        x, ys, gxs, gy = (x_view(t) for t in (x, ys, gxs, gy))
    x, ys, w = x.requires_grad_(), ys.requires_grad_(), w.requires_grad_()
    route = fitnet.route(index.cuda(), experts)
    xs, y = fitnet.dispatch(x, route), fitnet.combine(ys, w, route)
    gx, gys, gw = torch.autograd.grad((xs, y), (x, ys, w), (gxs, gy))
    return dict(x=x, ys=ys, w=w, gxs=gxs, gy=gy), dict(xs=xs, y=y, gx=gx, gys=gys, gw=gw)


def check_all(index, inputs, out):
    """Against loops over the slots: copies are exact; sums of k terms have an error of (k + 1) 2^-24 of their magnitudes and one rounding."""
    tokens, k = index.shape
    dtype = out["y"].dtype
    u, tiny = ref.U[dtype], ref.TINY[dtype]
    experts = int(index.max().clamp(min=0)) + 1
    order, _, _ = ref.route(index.reshape(-1).tolist(), experts)
    kept = [s for s in order if s >= 0]
    rows, n = torch.tensor(kept, dtype=torch.int64).cuda(), len(kept)
    token = rows // k
    d = {key: v.detach().double() for key, v in inputs.items()}
    w = d["w"].reshape(-1)[rows, None]
    width = d["x"].shape[1]
    want_xs = torch.zeros(tokens * k, width, dtype=torch.float64, device="cuda")
    want_xs[:n] = d["x"][token]
    assert torch.equal(out["xs"].double(), want_xs)
    want_gys = torch.zeros_like(want_xs)
    want_gys[:n] = w * d["gy"][token]
    assert bool(((out["gys"].double() - want_gys).abs() <= (u + 2 * ref.U32) * want_gys.abs() + tiny).all())
    assert not bool(out["gys"][n:].any())
    for name, terms in (("y", w * d["ys"][:n]), ("gx", d["gxs"][:n])):
        want, mag = (torch.zeros(tokens, width, dtype=torch.float64, device="cuda").index_add_(0, token, t) for t in (terms, terms.abs()))
        assert bool(((out[name].double() - want).abs() <= u * want.abs() + 2 * (k + 1) * ref.U32 * mag + tiny).all()), name
    want, mag = (torch.zeros(tokens * k, dtype=torch.float64, device="cuda").index_put_((rows,), t.sum(1)) for t in
                 (d["gy"][token] * d["ys"][:n], (d["gy"][token] * d["ys"][:n]).abs()))
    assert bool(((out["gw"].reshape(-1).double() - want).abs() <= (width + 2) * ref.U32 * mag).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,k,experts,width,dropped", [
    (1, 1, 1, 1, 0.0), (1, 4, 2, 1024, 0.5), (216, 1, 3, 20, 0.0), (77, 2, 5, 131, 0.3), (1157, 3, 4, 30, 0.2), (64, 5, 3, 7, 1.0), (3000, 8, 16, 64, 0.1),
    (513, 1, 2, 1000, 0.0), (40, 2, 2, 2050, 0.2)])
def test_dispatch_and_combine(tokens, k, experts, width, dropped, dtype):
    index = make_index(tokens, k, experts, dropped, 3 * tokens + width)
    check_all(index, *run_all(index, experts, width, dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_alignment(dtype):
    index = make_index(300, 2, 4, 0.2, 5)
    pad = lambda left, right: lambda t: torch.nn.functional.pad(t, (left, right))[:, left:t.shape[1] + left].detach()
    for view in (pad(0, 3), pad(1, 7), pad(8, 8), lambda t: t.T.contiguous().T, lambda t: t[:1].expand(t.shape[0], t.shape[1])):
        check_all(index, *run_all(index, 4, 48, dtype, x_view=view))


def test_no_tokens():
    index = torch.zeros(0, 2, dtype=torch.int32)
    inputs, out = run_all(index, 3, 8, torch.float32)
    assert out["xs"].shape == (0, 8) and out["y"].shape == (0, 8) and out["gw"].shape == (0, 2) and out["gys"].shape == (0, 8)


def test_dropped_slots_do_not_read_what_they_hold():
    """Weights and rows of dropped slots may hold anything: neither sums nor gradients see them."""
    index = torch.tensor([[0, -1], [-1, -1], [1, 0]], dtype=torch.int32)
    route = fitnet.route(index.cuda(), 2)
    ys, w = torch.ones(6, 8, device="cuda"), torch.ones(3, 2, device="cuda")
    ys[3:] = float("nan")
    w[0, 1] = w[1, 0] = w[1, 1] = float("inf")
    ys.requires_grad_(), w.requires_grad_()
    y = fitnet.combine(ys, w, route)
    assert torch.equal(y, torch.tensor([1.0, 0.0, 2.0], device="cuda")[:, None].expand(3, 8))
    gys, gw = torch.autograd.grad(y, (ys, w), torch.ones_like(y))
    assert torch.equal(gys, torch.tensor([1.0, 1, 1, 0, 0, 0], device="cuda")[:, None].expand(6, 8))
    assert gw.tolist() == [[8, 0], [0, 0], [8, 8]]


def test_gradients_against_differences():
    """combine is linear in each argument: a difference over a step of one has rounding errors only."""
    index = make_index(50, 3, 4, 0.2, 9)
    inputs, out = run_all(index, 4, 24, torch.float32)
    route = fitnet.route(index.cuda(), 4)
    gy, gxs = inputs["gy"].double(), inputs["gxs"].double()
    with torch.no_grad():
        for name, f, up, grad in (("ys", lambda v: fitnet.combine(v, inputs["w"], route), gy, out["gys"]), ("w", lambda v: fitnet.combine(inputs["ys"], v, route), gy, out["gw"]),
                                  ("x", lambda v: fitnet.dispatch(v, route), gxs, out["gx"])):
            v = inputs[name].detach()
            step = torch.randn(v.shape, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
            plus, minus = f(v + step).double(), f(v - step).double()
            diff, mag = ((plus - minus) * up).sum() / 2, ((plus.abs() + minus.abs()) * up.abs()).sum()
            assert abs(float(diff - (grad.double() * step.double()).sum())) <= 16 * ref.U32 * float(mag), name


def test_results_are_the_same_bits_every_time():
    index = make_index(50000, 2, 8, 0.1, 11)
    first = run_all(index, 8, 64, torch.bfloat16)[1]
    for _ in range(3):
        again = run_all(index, 8, 64, torch.bfloat16)[1]
        assert all(torch.equal(first[key], again[key]) for key in first)


def test_rows_beyond_32_bit_offsets():
    """2.2e9 elements: rows at the far end are those of the slots that they belong to."""
    tokens, width = 1_100_000, 2048
    index = torch.full((tokens,), 1, dtype=torch.int32, device="cuda")
    index[-3:] = 0
    route = fitnet.route(index, 2)
    x = torch.empty(tokens, width, dtype=torch.bfloat16, device="cuda")
    x[:, 0] = (torch.arange(tokens, device="cuda") % 256).bfloat16()
    x[:, 1:] = 1
    xs = fitnet.dispatch(x, route)
    want = torch.cat([torch.arange(tokens - 3, tokens, device="cuda"), torch.arange(tokens - 3, device="cuda")]) % 256
    assert torch.equal(xs[:, 0].float(), want.float()) and bool((xs[-1000:, 1:] == 1).all())
    y = fitnet.combine(xs, torch.ones(tokens, 1, device="cuda"), route)
    assert torch.equal(y[:, 0], x[:, 0]) and bool((y[-1000:] == x[-1000:]).all())


def test_on_another_stream():
    index = make_index(5000, 2, 4, 0.1, 13)
    want = run_all(index, 4, 96, torch.float32)[1]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = run_all(index, 4, 96, torch.float32)[1]
    side.synchronize()
    assert all(torch.equal(want[key], got[key]) for key in want)


def test_refusals():
    index = make_index(10, 2, 3, 0.0, 1).cuda()
    route = fitnet.route(index, 3)
    x, ys, w = torch.ones(10, 4, device="cuda"), torch.ones(20, 4, device="cuda"), torch.ones(10, 2, device="cuda")
    for call, text in [
            (lambda: fitnet.route(index.float(), 3), "int32 or int64"), (lambda: fitnet.route(index, 0), "between 1 and 1024"), (lambda: fitnet.route(index, 1025), "between 1 and 1024"),
            (lambda: fitnet.route(index[None], 3), r"\[tokens\]"), (lambda: fitnet.route(index.cpu(), 3), "CUDA"), (lambda: fitnet.dispatch(x[:9], route), r"x must be \[10"),
            (lambda: fitnet.dispatch(x.double(), route), "float32, bfloat16 or float16"), (lambda: fitnet.dispatch(x.cpu(), route), "CUDA"),
            (lambda: fitnet.combine(ys[:19], w, route), r"ys must be \[20"), (lambda: fitnet.combine(ys, w[:, :1], route), "weights must be float32"),
            (lambda: fitnet.combine(ys, w.half(), route), "weights must be float32"), (lambda: fitnet.combine(ys, w, route._replace(position=route.position.long())), "int32"),
            (lambda: fitnet.dispatch(x, route._replace(order=route.order[:5])), "one route")]:
        with pytest.raises(RuntimeError, match=text):
            call()
    y = fitnet.combine(ys.requires_grad_(), w, route)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(y.sum(), ys, create_graph=True)
    xs = fitnet.dispatch(x.requires_grad_(), route)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(xs.sum(), x, create_graph=True)
