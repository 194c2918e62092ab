"""One layer of all networks (fitnet.dense) and its gradients against the formulas in 64 bits, with elementwise bounds (fitnet_ref)."""
import pytest
import torch

import fitnet_ref as ref

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from ai2pot_b200 import fitnet


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    fitnet.check()

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(rows, groups, inner, outer, dtype, bias=True, residual=True, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + rows + 7 * inner + 13 * outer)
    normal = lambda *s, scale=1.0: (torch.randn(*s, generator=g, device="cuda") * scale).to(dtype)
    stack = (groups,) if groups else ()
    return dict(x=normal(rows, inner), weight=normal(*stack, outer, inner, scale=inner ** -0.5), bias=normal(*stack, outer, scale=0.5) if bias else None,
                residual=normal(rows, outer) if residual else None), normal(rows, outer)


def run(t, activation, offsets, gy):
    leaves = {key: v.detach().requires_grad_() for key, v in t.items() if v is not None}
    y = fitnet.dense(leaves["x"], leaves["weight"], bias=leaves.get("bias"), residual=leaves.get("residual"), activation=activation, offsets=offsets)
    grads = torch.autograd.grad(y, list(leaves.values()), gy)
    with torch.no_grad():
        assert torch.equal(fitnet.dense(t["x"], t["weight"], t["bias"], t["residual"], activation, offsets).nan_to_num(), y.nan_to_num())   # an evaluation gives the same
    return dict(zip(["y"] + ["g" + key for key in leaves], (y.detach(),) + grads))


def check(t, activation, offsets, gy, got=None):
    got = run(t, activation, offsets, gy) if got is None else got
    want = ref.dense(t["x"], t["weight"], t["bias"], t["residual"], activation, None if offsets is None else offsets.tolist(), gy)
    for key, v in got.items():
        value, bound = want[key]
        assert v.shape == value.shape and v.dtype == t["x"].dtype, key
        over = (v.double() - value).abs() - bound
        assert bool((over <= 0).all()), (key, float(over.max()), float(bound.max()), int((over > 0).sum()))
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("activation", ["none", "tanh", "silu", "gelu"])
@pytest.mark.parametrize("rows,inner,outer", [(1, 1, 1), (1, 1024, 1024), (3, 20, 30), (7, 64, 8), (65, 131, 97), (216, 20, 30), (300, 240, 240), (129, 64, 257)])
def test_one_network(rows, inner, outer, activation, dtype):
    t, gy = make(rows, 0, inner, outer, dtype)
    check(t, activation, None, gy)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("sizes,dropped", [([216], 0), ([0, 5, 0], 3), ([1, 1, 1, 1], 0), ([64, 128, 1, 63, 200], 7), ([0, 0], 10), ([700, 0, 129], 0)])
def test_groups(sizes, dropped, bias, residual, dtype):
    rows = sum(sizes) + dropped
    offsets = torch.tensor([0] + sizes).cumsum(0).int().cuda()
    for inner, outer, activation in [(20, 30, "tanh"), (72, 136, "silu")]:
        t, gy = make(rows, len(sizes), inner, outer, dtype, bias, residual)
        got = check(t, activation, offsets, gy)
        kept = sum(sizes)
        assert not bool(got["y"][kept:].any()) and not bool(got["gx"][kept:].any())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes,inner,outer", [([4000, 3000, 2300], 240, 240), ([5000, 0, 1200], 512, 256), ([2049], 1024, 512), ([3000, 1], 100, 520)])
def test_larger_layers(sizes, inner, outer, dtype):
    offsets = torch.tensor([0] + sizes).cumsum(0).int().cuda()
    t, gy = make(sum(sizes) + 31, len(sizes), inner, outer, dtype)
    check(t, "gelu", offsets, gy)


@pytest.mark.parametrize("dtype", TYPES)
def test_short_ragged_groups(dtype):
    """Groups of a few stages whose rows do not fill the last one, between long ones, in layers whose tiles are the largest: their ragged
    stages follow each other within the stages that are in flight."""
    sizes = [3000, 189, 23, 76, 5, 2100, 100, 63, 65, 1, 129, 2500, 47, 190, 33]
    offsets = torch.tensor([0] + sizes).cumsum(0).int().cuda()
    t, gy = make(sum(sizes), len(sizes), 1024, 1024, dtype)
    first = check(t, "gelu", offsets, gy)
    for _ in range(5):
        again = run(t, "gelu", offsets, gy)
        assert all(torch.equal(first[key], again[key]) for key in first)


@pytest.mark.parametrize("dtype", TYPES)
def test_many_groups(dtype):
    sizes = [(37 * e) % 19 for e in range(1024)]
    offsets = torch.tensor([0] + sizes).cumsum(0).int().cuda()
    t, gy = make(sum(sizes), 1024, 24, 40, dtype)
    check(t, "silu", offsets, gy)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_alignment_and_layouts(dtype):
    sizes = [100, 50, 90]
    offsets = torch.tensor([0] + sizes).cumsum(0).int().cuda()
    pad = lambda left, right: lambda t: torch.nn.functional.pad(t, (left, right))[:, left:t.shape[1] + left]
    for view in (pad(0, 5), pad(1, 2), pad(8, 8), lambda t: t.T.contiguous().T, lambda t: t[:1].expand(t.shape[0], t.shape[1])):
        t, gy = make(250, 3, 128, 96, dtype)
        t["x"], t["residual"], gy = view(t["x"]), view(t["residual"]), view(gy)
        t["weight"] = t["weight"].transpose(1, 2).contiguous().transpose(1, 2)
        check(t, "tanh", offsets, gy)
    # weights at an address that is a multiple of their element size only
    t, gy = make(250, 3, 128, 96, dtype)
    flat = torch.empty(t["weight"].numel() + 1, dtype=dtype, device="cuda")[1:]
    t["weight"] = flat.view(t["weight"].shape).copy_(t["weight"])
    check(t, "tanh", offsets, gy)


def test_more_dimensions():
    t, gy = make(60, 0, 24, 16, torch.float32)
    y = fitnet.dense(t["x"].view(3, 20, 24), t["weight"], t["bias"], t["residual"].view(3, 20, 16), "tanh")
    assert y.shape == (3, 20, 16) and torch.equal(y.view(60, 16), fitnet.dense(t["x"], t["weight"], t["bias"], t["residual"], "tanh"))
    assert fitnet.dense(t["x"][0], t["weight"], t["bias"], t["residual"][0]).shape == (16,)


@pytest.mark.parametrize("dtype", TYPES)
def test_no_rows(dtype):
    offsets = torch.zeros(4, dtype=torch.int32, device="cuda")
    t, gy = make(0, 3, 24, 40, dtype)
    got = check(t, "tanh", offsets, gy)
    assert not bool(got["gweight"].any()) and not bool(got["gbias"].any())
    t, gy = make(0, 0, 240, 256, dtype)
    got = check(t, "none", None, gy)
    assert not bool(got["gweight"].any())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("inner,outer", [(20, 30), (256, 192)])
def test_nothing_leaks_between_rows_and_groups(inner, outer, dtype):
    """NaN and infinities in the rows of one network and in rows of none leave every other row and every other network's gradient as
    they are."""
    sizes = [130, 70, 200]
    offsets = torch.tensor([0] + sizes).cumsum(0).int().cuda()
    t, gy = make(440, 3, inner, outer, dtype)
    clean = run(t, "tanh", offsets, gy)
    for bad in (float("nan"), float("inf")):
        dirty = {key: v.clone() for key, v in t.items()}
        dirty["x"][130:200] = bad
        dirty["x"][400:] = bad
        dirty["residual"][400:] = bad
        dirty["weight"][1] = bad
        gy2 = gy.clone()
        gy2[130:200], gy2[400:] = bad, bad
        got = run(dirty, "tanh", offsets, gy2)
        for key in ("y", "gx", "gresidual"):
            assert torch.equal(got[key][:130], clean[key][:130]) and torch.equal(got[key][200:], clean[key][200:]), (key, bad)
        for key in ("gweight", "gbias"):
            assert torch.equal(got[key][0], clean[key][0]) and torch.equal(got[key][2], clean[key][2]), (key, bad)
        assert bool(got["gweight"][1].isnan().all())


@pytest.mark.parametrize("activation", ["tanh", "silu", "gelu"])
def test_large_arguments(activation):
    """Activations far out: their limits, no overflow inside."""
    z = torch.tensor([-1e30, -300.0, -90.0, -20.0, 0.0, 20.0, 90.0, 300.0, 1e30], device="cuda")
    x = z[:, None].clone().requires_grad_()
    y = fitnet.dense(x, torch.ones(1, 1, device="cuda"), activation=activation)
    g, = torch.autograd.grad(y.sum(), x)
    a, s = ref.act(z.double(), activation)
    assert torch.allclose(y[:, 0].double(), a, rtol=1e-6, atol=1e-7) and torch.allclose(g[:, 0].double(), s, rtol=1e-6, atol=1e-7)


@pytest.mark.parametrize("activation", ["tanh", "silu", "gelu"])
@pytest.mark.parametrize("rows,inner,outer", [(40, 20, 30), (300, 128, 192)])
def test_gradients_against_differences(rows, inner, outer, activation):
    """(L(v + h d) - L(v - h d)) / 2h of L = <gy, y>. Third derivatives of the activations are at most 2, so the difference is off by at
    most h^2 / 3 <|gy|, |dz|^3>, and by the results' bounds over h."""
    h = 2.0 ** -7
    t, gy = make(rows, 0, inner, outer, torch.float32)
    got = run(t, activation, None, gy)
    for key in ("x", "weight", "bias"):
        d = torch.randn(t[key].shape, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda") * (0.1 if key == "weight" else 1.0)
        ends, bound = [], 0.0
        for sign in (1, -1):
            moved = dict(t, **{key: t[key] + sign * h * d})
            y = fitnet.dense(moved["x"], moved["weight"], moved["bias"], moved["residual"], activation).double()
            err = ref.dense(moved["x"], moved["weight"], moved["bias"], moved["residual"], activation, None)["y"][1]
            ends.append((y * gy.double()).sum())
            bound += float((err * gy.double().abs()).sum()) / (2 * h)
            # the step that was made, after rounding
            d_made = (moved[key].double() - t[key].double()) / (sign * h)
            bound += float(((d_made - d.double()).abs() * got["g" + key].double().abs()).sum())
        x, w = t["x"].double(), t["weight"].double()
        dz = d.double() @ w.T if key == "x" else x @ d.double().T if key == "weight" else d.double().expand(rows, outer)
        bound += h * h / 3 * float((gy.double().abs() * dz.abs() ** 3).sum())
        own = ref.dense(t["x"], t["weight"], t["bias"], t["residual"], activation, None, gy)["g" + key][1]
        bound += float((own * d.double().abs()).sum())
        diff = float(ends[0] - ends[1]) / (2 * h)
        exact = float((got["g" + key].double() * d.double()).sum())
        assert abs(diff - exact) <= bound, (key, diff, exact, bound)


@pytest.mark.parametrize("dtype", TYPES)
def test_results_are_the_same_bits_every_time(dtype):
    sizes = [3000, 100, 2000]
    offsets = torch.tensor([0] + sizes).cumsum(0).int().cuda()
    t, gy = make(sum(sizes), 3, 256, 384, dtype)
    first = run(t, "silu", offsets, gy)
    for _ in range(3):
        again = run(t, "silu", offsets, gy)
        assert all(torch.equal(first[key], again[key]) for key in first)


def test_rows_beyond_32_bit_offsets():
    """2.2e9 elements of x: the last rows are those of the layer, and so are their gradients."""
    rows, inner, outer = 1_100_000, 2048, 16
    x = torch.zeros(rows, inner, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(4)
    x[-300:] = torch.randn(300, inner, generator=g, device="cuda").bfloat16()
    w = (torch.randn(outer, inner, generator=g, device="cuda") * inner ** -0.5).bfloat16().requires_grad_()
    gy = torch.zeros(rows, outer, dtype=torch.bfloat16, device="cuda")
    gy[-300:] = torch.randn(300, outer, generator=g, device="cuda").bfloat16()
    x.requires_grad_()
    y = fitnet.dense(x, w, activation="tanh")
    gx, gw = torch.autograd.grad(y, (x, w), gy)
    want = ref.dense(x[-300:], w, None, None, "tanh", None, gy[-300:])
    for got, key in ((y[-300:], "y"), (gx[-300:], "gx"), (gw, "gweight")):
        assert bool(((got.double() - want[key][0]).abs() <= want[key][1]).all()), key
    assert not bool(gx[:1000].any())


def test_on_another_stream():
    offsets = torch.tensor([0, 2000, 3000]).int().cuda()
    t, gy = make(3100, 2, 256, 256, torch.bfloat16)
    want = run(t, "gelu", offsets, gy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(t, "gelu", offsets, gy)
    side.synchronize()
    assert all(torch.equal(want[key], got[key]) for key in want)


def test_gradients_of_some_inputs_only():
    t, gy = make(200, 0, 64, 64, torch.float32)
    full = run(t, "tanh", None, gy)
    for key in ("x", "weight", "bias", "residual"):
        leaves = {k2: v.detach().requires_grad_(k2 == key) for k2, v in t.items()}
        y = fitnet.dense(leaves["x"], leaves["weight"], leaves["bias"], leaves["residual"], "tanh")
        g, = torch.autograd.grad(y, leaves[key], gy)
        assert torch.equal(g, full["g" + key]), key


@pytest.mark.parametrize("key", ["x", "weight", "bias", "residual"])
def test_gradients_of_some_inputs_of_groups(key):
    """One input's gradient alone, rows of no network at the end: the residual's needs no slopes, which are not kept then."""
    offsets = torch.tensor([0, 90, 90, 180], device="cuda").int()
    t, gy = make(200, 3, 64, 48, torch.bfloat16)
    full = run(t, "tanh", offsets, gy)
    leaves = {k2: v.detach().requires_grad_(k2 == key) for k2, v in t.items()}
    y = fitnet.dense(leaves["x"], leaves["weight"], leaves["bias"], leaves["residual"], "tanh", offsets)
    g, = torch.autograd.grad(y, leaves[key], gy)
    assert torch.equal(g, full["g" + key])


def test_recorded_in_a_graph():
    """Layers, routing and updates recorded once and replayed on other values give the results of direct calls."""
    g = torch.Generator(device="cuda").manual_seed(8)
    types = torch.randint(-1, 3, (2000,), generator=g, device="cuda", dtype=torch.int32)
    x, w = torch.randn(2000, 96, generator=g, device="cuda"), torch.randn(3, 160, 96, generator=g, device="cuda") * 0.1
    ones = torch.ones(2000, 1, device="cuda")

    def call():
        route = fitnet.route(types, 3)
        h = fitnet.dense(fitnet.dispatch(x, route), w, activation="gelu", offsets=route.offsets)
        return fitnet.combine(h, ones, route), fitnet.orthogonalize(w)

    with torch.no_grad():
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        for seed in (1, 2):
            g.manual_seed(seed)
            x.copy_(torch.randn(2000, 96, generator=g, device="cuda"))
            types.copy_(torch.randint(-1, 3, (2000,), generator=g, device="cuda", dtype=torch.int32))
            w.copy_(torch.randn(3, 160, 96, generator=g, device="cuda") * 0.1)
            graph.replay()
            want = call()
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_refusals():
    t, gy = make(20, 3, 8, 12, torch.float32)
    offsets = torch.tensor([0, 5, 10, 20]).int().cuda()
    x, w, b, r = t["x"], t["weight"], t["bias"], t["residual"]
    for call, text in [
            (lambda: fitnet.dense(x, w, offsets=None), r"must be \[outer, inner\]"), (lambda: fitnet.dense(x, w[0], offsets=offsets), r"must be \[groups, outer, inner\]"),
            (lambda: fitnet.dense(x[:, :7], w, offsets=offsets), "last dimension of x must be 8"), (lambda: fitnet.dense(x, w, b[0], offsets=offsets), "bias must be"),
            (lambda: fitnet.dense(x, w, b, r[:, :11], offsets=offsets), "residual must have"), (lambda: fitnet.dense(x, w, b, r[:19], offsets=offsets), "residual must have"),
            (lambda: fitnet.dense(x, w, activation="relu", offsets=offsets), "activation must be"), (lambda: fitnet.dense(x, w, offsets=offsets[:3]), r"offsets must be \[4\]"),
            (lambda: fitnet.dense(x, w, offsets=offsets.long()), "int32"), (lambda: fitnet.dense(x, w, offsets=offsets.cpu()), "CUDA"),
            (lambda: fitnet.dense(x.half(), w, offsets=offsets), "weight must be"), (lambda: fitnet.dense(x.double(), w.double(), offsets=offsets), "float32, bfloat16 or float16"),
            (lambda: fitnet.dense(x.cpu(), w[0].cpu()), "CUDA"), (lambda: fitnet.dense(x, w.bfloat16(), offsets=offsets), "weight must be"),
            (lambda: fitnet.dense(x, w, b.half(), offsets=offsets), "bias must be")]:
        with pytest.raises(RuntimeError, match=text):
            call()
    y = fitnet.dense(x.detach().requires_grad_(), w, offsets=offsets)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(y.sum(), y.grad_fn.next_functions[0][0].variable, create_graph=True)


@pytest.mark.parametrize("values", [[0, -5, 2 ** 31 - 1, 40], [300, 200, 100, 0], [-2 ** 31, 250, 10, 260], [0, 300, 0, 300]])
def test_offsets_that_do_not_ascend(values):
    """Whatever offsets hold, no access leaves the rows and the workspace (results of such offsets have no meaning)."""
    offsets = torch.tensor(values, device="cuda").int()
    for inner, outer, dtype in [(24, 40, torch.float32), (256, 320, torch.bfloat16), (128, 136, torch.float32)]:
        t, gy = make(300, 3, inner, outer, dtype)
        leaves = {k: v.detach().requires_grad_() for k, v in t.items()}
        y = fitnet.dense(leaves["x"], leaves["weight"], leaves["bias"], leaves["residual"], "tanh", offsets)
        torch.autograd.grad(y, list(leaves.values()), gy)
    torch.cuda.synchronize()
