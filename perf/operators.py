"""The operators of per-species fitting networks, as cases that can be timed and compared.

Operators (ai2pot_b200.fitnet):
  route          atoms (tokens) sorted by the network (expert) that they belong to and back, with weights applied: route(),
                 dispatch(), combine(). An atom has k slots; a slot whose index names no network is dropped (padding).
  dense          one layer of all networks: residual + act(x W^T + b), rows grouped by network through device offsets
  orthogonalize  Newton-Schulz orthogonalisation of an update, as the Muon optimiser applies it to the layers' weights
Directions: "forward" is an evaluation, "train" a forward and the gradients of every differentiable input.

The framework's own sizes: 216 and 13,824 atoms (structures of its benchmark), 1,048,576 atoms (its largest), 9,323 atoms (its
ragged training batch), 3 species, 20 descriptors and 30 neurons (its NEP model), 1,157 atoms (a cell that is not a full lattice).
The others are generic."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
EPS = 1e-7


def listed():
    return [
        # one small structure, one network per species, descriptors of the NEP model: latency counts
        {"name": "route_f32_216x20_e3", "op": "route", "direction": "forward", "dtype": "f32", "tokens": 216, "k": 1, "experts": 3, "width": 20, "dropped": 0.0},
        # a padded training batch: a third of the slots are padding, two networks share every atom
        {"name": "route_bf16_9323x240_k2_train", "op": "route", "direction": "train", "dtype": "bf16", "tokens": 9323, "k": 2, "experts": 8, "width": 240,
         "dropped": 0.33},
        # the largest structure, sorted by species
        {"name": "route_f32_1048576x64_e4", "op": "route", "direction": "forward", "dtype": "f32", "tokens": 1048576, "k": 1, "experts": 4, "width": 64,
         "dropped": 0.0},
        # one atom moved (a Monte Carlo step): a layer for a single row
        {"name": "dense_bf16_1x1024x1024", "op": "dense", "direction": "forward", "dtype": "bf16", "rows": 1, "groups": 0, "inner": 1024, "outer": 1024,
         "act": "silu", "bias": True, "residual": True, "dropped": 0.0},
        # the NEP model's hidden layer on the smallest structure
        {"name": "dense_f32_216x20x30_e3", "op": "dense", "direction": "forward", "dtype": "f32", "rows": 216, "groups": 3, "inner": 20, "outer": 30,
         "act": "tanh", "bias": True, "residual": False, "dropped": 0.0},
        # a layer shared by all species, odd widths
        {"name": "dense_f16_1157x131x97_train", "op": "dense", "direction": "train", "dtype": "f16", "rows": 1157, "groups": 0, "inner": 131, "outer": 97,
         "act": "gelu", "bias": True, "residual": False, "dropped": 0.0},
        # a residual hidden layer of three species in single precision on the ragged training batch, padding at the end
        {"name": "dense_f32_9323x240x240_e3_train", "op": "dense", "direction": "train", "dtype": "f32", "rows": 9323, "groups": 3, "inner": 240,
         "outer": 240, "act": "tanh", "bias": True, "residual": True, "dropped": 0.1},
        # the evaluation of a wider layer on the structure of the benchmark
        {"name": "dense_bf16_13824x512x512_e4", "op": "dense", "direction": "forward", "dtype": "bf16", "rows": 13824, "groups": 4, "inner": 512,
         "outer": 512, "act": "silu", "bias": True, "residual": True, "dropped": 0.0},
        # a mixture of wide networks, the largest training step
        {"name": "dense_bf16_65536x1024x1024_e8_train", "op": "dense", "direction": "train", "dtype": "bf16", "rows": 65536, "groups": 8, "inner": 1024,
         "outer": 1024, "act": "gelu", "bias": True, "residual": True, "dropped": 0.05},
        # the update of the NEP model's hidden layer
        {"name": "orthogonalize_f32_3x30x20", "op": "orthogonalize", "dtype": "f32", "batch": 3, "m": 30, "n": 20},
        # the update of a hidden layer of eight networks
        {"name": "orthogonalize_bf16_8x512x512", "op": "orthogonalize", "dtype": "bf16", "batch": 8, "m": 512, "n": 512},
        # the largest single matrix, odd, in single precision
        {"name": "orthogonalize_f32_1x2048x1537", "op": "orthogonalize", "dtype": "f32", "batch": 1, "m": 2048, "n": 1537},
    ]


def draw(rng):
    def size(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["route", "dense", "dense", "orthogonalize"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "route":
        case = {"op": op, "direction": rng.choice(["forward", "train"]), "dtype": dtype, "k": rng.choice([1, 1, 2, 3, 4, 8]), "experts": size(1, 128),
                "width": size(1, 1024), "dropped": rng.choice([0.0, 0.0, 0.3, 0.9])}
        case["tokens"] = size(1, max(1, min(262144, 40_000_000 // (case["k"] * case["width"]))))
        return case
    if op == "dense":
        case = {"op": op, "direction": rng.choice(["forward", "train"]), "dtype": dtype, "groups": rng.choice([0, 1, 2, 3, 4, 8, 16]), "inner": size(1, 2048),
                "outer": size(1, 2048), "act": rng.choice(["none", "tanh", "silu", "gelu"]), "bias": rng.random() < 0.8, "dropped": 0.0}
        if case["groups"]:
            case["dropped"] = rng.choice([0.0, 0.2])
        case["residual"] = rng.random() < 0.5
        limit = 65536 * 1024 * 1024 // (case["inner"] * case["outer"])
        if dtype == "f32":
            limit //= 4
        case["rows"] = size(1, max(1, min(131072, limit, 60_000_000 // max(case["inner"], case["outer"]))))
        return case
    batch = rng.choice([1, 1, 2, 3, 4, 8])
    top = 2048 if batch == 1 else 1024 if batch < 4 else 640
    return {"op": op, "dtype": dtype, "batch": batch, "m": size(1, top), "n": size(1, min(top, 1537))}


# ---- inputs ---------------------------------------------------------------------------------------------------------------


def group_sizes(rows, groups, dropped, seed):
    """Rows of each group: uneven, one group empty where there are several; the rows that are left over belong to none."""
    g = torch.Generator().manual_seed(seed)
    kept = rows - int(rows * dropped)
    share = torch.rand(groups, generator=g) + 0.25
    if groups >= 4:
        share[int(torch.randint(groups, (1,), generator=g))] = 0.0
    sizes = [int(v) for v in (share / share.sum() * kept).floor()]
    sizes[max(range(groups), key=lambda e: sizes[e])] += kept - sum(sizes)
    return sizes


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=dtype):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    state = dict(case)
    if case["op"] == "route":
        t, k, e, width = (case[key] for key in ("tokens", "k", "experts", "width"))
        index = (torch.rand(t, k, generator=g, device="cuda") ** 1.5 * e).long().clamp_(max=e - 1)      # some networks get more atoms than others
        index[torch.rand(t, k, generator=g, device="cuda") < case["dropped"]] = -1
        weights = torch.softmax(torch.randn(t, k, generator=g, device="cuda"), dim=1)
        state.update(index=index.int(), x=normal(t, width), ys=normal(t * k, width), weights=weights)
        if case["direction"] == "train":
            state.update(gxs=normal(t * k, width), gy=normal(t, width))
            for key in ("x", "ys", "weights"):
                state[key].requires_grad_()
    elif case["op"] == "dense":
        m, k, n, e = (case[key] for key in ("rows", "inner", "outer", "groups"))
        stack = (e,) if e else ()
        state.update(x=normal(m, k), weight=normal(*stack, n, k, scale=k ** -0.5), bias=normal(*stack, n, scale=0.3) if case["bias"] else None,
                     residual=normal(m, n) if case["residual"] else None, sizes=None, offsets=None)
        if e:
            sizes = group_sizes(m, e, case["dropped"], seed)
            state["sizes"] = sizes
            state["offsets"] = torch.tensor([0] + sizes).cumsum(0).int().cuda()
        if case["direction"] == "train":
            state["gy"] = normal(m, n)
            for key in ("x", "weight", "bias", "residual"):
                if state[key] is not None:
                    state[key].requires_grad_()
    else:
        b, m, n = case["batch"], case["m"], case["n"]
        rows = 2 * max(m, n)
        # what a layer's gradient is: a sum of outer products, its inputs' scales spread over two decades
        gz, x = normal(b, rows, m, dtype=torch.float32), normal(b, rows, n, dtype=torch.float32)
        x *= 10.0 ** (-2.0 * torch.rand(n, generator=g, device="cuda"))
        state["g"] = (gz.transpose(1, 2) @ x / rows).to(dtype)
    return state


# ---- one pass -------------------------------------------------------------------------------------------------------------


def run(state):
    if own:
        return run_own(state)
    with torch.no_grad():
        return {"route": plain_route, "dense": plain_dense, "orthogonalize": plain_orthogonalize}[state["op"]](state)


def run_own(s):
    from ai2pot_b200 import fitnet
    if s["op"] == "route":
        route = fitnet.route(s["index"], s["experts"])
        xs = fitnet.dispatch(s["x"], route)
        y = fitnet.combine(s["ys"], s["weights"], route)
        out = {"order": route.order, "position": route.position, "offsets": route.offsets, "xs": xs.detach(), "y": y.detach()}
        if s["direction"] == "train":
            out["gx"], out["gys"], out["gw"] = torch.autograd.grad((xs, y), (s["x"], s["ys"], s["weights"]), (s["gxs"], s["gy"]))
        return out
    if s["op"] == "dense":
        y = fitnet.dense(s["x"], s["weight"], bias=s["bias"], residual=s["residual"], activation=s["act"], offsets=s["offsets"])
        out = {"y": y.detach()}
        if s["direction"] == "train":
            wanted = [key for key in ("x", "weight", "bias", "residual") if s[key] is not None]
            out.update(zip(["g" + key for key in wanted], torch.autograd.grad(y, [s[key] for key in wanted], s["gy"])))
        return out
    return {"x": fitnet.orthogonalize(s["g"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)}


def plain_route(s):
    t, k, e = s["tokens"], s["k"], s["experts"]
    index = s["index"].reshape(-1).long()
    kept = (index >= 0) & (index < e)
    key = torch.where(kept, index, e)
    order = torch.argsort(key, stable=True)
    position = torch.empty_like(order)
    position[order] = torch.arange(t * k, device=order.device)
    offsets = (key[:, None] < torch.arange(e + 1, device=key.device)).sum(0)
    kept_row = kept[order]
    token = order // k
    dtype, f = s["x"].dtype, torch.float32
    xs = s["x"][token] * kept_row[:, None]
    w = torch.where(kept, s["weights"].reshape(-1), 0.0)
    ys = s["ys"].to(f)[position].view(t, k, -1)
    y = (ys * w.view(t, k, 1)).sum(1)
    out = {"order": torch.where(kept_row, order, -1 - order).int(), "position": torch.where(kept, position, -1).int().view(t, k), "offsets": offsets.int(),
           "xs": xs, "y": y.to(dtype)}
    if s["direction"] == "train":
        gxs, gy = s["gxs"].to(f), s["gy"].to(f)
        out["gx"] = (gxs[position] * kept[:, None]).view(t, k, -1).sum(1).to(dtype)
        out["gys"] = (w[order][:, None] * gy[token]).to(dtype)
        out["gw"] = (ys * gy[:, None, :]).sum(2) * kept.view(t, k)
    return out


def plain_act(z, name):
    """The activation and its derivative."""
    if name == "tanh":
        y = torch.tanh(z)
        return y, 1.0 - y * y
    if name == "silu":
        p = 1.0 / (1.0 + torch.exp(-z))
        return z * p, p * (1.0 + z * (1.0 - p))
    if name == "gelu":
        p = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * p, p + z * torch.exp(-0.5 * z * z) * (0.5 / math.pi) ** 0.5
    return z, torch.ones_like(z)


def plain_dense(s):
    f, dtype = torch.float32, s["x"].dtype
    x, weight = s["x"].to(f), s["weight"].to(f)
    bias = None if s["bias"] is None else s["bias"].to(f)
    residual = None if s["residual"] is None else s["residual"].to(f)
    train = s["direction"] == "train"
    grouped = s["sizes"] is not None
    sizes = s["sizes"] if grouped else [x.shape[0]]
    if not grouped:
        weight, bias = weight[None], None if bias is None else bias[None]
    y = torch.zeros(x.shape[0], weight.shape[1], device=x.device)
    if train:
        gy = s["gy"].to(f)
        gx, gw, gb, gr = torch.zeros_like(x), torch.zeros_like(weight), torch.zeros_like(weight[:, :, 0]), torch.zeros_like(y)
    at = 0
    for e, rows in enumerate(sizes):
        part = slice(at, at + rows)
        at += rows
        z = x[part] @ weight[e].T
        if bias is not None:
            z = z + bias[e]
        a, slope = plain_act(z, s["act"])
        y[part] = a if residual is None else a + residual[part]
        if train:
            gz = gy[part] * slope
            gx[part], gw[e], gb[e], gr[part] = gz @ weight[e], gz.T @ x[part], gz.sum(0), gy[part]
    out = {"y": y.to(dtype)}
    if train:
        out["gx"] = gx.to(dtype)
        out["gweight"] = (gw if grouped else gw[0]).to(dtype)
        if bias is not None:
            out["gbias"] = (gb if grouped else gb[0]).to(dtype)
        if residual is not None:
            out["gresidual"] = gr.to(dtype)
    return out


def plain_orthogonalize(s):
    x = s["g"].to(torch.float32)
    x = x / ((x * x).sum((1, 2), keepdim=True).sqrt() + EPS)
    a, b, c = COEFFICIENTS
    wide = x.shape[1] <= x.shape[2]
    for _ in range(STEPS):
        if wide:
            gram = x @ x.transpose(1, 2)
            x = a * x + (b * gram + c * (gram @ gram)) @ x
        else:
            gram = x.transpose(1, 2) @ x
            x = a * x + x @ (b * gram + c * (gram @ gram))
    return {"x": x.to(s["g"].dtype)}


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "route":
        t, k, width = case["tokens"], case["k"], case["width"]
        nbytes = 4 * (3 * t * k + case["experts"] + 1) + 4 * t * k + size * width * (2 * t + 2 * t * k)        # index, order, position, offsets; weights; x, y, xs, ys
        flops = 2 * t * k * width
        if case["direction"] == "train":
            nbytes += 4 * t * k + size * width * (2 * t + 2 * t * k)                                           # gw; gx, gy, gxs, gys
            flops += 4 * t * k * width
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "dense":
        m, k, n, e = case["rows"], case["inner"], case["outer"], max(1, case["groups"])
        numbers = m * k + e * n * k + m * n + (e * n if case["bias"] else 0) + (m * n if case["residual"] else 0)
        flops = 2 * m * k * n
        if case["direction"] == "train":
            numbers += m * k + e * n * k + m * n + (e * n if case["bias"] else 0) + (m * n if case["residual"] else 0)
            flops *= 3
        return {"bytes": size * numbers, "flops": flops}
    b, short, long = case["batch"], min(case["m"], case["n"]), max(case["m"], case["n"])
    return {"bytes": size * 2 * b * short * long, "flops": STEPS * b * (short * short * long + short ** 3 + 2 * short * short * long)}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------


def exact(case, seed):
    with torch.no_grad():
        s = {key: v.detach() if isinstance(v, torch.Tensor) else v for key, v in prepare(case, seed).items()}
        return {"route": exact_route, "dense": exact_dense, "orthogonalize": exact_orthogonalize}[case["op"]](s)


def exact_route(s):
    t, k, e = s["tokens"], s["k"], s["experts"]
    flat = s["index"].cpu().reshape(-1).tolist()
    bins = [[] for _ in range(e + 1)]
    for slot, expert in enumerate(flat):
        bins[expert if 0 <= expert < e else e].append(slot)
    kept = [slot for b in bins[:e] for slot in b]
    position = torch.full((t * k,), -1, dtype=torch.int64)
    position[torch.tensor(kept, dtype=torch.int64)] = torch.arange(len(kept))
    offsets = [0]
    for b in bins[:e]:
        offsets.append(offsets[-1] + len(b))
    rows = torch.tensor(kept, dtype=torch.int64).cuda()
    position = position.cuda()
    x, ys, w = s["x"].double(), s["ys"].double(), s["weights"].double()
    xs = torch.zeros(t * k, x.shape[1], dtype=torch.float64, device="cuda")
    xs[:len(kept)] = x[rows // k]
    y = torch.zeros_like(x)
    y.index_add_(0, rows // k, ys[:len(kept)] * w.reshape(-1)[rows, None])
    out = {"order": torch.tensor(kept + [-1 - slot for slot in bins[e]], dtype=torch.int32).cuda(), "position": position.int().view(t, k),
           "offsets": torch.tensor(offsets, dtype=torch.int32).cuda(), "xs": xs, "y": y}
    if s["direction"] == "train":
        gxs, gy = s["gxs"].double(), s["gy"].double()
        gx = torch.zeros_like(x)
        gx.index_add_(0, rows // k, gxs[:len(kept)])
        gys = torch.zeros_like(ys)
        gys[:len(kept)] = w.reshape(-1)[rows, None] * gy[rows // k]
        gw = torch.zeros(t * k, dtype=torch.float64, device="cuda")
        gw[rows] = torch.einsum("rd,rd->r", gy[rows // k], ys[:len(kept)])
        out.update(gx=gx, gys=gys, gw=gw.view(t, k))
    return out


def exact_dense(s):
    x, n = s["x"].double(), s["outer"]
    grouped = s["sizes"] is not None
    weight = s["weight"].double().reshape(-1, n, x.shape[1])
    ends = torch.tensor(s["sizes"] if grouped else [x.shape[0]]).cumsum(0).tolist()
    y = torch.zeros(x.shape[0], n, dtype=torch.float64, device="cuda")
    slope = torch.zeros_like(y)
    first = 0
    for e, last in enumerate(ends):
        z = torch.einsum("mk,nk->mn", x[first:last], weight[e])
        if s["bias"] is not None:
            z = z + s["bias"].double().reshape(-1, n)[e]
        if s["act"] == "tanh":
            a, d = torch.tanh(z), torch.cosh(z) ** -2
        elif s["act"] == "silu":
            p = torch.sigmoid(z)
            a, d = z * p, p + z * p * torch.sigmoid(-z)
        elif s["act"] == "gelu":
            p = 0.5 * torch.erfc(-z / math.sqrt(2.0))
            a, d = z * p, p + z * torch.exp(-z * z / 2.0) / math.sqrt(2.0 * math.pi)
        else:
            a, d = z, torch.ones_like(z)
        y[first:last], slope[first:last] = a, d
        first = last
    kept = ends[-1]
    if s["residual"] is not None:
        y[:kept] += s["residual"][:kept].double()
    out = {"y": y}
    if s["direction"] == "train":
        gy = s["gy"].double()
        gz = gy * slope
        gx, gw = torch.zeros_like(x), torch.zeros_like(weight)
        gb = torch.zeros(len(ends), n, dtype=torch.float64, device="cuda")
        first = 0
        for e, last in enumerate(ends):
            gx[first:last] = torch.einsum("mn,nk->mk", gz[first:last], weight[e])
            gw[e] = torch.einsum("mn,mk->nk", gz[first:last], x[first:last])
            gb[e] = gz[first:last].sum(0)
            first = last
        out["gx"], out["gweight"] = gx, gw if grouped else gw[0]
        if s["bias"] is not None:
            out["gbias"] = gb if grouped else gb[0]
        if s["residual"] is not None:
            gr = torch.zeros_like(gy)
            gr[:kept] = gy[:kept]
            out["gresidual"] = gr
    return out


def exact_orthogonalize(s):
    out = []
    for g in s["g"].double():
        # the polynomial acts on the singular values alone
        u, sigma, vt = torch.linalg.svd(g.cpu() if min(g.shape) < 64 else g, full_matrices=False)
        sigma = sigma / (torch.linalg.vector_norm(g).to(sigma.device) + EPS)
        for _ in range(STEPS):
            sigma = sum(c * sigma ** (2 * i + 1) for i, c in enumerate(COEFFICIENTS))
        out.append(((u * sigma) @ vt).cuda())
    return {"x": torch.stack(out)}
