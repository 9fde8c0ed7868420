"""The operators of a layer of experts and of its training step, as one file that a measurement calls: the cases, their inputs, the
plain form of each operator in elementary torch operations, the call a program makes of spla_amd.kernels, and the definition in 64 bits.

    sort          entries (token, choice) sorted by expert: offsets, order, place
    rows          token rows gathered into expert order, times the routing weight
    back          expert rows summed back into token order with the routing weights
    back_grad     the gradient of `back` for the expert rows and for the weights
    product       every expert's row range times that expert's matrix
    product_grad  the gradients of `product` for the rows and for the matrices
    norm          the global norm over many tensors
    clip          the same and the tensors scaled down to a largest norm
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # one decoding step of a small batch: the launch is everything
        {"name": "sort_step", "kind": "sort", "tokens": 64, "per_token": 2, "experts": 8, "skew": 0.0, "padding": 0.0},
        # a long training batch over many experts, a tenth of the tokens padding
        {"name": "sort_batch", "kind": "sort", "tokens": 131072, "per_token": 8, "experts": 128, "skew": 0.5, "padding": 0.1},
        # the tokens of a training step on their way to the experts
        {"name": "rows_batch", "kind": "rows", "tokens": 16384, "per_token": 4, "experts": 32, "skew": 0.3, "padding": 0.0, "width": 2048, "dtype": "bf16",
         "weighted": False},
        # the way back at an odd width and odd counts, full precision, some rows padding
        {"name": "back_odd", "kind": "back", "tokens": 10007, "per_token": 3, "experts": 13, "skew": 0.5, "padding": 0.05, "width": 1001, "dtype": "fp32",
         "weighted": True},
        # the way back's gradient in a training step
        {"name": "back_grad_batch", "kind": "back_grad", "tokens": 16384, "per_token": 4, "experts": 32, "skew": 0.3, "padding": 0.0, "width": 2048,
         "dtype": "bf16", "weighted": True},
        # decoding one token: two experts' matrices are read once
        {"name": "product_token", "kind": "product", "tokens": 1, "per_token": 2, "experts": 8, "skew": 0.0, "padding": 0.0, "n_in": 2048, "n_out": 4096,
         "dtype": "bf16"},
        # decoding a batch: every matrix is read, each for a few rows
        {"name": "product_step", "kind": "product", "tokens": 64, "per_token": 4, "experts": 32, "skew": 0.3, "padding": 0.0, "n_in": 2048, "n_out": 2048,
         "dtype": "bf16"},
        # a prompt or the forward pass of a training step
        {"name": "product_batch", "kind": "product", "tokens": 16384, "per_token": 2, "experts": 8, "skew": 0.3, "padding": 0.0, "n_in": 2048, "n_out": 4096,
         "dtype": "bf16"},
        # the backward pass over more and smaller experts, unevenly loaded, some padding
        {"name": "product_grad_batch", "kind": "product_grad", "tokens": 8192, "per_token": 4, "experts": 32, "skew": 0.7, "padding": 0.03, "n_in": 2048,
         "n_out": 1024, "dtype": "bf16"},
        # a small model trained in full precision at sizes that are no multiple of anything
        {"name": "product_grad_odd", "kind": "product_grad", "tokens": 1777, "per_token": 3, "experts": 5, "skew": 0.5, "padding": 0.1, "n_in": 250, "n_out": 333,
         "dtype": "fp32"},
        # the gradients of one small layer
        {"name": "norm_layer", "kind": "norm", "tensors": 12, "elements": 300001, "dtype": "fp32", "limit": 0.0},
        # the gradients of a whole model, 16-bit and 32-bit tensors mixed, a sixth as many vectors as matrices
        {"name": "clip_model", "kind": "clip", "tensors": 300, "elements": 400000000, "dtype": "mixed", "limit": 1.0},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    """mostly multiples of 64, as layers have them; else anything"""
    n = _log_int(rng, low, high)
    return max(64, n // 64 * 64) if rng.random() < 0.7 else n


def draw(rng):
    kind = rng.choice(["sort", "rows", "back", "back_grad", "product", "product", "product_grad", "product_grad", "norm", "clip"])
    if kind in ("norm", "clip"):
        return {"kind": kind, "tensors": _log_int(rng, 1, 400), "elements": _log_int(rng, 1000, 400000000), "dtype": rng.choice(["fp32", "bf16", "fp16", "mixed"]),
                "limit": rng.choice([0.5, 1.0, 1e6]) if kind == "clip" else 0.0}
    case = {"kind": kind, "tokens": _log_int(rng, 1, 131072), "per_token": rng.randint(1, 8), "experts": _log_int(rng, 8, 128),
            "skew": rng.choice([0.0, 0.3, 0.7, 1.5]), "padding": rng.choice([0.0, 0.0, 0.1])}
    if kind in ("rows", "back", "back_grad"):
        case["tokens"] = min(case["tokens"], 32768)
        case["width"] = _width(rng, 64, 4096)
        case["dtype"] = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        case["weighted"] = True if kind == "back_grad" else rng.random() < 0.5
        limit = 16384 * 4 * 2048
        case["tokens"] = max(1, min(case["tokens"], limit // (case["per_token"] * case["width"])))
    if kind in ("product", "product_grad"):
        case["experts"] = min(case["experts"], 64)
        case["n_in"] = _width(rng, 64, 4096)
        case["n_out"] = _width(rng, 64, 4096)
        case["dtype"] = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        flops = 2 * 32768 * 2048 * 4096 // (2 if kind == "product_grad" else 1) // (8 if case["dtype"] == "fp32" else 1)
        case["tokens"] = max(1, min(case["tokens"], flops // (2 * case["per_token"] * case["n_in"] * case["n_out"])))
    return case


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _choices(case, g):
    """k different experts a token by random scores with a popularity of each expert, padding tokens -1: what a router hands over"""
    t, k, e = case["tokens"], case["per_token"], case["experts"]
    scores = torch.rand(t, e, generator=g, device="cuda") + case["skew"] * torch.rand(e, generator=g, device="cuda")
    weights, experts = torch.topk(scores, k, dim=1)
    weights = weights / weights.sum(1, keepdim=True)
    if case["padding"]:
        experts[torch.rand(t, generator=g, device="cuda") < case["padding"]] = -1
    return experts.to(torch.int32).contiguous(), weights.contiguous()


def _sizes(case):
    """the tensors' shapes: mostly matrices of one width, every seventh a vector, the last takes the rest"""
    n, left, shapes = case["tensors"], case["elements"], []
    each = max(1, left // n)
    for i in range(n - 1):
        rows = max(1, math.isqrt(each))
        shape = (min(each, 4 * rows),) if i % 7 == 6 else (max(1, each // rows), rows)
        shapes.append(shape)
        left -= math.prod(shape)
    return shapes + [(max(left, 1),)] if n > 1 else [(left,)]


def _tensor_dtype(case, i):
    return _DTYPES[("bf16", "fp32", "bf16", "fp16")[i % 4]] if case["dtype"] == "mixed" else _DTYPES[case["dtype"]]


def _bucket_places(case):
    """(type, first element, shape) of every tensor in the bucket of its type, each starting at a multiple of 64 elements, and the buckets' lengths"""
    places, lengths = [], {}
    for i, shape in enumerate(_sizes(case)):
        dtype = _tensor_dtype(case, i)
        places.append((dtype, lengths.get(dtype, 0), shape))
        lengths[dtype] = places[-1][1] + (math.prod(shape) + 63) // 64 * 64
    return places, lengths


def _inputs(case, seed):
    g = _generator(seed)
    kind = case["kind"]
    if kind in ("norm", "clip"):
        # gradients: small values whose size differs from tensor to tensor
        shapes = _sizes(case)
        return {"tensors": [(torch.randn(s, generator=g, device="cuda") * (1e-3 * (1 + i % 5))).to(_tensor_dtype(case, i)) for i, s in enumerate(shapes)]}
    s = {}
    s["experts"], s["weights"] = _choices(case, g)
    if kind == "sort":
        return s
    dtype = _DTYPES[case["dtype"]]
    t, places = case["tokens"], case["tokens"] * case["per_token"]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    if kind == "rows":
        s["x"] = normal(t, case["width"])
    elif kind == "back":
        s["y"] = normal(places, case["width"])
    elif kind == "back_grad":
        s["y"] = normal(places, case["width"])
        s["dout"] = normal(t, case["width"])
    else:
        s["x"] = normal(places, case["n_in"])
        s["w"] = normal(case["experts"], case["n_out"], case["n_in"], scale=case["n_in"] ** -0.5)
        if kind == "product_grad":
            s["dy"] = normal(places, case["n_out"])
    return s


def _plain_sort(experts, n_experts):
    flat = experts.reshape(-1).long()
    routed = (flat >= 0) & (flat < n_experts)
    key, order = torch.sort(torch.where(routed, flat, torch.full_like(flat, n_experts)), stable=True)
    offsets = torch.searchsorted(key, torch.arange(n_experts + 1, device=flat.device))
    position = torch.arange(flat.numel(), device=flat.device)
    place = torch.empty_like(flat)
    place[order] = torch.where(key < n_experts, position, torch.full_like(position, -1))
    order = torch.where(key < n_experts, order, torch.full_like(order, -1))
    return offsets.to(torch.int32), order.to(torch.int32), place.to(torch.int32).reshape(experts.shape)


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if case["kind"] == "clip":
        # the clipped gradients go into one flat bucket a type, as a program exchanges them
        places, lengths = _bucket_places(case)
        state["buckets"] = {d: torch.zeros(n, dtype=d, device="cuda") for d, n in lengths.items()}
        state["out"] = [state["buckets"][d][a:a + math.prod(shape)].view(shape) for d, a, shape in places]
    elif case["kind"] not in ("norm", "sort"):
        # the plan of the step's routing, which the program made once for all the calls of the layer
        if own:
            from spla_amd import kernels
            state["plan"] = kernels.route_sort(state["experts"], case["experts"])
        else:
            state["offsets"], state["order"], state["place"] = _plain_sort(state["experts"], case["experts"])
            if "w" in state:
                state["bounds"] = state["offsets"].tolist()
    return state


def _run_own(state):
    from spla_amd import kernels
    case, kind = state["case"], state["case"]["kind"]
    if kind == "sort":
        plan = kernels.route_sort(state["experts"], case["experts"])
        return [plan.offsets, plan.order, plan.place]
    if kind == "rows":
        return kernels.route_rows(state["plan"], state["x"], state["weights"] if case["weighted"] else None)
    if kind == "back":
        return kernels.route_back(state["plan"], state["y"], state["weights"] if case["weighted"] else None)
    if kind == "back_grad":
        return list(kernels.route_back_grad(state["plan"], state["y"], state["weights"], state["dout"]))
    if kind == "product":
        return kernels.expert_product(state["plan"], state["x"], state["w"])
    if kind == "product_grad":
        return list(kernels.expert_product_grad(state["plan"], state["x"], state["w"], state["dy"]))
    if kind == "norm":
        return kernels.global_norm(state["tensors"])
    return [kernels.clip_global_norm(state["tensors"], case["limit"], out=state["out"])] + list(state["buckets"].values())


def run(state):
    if own:
        return _run_own(state)
    case, kind = state["case"], state["case"]["kind"]
    if kind == "sort":
        return list(_plain_sort(state["experts"], case["experts"]))
    if kind == "rows":
        order = state["order"].long()
        entry = order.clamp(min=0)
        rows = state["x"].float()[entry // case["per_token"]]
        if case["weighted"]:
            rows = rows * state["weights"].reshape(-1)[entry, None]
        return torch.where(order[:, None] >= 0, rows, torch.zeros((), device=rows.device)).to(state["x"].dtype)
    if kind in ("back", "back_grad"):
        place = state["place"].long()
        factor = (place >= 0).float()
        if case["weighted"]:
            factor = factor * state["weights"]
        y = state["y"].float()[place.clamp(min=0)]
        if kind == "back":
            return (y * factor[:, :, None]).sum(1).to(state["y"].dtype)
        dout = state["dout"].float()
        dweights = (y * dout[:, None, :]).sum(2) * (place >= 0)
        order = state["order"].long()
        entry = order.clamp(min=0)
        dy = dout[entry // case["per_token"]] * (factor.reshape(-1)[entry] * (order >= 0))[:, None]
        return [dy.to(state["y"].dtype), dweights]
    if kind in ("product", "product_grad"):
        x, w, bounds = state["x"], state["w"], state["bounds"]
        if kind == "product":
            y = torch.zeros(x.shape[0], w.shape[1], dtype=x.dtype, device=x.device)
            for e in range(w.shape[0]):
                a, b = bounds[e], bounds[e + 1]
                if b > a:
                    y[a:b] = torch.matmul(x[a:b].float(), w[e].float().t()).to(x.dtype)
            return y
        dy, dx, dw = state["dy"], torch.zeros_like(x), torch.zeros_like(w)
        for e in range(w.shape[0]):
            a, b = bounds[e], bounds[e + 1]
            if b > a:
                dx[a:b] = torch.matmul(dy[a:b].float(), w[e].float()).to(x.dtype)
                dw[e] = torch.matmul(dy[a:b].float().t(), x[a:b].float()).to(w.dtype)
        return [dx, dw]
    # squares summed in 64 bits: a sum of 1e8 squares
    norm = torch.stack([t.double().square().sum() for t in state["tensors"]]).sum().sqrt()
    if kind == "norm":
        return norm.float()
    scale = torch.clamp(case["limit"] / norm, max=1.0).float()
    for t, out in zip(state["tensors"], state["out"]):
        out.copy_(t.float() * scale)
    return [norm.float()] + list(state["buckets"].values())


def work(case):
    kind = case["kind"]
    if kind in ("norm", "clip"):
        size = sum(math.prod(s) * (2 if _tensor_dtype(case, i) != torch.float32 else 4) for i, s in enumerate(_sizes(case)))
        n = sum(math.prod(s) for s in _sizes(case))
        return {"bytes": size + 4, "flops": 2 * n} if kind == "norm" else {"bytes": 2 * size + 4, "flops": 3 * n}
    t, places, e = case["tokens"], case["tokens"] * case["per_token"], case["experts"]
    if kind == "sort":
        return {"bytes": 12 * places + 4 * (e + 1), "flops": 0}
    s, routed = _SIZE[case["dtype"]], max(1, round(places * (1 - case["padding"])))
    if kind == "rows":
        return {"bytes": (t + places) * case["width"] * s + (8 if case["weighted"] else 4) * places, "flops": routed * case["width"] if case["weighted"] else 0}
    if kind == "back":
        return {"bytes": (t + routed) * case["width"] * s + (8 if case["weighted"] else 4) * places, "flops": 2 * routed * case["width"]}
    if kind == "back_grad":
        return {"bytes": (t + routed + places) * case["width"] * s + 12 * places, "flops": 3 * routed * case["width"]}
    used = min(e, routed) * case["n_in"] * case["n_out"] * s
    if kind == "product":
        return {"bytes": (routed * case["n_in"] + places * case["n_out"]) * s + used, "flops": 2 * routed * case["n_in"] * case["n_out"]}
    return {"bytes": (routed * (case["n_in"] + case["n_out"]) + places * case["n_in"]) * s + used + e * case["n_in"] * case["n_out"] * s,
            "flops": 4 * routed * case["n_in"] * case["n_out"]}


def exact(case, seed):
    kind = case["kind"]
    data = _inputs(case, seed)
    if kind == "norm" or kind == "clip":
        total = sum(float((t.double() ** 2).sum()) for t in data["tensors"])
        norm = math.sqrt(total)
        if kind == "norm":
            return torch.tensor(norm, dtype=torch.float64)
        factor = min(1.0, case["limit"] / norm)
        places, lengths = _bucket_places(case)
        buckets = {d: torch.zeros(n, dtype=torch.float64, device="cuda") for d, n in lengths.items()}
        for (d, a, shape), t in zip(places, data["tensors"]):
            buckets[d][a:a + t.numel()] = t.double().reshape(-1) * factor
        return [torch.tensor(norm, dtype=torch.float64)] + list(buckets.values())
    experts = data["experts"].cpu().reshape(-1)
    k = case["per_token"]
    # entry lists of the experts, in entry order
    lists = [torch.nonzero(experts == e).reshape(-1) for e in range(case["experts"])]
    bounds = [0]
    for entries in lists:
        bounds.append(bounds[-1] + entries.numel())
    order = torch.cat(lists) if lists else experts.new_empty(0)
    if kind == "sort":
        full = torch.full((experts.numel(),), -1, dtype=torch.int32)
        full[:order.numel()] = order.to(torch.int32)
        place = torch.full((experts.numel(),), -1, dtype=torch.int32)
        place[order] = torch.arange(order.numel(), dtype=torch.int32)
        return [torch.tensor(bounds, dtype=torch.int32), full, place.reshape(-1, k)]
    order = order.cuda()
    places = experts.numel()
    weights = data["weights"].double().reshape(-1)
    if not case.get("weighted", True):
        weights = torch.ones_like(weights)
    if kind == "rows":
        out = torch.zeros(places, case["width"], dtype=torch.float64, device="cuda")
        out[:order.numel()] = data["x"].double()[order // k] * weights[order][:, None]
        return out
    if kind == "back":
        out = torch.zeros(case["tokens"], case["width"], dtype=torch.float64, device="cuda")
        for j in range(k):
            mine = torch.nonzero(order % k == j).reshape(-1)
            out[order[mine] // k] += data["y"][mine].double() * weights[order[mine]][:, None]
        return out
    if kind == "back_grad":
        dy = torch.zeros(places, case["width"], dtype=torch.float64, device="cuda")
        dweights = torch.zeros(places, dtype=torch.float64, device="cuda")
        routed = order.numel()
        token_rows = data["dout"].double()[order // k]
        dy[:routed] = token_rows * weights[order][:, None]
        dweights[order] = (token_rows * data["y"][:routed].double()).sum(1)
        return [dy, dweights.reshape(-1, k)]
    x, w = data["x"], data["w"]
    if kind == "product":
        y = torch.zeros(places, case["n_out"], dtype=torch.float64, device="cuda")
        for e, (a, b) in enumerate(zip(bounds, bounds[1:])):
            if a < b:
                y[a:b] = x[a:b].double() @ w[e].double().t().contiguous()
        return y
    dx = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    dw = torch.zeros(w.shape, dtype=torch.float64, device="cuda")
    for e, (a, b) in enumerate(zip(bounds, bounds[1:])):
        if a < b:
            rows = data["dy"][a:b].double()
            dx[a:b] = rows @ w[e].double()
            dw[e] = rows.t().contiguous() @ x[a:b].double()
    return [dx, dw]
