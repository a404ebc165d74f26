"""The operators of an expert feed-forward block over voxel features, as they are measured.

A block of that kind is, per voxel row of a sparse tensor:

    stream, h = residual_norm(x, block)             norm after the previous block, its gate, the residual, the next norm
    routing   = expert_route(logits(h), k)          the k experts of every row, and the place of every (row, expert) pair
    rows      = expert_dispatch(h, routing)         the rows in expert order
    rows      = grouped_linear(rows, W, offsets)    one weight matrix per expert, ragged groups of rows
    block     = expert_combine(rows, routing)       back to voxel order, weighted

``run`` makes one pass through one of them: the framework's calls where ``own`` is set, otherwise the same formulas in
elementary torch operations on 32 bits, rounded once at the end.  ``exact`` states them once more in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases
def _route(rows, experts, k, dtype, renormalize=True, padded=0.0, train=False):
    return {"op": "route", "rows": rows, "experts": experts, "k": k, "dtype": dtype, "renormalize": renormalize, "padded": padded, "train": train}


def _exchange(rows, channels, experts, k, dtype, padded=0.0, train=False):
    return {"op": "exchange", "rows": rows, "channels": channels, "experts": experts, "k": k, "dtype": dtype, "padded": padded, "train": train}


def _products(rows, experts, c_in, c_out, dtype, bias=False, relu=False, behind=0.0, train=False):
    return {"op": "products", "rows": rows, "experts": experts, "c_in": c_in, "c_out": c_out, "dtype": dtype, "bias": bias, "relu": relu,
            "behind": behind, "train": train}


def _norm(rows, channels, dtype, kind="rms", post=False, gate="none", params=None, residual_scale=1.0, block_scale=1.0, train=False):
    return {"op": "norm", "rows": rows, "channels": channels, "dtype": dtype, "kind": kind, "post": post, "gate": gate, "params": params or dtype,
            "residual_scale": residual_scale, "block_scale": block_scale, "train": train}


def listed():
    """Row counts are voxel counts of the framework's scenes (one voxel, a deep level of 1961, the 40 k level, the 127 363 voxels
    of a LiDAR scene), widths those of its networks and their usual four-fold expansion."""
    return [
        # one voxel (or one query row) asked for its experts: launches and host time are everything
        dict(_route(1, 8, 2, "float32"), name="route one voxel"),
        # every voxel of a scene over many small experts, with some padding rows whose mask leaves no expert
        dict(_route(127363, 64, 4, "float16", padded=0.02), name="route scene"),
        # a training step of the router: softmax over all experts, gradient of the logits
        dict(_route(40013, 16, 2, "float32", renormalize=False, train=True), name="route train"),
        # a scene's rows to two experts each and back, narrow rows
        dict(_exchange(127363, 96, 8, 2, "float16"), name="exchange scene"),
        # the same in training, with the gradients of rows and of routing weights; padding rows go nowhere
        dict(_exchange(40013, 256, 16, 2, "bfloat16", padded=0.02, train=True), name="exchange train"),
        # the two experts of one voxel: as long as it takes to read their weights
        dict(_products(2, 8, 256, 1024, "float16"), name="products one voxel"),
        # first half of the experts of a scene: narrow rows, bound by memory, bias and ReLU in the same pass
        dict(_products(254726, 8, 96, 384, "float16", bias=True, relu=True), name="products scene"),
        # a training step of wide experts on the 40 k level: three large ragged products
        dict(_products(80026, 16, 512, 2048, "bfloat16", bias=True, relu=True, behind=0.02, train=True), name="products train"),
        # channel counts that no tile divides, on a deep level, few rows an expert
        dict(_products(3922, 5, 19, 100, "float16", bias=True, train=True), name="products odd"),
        # the norms around one voxel's block
        dict(_norm(1, 256, "float16", post=True, gate="channel"), name="norm one voxel"),
        # pre-norm residual of a whole scene at the narrow width
        dict(_norm(127363, 96, "float16", gate="channel", params="float32", block_scale=0.5), name="norm scene"),
        # norms on both sides of the block with a gate per element, trained with 32-bit parameters
        dict(_norm(127363, 256, "bfloat16", kind="layer", post=True, gate="full", params="float32", train=True), name="norm train"),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return max(low, min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def _width(rng, low, high):
    """A channel count: mostly a multiple of 16 or 8, sometimes any number."""
    c = _spread(rng, low, high)
    step = rng.choice([16, 16, 8, 1])
    return max(low, c // step * step)


def draw(rng):
    op = rng.choice(["route", "exchange", "products", "norm"])
    train = rng.random() < 0.5
    padded = rng.choice([0.0, 0.02, 0.3])
    experts = _spread(rng, 2, 64)
    k = min(experts, rng.choice([1, 2, 2, 3, 4, 8]))
    half = rng.choice(["float16", "bfloat16"])
    if op == "route":
        return _route(_spread(rng, 1, 127363), experts, min(k, 4), rng.choice(["float16", "bfloat16", "float32"]), rng.random() < 0.5, padded, train)
    if op == "exchange":
        channels = _width(rng, 8, 1024)
        most = 2 * 40013 * 256 // (channels * k) if train else 2 * 127363 * 96 // (channels * k)
        return _exchange(_spread(rng, 1, min(127363, most)), channels, experts, k, rng.choice([half, half, "float32"]) if not train else half, padded, train)
    if op == "products":
        c_in, c_out = _width(rng, 16, 2048), _width(rng, 16, 2048)
        rows = _spread(rng, 1, 254726)
        passes = 3 if train else 1
        while rows > 1 and (rows * c_in * c_out * passes > 3 * 80026 * 512 * 2048 or rows * (c_in + c_out) * passes > 254726 * 480):
            rows = (rows + 1) // 2
        return _products(rows, experts, c_in, c_out, half, rng.random() < 0.5, rng.random() < 0.5, padded, train)
    channels = _width(rng, 8, 4096)
    dtype = rng.choice([half, half, "float32"])
    most = max(1, 127363 * 256 // (channels * (2 if dtype == "float32" else 1)))
    return _norm(_spread(rng, 1, min(127363, most)), channels, dtype, rng.choice(["rms", "layer"]), rng.random() < 0.5,
                 rng.choice(["none", "channel", "row", "full"]), rng.choice([dtype, "float32"]), rng.choice([1.0, 0.7]), rng.choice([1.0, 0.25]), train)


# ------------------------------------------------------------------------------------------------ inputs
def _normal(g, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype)


def _logits(c, g, dtype):
    """Router logits: some experts are preferred; rows of padding are masked everywhere, single entries here and there."""
    n, e = c["rows"], c["experts"]
    l = torch.randn(n, e, generator=g, device="cuda") * 1.5 + torch.randn(e, generator=g, device="cuda") * 0.7
    if c["padded"]:
        l[torch.rand(n, generator=g, device="cuda") < c["padded"]] = float("-inf")
        l[torch.rand(n, e, generator=g, device="cuda") < 0.01] = float("-inf")
    return l.to(dtype)


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    t = DTYPES[c["dtype"]]
    s = {"case": c}
    leaves = []
    if c["op"] == "route":
        s["logits"] = _logits(c, g, t)
        leaves = ["logits"]
        if c["train"]:
            s["dweights"] = _normal(g, c["rows"], c["k"])
    elif c["op"] == "exchange":
        with torch.no_grad():
            weights, experts, slots, order, offsets = _plain_route(_logits(c, g, torch.float32), c["k"], True)
        s.update(weights=weights, experts=experts, slots=slots, order=order, offsets=offsets)
        s["x"] = _normal(g, c["rows"], c["channels"], dtype=t)
        s["y"] = _normal(g, c["rows"] * c["k"], c["channels"], dtype=t)
        leaves = ["x", "y", "weights"]
        if c["train"]:
            s["drows"] = _normal(g, c["rows"] * c["k"], c["channels"], dtype=t, scale=0.1)
            s["dout"] = _normal(g, c["rows"], c["channels"], dtype=t, scale=0.1)
    elif c["op"] == "products":
        n, e, ci, co = c["rows"], c["experts"], c["c_in"], c["c_out"]
        liking = torch.randn(e, generator=g, device="cuda") * 0.6
        if e > 3:
            liking[int(seed) % e] = float("-inf")                       # an expert that nobody asked for
        expert = torch.multinomial(torch.softmax(liking, 0), n, replacement=True, generator=g)
        expert = expert[torch.rand(n, generator=g, device="cuda") >= c["behind"]]   # the other rows lie behind the last group
        counts = torch.bincount(expert, minlength=e)
        s["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
        s["most"] = int(counts.max())
        s["x"] = _normal(g, n, ci, dtype=t)
        s["w"] = _normal(g, e, ci, co, dtype=t, scale=1 / math.sqrt(ci))
        s["b"] = _normal(g, e, co, dtype=t, scale=0.1) if c["bias"] else None
        leaves = ["x", "w"] + (["b"] if c["bias"] else [])
        if c["train"]:
            s["dy"] = _normal(g, n, co, dtype=t, scale=0.1)
    else:
        n, ch, p = c["rows"], c["channels"], DTYPES[c["params"]]
        s["x"] = _normal(g, n, ch, dtype=t, shift=0.1)
        s["block"] = _normal(g, n, ch, dtype=t, scale=0.6, shift=-0.05)
        leaves = ["x", "block"]

        def param(name, shift):
            s[name] = _normal(g, ch, dtype=p, scale=0.2, shift=shift)
            leaves.append(name)
        param("weight", 1.0)
        if c["kind"] == "layer":
            param("bias", 0.0)
        if c["post"]:
            param("post_weight", 1.0)
            if c["kind"] == "layer":
                param("post_bias", 0.0)
        if c["gate"] != "none":
            s["gate"] = {"channel": lambda: _normal(g, ch, dtype=p, scale=0.3, shift=0.5),
                         "row": lambda: _normal(g, n, 1, dtype=t, scale=0.3, shift=0.5),
                         "full": lambda: _normal(g, n, ch, dtype=t, scale=0.3, shift=0.5)}[c["gate"]]()
            leaves.append("gate")
        if c["train"]:
            s["dstream"] = _normal(g, n, ch, dtype=t, scale=0.1)
            s["dnormed"] = _normal(g, n, ch, dtype=t, scale=0.1)
    if c["train"]:
        for name in leaves:
            s[name].requires_grad_(True)
        s["leaves"] = [s[name] for name in leaves]
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _PLAIN[state["case"]["op"]](state, state["case"])


def _own(s):
    from spira_b200.nn import functional as F
    c = s["case"]
    if c["op"] == "route":
        r = F.expert_route(s["logits"], c["k"], renormalize=c["renormalize"])
        out = [r.weights, r.experts, r.slots, r.order, r.offsets]
        tops, douts = [r.weights], [s.get("dweights")]
    elif c["op"] == "exchange":
        r = F.ExpertRouting(s["weights"], s["experts"], s["slots"], s["order"], s["offsets"])
        out = [F.expert_dispatch(s["x"], r), F.expert_combine(s["y"], r)]
        tops, douts = out, [s.get("drows"), s.get("dout")]
    elif c["op"] == "products":
        out = [F.grouped_linear(s["x"], s["w"], s["offsets"], s["b"], relu=c["relu"])]
        tops, douts = out, [s.get("dy")]
    else:
        out = list(F.residual_norm(s["x"], s["block"], kind=c["kind"], weight=s["weight"], bias=s.get("bias"), post=c["post"],
                                   post_weight=s.get("post_weight"), post_bias=s.get("post_bias"), gate=s.get("gate"),
                                   residual_scale=c["residual_scale"], block_scale=c["block_scale"], eps=1e-5))
        tops, douts = out, [s.get("dstream"), s.get("dnormed")]
    if c["train"]:
        return out + list(torch.autograd.grad(tops, s["leaves"], douts))
    return out


def _plain_route(logits, k, renormalize):
    l = logits.float()
    n, e = l.shape
    values, index = torch.sort(l, dim=1, descending=True, stable=True)
    chosen = values[:, :k] > float("-inf")
    top = torch.where(chosen[:, :1], values[:, :1], 0.0)
    scores = torch.exp(values - top)                                   # 0 where a logit is -inf
    total = (scores[:, :k] if renormalize else scores).sum(1, keepdim=True)
    weights = torch.where(chosen, scores[:, :k] / total, 0.0)
    experts = torch.where(chosen, index[:, :k], -1)
    flat = experts.reshape(-1)
    of_expert = flat[:, None] == torch.arange(e, device=l.device)
    ends = of_expert.sum(0).cumsum(0)
    offsets = torch.cat([ends.new_zeros(1), ends])
    order = torch.argsort(torch.where(flat < 0, e, flat), stable=True)
    slots = torch.empty_like(order)
    slots[order] = torch.arange(n * k, device=l.device)
    slots = torch.where(flat < 0, -1, slots).view(n, k)
    order = torch.where(torch.arange(n * k, device=l.device) < offsets[-1], order, -1)
    return weights, experts.int(), slots.int(), order.int(), offsets.int()


def _plain_route_case(s, c):
    out = list(_plain_route(s["logits"], c["k"], c["renormalize"]))
    if c["train"]:
        weights, experts = out[0], out[1]
        u = s["dweights"] * (experts >= 0)
        dot = (u * weights).sum(1, keepdim=True)
        if c["renormalize"]:
            d = torch.zeros_like(s["logits"], dtype=torch.float32)
        else:
            l = s["logits"].float()
            top = l.amax(1, keepdim=True)
            scores = torch.exp(l - torch.where(top > float("-inf"), top, 0.0))
            d = -dot * scores / scores.sum(1, keepdim=True).clamp_min(1e-30)
        add = weights * (u - dot) if c["renormalize"] else weights * u
        d.scatter_add_(1, experts.clamp_min(0).long(), torch.where(experts >= 0, add, 0.0))
        out.append(d.to(s["logits"].dtype))
    return out


def _plain_exchange(s, c):
    n, k, ch = c["rows"], c["k"], c["channels"]
    t = s["x"].dtype
    order, slots = s["order"].long(), s["slots"].long()
    there, taken = (order >= 0)[:, None], (slots >= 0)[:, :, None]
    place = slots.clamp_min(0)
    rows = torch.where(there, s["x"][order.clamp_min(0) // k], 0.0).to(t)
    y = s["y"].float()[place]                                         # [n, k, channels]
    w = torch.where(taken, s["weights"][:, :, None], 0.0)
    out = [rows, (torch.where(taken, y, 0.0) * w).sum(1).to(t)]
    if c["train"]:
        dout = s["dout"].float()
        dx = torch.where(taken, s["drows"].float()[place], 0.0).sum(1)
        dy = torch.where(there, dout[order.clamp_min(0) // k] * s["weights"].reshape(-1)[order.clamp_min(0)][:, None], 0.0)
        dw = torch.where(taken, y * dout[:, None, :], 0.0).sum(2)
        out += [dx.to(t), dy.to(t), dw]
    return out


def _plain_products(s, c):
    n, t = c["rows"], s["x"].dtype
    begin, end = s["offsets"][:-1].long(), s["offsets"][1:].long()
    place = begin[:, None] + torch.arange(s["most"], device="cuda")    # [experts, most]: every group padded to the longest
    inside = place < end[:, None]
    place = place.clamp_max(n - 1)
    x = torch.where(inside[:, :, None], s["x"].float()[place], 0.0)
    w = s["w"].float()
    z = torch.bmm(x, w)
    if s["b"] is not None:
        z = z + s["b"].float()[:, None, :]
    if c["relu"]:
        z = z.clamp_min(0.0)
    at = place[inside]
    y = torch.zeros(n, c["c_out"], device="cuda")
    y[at] = z[inside]
    out = [y.to(t)]
    if c["train"]:
        dz = torch.where(inside[:, :, None], s["dy"].float()[place], 0.0)
        if c["relu"]:
            dz = dz * (z > 0)
        dx = torch.zeros(n, c["c_in"], device="cuda")
        dx[at] = torch.bmm(dz, w.transpose(1, 2))[inside]
        out += [dx.to(t), torch.bmm(x.transpose(1, 2), dz).to(t)]
        if s["b"] is not None:
            out.append(dz.sum(1).to(t))
    return out


def _plain_norm_parts(v, kind, eps=1e-5):
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    r = torch.rsqrt((v * v).mean(1, keepdim=True) + eps)
    return v * r, r


def _plain_norm(s, c):
    t, p, kind = s["x"].dtype, s["weight"].dtype, c["kind"]
    f = {name: s[name].float() for name in ("x", "block", "weight", "bias", "post_weight", "post_bias", "gate") if name in s}
    a, b = c["residual_scale"], c["block_scale"]
    block = f["block"]
    if c["post"]:
        bhat, rb = _plain_norm_parts(block, kind)
        block = bhat * f["post_weight"]
        if "post_bias" in f:
            block = block + f["post_bias"]
    gated = block * f["gate"] if "gate" in f else block
    stream = a * f["x"] + b * gated
    hat, r = _plain_norm_parts(stream, kind)
    normed = hat * f["weight"]
    if "bias" in f:
        normed = normed + f["bias"]
    out = [stream.to(t), normed.to(t)]
    if c["train"]:
        dh = s["dnormed"].float()
        u = dh * f["weight"]
        back = u - hat * (u * hat).mean(1, keepdim=True)
        if kind == "layer":
            back = back - u.mean(1, keepdim=True)
        d = s["dstream"].float() + r * back
        grads = {"x": a * d, "weight": (dh * hat).sum(0), "bias": dh.sum(0)}
        dp = b * d
        if "gate" in f:
            dg = dp * block
            grads["gate"] = dg.sum(0) if c["gate"] == "channel" else dg.sum(1, keepdim=True) if c["gate"] == "row" else dg
            dp = dp * f["gate"]
        if c["post"]:
            grads["post_weight"], grads["post_bias"] = (dp * bhat).sum(0), dp.sum(0)
            u = dp * f["post_weight"]
            back = u - bhat * (u * bhat).mean(1, keepdim=True)
            if kind == "layer":
                back = back - u.mean(1, keepdim=True)
            dp = rb * back
        grads["block"] = dp
        out += [grads[name].to(s[name].dtype) for name in ("x", "block", "weight", "bias", "post_weight", "post_bias", "gate") if name in f]
    return out


_PLAIN = {"route": _plain_route_case, "exchange": _plain_exchange, "products": _plain_products, "norm": _plain_norm}


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    s = {"float16": 2, "bfloat16": 2, "float32": 4}
    t, n = s[c["dtype"]], c["rows"]
    if c["op"] == "route":
        k, e = c["k"], c["experts"]
        forward = n * e * t + n * k * 16 + (e + 1) * 4
        return {"bytes": forward + (n * e * t * (1 if c["renormalize"] else 2) + n * k * 4 if c["train"] else 0), "flops": n * e * (12 if c["train"] else 4)}
    if c["op"] == "exchange":
        ch, k = c["channels"], c["k"]
        forward = n * ch * t * (1 + k) + n * k * 4 + n * ch * t * (k + 1) + n * k * 8
        backward = n * ch * t * (k + 1) + n * ch * t * (2 * k + 1) + n * k * 8
        return {"bytes": forward + (backward if c["train"] else 0), "flops": n * ch * k * (8 if c["train"] else 2)}
    if c["op"] == "products":
        ci, co = c["c_in"], c["c_out"]
        live = min(c["experts"], n)                                    # an expert without rows is not read
        weights = live * ci * co * t
        forward = n * (ci + co) * t + weights
        backward = n * (ci + co) * t + weights + c["experts"] * ci * co * t
        return {"bytes": forward + (backward if c["train"] else 0), "flops": 2 * n * ci * co * (3 if c["train"] else 1)}
    ch = c["channels"]
    gate = {"none": 0, "channel": 0, "row": n * t, "full": n * ch * t}[c["gate"]]
    forward = 4 * n * ch * t + gate
    backward = 6 * n * ch * t + 2 * gate - (4 * n * ch * t if c["train"] else 0) + 2 * n * ch * t     # x, block, gate are read once
    return {"bytes": forward + (backward if c["train"] else 0) + 5 * ch * s[c["params"]], "flops": n * ch * (40 if c["train"] else 14)}


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"route": _exact_route, "exchange": _exact_exchange, "products": _exact_products, "norm": _exact_norm}[case["op"]](s, case)


def _exact_route(s, c):
    l = s["logits"].detach().double()
    n, e = l.shape
    column = torch.arange(e, device=l.device)
    left, picked, any_left = l.clone(), torch.zeros_like(l, dtype=torch.bool), []
    firsts = []
    for _ in range(c["k"]):                                            # the largest that is left, the lowest index of equals
        best = left.max(1, keepdim=True).values
        first = torch.where(left == best, column, e).min(1).values
        alive = best[:, 0] > -math.inf
        firsts.append(first)
        any_left.append(alive)
        hit = (column == first[:, None]) & alive[:, None]
        picked |= hit
        left = torch.where(hit, -math.inf, left)
    basis = torch.where(picked, l, -math.inf) if c["renormalize"] else l
    softmax = torch.nan_to_num(torch.softmax(basis, 1), nan=0.0)       # a row without experts has no weights
    weights = torch.stack([torch.where(a, softmax.gather(1, f.clamp_max(e - 1)[:, None])[:, 0], 0.0) for f, a in zip(firsts, any_left)], 1)
    out = [weights, None, None, None, None]
    if c["train"]:
        du = torch.zeros_like(l)
        for j, (f, a) in enumerate(zip(firsts, any_left)):
            du.scatter_add_(1, f.clamp_max(e - 1)[:, None], torch.where(a, s["dweights"][:, j].double(), 0.0)[:, None])
        out.append(softmax * (du - (du * softmax).sum(1, keepdim=True)))
    return out


def _exact_exchange(s, c):
    n, k = c["rows"], c["k"]
    x, y, w = s["x"].detach().double(), s["y"].detach().double(), s["weights"].detach().double()
    rows, out = torch.zeros_like(y), torch.zeros_like(x)
    dx, dy, dw = torch.zeros_like(x), torch.zeros_like(y), torch.zeros_like(w)
    for j in range(k):
        slot = s["slots"][:, j].long()
        voxel = torch.nonzero(slot >= 0)[:, 0]
        slot = slot[voxel]
        rows[slot] = x[voxel]
        out[voxel] += w[voxel, j, None] * y[slot]
        if c["train"]:
            dx[voxel] += s["drows"][slot].double()
            dy[slot] = w[voxel, j, None] * s["dout"][voxel].double()
            dw[voxel, j] = torch.einsum("nc,nc->n", y[slot], s["dout"][voxel].double())
    return [rows, out] + ([dx, dy, dw] if c["train"] else [])


def _exact_products(s, c):
    x, w = s["x"].detach().double(), s["w"].detach().double()
    y = torch.zeros(c["rows"], c["c_out"], dtype=torch.float64, device="cuda")
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros(c["experts"], c["c_out"], dtype=torch.float64, device="cuda")
    o = s["offsets"].tolist()
    for e in range(c["experts"]):
        group = slice(o[e], o[e + 1])
        z = x[group] @ w[e]
        if c["bias"]:
            z += s["b"][e].detach().double()
        live = z > 0 if c["relu"] else torch.ones_like(z, dtype=torch.bool)
        y[group] = torch.where(live, z, 0.0)
        if c["train"]:
            dz = torch.where(live, s["dy"][group].double(), 0.0)
            dx[group], dw[e], db[e] = dz @ w[e].T, x[group].T @ dz, dz.sum(0)
    return [y] + (([dx, dw] + ([db] if c["bias"] else [])) if c["train"] else [])


def _exact_norm(s, c):
    """The forward pass in 64 bits, its gradients from torch's differentiation of it, some rows at a time."""
    names = [n for n in ("x", "block", "weight", "bias", "post_weight", "post_bias", "gate") if n in s]
    per_row = {"x", "block"} | ({"gate"} if c["gate"] in ("row", "full") else set())
    parts, sums = {n: [] for n in ["stream", "normed"] + names}, {}

    def norm(v, w, b):
        if c["kind"] == "layer":
            v = v - v.mean(dim=-1, keepdim=True)
        v = v / (v.pow(2).mean(dim=-1, keepdim=True) + 1e-5).sqrt() * w
        return v if b is None else v + b

    for low in range(0, c["rows"], 16384):
        q = {n: (s[n][low:low + 16384] if n in per_row else s[n]).detach().double().requires_grad_(c["train"]) for n in names}
        with torch.enable_grad():
            block = norm(q["block"], q["post_weight"], q.get("post_bias")) if c["post"] else q["block"]
            stream = c["residual_scale"] * q["x"] + c["block_scale"] * (block * q["gate"] if "gate" in q else block)
            normed = norm(stream, q["weight"], q.get("bias"))
        parts["stream"].append(stream.detach())
        parts["normed"].append(normed.detach())
        if c["train"]:
            d = torch.autograd.grad([stream, normed], [q[n] for n in names], [s["dstream"][low:low + 16384].double(), s["dnormed"][low:low + 16384].double()])
            for n, v in zip(names, d):
                if n in per_row:
                    parts[n].append(v)
                else:
                    sums[n] = sums[n] + v if n in sums else v
    out = [torch.cat(parts["stream"]), torch.cat(parts["normed"])]
    if c["train"]:
        out += [torch.cat(parts[n]) if n in per_row else sums[n] for n in names]
    return out
