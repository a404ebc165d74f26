"""GPU: routing, row exchange, ragged products and gated residual norms against plain 64-bit forms.

Tolerances.  A result rounded to type t is off by at most half a step, eps(t)/2 relative.  A sum of n fp32 terms is off
by at most n * 2^-24 * (sum of the terms' absolute values), whatever its order; every elementary fp32 operation in front of
it adds 2^-24 relative of its own result.  `close` takes the exact value, the sum of absolute values ("size") and n.
Products with integer inputs are exact in fp32, so those tests ask for equal bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
HALF = [torch.float16, torch.bfloat16]
ANY = HALF + [torch.float32]


def half_step(t):
    return torch.finfo(t).eps / 2


def close(got, exact, size, terms, name=""):
    """|got - exact| <= eps/2 |exact| + terms 2^-24 size (both scaled by the rounding) + the smallest step of the type."""
    assert got.shape == exact.shape, (name, got.shape, exact.shape)
    u = half_step(got.dtype)
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps / 2
    tol = u * exact.abs() + (1 + u) * terms * U32 * size + tiny
    err = (got.double() - exact).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (name, int(bad.sum()), float((err / tol.clamp_min(1e-300)).max()))


def rand(*shape, dtype=torch.float32, scale=1.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + sum(shape))
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def whole(*shape, dtype, top=2, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + sum(shape))
    return torch.randint(-top, top + 1, shape, generator=g, device="cuda").to(dtype)


# ------------------------------------------------------------------------------------------------ routing
def plain_route(logits, k, renormalize):
    l = logits.double().cpu()
    n, e = l.shape
    weights, experts = torch.zeros(n, k, dtype=torch.float64), torch.full((n, k), -1, dtype=torch.int32)
    for t in range(n):
        row = [(-(math.inf if math.isnan(v) else v), not math.isnan(v), i) for i, v in enumerate(l[t].tolist()) if v != -math.inf]
        best = [i for _, _, i in sorted(row, key=lambda q: (q[1], q[0], q[2]))[:k]]
        experts[t, :len(best)] = torch.tensor(best, dtype=torch.int32)
        if best:
            over = l[t, best] if renormalize else l[t]
            p = torch.exp(l[t, best] - l[t].max()) / torch.exp(over - l[t].max()).sum()
            weights[t, :len(best)] = p
    flat = experts.view(-1).tolist()
    order = [i for e_ in range(e) for i, v in enumerate(flat) if v == e_]
    slots = torch.full((n * k,), -1, dtype=torch.int32)
    slots[torch.tensor(order, dtype=torch.long)] = torch.arange(len(order), dtype=torch.int32)
    counts = [flat.count(e_) for e_ in range(e)]
    offsets = torch.tensor([0] + counts, dtype=torch.int32).cumsum(0).int()
    order = torch.tensor(order + [-1] * (n * k - len(order)), dtype=torch.int32)
    return weights, experts, slots.view(n, k), order, offsets


def check_route(logits, k, renormalize):
    from spira_b200.nn import functional as F
    r = F.expert_route(logits, k, renormalize=renormalize)
    weights, experts, slots, order, offsets = plain_route(logits, k, renormalize)
    assert torch.equal(r.experts.cpu(), experts)
    assert torch.equal(r.slots.cpu(), slots)
    assert torch.equal(r.order.cpu(), order)
    assert torch.equal(r.offsets.cpu(), offsets)
    # exp of a difference d that is rounded once: relative error d 2^-24 and 2 steps of exp; a sum and a division
    spread = logits.double().cpu().nan_to_num(0, 0, 0)
    d = float(spread.max() - spread.min()) if spread.numel() else 0.0
    got = r.weights.double().cpu()
    assert torch.equal(got.isnan(), weights.isnan())
    assert bool(((got - weights).abs() <= (2 * (d + 4) + logits.shape[1] + 2) * U32 * weights.abs() + 1e-37)[~weights.isnan()].all())
    return r


@pytest.mark.parametrize("dtype", ANY)
@pytest.mark.parametrize("n,e,k", [(0, 4, 2), (1, 1, 1), (1, 8, 2), (3, 5, 5), (37, 16, 3), (255, 33, 4), (64, 64, 8), (129, 128, 2), (40, 200, 7),
                                   (19, 512, 32), (200, 40, 32), (1500, 7, 3), (2049, 9, 2), (2500, 65, 2)])
@pytest.mark.parametrize("renormalize", [True, False])
def test_route(dtype, n, e, k, renormalize):
    logits = rand(n, e, dtype=dtype, scale=2.0)
    if n > 2:
        logits[n // 2] = float("-inf")                     # a row that goes nowhere
        logits[::3, e // 2] = float("-inf")
        logits[1, : max(1, e - 1)] = float("-inf")         # one expert left
        logits[n // 3] = 1.0                               # all equal
    check_route(logits, k, renormalize)


@pytest.mark.parametrize("dtype", ANY)
def test_route_ties_zeros_lowest_values_and_nan(dtype):
    low, tiny = torch.finfo(dtype).min, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps      # the smallest step above zero
    rows = torch.tensor([[0.0, -0.0, 0.0, -0.0, -1.0], [low, low, low, low, low], [low, 3.0, low, 3.0, low], [-math.inf] * 5,
                         [1.0, math.nan, 2.0, math.nan, 0.0], [1.0, -math.nan, 2.0, 3.0, 0.0], [-math.inf, low, -math.inf, -math.inf, -math.inf],
                         [5.0, tiny, -tiny, 0.0, 5.0], [-tiny, tiny, -0.0, 0.0, -2.0]], dtype=torch.float64).to(dtype)
    for k in (1, 2, 4, 5):
        for renormalize in (True, False):
            check_route(rows.cuda(), k, renormalize)


def test_route_infinite_logit_gives_nan_weights_like_a_softmax():
    from spira_b200.nn import functional as F
    r = F.expert_route(torch.tensor([[math.inf, 0.0, 1.0], [0.0, 1.0, 2.0]], device="cuda"), 2)
    assert r.experts.tolist() == [[0, 2], [2, 1]]
    assert bool(r.weights[0].isnan().any()) and bool(r.weights[1].isfinite().all())


def test_route_strided_and_misaligned_rows():
    base = rand(300, 80)
    check_route(base[:, 3:67], 4, True)
    check_route(base[::2, :64], 4, False)
    check_route(rand(64, 300).t(), 2, True)
    check_route(rand(1, 32).expand(70, 32), 3, True)


@pytest.mark.parametrize("dtype", ANY)
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("n,e,k", [(1, 4, 2), (77, 16, 2), (300, 70, 5), (2100, 8, 2)])
def test_route_gradient(dtype, renormalize, n, e, k):
    from spira_b200.nn import functional as F
    logits = rand(n, e, dtype=dtype)
    if n > 10:
        logits[4] = float("-inf")
        logits[6, 1:] = float("-inf")
    logits.requires_grad_(True)
    r = F.expert_route(logits, k, renormalize=renormalize)
    dw = rand(k, n).t()                                    # a strided gradient
    got, = torch.autograd.grad(r.weights, logits, dw)
    l = logits.detach().double().requires_grad_(True)
    there = r.experts >= 0
    picked = torch.zeros(n, e, dtype=torch.bool, device="cuda").scatter_(1, r.experts.clamp_min(0).long(), there)
    # scatter writes False for missing experts at column 0: put the chosen ones back
    for j in range(k):
        rows = there[:, j].nonzero()[:, 0]
        picked[rows, r.experts[rows, j].long()] = True
    alive = picked.any(1)
    basis = torch.where(picked if renormalize else torch.ones_like(picked), l, -math.inf)
    p = torch.softmax(basis[alive], 1)
    w = torch.where(there[alive], p.gather(1, r.experts[alive].clamp_min(0).long()), 0.0)
    exact, = torch.autograd.grad(w, l, dw[alive].double())
    size = dw.double().abs().sum(1, keepdim=True).expand(n, e)
    close(got, exact, size, 8 * (e + 20), "dlogits")


@pytest.mark.parametrize("e,k,dtype", [(64, 4, torch.float16), (20, 3, torch.bfloat16), (32, 32, torch.float16), (128, 2, torch.bfloat16), (250, 9, torch.float16),
                                       (512, 8, torch.bfloat16), (64, 4, torch.float32), (9, 9, torch.float32)])
def test_route_many_rows_against_torch(e, k, dtype):
    """A whole scene over many CTAs: places from a stable sort of the choices."""
    from spira_b200.nn import functional as F
    logits = rand(127363, e, dtype=dtype)
    logits[::50] = float("-inf")
    logits[1::50, : e - 1] = float("-inf")
    r = F.expert_route(logits, k)
    values, index = torch.sort(logits.float(), dim=1, descending=True, stable=True)
    experts = torch.where(values[:, :k] > -math.inf, index[:, :k], -1)
    assert torch.equal(r.experts, experts.int())
    flat = experts.reshape(-1)
    order = torch.argsort(torch.where(flat < 0, e, flat), stable=True)
    total = int((flat >= 0).sum())
    assert torch.equal(r.order[:total], order[:total].int()) and bool((r.order[total:] == -1).all())
    assert torch.equal(r.offsets.cpu(), torch.cat([torch.zeros(1, dtype=torch.long), torch.bincount(flat[flat >= 0], minlength=e).cumsum(0).cpu()]).int())
    top = torch.where(values[:, :1] > -math.inf, values[:, :1], 0.0).double()
    p = torch.where(experts >= 0, torch.exp(values[:, :k].double() - top), 0.0)
    exact = p / p.sum(1, keepdim=True).clamp_min(1e-300)
    assert bool(((r.weights.double() - exact).abs() <= (2 * (14 + 4) + k + 2) * U32 * exact + 1e-37).all())       # (differences of logits below 14)
    assert torch.equal(r.slots.view(-1)[order[:total]], torch.arange(total, device="cuda", dtype=torch.int32))


# ------------------------------------------------------------------------------------------------ exchange
def some_routing(n, e, k, dead=0.1, seed=0):
    from spira_b200.nn import functional as F
    logits = rand(n, e, seed=seed)
    if n:
        logits[torch.rand(n, generator=torch.Generator().manual_seed(seed)) < dead] = float("-inf")
    return F.expert_route(logits, k)


@pytest.mark.parametrize("dtype", ANY)
@pytest.mark.parametrize("n,c,e,k", [(0, 8, 4, 2), (1, 1, 3, 1), (1, 256, 8, 2), (5, 7, 4, 4), (300, 96, 8, 2), (257, 100, 16, 5), (90, 1024, 9, 3), (64, 2056, 4, 2)])
def test_dispatch_and_combine(dtype, n, c, e, k):
    from spira_b200.nn import functional as F
    r = some_routing(n, e, k)
    x, y = whole(n, c, dtype=dtype, seed=1).requires_grad_(True), whole(n * k, c, dtype=dtype, top=8, seed=2).requires_grad_(True)
    w = (2.0 ** -torch.randint(0, 4, (n, k), device="cuda").float()).requires_grad_(True)
    r = r._replace(weights=w)
    rows, out = F.expert_dispatch(x, r), F.expert_combine(y, r)
    drows, dout = whole(n * k, c, dtype=dtype, seed=3), whole(n, c, dtype=dtype, seed=4)
    dx, dy, dw = torch.autograd.grad([rows, out], [x, y, w], [drows, dout])
    slots = r.slots.long()
    want_rows, want_out = torch.zeros(n * k, c, dtype=torch.float64, device="cuda"), torch.zeros(n, c, dtype=torch.float64, device="cuda")
    want_dx, want_dy, want_dw = torch.zeros_like(want_out), torch.zeros_like(want_rows), torch.zeros(n, k, dtype=torch.float64, device="cuda")
    for j in range(k):
        t = (slots[:, j] >= 0).nonzero()[:, 0]
        s = slots[t, j]
        want_rows[s] = x.detach()[t].double()
        want_out[t] += w.detach()[t, j, None].double() * y.detach()[s].double()
        want_dx[t] += drows[s].double()
        want_dy[s] = w.detach()[t, j, None].double() * dout[t].double()
        want_dw[t, j] = (y.detach()[s].double() * dout[t].double()).sum(1)
    # whole numbers and powers of two: every fp32 sum is exact
    for got, want in ((rows, want_rows), (out, want_out), (dx, want_dx), (dy, want_dy), (dw, want_dw)):
        assert torch.equal(got, want.to(got.dtype))


def test_exchange_strides_and_alignment():
    from spira_b200.nn import functional as F
    n, c, k = 200, 64, 2
    r = some_routing(n, 8, k)
    wide = whole(n, c + 5, dtype=torch.float16)
    for x in (wide[:, 5:], wide[:, :c], wide[:, 3:3 + c].t().contiguous().t(), whole(1, c, dtype=torch.float16).expand(n, c)):
        dense = x.contiguous()
        assert torch.equal(F.expert_dispatch(x, r), F.expert_dispatch(dense, r))
    rows = whole(n * k, c + 3, dtype=torch.bfloat16)
    assert torch.equal(F.expert_combine(rows[:, 3:], r), F.expert_combine(rows[:, 3:].contiguous(), r))
    w = torch.rand(k, n, device="cuda").t()
    assert torch.equal(F.expert_combine(rows[:, 3:], r._replace(weights=w)), F.expert_combine(rows[:, 3:].contiguous(), r._replace(weights=w.contiguous())))


def test_combine_rounds_once():
    from spira_b200.nn import functional as F
    n, c, k = 500, 72, 3
    r = some_routing(n, 8, k)
    for dtype in ANY:
        y = rand(n * k, c, dtype=dtype)
        terms = torch.where((r.slots >= 0)[:, :, None], y[r.slots.clamp_min(0).long()].double() * r.weights[:, :, None].double(), 0.0)
        close(F.expert_combine(y, r), terms.sum(1), terms.abs().sum(1), k + 1, "combine")


def test_places_outside_the_rows_are_skipped():
    """A routing that was not made by expert_route cannot make the kernels reach outside their tensors."""
    from spira_b200.nn import functional as F
    n, c, k = 33, 24, 2
    r = some_routing(n, 4, k, dead=0.0)
    slots = r.slots.clone()
    slots[3, 0], slots[7, 1], slots[9, 0] = n * k, -5, 1 << 30
    bad = r._replace(slots=slots, offsets=torch.full_like(r.offsets, 1 << 30))
    x = rand(n, c, dtype=torch.float16).requires_grad_(True)
    y = rand(n * k, c, dtype=torch.float16).requires_grad_(True)
    out = F.expert_combine(y, bad)
    good = F.expert_combine(y, r)
    same = torch.ones(n, dtype=torch.bool)
    same[[3, 7, 9]] = False
    assert torch.equal(out[same.cuda()], good[same.cuda()])
    torch.autograd.grad([F.expert_dispatch(x, bad), out], [x, y], [torch.ones(n * k, c, dtype=torch.float16, device="cuda"), torch.ones_like(out)])
    torch.cuda.synchronize()


# ------------------------------------------------------------------------------------------------ ragged products
def some_offsets(n, e, seed=0, first=0, behind=0):
    g = torch.Generator().manual_seed(seed + n + e)
    cuts = torch.sort(torch.randint(0, max(1, n - behind - first + 1), (e - 1,), generator=g)).values + first
    o = torch.cat([torch.tensor([first]), cuts, torch.tensor([max(first, n - behind)])])
    return o.clamp_max(n).to(torch.int32).cuda()


def plain_products(x, w, offsets, b, relu, dy, y_own):
    x, w, dy = x.detach().double(), w.detach().double(), dy.double()
    o = offsets.tolist()
    y = torch.zeros(x.shape[0], w.shape[2], dtype=torch.float64, device="cuda")
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros(w.shape[0], w.shape[2], dtype=torch.float64, device="cuda")
    for e in range(w.shape[0]):
        s = slice(o[e], o[e + 1])
        z = x[s] @ w[e] + (0 if b is None else b.detach()[e].double())
        y[s] = z.clamp_min(0) if relu else z
        dz = dy[s] * (y_own[s] > 0) if relu else dy[s]
        dx[s], dw[e], db[e] = dz @ w[e].T, x[s].T @ dz, dz.sum(0)
    return y, dx, dw, db


SHAPES = [(1, 1, 1, 1), (2, 8, 256, 1024), (5, 3, 19, 100), (130, 4, 16, 16), (129, 1, 64, 64), (300, 7, 20, 33), (257, 5, 40, 24), (1000, 3, 96, 384),
          (777, 6, 72, 264), (512, 2, 136, 520), (2000, 2, 512, 48), (640, 9, 8, 8), (4100, 4, 32, 32), (33, 40, 48, 80), (1500, 3, 17, 64), (1500, 3, 64, 17),
          (20000, 3, 256, 512), (19001, 7, 264, 392), (30000, 2, 200, 136), (9000, 5, 384, 192),
          (6000, 3, 201, 227), (9000, 2, 200, 151), (9000, 2, 151, 200), (20000, 1, 121, 129)]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("n,e,ci,co", SHAPES)
def test_products_exact(dtype, n, e, ci, co):
    """Small whole numbers: every sum is exact in fp32, so forward and gradients equal the rounded 64-bit values bit for bit."""
    from spira_b200.nn import functional as F
    for variant in range(3):
        bias, relu = variant >= 1, variant == 2
        offsets = some_offsets(n, e, seed=variant, first=min(n, 3 * (variant == 1)), behind=min(n, 5 * (variant >= 1)))
        x = whole(n, ci, dtype=dtype, seed=variant).requires_grad_(True)
        w = whole(e, ci, co, dtype=dtype, seed=7).requires_grad_(True)
        b = whole(e, co, dtype=dtype, seed=9).requires_grad_(True) if bias else None
        dy = whole(n, co, dtype=dtype, top=1, seed=11)
        y = F.grouped_linear(x, w, offsets, b, relu=relu)
        grads = torch.autograd.grad(y, [x, w] + ([b] if bias else []), dy)
        want = plain_products(x, w, offsets, b, relu, dy, y.detach())
        for name, got, ref in zip(("y", "dx", "dw", "db"), (y,) + grads, want):
            assert torch.equal(got, ref.to(dtype)), (name, variant, float((got.double() - ref).abs().max()))


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("n,e,ci,co", [(3000, 4, 96, 384), (3000, 5, 100, 39), (20000, 3, 64, 128)])
def test_products_rounding(dtype, n, e, ci, co):
    from spira_b200.nn import functional as F
    offsets = some_offsets(n, e, behind=11)
    x, w, b = rand(n, ci, dtype=dtype).requires_grad_(True), rand(e, ci, co, dtype=dtype, scale=ci ** -0.5).requires_grad_(True), rand(e, co, dtype=dtype).requires_grad_(True)
    dy = rand(n, co, dtype=dtype, seed=5)
    y = F.grouped_linear(x, w, offsets, b, relu=True)
    grads = torch.autograd.grad(y, [x, w, b], dy)
    want = plain_products(x, w, offsets, b, True, dy, y.detach())
    zero = torch.zeros_like
    size = plain_products(x.detach().abs(), w.detach().abs(), offsets, b.detach().abs(), True, dy.abs(), torch.ones_like(y))
    for name, got, ref, s, terms in zip(("y", "dx", "dw", "db"), (y,) + grads, want, size, (ci + 1, co, n, n)):
        close(got, ref, s, terms, name)


def test_products_strided_misaligned_and_foreign_rows():
    """Views with other strides and alignments give what dense copies give; NaN and infinity in rows of no group, or of
    another group, reach nothing else."""
    from spira_b200.nn import functional as F
    n, e, ci, co = 700, 5, 64, 96
    offsets = some_offsets(n, e, first=4, behind=9)
    w = whole(e, ci, co, dtype=torch.float16)
    base = whole(n, ci + 9, dtype=torch.float16)
    for x in (base[:, 8:72], base[:, 1:65], base[:, :ci], whole(ci, n, dtype=torch.float16).t(), whole(1, ci, dtype=torch.float16).expand(n, ci)):
        assert torch.equal(F.grouped_linear(x, w, offsets), F.grouped_linear(x.contiguous(), w, offsets))
    x = whole(n, ci, dtype=torch.float16)
    o = offsets.tolist()
    dirty = x.clone()
    dirty[:4], dirty[n - 9:] = math.nan, math.inf
    big = max(range(e), key=lambda i: o[i + 1] - o[i])
    others = [i for i in range(e) if i != big and o[i + 1] > o[i]]
    for i in others:
        dirty[o[i]:o[i + 1]] = math.nan
    clean, got = F.grouped_linear(x, w, offsets), F.grouped_linear(dirty, w, offsets)
    assert torch.equal(got[o[big]:o[big + 1]], clean[o[big]:o[big + 1]])
    assert bool((got[:4] == 0).all()) and bool((got[n - 9:] == 0).all())
    dy = whole(n, co, dtype=torch.float16, top=1)
    ddirty = torch.where(dirty[:, :1].isfinite(), dy, math.nan)
    grads = []
    for xx, dd in ((x, dy), (dirty, ddirty)):
        xx, ww = xx.clone().requires_grad_(True), w.clone().requires_grad_(True)
        grads.append(torch.autograd.grad(F.grouped_linear(xx, ww, offsets), [xx, ww], dd))
    assert torch.equal(grads[0][0][o[big]:o[big + 1]], grads[1][0][o[big]:o[big + 1]])
    assert torch.equal(grads[0][1][big], grads[1][1][big])
    assert bool((grads[1][0][:4] == 0).all()) and bool((grads[1][0][n - 9:] == 0).all())


@pytest.mark.parametrize("relu", [False, True])
def test_large_products_on_misaligned_rows(relu):
    """Rows off the 16-byte boundaries of products large enough to be copied for the tensor cores, gradients included."""
    from spira_b200.nn import functional as F
    n, e, ci, co = 9000, 3, 200, 152
    offsets = some_offsets(n, e, first=2, behind=7)
    base, dbase = whole(n, ci + 3, dtype=torch.bfloat16), whole(n, co + 5, dtype=torch.bfloat16, top=1, seed=4)
    w = whole(e, ci, co, dtype=torch.bfloat16, seed=2).requires_grad_(True)
    out = []
    for x, dy in ((base[:, 1:1 + ci], dbase[:, 3:3 + co]), (base[:, 1:1 + ci].contiguous(), dbase[:, 3:3 + co].contiguous())):
        x = x.detach().requires_grad_(True)
        y = F.grouped_linear(x, w, offsets, relu=relu)
        out.append((y,) + torch.autograd.grad(y, [x, w], dy))
    assert all(torch.equal(a, b) for a, b in zip(*out))


def test_products_nan_passes_the_relu():
    from spira_b200.nn import functional as F
    for ci, co in ((64, 64), (20, 30)):
        x, w = torch.ones(40, ci, dtype=torch.float16, device="cuda"), torch.ones(2, ci, co, dtype=torch.float16, device="cuda")
        x[3, 5] = math.nan
        y = F.grouped_linear(x, -w, torch.tensor([0, 10, 40], dtype=torch.int32, device="cuda"), relu=True)
        assert bool(y[3].isnan().all()) and bool((y[torch.arange(40, device="cuda") != 3] == 0).all())


def test_products_empty():
    from spira_b200.nn import functional as F
    for n, offsets in ((0, [0, 0, 0]), (5, [0, 0, 0]), (5, [5, 5, 5]), (5, [2, 2, 2])):
        x = rand(n, 24, dtype=torch.float16).requires_grad_(True)
        w, b = rand(2, 24, 40, dtype=torch.float16).requires_grad_(True), rand(2, 40, dtype=torch.float16).requires_grad_(True)
        y = F.grouped_linear(x, w, torch.tensor(offsets, dtype=torch.int32, device="cuda"), b, relu=True)
        assert y.shape == (n, 40) and bool((y == 0).all())
        for g, t in zip(torch.autograd.grad(y, [x, w, b], torch.ones_like(y)), (x, w, b)):
            assert g.shape == t.shape and bool((g == 0).all())


@pytest.mark.parametrize("ci,co", [(64, 64), (20, 30)])
def test_products_bad_offsets_stay_inside(ci, co):
    """Offsets that fall, or lie outside the rows, count as the largest before them and as N at most."""
    from spira_b200.nn import functional as F
    n = 300
    x, w = whole(n, ci, dtype=torch.float16).requires_grad_(True), whole(3, ci, co, dtype=torch.float16).requires_grad_(True)
    for bad, good in (([-7, 100, 50, 1 << 30], [0, 100, 100, n]), ([10, 5, 200, 150], [10, 10, 200, 200]), ([1 << 30, 0, 0, 0], [n, n, n, n])):
        o = [torch.tensor(v, dtype=torch.int32, device="cuda") for v in (bad, good)]
        ys = [F.grouped_linear(x, w, v) for v in o]
        gs = [torch.autograd.grad(y, [x, w], torch.ones_like(y)) for y in ys]
        assert torch.equal(ys[0], ys[1]) and all(torch.equal(a, b) for a, b in zip(*gs))


# ------------------------------------------------------------------------------------------------ norms
def plain_norm(x, block, weight, bias, post, post_weight, post_bias, gate, kind, a, s, eps, pre=True):
    def norm(v, w, b):
        c = v - v.mean(1, keepdim=True) if kind == "layer" else v
        h = c / (c.pow(2).mean(1, keepdim=True) + eps).sqrt()
        h = h if w is None else h * w
        return h if b is None else h + b
    if block is None:
        return x, norm(x, weight, bias)
    p = norm(block, post_weight, post_bias) if post else block
    stream = a * x + s * (p if gate is None else gate * p)
    return stream, norm(stream, weight, bias) if pre else None


NORM_SHAPES = [(0, 16), (1, 1), (1, 256), (3, 7), (70, 8), (65, 96), (21, 192), (19, 384), (33, 100), (129, 256), (20, 257), (40, 512), (9, 1000), (7, 1030), (5, 2048), (5, 4096), (3, 5001), (3, 8192)]


@pytest.mark.parametrize("dtype", ANY)
@pytest.mark.parametrize("n,c", NORM_SHAPES)
def test_norm(dtype, n, c):
    from spira_b200.nn import functional as F
    for variant in range(6):
        kind = ("rms", "layer")[variant % 2]
        post, gate_kind = variant in (1, 2, 5), ("none", "channel", "row", "full", "channel", "none")[variant]
        pdtype = torch.float32 if variant in (0, 3, 5) else dtype
        a, s, eps = (1.0, 0.7)[variant % 2], (1.0, 0.25)[variant // 3], 1e-5
        t = dict(x=rand(n, c, dtype=dtype, seed=variant), block=rand(n, c, dtype=dtype, seed=20 + variant),
                 weight=1 + rand(c, scale=0.2), gate=None, bias=None, post_weight=None, post_bias=None)
        if kind == "layer":
            t["bias"] = rand(c, scale=0.2, seed=1)
        if post:
            t["post_weight"] = 1 + rand(c, scale=0.2, seed=2)
            t["post_bias"] = rand(c, scale=0.2, seed=3) if kind == "layer" else None
        for name in ("weight", "bias", "post_weight", "post_bias"):
            t[name] = None if t[name] is None else t[name].to(pdtype)
        if gate_kind == "channel":
            t["gate"] = rand(c, scale=0.5, seed=4).to(pdtype)
        elif gate_kind != "none":
            t["gate"] = rand(n, 1 if gate_kind == "row" else c, dtype=dtype, scale=0.5, seed=5)
        leaves = {k: v.requires_grad_(True) for k, v in t.items() if v is not None}
        x, block, kw = t["x"], t["block"], {k: v for k, v in t.items() if k not in ("x", "block")}
        stream, normed = F.residual_norm(x, block, kind=kind, post=post, residual_scale=a, block_scale=s, eps=eps, **kw)
        ds, dh = rand(n, c, dtype=dtype, seed=6), rand(n, c, dtype=dtype, seed=7)
        got = dict(zip(leaves, torch.autograd.grad([stream, normed], list(leaves.values()), [ds, dh])))
        q = {k: v.detach().double().requires_grad_(True) for k, v in leaves.items()}
        es, eh = plain_norm(q["x"], q["block"], q.get("weight"), q.get("bias"), post, q.get("post_weight"), q.get("post_bias"), q.get("gate"), kind, a, s, eps)
        want = dict(zip(q, torch.autograd.grad([es, eh], list(q.values()), [ds.double(), dh.double()])))
        # sizes: what the cancelling parts of each result add up to.  A row statistic is a sum over the row held by the
        # threads as a tree (at most 40 additions a path), a normalised value takes some ten operations: 128 roundings
        # cover the forward pass, 256 what the backward pass adds to it.
        with torch.no_grad():
            r = 1 / ((es - es.mean(1, keepdim=True) if kind == "layer" else es).pow(2).mean(1, keepdim=True) + eps).sqrt()
            b_in = q["block"]
            rb = 1 / ((b_in - b_in.mean(1, keepdim=True) if kind == "layer" else b_in).pow(2).mean(1, keepdim=True) + eps).sqrt()
            one = torch.ones(c, dtype=torch.float64, device="cuda")
            w, pw = q.get("weight", one).abs(), q.get("post_weight", one).abs()
            p_size = (b_in.abs() + b_in.abs().mean(1, keepdim=True)) * rb if post else b_in.abs()
            p_aff = p_size * pw + q["post_bias"].abs() if "post_bias" in q else p_size * pw if post else p_size
            g = q["gate"].abs() if "gate" in q else torch.ones_like(b_in)
            s_size = a * q["x"].abs() + s * g * p_aff
            hat = (s_size + s_size.mean(1, keepdim=True)) * r
            h_size = hat * w + (q["bias"].abs() if "bias" in q else 0)
            close(stream, es, s_size, 128, "stream")
            close(normed, eh, h_size, 128, "normed")
            u = dh.double().abs() * w
            d_size = ds.double().abs() + r * (u + hat * (u * hat).mean(1, keepdim=True) + u.mean(1, keepdim=True))
            v = s * g * d_size
            u2 = v * pw
            sizes = {"x": a * d_size, "weight": (dh.double().abs() * hat).sum(0), "bias": dh.double().abs().sum(0),
                     "block": rb * (u2 + p_size * (u2 * p_size).mean(1, keepdim=True) + u2.mean(1, keepdim=True)) if post else v,
                     "post_weight": (v * p_size).sum(0), "post_bias": v.sum(0)}
            dg = s * d_size * p_aff
            sizes["gate"] = dg.sum(0) if gate_kind == "channel" else dg.sum(1, keepdim=True) if gate_kind == "row" else dg
            for name in leaves:
                close(got[name], want[name], sizes[name], 256 + (n if want[name].dim() == 1 else 0), f"{variant} d{name}")


@pytest.mark.parametrize("dtype", ANY)
def test_norm_alone_and_without_pre(dtype):
    from spira_b200.nn import functional as F
    x, b = rand(50, 96, dtype=dtype).requires_grad_(True), rand(50, 96, dtype=dtype, seed=1).requires_grad_(True)
    stream, normed = F.residual_norm(x)
    assert stream is x
    dh = rand(50, 96, dtype=dtype, seed=2)
    dx, = torch.autograd.grad(normed, x, dh)
    q = x.detach().double().requires_grad_(True)
    _, want = plain_norm(q, None, None, None, False, None, None, None, "rms", 1, 1, 1e-6)
    wx, = torch.autograd.grad(want, q, dh.double())
    r = 1 / (q.detach().pow(2).mean(1, keepdim=True) + 1e-6).sqrt()
    close(normed, want.detach(), q.detach().abs() * r, 128)
    u, hat = dh.double().abs(), q.detach().abs() * r
    close(dx, wx, r * (u + hat * (u * hat).mean(1, keepdim=True)), 256)
    stream, none = F.residual_norm(x, b, pre=False, residual_scale=0.5)
    assert none is None
    ds = rand(50, 96, dtype=dtype, seed=3)
    gx, gb = torch.autograd.grad(stream, [x, b], ds)
    assert torch.equal(gb, ds) and torch.equal(gx, (0.5 * ds.float()).to(dtype))
    # one output used: the other has no gradient
    stream, normed = F.residual_norm(x, b)
    gx, = torch.autograd.grad(stream, x, ds, retain_graph=True)
    assert torch.equal(gx, ds)
    a1 = torch.autograd.grad(normed, [x, b], dh)
    assert torch.equal(a1[0], a1[1])


def test_norm_strides_alignment_and_odd_rows():
    from spira_b200.nn import functional as F
    base, other = rand(300, 110, dtype=torch.float16), rand(300, 110, dtype=torch.float16, seed=1)
    w = rand(97, seed=2)
    for lo, hi in ((8, 104), (3, 99), (0, 97)):
        x, b = base[:, lo:hi], other[:, lo:hi]
        ww = w[1:97] if hi - lo == 96 else w
        got = F.residual_norm(x, b, weight=ww, post=True, gate=other[:, :1])
        want = F.residual_norm(x.contiguous(), b.contiguous(), weight=ww.clone(), post=True, gate=other[:, :1].contiguous())
        for p, q in zip(got, want):
            size = want[0].double().abs() + want[1].double().abs() + x.double().abs() + b.double().abs() + 3
            close(p, q.double(), size, 1024 * 16, "views")     # (another split of the row sums: one rounding of fp16 apart)
    x = torch.zeros(5, 64, dtype=torch.float16, device="cuda")
    assert bool((F.residual_norm(x)[1] == 0).all()) and bool((F.residual_norm(x, kind="layer")[1] == 0).all())
    x[2] = math.nan
    y = F.residual_norm(x + 1)[1]
    assert bool(y[2].isnan().all()) and bool(y[[0, 1, 3, 4]].isfinite().all())


def test_norm_gradient_against_differences():
    """Directional derivatives in fp32: central differences are off by h^2/6 f''' and 2^-24 |f| / h."""
    from spira_b200.nn import functional as F
    n, c = 12, 40
    t = {k: v.requires_grad_(True) for k, v in dict(x=rand(n, c), block=rand(n, c, seed=1), weight=1 + rand(c, scale=0.2), bias=rand(c, seed=2),
                                                    post_weight=1 + rand(c, scale=0.2, seed=3), post_bias=rand(c, seed=4), gate=rand(c, seed=5)).items()}
    ds, dh = rand(n, c, seed=6), rand(n, c, seed=7)

    def value(q):
        s, h = F.residual_norm(q["x"], q["block"], weight=q["weight"], bias=q["bias"], post=True, post_weight=q["post_weight"], post_bias=q["post_bias"],
                               gate=q["gate"], kind="layer")
        return float((s.double() * ds.double()).sum() + (h.double() * dh.double()).sum())
    s, h = F.residual_norm(t["x"], t["block"], weight=t["weight"], bias=t["bias"], post=True, post_weight=t["post_weight"], post_bias=t["post_bias"],
                           gate=t["gate"], kind="layer")
    grads = dict(zip(t, torch.autograd.grad([s, h], list(t.values()), [ds, dh])))
    step = 2.0 ** -8
    for name in t:
        v = rand(*t[name].shape, seed=11)
        up, down = ({k: (q.detach() + (sign * step * v if k == name else 0)) for k, q in t.items()} for sign in (1, -1))
        slope = (value(up) - value(down)) / (2 * step)
        exact = float((grads[name].double() * v.double()).sum())
        # rounding: n c values of size ~2, each off by ~16 roundings, as independent errors; truncation: 2^-16 / 6 of a third
        # derivative that is ~100 times the slope's parts
        noise = 16 * U32 * 2 * math.sqrt(2 * n * c) * 3 / step
        size = float((grads[name].double().abs() * v.double().abs()).sum())
        assert abs(slope - exact) <= noise + 100 * step * step / 6 * size, (name, slope, exact)


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals():
    from spira_b200.nn import functional as F
    x = rand(6, 8, dtype=torch.float16)
    r = some_routing(6, 4, 2, dead=0.0)
    o = torch.tensor([0, 3, 6], dtype=torch.int32, device="cuda")
    w = rand(2, 8, 16, dtype=torch.float16)
    bad = [(lambda: F.expert_route(x, 9), "top_k"), (lambda: F.expert_route(x, 0), "top_k"), (lambda: F.expert_route(x[0], 1), "logits"),
           (lambda: F.expert_route(x.double(), 1), "logits"), (lambda: F.expert_route(rand(2, 513), 1), "experts"),
           (lambda: F.expert_dispatch(x[:5], r), "dimension 0"), (lambda: F.expert_dispatch(x.double(), r), "feats"),
           (lambda: F.expert_dispatch(x, r._replace(slots=r.slots.long())), "int32"), (lambda: F.expert_combine(x, r), "dimension 0"),
           (lambda: F.expert_combine(rand(12, 8), r._replace(weights=r.weights.half())), "float32"),
           (lambda: F.grouped_linear(x, w.bfloat16(), o), "both"), (lambda: F.grouped_linear(x.float(), w.float(), o), "float16"),
           (lambda: F.grouped_linear(x[:, :7], w, o), "dimension 1"), (lambda: F.grouped_linear(x, w, o.long()), "offsets"),
           (lambda: F.grouped_linear(x, w, o[:2]), "offsets"), (lambda: F.grouped_linear(x, w, o, w[0, :3]), "bias"),
           (lambda: F.grouped_linear(x, w[0], o), "weights"), (lambda: F.residual_norm(x, x[:5]), "block"), (lambda: F.residual_norm(x, x, kind="l2"), "kind"),
           (lambda: F.residual_norm(x, x, eps=0), "eps"), (lambda: F.residual_norm(x, gate=rand(8)), "needs a block"),
           (lambda: F.residual_norm(x, x, gate=rand(7)), "gate"), (lambda: F.residual_norm(x, x, gate=rand(6, 8)), "type"),
           (lambda: F.residual_norm(x, x, weight=rand(8), bias=rand(8, dtype=torch.float16)), "one type"), (lambda: F.residual_norm(x, pre=False), "nothing"),
           (lambda: F.residual_norm(x, x, post_weight=rand(8)), "post=True"), (lambda: F.residual_norm(x, x, weight=rand(8), pre=False), "pre=False"),
           (lambda: F.residual_norm(rand(2, 8193)), "channels"), (lambda: F.residual_norm(x, x, weight=rand(8).double()), "float32")]
    for call, word in bad:
        with pytest.raises(RuntimeError, match=word):
            call()


def test_second_derivatives_are_refused():
    from spira_b200.nn import functional as F
    x = rand(6, 8, dtype=torch.float16).requires_grad_(True)
    w, o = rand(2, 8, 16, dtype=torch.float16), torch.tensor([0, 3, 6], dtype=torch.int32, device="cuda")
    r = some_routing(6, 4, 2, dead=0.0)
    for y in (F.grouped_linear(x, w, o), F.residual_norm(x)[1], F.expert_dispatch(x, r), F.expert_combine(x.repeat(2, 1), r), F.expert_route(x, 2).weights):
        with pytest.raises(RuntimeError, match="once only"):
            torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)


# ------------------------------------------------------------------------------------------------ together
def small_block(dtype=torch.float16, experts=6, c=64):
    import spira_b200 as sp
    from spira_b200 import nn as spnn
    torch.manual_seed(3)
    first, moe, last = spnn.ResidualNorm(c), spnn.SparseExperts(c, 2 * c, experts, top_k=2), spnn.ResidualNorm(c, kind="layer", post=True, gate=True, gate_init=0.5)
    for m in (first, moe, last):
        m.cuda().to(dtype)
    return sp, first, moe, last


def test_block_forward_and_gradients():
    """Norm, experts, gated residual norm on a SparseTensor, against the same formulas in 64 bits on the kernels' choices."""
    sp, first, moe, last = small_block()
    from spira_b200.nn import functional as F
    n, c = 700, 64
    x = sp.SparseTensor(torch.arange(n, dtype=torch.int32, device="cuda"), rand(n, c, dtype=torch.float16))
    mask = torch.rand(n, generator=torch.Generator().manual_seed(1)).cuda() > 0.1
    stream, h = first(x)
    block = moe(h, mask)
    stream, out = last(stream, block)
    assert out._coordinates is x._coordinates and out._features.dtype == torch.float16
    assert bool((block._features[~mask] == 0).all())
    params = [p for m in (first, moe, last) for p in m.parameters()]
    loss_grad = rand(n, c, dtype=torch.float16, seed=9)
    grads = torch.autograd.grad([stream._features, out._features], params, [loss_grad, loss_grad], allow_unused=True)
    # the same in 64 bits
    q = [p.detach().double().requires_grad_(True) for p in params]
    names = [f"{i}.{k}" for i, m in enumerate((first, moe, last)) for k, _ in m.named_parameters()]
    d = dict(zip(names, q))
    xf = x._features.double()
    _, hh = plain_norm(xf, None, d["0.weight"], None, False, None, None, None, "rms", 1, 1, 1e-6)
    with torch.no_grad():
        r = F.expert_route(moe.logits(h._features).masked_fill(~mask[:, None], float("-inf")), 2)
    logits = hh @ d["1.router"]
    chosen = r.experts.clamp_min(0).long()
    w = torch.where((r.experts >= 0), torch.softmax(logits.gather(1, chosen), 1), 0.0)
    bb = torch.zeros(n, c, dtype=torch.float64, device="cuda")
    for e in range(6):
        for j in range(2):
            t = (r.experts[:, j] == e).nonzero()[:, 0]
            z = torch.relu(hh[t] @ d["1.kernel1"][e] + d["1.bias1"][e]) @ d["1.kernel2"][e] + d["1.bias2"][e]
            bb = bb.index_add(0, t, z * w[t, j, None])
    ss, oo = plain_norm(xf, bb, d["2.weight"], d["2.bias"], True, d["2.post_weight"], d["2.post_bias"], d["2.gate"], "layer", 1, 1, 1e-6)
    want = torch.autograd.grad([ss, oo], q, [loss_grad.double()] * 2, allow_unused=True)
    # every tensor between the operators is rounded to fp16 (2^-11 relative) and a chain of five such roundings, amplified by
    # the norms' division, stays below 5 * 4 half steps in the 2-norm
    def off(a, b):
        return float(((a.double() - b).norm() / b.norm().clamp_min(1e-30)).detach())
    assert off(out._features, oo.detach()) < 20 * 2.0 ** -11 and off(stream._features, ss.detach()) < 20 * 2.0 ** -11
    for name, g, e in zip(names, grads, want):
        assert (g is None) == (e is None), name
        if g is not None:
            assert off(g, e) < 40 * 2.0 ** -11, (name, off(g, e))


@pytest.mark.parametrize("renormalize", [True, False])
def test_masked_voxels_reach_nothing(renormalize):
    """What masked voxels hold (NaN, infinities) shows in no result and no gradient: the same bits as with zeros there."""
    import spira_b200 as sp
    from spira_b200 import nn as spnn
    torch.manual_seed(4)
    moe = spnn.SparseExperts(32, 64, 5, top_k=2, renormalize=renormalize).cuda().half()
    n = 300
    mask = torch.rand(n, generator=torch.Generator().manual_seed(2)).cuda() > 0.3
    clean = rand(n, 32, dtype=torch.float16).masked_fill(~mask[:, None], 0.0)
    dirty = clean.clone()
    dirty[~mask] = float("nan")
    dirty[torch.nonzero(~mask)[0, 0]] = float("inf")
    results = []
    for feats in (clean, dirty):
        feats.requires_grad_(True)
        y = moe(sp.SparseTensor(torch.arange(n, dtype=torch.int32, device="cuda"), feats), mask)._features
        results.append([y.detach(), *torch.autograd.grad(y, [feats, *moe.parameters()], rand(n, 32, dtype=torch.float16, seed=7))])
    for a, b in zip(*results):
        assert bool(torch.isfinite(b).all()) and torch.equal(a, b)
    assert not bool(results[1][1][~mask].any())


def test_block_behind_a_sparse_convolution_compiles():
    """The modules as layers of a network: eager, recorded and replayed on another scene, the same bits."""
    import spira_oracle as O  # noqa: F401
    from helpers import surface
    sp, first, moe, last = small_block(c=32)
    from spira_b200 import nn as spnn

    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.conv, self.first, self.moe, self.last = spnn.SparseConv(4, 32, 3).cuda().half(), first, moe, last

        def forward(self, x):
            stream, h = self.first(self.conv(x))
            stream, h = self.last(stream, self.moe(h))
            return [stream, h]
    net = Net().eval()
    net.conv._tunable_config["map_dataflow"] = 0
    cache = spnn.KernelMapCache()
    sp.set_kernel_map_cache(net, cache)
    compiled = None
    for seed in (1, 2):
        c = torch.from_numpy(surface(seed, 3000)).cuda()
        x = sp.SparseTensor(c, rand(len(c), 4, dtype=torch.float16)).order()
        cache.reset()
        cache.add_all_kernel_maps(x._coordinates, [(3, 3, 3)], [(1, 1, 1)] * 2, [], (1, 1, 1), [0])
        with torch.no_grad():
            eager = net(x)
        if compiled is None:
            compiled = sp.compile_model(net, x, cache)
        replayed = compiled(x)
        for a, b in zip(eager, replayed):
            assert torch.equal(a._features, b._features)


@pytest.mark.parametrize("n", [1, 300, 70_000])
@pytest.mark.parametrize("step", [0, 8])
def test_rows_that_overlap(n, step):
    """Broadcast rows (all of them one row) and rows that start inside the one before: the same bits as of dense copies."""
    from spira_b200.nn import functional as F
    c = 64
    base = whole(n * step + c, dtype=torch.float16, top=2)
    lapped = base.as_strided((n, c), (step, 1))
    dense = lapped.contiguous()
    w = whole(3, c, c, dtype=torch.float16, top=1, seed=1)
    o = torch.tensor([0, n // 3, n // 2, n], dtype=torch.int32, device="cuda")
    r = F.expert_route(rand(n, 3), 2)
    dy = whole(n, c, dtype=torch.float16, seed=2)
    for relu in (False, True):
        assert torch.equal(F.grouped_linear(lapped, w, o, relu=relu), F.grouped_linear(dense, w, o, relu=relu))
    assert torch.equal(F.expert_dispatch(lapped, r), F.expert_dispatch(dense, r))
    assert torch.equal(F.expert_route(lapped, 2).experts, F.expert_route(dense, 2).experts)
    for a, b in zip(F.residual_norm(lapped, lapped, gate=lapped), F.residual_norm(dense, dense, gate=dense)):
        assert torch.equal(a, b)
    grads = []
    for x, g in ((lapped, dy), (dense, dy), (dense, lapped)):
        x, v = x.detach(), w.clone().requires_grad_(True)
        x.requires_grad_(True)
        grads.append(torch.autograd.grad(F.grouped_linear(x, v, o, relu=True), [x, v], g))
    grads.append(torch.autograd.grad(F.grouped_linear(x, v, o, relu=True), [x, v], dense))
    for a, b in (grads[0:2], grads[2:4]):
        assert torch.equal(a[1], b[1]) and torch.equal(a[0], b[0])


def test_offsets_past_32_bits():
    """Tensors of more than 2^31 elements: the last rows are what the same rows give on their own."""
    from spira_b200.nn import functional as F
    n, c = 1_060_000, 2048                                   # 2.17e9 elements, 4.3 GB
    tail = 600
    x = whole(1, c, dtype=torch.float16).expand(n, c).contiguous()
    x[-tail:] = whole(tail, c, dtype=torch.float16, seed=1)
    assert x.numel() > 1 << 31
    stream, normed = F.residual_norm(x, x, gate=x)
    want = F.residual_norm(x[-tail:].clone(), x[-tail:].clone(), gate=x[-tail:].clone())
    assert torch.equal(stream[-tail:], want[0]) and torch.equal(normed[-tail:], want[1])
    del stream, normed
    logits = torch.zeros(n, 2, device="cuda")
    logits[1::2, 1] = 1.0
    r = F.expert_route(logits, 1)
    rows = F.expert_dispatch(x, r)
    back = F.expert_combine(rows, r)
    assert torch.equal(back[-tail:], x[-tail:]) and torch.equal(back[:tail], x[:tail])
    del back
    w = whole(2, c, 24, dtype=torch.float16, top=1, seed=2)
    y = F.grouped_linear(rows, w, r.offsets)
    last = rows[-tail:].double() @ w[1].double()             # (sums below 2^24: exact in fp32)
    assert torch.equal(y[-tail:], last.to(torch.float16))
    del rows
    wide = F.grouped_linear(y[:, :8].contiguous(), whole(2, 8, c, dtype=torch.float16, top=1, seed=3), r.offsets)
    assert wide.numel() > 1 << 31
    last = y[-tail:, :8].double() @ whole(2, 8, c, dtype=torch.float16, top=1, seed=3)[1].double()
    assert torch.equal(wide[-tail:], last.to(torch.float16))


# ------------------------------------------------------------------------------------------------ streams, graphs, repetition
def one_pass(x, logits, w1, b1, w2, gate):
    from spira_b200.nn import functional as F
    r = F.expert_route(logits, 2)
    rows = F.grouped_linear(F.expert_dispatch(x, r), w1, r.offsets, b1, relu=True)
    block = F.expert_combine(F.grouped_linear(rows, w2, r.offsets), r)
    return F.residual_norm(x, block, gate=gate, post=True)


def pass_inputs(n=900, c=64, e=5, seed=0):
    return [rand(n, c, dtype=torch.float16, seed=seed), rand(n, e, seed=seed + 1), rand(e, c, 2 * c, dtype=torch.float16, scale=0.1, seed=seed + 2),
            rand(e, 2 * c, dtype=torch.float16, seed=seed + 3), rand(e, 2 * c, c, dtype=torch.float16, scale=0.1, seed=seed + 4), rand(c, dtype=torch.float16, seed=seed + 5)]


def test_same_bits_every_time_and_on_other_streams():
    ins = [t.requires_grad_(True) for t in pass_inputs(20000)]
    d = rand(20000, 64, dtype=torch.float16, seed=8)

    def everything():
        out = one_pass(*ins)
        return list(out) + list(torch.autograd.grad(out, ins, [d, d]))
    first = everything()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = everything()
    third = everything()
    torch.cuda.synchronize()
    for a, b, c in zip(first, second, third):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_threads_without_a_context():
    """The first CUDA call of a thread may be the product's (autograd runs backward passes in a thread of its own)."""
    import threading
    from spira_b200.nn import functional as F
    x, w, o = whole(300, 64, dtype=torch.float16), whole(2, 64, 64, dtype=torch.float16), torch.tensor([0, 100, 300], dtype=torch.int32, device="cuda")
    want = F.grouped_linear(x, w, o)
    got, errors = [], []

    def work():
        try:
            got.append(F.grouped_linear(x, w, o))
        except Exception as e:
            errors.append(e)
    for _ in range(2):
        t = threading.Thread(target=work)
        t.start()
        t.join()
    assert not errors and len(got) == 2 and all(torch.equal(g, want) for g in got)


LIVING_GRAPH = """
import torch
from spira_b200.nn import functional as F
x, o = torch.ones(300, 64, device="cuda", dtype=torch.float16), torch.tensor([0, 100, 300], dtype=torch.int32, device="cuda")
w = torch.ones(2, 64, 64, device="cuda", dtype=torch.float16, requires_grad=True)
d = torch.ones(300, 64, device="cuda", dtype=torch.float16)
alive = F.grouped_linear(x, w, o)
want, = torch.autograd.grad(alive, w, d, retain_graph=True)
before = torch.cuda.current_stream()
graph = torch.cuda.CUDAGraph()
try:
    with torch.cuda.graph(graph):
        got, = torch.autograd.grad(F.grouped_linear(x, w, o), w, d)
    graph.replay()
    assert torch.equal(got, want)
except RuntimeError as e:
    assert "capture" in str(e)
torch.cuda.set_stream(before)
torch.cuda.synchronize()
again, = torch.autograd.grad(F.grouped_linear(x, w, o), w, d)
assert torch.equal(again, want)
print("alive")
"""


def test_capture_beside_a_living_eager_graph_ends_in_an_exception_at_most():
    """Autograd refuses such a capture itself (the leaves' accumulators belong to another stream).  The refusal arrives as an
    exception and the operators work afterwards; in a process of its own, because a failed capture leaves torch's
    stream and allocator in the middle of it."""
    import subprocess
    import sys
    from pathlib import Path
    r = subprocess.run([sys.executable, "-c", LIVING_GRAPH], capture_output=True, text=True, timeout=300, cwd=Path(__file__).resolve().parents[1])
    assert r.returncode == 0 and "alive" in r.stdout, (r.returncode, r.stderr[-2000:])


def test_two_streams_at_once():
    sets = [pass_inputs(6000, seed=s) for s in (0, 100)]
    with torch.no_grad():
        want = [one_pass(*s) for s in sets]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in sets]
        got = [[], []]
        for _ in range(5):
            for i, st in enumerate(streams):
                with torch.cuda.stream(st):
                    got[i].append(one_pass(*sets[i]))
        torch.cuda.synchronize()
    for w, gs in zip(want, got):
        for g in gs:
            assert all(torch.equal(a, b) for a, b in zip(w, g))


def test_two_captured_graphs_share_nothing():
    sets = [pass_inputs(5000, seed=s) for s in (0, 100)]
    graphs, outs = [], []
    with torch.no_grad():
        one_pass(*sets[0])
        torch.cuda.synchronize()
        for s in sets:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                outs.append(one_pass(*s))
            graphs.append(g)
        for s in sets:                                     # new values in the same buffers
            for t, v in zip(s, pass_inputs(5000, seed=777)):
                t.copy_(v)
        sets[1][0].neg_()
        want = [one_pass(*s) for s in sets]
        for _ in range(3):
            for g in graphs:
                g.replay()
        torch.cuda.synchronize()
    for w, o in zip(want, outs):
        assert all(torch.equal(a, b) for a, b in zip(w, o))


def test_captured_training_step():
    """Forward and backward in one graph, leaves and all made on the capturing side stream as torch asks for."""
    ins = [t.requires_grad_(True) for t in pass_inputs(3000)]
    d = rand(3000, 64, dtype=torch.float16, seed=8)

    def step():
        out = one_pass(*ins)
        return torch.autograd.grad(out, ins, [d, d])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        got = step()
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
