"""GPU: the expert and norm operators called in ways that a program may call them: from several threads at once, with a routing
that the caller changed, under forward-mode differentiation, on every kernel that the sizes choose between."""
import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

from test_gpu_experts import ANY, HALF, plain_products, rand, whole

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parents[1]


# ------------------------------------------------------------------------------------------------ threads
# Two threads call one function of the library as fast as they can, without Python between the calls.
TWO_THREADS = r"""
#include <atomic>
#include <cstring>
#include <thread>
#include "spira_b200.h"
struct Route { const void *logits; int64_t n; int32_t experts, k; float *weights; int32_t *chosen, *slots, *order, *offsets; };
extern "C" int two_threads(const char *name, void *fn, const char *(*last_error)(void), const void *const *calls, void *const *streams, int32_t *status,
                           int rounds, char *message) {
  std::atomic<int> failed(0), ready(0);
  auto one = [&](int i) -> int {
    if (std::strcmp(name, "norm") == 0)
      return reinterpret_cast<decltype(&spira_b200_residual_norm)>(fn)(static_cast<const spira_b200_norm_desc *>(calls[i]), streams[i]);
    if (std::strcmp(name, "products") == 0)
      return reinterpret_cast<decltype(&spira_b200_grouped_linear)>(fn)(static_cast<const spira_b200_grouped_desc *>(calls[i]), nullptr, 0, status, streams[i]);
    const Route &q = *static_cast<const Route *>(calls[i]);
    return reinterpret_cast<decltype(&spira_b200_expert_route)>(fn)(q.logits, SPIRA_B200_F32, q.n, q.experts, q.experts, q.k, 1, q.weights, q.chosen,
                                                                     q.slots, q.order, q.offsets, nullptr, 0, streams[i]);
  };
  auto work = [&](int i) {
    ++ready;
    while (ready < 2) {}
    for (int r = 0; r < rounds; ++r)
      if (one(i) != 0 && failed++ == 0) std::strncpy(message, last_error(), 255);
  };
  std::thread a(work, 0), b(work, 1);
  a.join();
  b.join();
  return failed;
}
"""


class RouteCall(ctypes.Structure):
    _fields_ = [("logits", ctypes.c_void_p), ("n", ctypes.c_int64), ("experts", ctypes.c_int32), ("k", ctypes.c_int32)] + \
               [(q, ctypes.c_void_p) for q in ("weights", "chosen", "slots", "order", "offsets")]


@pytest.mark.parametrize("kind", ["norm", "products", "routing"])
def test_threads_that_launch_one_kernel_with_different_sizes(kind, tmp_path):
    """Calls of one kernel that take different amounts of shared memory do not disturb each other, and each has its own result."""
    from spira_b200 import _lib
    from spira_b200.nn import functional as F
    from spira_b200.nn.functional import _C, experts, norms
    (tmp_path / "threads.cpp").write_text(TWO_THREADS)
    subprocess.run(["g++", "-O2", "-shared", "-fPIC", "-pthread", "-I", str(ROOT / "include"), "-o", str(tmp_path / "threads.so"),
                    str(tmp_path / "threads.cpp")], check=True)
    run = ctypes.CDLL(str(tmp_path / "threads.so")).two_threads
    lib, calls, keep, pairs = _lib.load(), [], [], []
    if kind == "norm":                       # rows of three and of two tensors on their way
        fn, x = lib.spira_b200_residual_norm, rand(64, 96, dtype=torch.float16)
        for gate, gate_kind in ((x, norms.GATE_FULL), (None, norms.GATE_NONE)):
            out = torch.empty_like(x), torch.empty_like(x)
            spec = norms._Spec(False, False, True, False, gate_kind, 1.0, 1.0, 1e-6)
            calls.append(ctypes.create_string_buffer(norms._desc(spec, x, (x, gate, None, None, None, None), *out)))
            pairs.append((out, F.residual_norm(x, x, gate=gate)))
    elif kind == "products":                 # few and many groups, narrow and wide tiles
        fn = lib.spira_b200_grouped_linear
        for e, c in ((2, 64), (900, 256)):
            x, w, y = rand(64, 64, dtype=torch.float16), rand(e, 64, c, dtype=torch.float16), torch.empty(64, c, dtype=torch.float16, device="cuda")
            o = torch.full((e + 1,), 64, dtype=torch.int32, device="cuda")
            o[0] = 0
            calls.append(ctypes.create_string_buffer(experts._grouped_desc(64, w, o, 0, x, None, y=y)))
            pairs.append(((y,), (F.grouped_linear(x, w, o),)))
            keep.append((x, w, o))
    else:                                    # different numbers of experts and choices
        fn = lib.spira_b200_expert_route
        for e, k in ((512, 32), (400, 2)):
            logits = rand(16, e)
            want = F.expert_route(logits, k)
            got = [torch.empty_like(t) for t in want]
            calls.append(RouteCall(logits.data_ptr(), 16, e, k, *(t.data_ptr() for t in got)))
            pairs.append((got, want))
            keep.append(logits)
    streams = [torch.cuda.Stream() for _ in calls]
    status, message = _C.status_word(torch.device("cuda", torch.cuda.current_device())), ctypes.create_string_buffer(256)
    torch.cuda.synchronize()
    failed = run(kind.encode(), ctypes.cast(fn, ctypes.c_void_p), ctypes.cast(lib.spira_b200_last_error, ctypes.c_void_p),
                 (ctypes.c_void_p * 2)(*(ctypes.addressof(c) for c in calls)), (ctypes.c_void_p * 2)(*(s.cuda_stream for s in streams)),
                 ctypes.c_void_p(status.data_ptr()), 10000, message)
    torch.cuda.synchronize()
    assert failed == 0, (failed, message.value)
    for got, want in pairs:
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------------------------------------------------ forward mode
def test_forward_mode_tangents_are_refused():
    """Inputs with a tangent, and gradients with one on their way back, are refused; a level without tangents changes nothing."""
    import torch.autograd.forward_ad as fw
    from spira_b200.nn import functional as F
    x, w = rand(6, 8, dtype=torch.float16).requires_grad_(True), rand(2, 8, 8, dtype=torch.float16)
    o = torch.tensor([0, 3, 6], dtype=torch.int32, device="cuda")
    r = F.expert_route(rand(6, 4), 2)
    calls = [lambda t: F.expert_route(t, 2).weights, lambda t: F.expert_dispatch(t, r), lambda t: F.expert_combine(t.repeat(2, 1), r),
             lambda t: F.grouped_linear(t, w, o), lambda t: F.residual_norm(t)[1], lambda t: F.residual_norm(t, t, pre=False)[0]]
    for call in calls:
        y = call(x)
        want, = torch.autograd.grad(y, x, torch.ones_like(y), retain_graph=True)
        with fw.dual_level():
            for t in (fw.make_dual(x.detach(), torch.ones_like(x)), fw.make_dual(x, torch.ones_like(x))):
                with pytest.raises(RuntimeError):
                    call(t)
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y, x, fw.make_dual(torch.ones_like(y), torch.ones_like(y)), retain_graph=True)
            assert torch.equal(call(x.detach()), y)
            got, = torch.autograd.grad(y, x, torch.ones_like(y), retain_graph=True)
        assert torch.equal(got, want)


# ------------------------------------------------------------------------------------------------ a routing that the caller changed
def stale_memory(n, c, dtype):
    """Leaves NaN in the memory that the next tensors of this size get."""
    t = [torch.full((n, c), float("nan"), dtype=dtype, device="cuda") for _ in range(6)]
    torch.cuda.synchronize()
    del t


@pytest.mark.parametrize("dtype", ANY)
@pytest.mark.parametrize("n,c,e,k", [(1, 8, 4, 2), (17, 33, 5, 3), (700, 96, 8, 2), (90, 1028, 9, 4), (3000, 7, 16, 2)])
def test_rows_that_no_slot_names_are_zero(dtype, n, c, e, k):
    """Pairs taken out of a routing, places exchanged, an order that is older than the slots, senseless or absent: rows and
    gradients are those of the slots, and zero where there is none."""
    from spira_b200.nn import functional as F
    logits = rand(n, e)
    if n > 1:
        logits[n // 2:n // 2 + n // 8] = float("-inf")
    r = F.expert_route(logits, k)
    g = torch.Generator().manual_seed(n + c)
    dropped = r.slots.masked_fill((torch.rand(n, k, generator=g) < 0.2).cuda(), -1)
    none = torch.full_like(r.slots, -1)
    shuffle = torch.randperm(n * k, generator=g).int().cuda()
    moved = torch.where(r.slots >= 0, shuffle[r.slots.clamp_min(0).long()], -1)           # (places that the order does not know)
    odd = torch.randint(-5, 2 * n * k, (n * k,), generator=g).int().cuda()
    x, y = whole(n, c, dtype=dtype, seed=1).requires_grad_(True), whole(n * k, c, dtype=dtype, top=8, seed=2).requires_grad_(True)
    w = (2.0 ** -torch.randint(0, 4, (n, k), device="cuda").float()).requires_grad_(True)
    drows, dout = whole(n * k, c, dtype=dtype, seed=3), whole(n, c, dtype=dtype, seed=4)
    for slots in (r.slots, dropped, none, moved, moved.masked_fill(dropped < 0, -1)):
        for order in (r.order, odd, torch.full_like(r.order, -1), None, r.order[:-1], r.order.long()):
            q = r._replace(slots=slots, weights=w, order=order)
            stale_memory(n * k, c, dtype)
            rows, out = F.expert_dispatch(x, q), F.expert_combine(y, q)
            stale_memory(n * k, c, dtype)
            dx, dy, dw = torch.autograd.grad([rows, out], [x, y, w], [drows, dout])
            want_rows, want_out = torch.zeros(n * k, c, dtype=torch.float64, device="cuda"), torch.zeros(n, c, dtype=torch.float64, device="cuda")
            want_dx, want_dy, want_dw = torch.zeros_like(want_out), torch.zeros_like(want_rows), torch.zeros(n, k, dtype=torch.float64, device="cuda")
            for j in range(k):
                t = (slots[:, j] >= 0).nonzero()[:, 0]
                s = slots[t, j].long()
                want_rows[s] = x.detach()[t].double()
                want_out[t] += w.detach()[t, j, None].double() * y.detach()[s].double()
                want_dx[t] += drows[s].double()
                want_dy[s] = w.detach()[t, j, None].double() * dout[t].double()
                want_dw[t, j] = (y.detach()[s].double() * dout[t].double()).sum(1)
            # whole numbers and powers of two: every fp32 sum is exact
            for got, want in ((rows, want_rows), (out, want_out), (dx, want_dx), (dy, want_dy), (dw, want_dw)):
                assert torch.equal(got, want.to(got.dtype))


def test_capacity_limit_reaches_the_products():
    """An expert's pairs behind its capacity taken out by their slots: the products and their gradients are those of the kept rows."""
    from spira_b200.nn import functional as F
    n, c, e, k, room = 900, 64, 4, 2, 300
    r = F.expert_route(rand(n, e), k)
    x, w = whole(n, c, dtype=torch.float16).requires_grad_(True), whole(e, c, c, dtype=torch.float16, top=1, seed=1).requires_grad_(True)
    first = r.offsets[:-1].long()[r.experts.long()]
    slots = r.slots.masked_fill(r.slots - first >= room, -1)
    assert int((slots < 0).sum()) > 100
    stale_memory(n * k, c, torch.float16)
    rows = F.expert_dispatch(x, r._replace(slots=slots))
    stale_memory(n * k, c, torch.float16)
    y = F.expert_combine(F.grouped_linear(rows, w, r.offsets), r._replace(slots=slots, weights=torch.ones_like(r.weights)))
    d = whole(n, c, dtype=torch.float16, top=1, seed=2)
    dx, dw = torch.autograd.grad(y, [x, w], d)
    want, q, v = torch.zeros(n, c, dtype=torch.float64, device="cuda"), x.detach().double(), w.detach().double()
    want_dx, want_dw = torch.zeros_like(q), torch.zeros_like(v)
    for t, j in (slots >= 0).nonzero().tolist():
        i = int(r.experts[t, j])
        want[t] += (q[t] @ v[i]).half().double()
        want_dx[t] += (v[i] @ d[t].double()).half().double()
        want_dw[i] += q[t, :, None] * d[t].double()
    assert torch.equal(y, want.half()) and torch.equal(dx, want_dx.half()) and torch.equal(dw, want_dw.half())


@pytest.mark.parametrize("c", [96, 33])
def test_library_forms_for_complete_routings(c):
    """The calls without a clear: for slots as the routing made them, rows behind the last place are cleared by the call itself."""
    from spira_b200 import _lib
    from spira_b200.nn import functional as F
    n, k = 700, 2
    logits = rand(n, 8)
    logits[100:180] = float("-inf")
    r = F.expert_route(logits, k)
    x, y, dout = rand(n, c, dtype=torch.float16), rand(n * k, c, dtype=torch.float16, seed=1).requires_grad_(True), rand(n, c, dtype=torch.float16, seed=2)
    w = r.weights.clone().requires_grad_(True)
    dy, dw = torch.autograd.grad(F.expert_combine(y, r._replace(weights=w)), [y, w], dout)
    rows, drows, dweights = torch.full((n * k, c), float("nan"), dtype=torch.float16, device="cuda"), torch.full_like(y, float("nan")), torch.empty_like(w)
    stream = torch.cuda.current_stream().cuda_stream
    _lib.call("spira_b200_expert_dispatch", x.data_ptr(), _lib.F16, n, c, c, r.slots.data_ptr(), k, r.offsets.data_ptr(), 8, rows.data_ptr(), stream)
    _lib.call("spira_b200_expert_combine_backward", y.data_ptr(), dout.data_ptr(), _lib.F16, n, c, c, c, w.data_ptr(), k, 1, r.slots.data_ptr(), k,
              r.offsets.data_ptr(), 8, drows.data_ptr(), dweights.data_ptr(), stream)
    assert torch.equal(rows, F.expert_dispatch(x, r)) and torch.equal(drows, dy) and torch.equal(dweights, dw)


# ------------------------------------------------------------------------------------------------ bounded waits
@pytest.mark.parametrize("c_in,c_out", [(256, 512), (64, 512)])
def test_a_long_group_does_not_run_out_of_a_bounded_wait(c_in, c_out):
    """All rows in one of many groups: the weight gradient is one sum over 10^6 rows, which takes several times the limit set here.
    (256 channels run on pairs of CTAs.)"""
    from spira_b200.nn import functional as F
    from spira_b200.nn.functional import _C
    n, e = 1_000_000, 160
    x, dy = whole(n, c_in, dtype=torch.bfloat16, top=1), whole(n, c_out, dtype=torch.bfloat16, top=1, seed=1)
    w = whole(e, c_in, c_out, dtype=torch.bfloat16, top=1, seed=2).requires_grad_(True)
    offsets = torch.full((e + 1,), n, dtype=torch.int32, device="cuda")
    offsets[:3] = 0
    y = F.grouped_linear(x, w, offsets)
    _C.check_status()
    default = _C.get_option("wait_limit_us")
    _C.set_option("wait_limit_us", 1000)
    try:
        dw, = torch.autograd.grad(y, w, dy)
        torch.cuda.synchronize()
    finally:
        _C.set_option("wait_limit_us", default)
    _C.check_status()
    want = torch.zeros(c_in, c_out, dtype=torch.float64, device="cuda")
    for part in range(0, n, 250_000):
        want += x[part:part + 250_000].double().T @ dy[part:part + 250_000].double()
    assert torch.equal(dw[2], want.to(torch.bfloat16))
    assert not bool(dw[:2].any()) and not bool(dw[3:].any())


# ------------------------------------------------------------------------------------------------ what the ReLU lets through
@pytest.mark.parametrize("ci,co", [(64, 64), (20, 30), (33, 72), (200, 152)])
def test_relu_gradient_goes_by_the_unrounded_value(ci, co):
    """Positive values that round to zero in fp16 let the gradient through on every kernel, as max(z, 0) does before its rounding."""
    from spira_b200.nn import functional as F
    n = 40
    sign = torch.where(torch.arange(n, device="cuda") % 3 == 0, -1.0, 1.0)
    x = (2.0 ** -14 * sign[:, None].expand(n, ci)).half().requires_grad_(True)
    w = torch.full((2, ci, co), 2.0 ** -21, device="cuda").half().requires_grad_(True)         # (a subnormal: ci 2^-35 rounds to zero)
    o = torch.tensor([0, 10, n - 1], dtype=torch.int32, device="cuda")
    b = torch.zeros(2, co, dtype=torch.float16, device="cuda").requires_grad_(True)
    y = F.grouped_linear(x, w, o, b, relu=True)
    assert not bool(y.any())
    dx, dw, db = torch.autograd.grad(y, [x, w, b], torch.ones_like(y))
    live = (sign > 0) & (torch.arange(n, device="cuda") < n - 1)
    assert torch.equal(dx, torch.where(live[:, None], float(co) * 2.0 ** -21, 0.0).half().expand(n, ci))
    counts = torch.stack([live[:10].sum(), live[10:].sum()])
    assert torch.equal(db, counts[:, None].half().expand(2, co)) and torch.equal(dw, (counts[:, None, None] * 2.0 ** -14).half().expand(2, ci, co))


@pytest.mark.parametrize("ci,co", [(64, 64), (20, 30)])
def test_library_backward_without_a_mask_goes_by_the_result(ci, co):
    """A caller of the library that kept y and no mask: y > 0 says what the ReLU let through."""
    from spira_b200 import _lib
    from spira_b200.nn import functional as F
    from spira_b200.nn.functional import experts
    n = 300
    o = torch.tensor([3, 100, 290], dtype=torch.int32, device="cuda")
    x, w, dy = whole(n, ci, dtype=torch.float16), whole(2, ci, co, dtype=torch.float16, seed=1), whole(n, co, dtype=torch.float16, top=1, seed=2)
    xg, wg = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y = F.grouped_linear(xg, wg, o, relu=True)
    want = torch.autograd.grad(y, [xg, wg], dy)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty(2, co, dtype=torch.float16, device="cuda")
    desc = experts._grouped_desc(n, w, o, 1, x, None, dy, y.detach(), None, dx, dw, db)
    experts._with_workspace(x.get_device(), x, "spira_b200_grouped_linear_backward", desc, experts._status(x.get_device()))
    dz = torch.where(y.detach() > 0, dy, 0.0).double()
    assert torch.equal(dx, want[0]) and torch.equal(dw, want[1]) and torch.equal(db, torch.stack([dz[3:100].sum(0), dz[100:290].sum(0)]).half())


# ------------------------------------------------------------------------------------------------ every kernel the sizes choose between
def cut(n, e, seed, first=0, behind=0, empty=(), most=0.0):
    """Offsets of uneven groups: random cuts, some groups empty, a share `most` of the rows in group 1."""
    g = torch.Generator().manual_seed(seed)
    share = torch.rand(e, generator=g) + 0.05
    share[list(empty)] = 0.0
    share = share / share.sum() * (1 - most)
    share[1] += most
    ends = first + ((n - first - behind) * share.cumsum(0)).round().long()
    ends[-1] = n - behind
    return torch.cat([torch.tensor([first]), ends]).to(torch.int32).cuda()


GENERAL, SINGLE, PAIR = 0, 1, 2
#         rows    groups  c_in  c_out  forward dx      dW      rows of a unit of dW: whole groups or pieces
PATHS = [(40000,  16,     512,  2048,  PAIR,   PAIR,   PAIR,   "whole"),       # long reductions: staged stores forward, direct ones in dx
         (20003,  7,      520,  1992,  PAIR,   PAIR,   PAIR,   "whole"),       # channels and rows that no tile divides, direct stores forward
         (24001,  20,     1992, 520,   PAIR,   PAIR,   PAIR,   "whole"),
         (20000,  80,     136,  264,   SINGLE, SINGLE, SINGLE, "whole"),       # more groups than are sorted by length
         (24007,  80,     136,  264,   SINGLE, SINGLE, PAIR,   "whole"),
         (9000,   50,     128,  520,   SINGLE, SINGLE, SINGLE, "whole"),       # sorted by length: 50 x 3 tiles fill 148 SMs
         (9000,   40,     128,  520,   SINGLE, SINGLE, SINGLE, "pieces"),      # 40 x 3 do not
         (30001,  2,      200,  136,   SINGLE, SINGLE, PAIR,   "pieces"),
         (9001,   5,      96,   192,   SINGLE, SINGLE, SINGLE, "pieces"),
         (500,    3,      33,   70,    GENERAL, GENERAL, GENERAL, "pieces"),
         (500,    90,     65,   70,    GENERAL, GENERAL, GENERAL, "whole")]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("n,e,ci,co,forward,dx,dw,unit", PATHS)
def test_products_exact_on_every_path(dtype, n, e, ci, co, forward, dx, dw, unit):
    """Whole numbers on uneven, empty and dominating groups, with and without bias and ReLU: the bits of the 64-bit values; and the
    sizes take the kernels that the list says."""
    from spira_b200 import _lib
    from spira_b200.nn import functional as F
    from spira_b200.nn.functional import experts
    x, w, b = whole(n, ci, dtype=dtype, seed=1), whole(e, ci, co, dtype=dtype, seed=2), whole(e, co, dtype=dtype, seed=3)
    dy = whole(n, co, dtype=dtype, top=1, seed=4)
    paths = (ctypes.c_int32 * 4)()
    _lib.call("spira_b200_grouped_linear_paths", experts._grouped_desc(n, w, torch.zeros(e + 1, dtype=torch.int32, device="cuda"), 1, x, b, dy, None, None, x, w, b), paths)
    assert list(paths)[:3] == [forward, dx, dw] and (paths[3] == 0) == (unit == "whole"), list(paths)
    variants = [(cut(n, e, 1, first=3, behind=5, empty=(0, e // 2)), True, True), (cut(n, e, 2, behind=1, empty=(e - 1,), most=0.8), False, False),
                (cut(n, e, 3, empty=(0,), most=0.97), True, False)]
    for offsets, bias, relu in variants:
        leaves = [t.clone().requires_grad_(True) for t in ([x, w, b] if bias else [x, w])]
        y = F.grouped_linear(leaves[0], leaves[1], offsets, leaves[2] if bias else None, relu=relu)
        grads = torch.autograd.grad(y, leaves, dy)
        want = plain_products(x, w, offsets, b if bias else None, relu, dy, y.detach())
        for name, got, ref in zip(("y", "dx", "dw", "db"), (y,) + grads, want):
            assert torch.equal(got, ref.to(dtype)), (name, bias, relu, float((got.double() - ref).abs().max()))


# ------------------------------------------------------------------------------------------------ launch counts
def test_launches_are_counted():
    """The counter against the number of kernels each call is made of."""
    from spira_b200 import _lib
    from spira_b200.nn import functional as F

    def count(call, *args, **kw):
        before = _lib.launches()
        out = call(*args, **kw)
        return _lib.launches() - before, out
    few, many = rand(8, 8).requires_grad_(True), rand(5000, 8)
    one, r = count(F.expert_route, few, 2)
    assert one == 1 and count(torch.autograd.grad, r.weights, few, torch.ones_like(r.weights))[0] == 1
    two, r = count(F.expert_route, many, 2)
    assert two == 2
    x, y, w = rand(5000, 64, dtype=torch.float16), rand(10000, 64, dtype=torch.float16), r.weights.clone().requires_grad_(True)
    n, rows = count(F.expert_dispatch, x.requires_grad_(True), r)
    assert n == 2 and count(torch.autograd.grad, rows, x, rows.detach())[0] == 1                              # clear and write; sums
    # (a function computes the gradients of all inputs that asked for one when it was called)
    n, out = count(F.expert_combine, y, r._replace(weights=w))
    assert n == 1 and count(torch.autograd.grad, out, w, out.detach())[0] == 1                                # no rows to clear
    n, out = count(F.expert_combine, y.requires_grad_(True), r)
    assert n == 1 and count(torch.autograd.grad, out, y, out.detach())[0] == 2
    v, b = rand(8, 64, 64, dtype=torch.float16).requires_grad_(True), rand(8, 64, dtype=torch.float16).requires_grad_(True)
    n, z = count(F.grouped_linear, y, v, r.offsets, b, relu=True)
    assert n == 1 and count(torch.autograd.grad, z, [y, v, b], z.detach())[0] == 5                            # dz, db, dx, dW in pieces, their sum
    n, z = count(F.grouped_linear, y, v.detach(), r.offsets)
    assert n == 1 and count(torch.autograd.grad, z, y, z.detach())[0] == 1
    base, u = rand(9000, 203, dtype=torch.float16), rand(3, 200, 151, dtype=torch.float16)
    o = torch.tensor([0, 3000, 4000, 9000], dtype=torch.int32, device="cuda")
    assert count(F.grouped_linear, base[:, 1:201], u, o)[0] == 4                                              # copies of x and W, product, copy of y
    weight = rand(64).requires_grad_(True)
    n, (_, h) = count(F.residual_norm, x, weight=weight.detach())
    assert n == 1 and count(torch.autograd.grad, h, x, h.detach())[0] == 1
    n, (_, h) = count(F.residual_norm, x, weight=weight)
    assert n == 1 and count(torch.autograd.grad, h, [x, weight], h.detach())[0] == 2


# ------------------------------------------------------------------------------------------------ the modules
def test_router_refuses_tensors_that_do_not_fit():
    """Features of another width, and weights that were not moved to the device, end in an error and not in a kernel."""
    import spira_b200 as sp
    from spira_b200 import nn as spnn
    moe = spnn.SparseExperts(64, 128, 8).cuda().half()
    n = 300
    coords = torch.arange(n, dtype=torch.int32, device="cuda")
    for c in (32, 72):
        with torch.no_grad(), pytest.raises(RuntimeError):
            moe(sp.SparseTensor(coords, rand(n, c, dtype=torch.float16)))
    with torch.no_grad(), pytest.raises(RuntimeError):
        spnn.SparseExperts(64, 128, 8).half()(sp.SparseTensor(coords, rand(n, 64, dtype=torch.float16)))
    with torch.no_grad():
        x = rand(n, 64, dtype=torch.float16)
        y = moe(sp.SparseTensor(coords, x))._features
        head = spnn.SparseConv(64, 8, 1, bias=True).cuda().half()
        z = head(sp.SparseTensor(coords, x))._features
        with pytest.raises(RuntimeError):
            head(sp.SparseTensor(coords, rand(n, 32, dtype=torch.float16)))
    assert bool(y.isfinite().all()) and bool(z.isfinite().all())
    torch.cuda.synchronize()


def test_the_readme_runs():
    """Its Python blocks, one after the other, on a small scene; the modules of the second one train."""
    import re
    from helpers import surface
    blocks = re.findall(r"```python\n(.*?)```", (ROOT / "README.md").read_text(), flags=re.S)
    assert len(blocks) >= 2 and "SparseExperts" in blocks[1]
    coords = torch.from_numpy(surface(3, 3000)).cuda()
    names = {"coords_int32_cuda": coords, "feats_fp16_cuda": rand(len(coords), 4, dtype=torch.float16)}
    for block in blocks:
        exec(block, names)
    stream, h = names["stream"]._features, names["h"]._features
    assert stream.shape == h.shape == (len(coords), 96) and bool(h.isfinite().all())
    h.float().square().mean().backward()
    assert all(p.grad is not None and bool(p.grad.isfinite().all()) for m in ("moe", "last") for p in names[m].parameters())


def test_few_rows_are_cleared_and_written_in_one_launch():
    """21 rows of 96 channels are the work of one CTA (256 pieces of 16 bytes), 22 are not; the rows are right on both sides."""
    from spira_b200 import _lib
    from spira_b200.nn import functional as F
    c, k = 96, 2
    for n, launches in ((1, 1), (21, 1), (22, 2)):
        r = F.expert_route(rand(n, 4), k)
        slots = r.slots.clone()
        slots[n // 2, 0] = -1
        x = whole(n, c, dtype=torch.float16)
        stale_memory(n * k, c, torch.float16)
        before = _lib.launches()
        rows = F.expert_dispatch(x, r._replace(slots=slots))
        assert _lib.launches() - before == launches
        want = torch.zeros_like(rows)
        for j in range(k):
            t = (slots[:, j] >= 0).nonzero()[:, 0]
            want[slots[t, j].long()] = x[t]
        assert torch.equal(rows, want)
