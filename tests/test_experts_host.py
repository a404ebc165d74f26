"""CPU: what the expert and norm operators refuse, and the layouts of their descriptors (no CUDA call is made)."""
import ctypes

import pytest
import torch


def test_descriptor_layouts_match_the_header():
    from spira_b200 import _lib
    assert ctypes.sizeof(_lib.GroupedDesc) == 6 * 4 + 3 * 8 + 10 * 8          # the library static_asserts the same sizes
    assert ctypes.sizeof(_lib.NormDesc) == 8 * 4 + 4 * 4 + 6 * 8 + 19 * 8


def test_cpu_tensors_are_refused():
    from spira_b200.nn import functional as F
    x = torch.zeros(4, 8)
    offsets = torch.zeros(3, dtype=torch.int32)
    routing = F.ExpertRouting(torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2, dtype=torch.int32),
                              torch.zeros(8, dtype=torch.int32), offsets)
    for call in (lambda: F.expert_route(x, 2), lambda: F.expert_dispatch(x, routing), lambda: F.expert_combine(torch.zeros(8, 8), routing),
                 lambda: F.grouped_linear(x.half(), torch.zeros(2, 8, 8).half(), offsets), lambda: F.residual_norm(x, x)):
        with pytest.raises(NotImplementedError, match="CUDA"):
            call()


def test_library_refuses_bad_arguments(lib):
    from spira_b200 import _lib
    n = ctypes.c_size_t()
    err = lib.spira_b200_last_error
    assert lib.spira_b200_expert_route_workspace(100000, 513, 2, ctypes.byref(n)) != 0 and b"experts=513" in err()
    assert lib.spira_b200_expert_route_workspace(100000, 8, 9, ctypes.byref(n)) != 0 and b"top_k=9" in err()
    assert lib.spira_b200_expert_route_workspace(-1, 8, 2, ctypes.byref(n)) != 0
    assert lib.spira_b200_expert_route_workspace((1 << 31) // 2, 8, 2, ctypes.byref(n)) != 0 and b"out of range" in err()
    assert lib.spira_b200_expert_route_workspace(100, 8, 2, ctypes.byref(n)) == 0 and n.value == 0
    assert lib.spira_b200_expert_route(None, 7, 1, 8, 8, 2, 1, None, None, None, None, None, None, 0, None) != 0 and b"element type" in err()
    assert lib.spira_b200_expert_route(None, 0, 1, 8, 8, 2, 1, None, None, None, None, None, None, 0, None) != 0 and b"null" in err()
    assert lib.spira_b200_expert_dispatch(None, 0, 4, 8, 8, None, 33, None, 2, None, None) != 0 and b"top_k=33" in err()
    assert lib.spira_b200_expert_combine(None, 0, 4, 8, 8, None, 0, 0, None, 2, None, None) != 0 and b"null" in err()
    assert lib.spira_b200_expert_combine_backward(None, None, 0, 0, 8, 8, 8, None, 0, 0, None, 2, None, 2, None, None, None) == 0   # no rows
    g = _lib.GroupedDesc(dtype=_lib.F32, experts=2, c_in=8, c_out=8, n=4)
    assert lib.spira_b200_grouped_linear(ctypes.byref(g), None, 0, None, None) != 0 and b"neither fp16 nor bf16" in err()
    assert lib.spira_b200_grouped_linear(None, None, 0, None, None) != 0
    assert lib.spira_b200_grouped_linear_backward(ctypes.byref(g), None, 0, None, None) != 0 and b"neither fp16 nor bf16" in err()
    assert lib.spira_b200_grouped_linear_backward_workspace(None, ctypes.byref(n)) != 0
    g.dtype = _lib.F16
    assert lib.spira_b200_grouped_linear(ctypes.byref(g), None, 0, None, None) != 0 and b"null pointer" in err()
    g.experts = 1025
    assert lib.spira_b200_grouped_linear(ctypes.byref(g), None, 0, None, None) != 0 and b"experts=1025" in err()
    g.experts, g.c_in = 2, 0
    assert lib.spira_b200_grouped_linear(ctypes.byref(g), None, 0, None, None) != 0 and b"channels" in err()
    g.c_in, g.offsets = 8, 4096
    assert lib.spira_b200_grouped_linear_backward(ctypes.byref(g), None, 0, None, None) != 0 and b"no gradient" in err()
    g.dweight = 4096
    assert lib.spira_b200_grouped_linear_backward(ctypes.byref(g), None, 0, None, None) != 0 and b"null pointer" in err()
    d = _lib.NormDesc(dtype=_lib.F16, channels=8193, pre=1, eps=1e-6, n=3)
    assert lib.spira_b200_residual_norm(ctypes.byref(d), None) != 0 and b"channels=8193" in err()
    d.channels = 64
    assert lib.spira_b200_residual_norm(ctypes.byref(d), None) != 0 and b"null pointer" in err()
    d.eps = 0.0
    assert lib.spira_b200_residual_norm(ctypes.byref(d), None) != 0 and b"eps" in err()
    d.eps, d.post = 1e-6, 1
    assert lib.spira_b200_residual_norm(ctypes.byref(d), None) != 0 and b"needs a block" in err()
    d.post, d.gate_kind = 0, 4
    assert lib.spira_b200_residual_norm(ctypes.byref(d), None) != 0 and b"gate" in err()


def test_modules_check_their_arguments():
    from spira_b200 import nn as spnn
    with pytest.raises(ValueError, match="top_k"):
        spnn.SparseExperts(16, 32, 4, top_k=5)
    with pytest.raises(ValueError, match="kind"):
        spnn.ResidualNorm(16, kind="batch")
    m = spnn.ResidualNorm(16, kind="layer", post=True, gate=True, gate_init=0.5)
    assert sorted(n for n, _ in m.named_parameters()) == ["bias", "gate", "post_bias", "post_weight", "weight"]
    assert sorted(n for n, _ in spnn.ResidualNorm(16).named_parameters()) == ["weight"]


def test_forward_mode_tangents_are_refused():
    """Any tensor argument may carry one; the refusal comes before everything else, so it needs no device."""
    import torch.autograd.forward_ad as fw
    from spira_b200.nn import functional as F
    x, w, o = torch.zeros(4, 8), torch.zeros(2, 8, 8), torch.zeros(3, dtype=torch.int32)
    routing = F.ExpertRouting(torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), o)
    with fw.dual_level():
        def dual(t):
            return fw.make_dual(t, torch.ones_like(t))
        calls = [lambda: F.expert_route(dual(x), 2), lambda: F.expert_dispatch(dual(x), routing), lambda: F.expert_combine(dual(torch.zeros(8, 8)), routing),
                 lambda: F.expert_combine(torch.zeros(8, 8), routing._replace(weights=dual(routing.weights))), lambda: F.grouped_linear(dual(x), w, o),
                 lambda: F.grouped_linear(x, dual(w), o), lambda: F.grouped_linear(x, w, o, dual(torch.zeros(2, 8))), lambda: F.residual_norm(dual(x)),
                 lambda: F.residual_norm(x, dual(x)), lambda: F.residual_norm(x, weight=dual(x[0])), lambda: F.residual_norm(x, bias=dual(x[0])),
                 lambda: F.residual_norm(x, x, gate=dual(x)), lambda: F.residual_norm(x, x, post=True, post_weight=dual(x[0])),
                 lambda: F.residual_norm(x, x, post=True, post_bias=dual(x[0]))]
        for call in calls:
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        with pytest.raises(NotImplementedError, match="CUDA"):      # (a level without tangents changes nothing)
            F.residual_norm(x)


def test_library_refuses_bad_arguments_of_the_cleared_forms(lib):
    err = lib.spira_b200_last_error
    dispatch, backward = lib.spira_b200_expert_dispatch_cleared, lib.spira_b200_expert_combine_backward_cleared
    assert dispatch(None, 0, 0, 8, 8, None, None, 2, None, None) == 0                      # no rows
    assert dispatch(None, 0, 4, 8, 8, None, None, 2, None, None) != 0 and b"null pointer" in err()
    assert dispatch(None, 0, 4, 8, 8, None, None, 33, None, None) != 0 and b"top_k=33" in err()
    assert dispatch(None, 3, 4, 8, 8, None, None, 2, None, None) != 0 and b"element type" in err()
    assert dispatch(None, 0, 1 << 30, 8, 8, None, None, 2, None, None) != 0 and b"out of range" in err()
    assert dispatch(None, 0, 4, 8, 0, None, None, 2, None, None) != 0 and b"channels" in err()
    assert dispatch(None, 0, 4, -8, 8, None, None, 2, None, None) != 0 and b"stride" in err()
    assert backward(None, None, 0, 0, 8, 8, 8, None, 0, 0, None, None, 2, None, None, None) == 0
    assert backward(None, None, 0, 4, 8, 8, 8, None, 0, 0, None, None, 2, None, None, None) != 0 and b"null pointer" in err()
    assert backward(None, None, 0, 4, 8, 8, 8, None, 0, 0, None, None, 0, None, None, None) != 0 and b"top_k=0" in err()


def test_paths_call_checks_its_arguments(lib):
    from spira_b200 import _lib
    paths, err = (ctypes.c_int32 * 4)(), lib.spira_b200_last_error
    g = _lib.GroupedDesc(dtype=_lib.F16, experts=2, c_in=8, c_out=8, n=0)
    assert lib.spira_b200_grouped_linear_paths(ctypes.byref(g), paths) != 0 and b"no rows" in err()
    g.n, g.offsets = 4, 4096
    assert lib.spira_b200_grouped_linear_paths(ctypes.byref(g), None) != 0 and b"null pointer" in err()
    assert lib.spira_b200_grouped_linear_paths(None, paths) != 0
    g.x_stride, g.c_in = 7, 7
    assert lib.spira_b200_grouped_linear_paths(ctypes.byref(g), paths) == 0 and list(paths) == [0, -1, -1, -1]


def test_pointwise_leaves_tensors_that_do_not_fit_to_the_library_product(monkeypatch):
    """Widths that differ, or a weight that was not moved to the device: None before any launch (the kernel would read outside)."""
    from types import SimpleNamespace
    from spira_b200 import _lib
    from spira_b200.nn.functional import _C

    def device_tensor(*shape, index=0):
        return SimpleNamespace(shape=torch.Size(shape), dtype=torch.float16, is_cuda=True, device=torch.device("cuda", index))
    monkeypatch.setattr(_lib, "load", lambda: pytest.fail("the library was called"))
    weight = device_tensor(64, 8)
    assert _C.pointwise(device_tensor(5, 32), weight, None) is None
    assert _C.pointwise(device_tensor(5, 72), weight, None) is None
    assert _C.pointwise(device_tensor(64), weight, None) is None
    assert _C.pointwise(device_tensor(5, 64), torch.zeros(64, 8, dtype=torch.float16), None) is None
    assert _C.pointwise(device_tensor(5, 64), device_tensor(64, 8, index=1), None) is None
    assert _C.pointwise(device_tensor(5, 64), weight, torch.zeros(8, dtype=torch.float16)) is None
    assert _C.pointwise(device_tensor(5, 64), weight, device_tensor(7)) is None


def test_experts_module_says_which_types_it_runs_in():
    import spira_b200 as sp
    from spira_b200 import nn as spnn
    x, coords = torch.zeros(4, 16), torch.arange(4, dtype=torch.int32)
    for module, feats in ((spnn.SparseExperts(16, 32, 4), x), (spnn.SparseExperts(16, 32, 4), x.half()), (spnn.SparseExperts(16, 32, 4).half(), x),
                          (spnn.SparseExperts(16, 32, 4).half(), x.bfloat16()), (spnn.SparseExperts(16, 32, 4).double(), x.double())):
        with pytest.raises(RuntimeError, match="float16 or bfloat16, module and features alike"):
            module(sp.SparseTensor(coords, feats))
    with pytest.raises(NotImplementedError, match="CUDA"):
        spnn.SparseExperts(16, 32, 4).half()(sp.SparseTensor(coords, x.half()))


def test_traffic_hash_follows_the_includes(tmp_path):
    """A header that a benchmarked kernel starts to include counts towards the hash of its sources; the operators' units do not."""
    import bench
    names = {f.name for f in bench.kernel_sources()}
    assert {"conv.cu", "common.cuh", "ptx.cuh"} <= names and not names & (bench.OTHER_UNITS | {"elem.cuh", "grouped.cuh"})
    for name, text in (("conv.cu", '#include "a.cuh"\n#include <cuda.h>\n'), ("a.cuh", '  #  include "elem.cuh"\n'), ("elem.cuh", '#include "a.cuh"\n'),
                       ("norm.cu", '#include "only.cuh"\n'), ("only.cuh", "")):
        (tmp_path / name).write_text(text)
    assert [f.name for f in bench.kernel_sources(tmp_path)] == ["a.cuh", "conv.cu", "elem.cuh"]
