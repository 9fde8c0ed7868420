"""Refusals of the panel operators (routing, experts' products, global norm): wrong types, shapes, layouts, devices and sizes raise before anything reaches a
GPU, in the Python face (ValueError) and at the C entry points (status 6)."""
import ctypes as C

import pytest
import torch

from spla_amd import _lib, kernels

INVALID = 6


def _plan(rows=4, k=2, experts=3):
    plan = kernels.RoutePlan.__new__(kernels.RoutePlan)  # a plan of CPU tensors: what the checks look at, without a GPU
    plan.offsets = torch.zeros(experts + 1, dtype=torch.int32)
    plan.order = torch.zeros(rows * k, dtype=torch.int32)
    plan.place = torch.zeros(rows, k, dtype=torch.int32)
    plan.n_rows, plan.per_row, plan.n_places, plan.n_experts, plan.device = rows, k, rows * k, experts, plan.offsets.device
    return plan


@pytest.mark.parametrize("experts,n", [
    (torch.zeros(4, 2, dtype=torch.int64), 3),       # type
    (torch.zeros(8, dtype=torch.int32), 3),          # one axis
    (torch.zeros(4, 2, dtype=torch.int32), 3),       # not on the GPU
    ([[0, 1]], 3),                                   # not a tensor
])
def test_sort_refuses(experts, n):
    with pytest.raises(ValueError):
        kernels.route_sort(experts, n)


def test_plan_refuses_mismatched_arrays():
    with pytest.raises(ValueError):
        kernels.RoutePlan(torch.zeros(4, dtype=torch.int32), torch.zeros(7, dtype=torch.int32), torch.zeros(4, 2, dtype=torch.int32))


@pytest.mark.parametrize("call", [
    lambda p: kernels.route_rows(p, torch.zeros(4, 8, dtype=torch.float64)),
    lambda p: kernels.route_rows(p, torch.zeros(5, 8)),
    lambda p: kernels.route_rows(p, torch.zeros(4, 2, 4)),
    lambda p: kernels.route_rows(p, torch.zeros(4, 8)),  # not on the GPU
    lambda p: kernels.route_back(p, torch.zeros(4, 8)),
    lambda p: kernels.route_back(p, torch.zeros(8, 8, dtype=torch.int32)),
    lambda p: kernels.route_back_grad(p, torch.zeros(8, 8), torch.zeros(4, 2), torch.zeros(4, 7)),
    lambda p: kernels.expert_product(p, torch.zeros(8, 5), torch.zeros(2, 7, 5)),
    lambda p: kernels.expert_product(p, torch.zeros(8, 5), torch.zeros(3, 7, 5, dtype=torch.float16)),
    lambda p: kernels.expert_product(p, torch.zeros(8, 5), torch.zeros(3, 7, 0)),
    lambda p: kernels.expert_product_grad(p, torch.zeros(8, 5), torch.zeros(3, 7, 5), torch.zeros(8, 6)),
    lambda p: kernels.global_norm([]),
    lambda p: kernels.global_norm([torch.zeros(3)]),
    lambda p: kernels.global_norm([torch.zeros(3, dtype=torch.int32)]),
    lambda p: kernels.clip_global_norm([torch.zeros(3)], 1.0, out=[]),
    lambda p: kernels.clip_global_norm([], 1.0),
])
def test_panel_calls_refuse(call):
    with pytest.raises(ValueError):
        call(_plan())


def _fails(name, *args):
    with pytest.raises(_lib.SplaHipError) as e:
        _lib.call(name, *args)
    assert e.value.status == INVALID, e.value


def test_c_entries_refuse():
    a = (C.c_uint32 * 64)()
    p = C.cast(a, C.c_void_p)  # never dereferenced: the checks come first
    big = 1 << 20
    _fails("splahip_route_sort", 4, 0, 3, p, p, p, p, p, big, None)           # no entry per row
    _fails("splahip_route_sort", 4, 2, 0, p, p, p, p, p, big, None)           # no expert
    _fails("splahip_route_sort", 4, 2, 2049, p, p, p, p, p, big, None)        # too many experts
    _fails("splahip_route_sort", 1 << 30, 2, 3, p, p, p, p, p, big, None)     # 2^31 entries
    _fails("splahip_route_sort", 4, 2, 3, None, p, p, p, p, big, None)        # null
    _fails("splahip_route_sort", 1 << 16, 2, 3, p, p, p, p, p, 8, None)       # workspace
    _fails("splahip_route_sort", 1 << 16, 2, 3, p, p, p, p, None, big, None)  # no workspace
    _fails("splahip_route_rows", 3, 4, 2, 3, 8, p, p, None, p, p, None)       # panel type
    _fails("splahip_route_rows", 0, 4, 2, 3, 1 << 30, p, p, None, p, p, None)  # width
    _fails("splahip_route_back", 0, 4, 2, 8, p, None, None, p, None)          # null
    _fails("splahip_route_back_grad", 0, 4, 2, 3, 8, p, p, None, p, p, p, p, None)  # no weights
    for name, more in (("splahip_expert_product", ()), ("splahip_expert_product_dx", ()), ("splahip_expert_product_dw", (p, big))):
        _fails(name, 7, 8, 3, 4, 4, p, p, p, p, *more, None)
        _fails(name, 0, 8, 0, 4, 4, p, p, p, p, *more, None)
        _fails(name, 0, 8, 3, 0, 4, p, p, p, p, *more, None)
        _fails(name, 0, 8, 3, 4, 1 << 21, p, p, p, p, *more, None)
        _fails(name, 0, 8, 3, 4, 4, None, p, p, p, *more, None)
        _fails(name, 0, 1 << 31, 3, 4, 4, p, p, p, p, *more, None)
    need = _lib.call("splahip_expert_product_dw_workspace", 0, 20000, 2, 40, 56)
    assert need >= 2 * 2 * 40 * 56 * 4
    _fails("splahip_expert_product_dw", 0, 20000, 2, 40, 56, p, p, p, p, p, need - 1, None)
    _fails("splahip_expert_product_dw", 0, 20000, 2, 40, 56, p, p, p, p, None, need, None)


def test_clip_refuses_overlaps_and_limits():
    base = 1 << 40  # addresses that nothing reads: the checks come first

    def clip(src, dst, n, types, limit=1.0, norm=1 << 30, given=0):
        k = len(src)
        work = (C.c_uint64 * 4096)()
        _fails("splahip_clip_global_norm", k, (C.c_void_p * k)(*src), (C.c_void_p * k)(*dst), (C.c_uint64 * k)(*n), (C.c_int * k)(*types), limit, given,
               C.cast(work, C.c_void_p), 4096 * 8, C.c_void_p(norm), None)

    clip([base, base], [base, base], [4, 4], [0, 0])                         # the same array twice, in place
    clip([base, base + 64], [base, base + 12], [4, 4], [0, 0])               # results overlap by an element
    clip([base, base + 4096], [base + 4100, base + 8192], [4, 4], [0, 0])    # a result over another array
    clip([base], [base + 2], [4], [1])                                       # a result shifted into its own array
    clip([base], [base], [4], [0], norm=base + 12, given=1)                  # the norm is one of the values it scales
    clip([base], [base], [4], [5])                                           # type
    clip([0], [base], [4], [0])                                              # null
    for limit in (-1.0, float("inf"), float("nan")):
        clip([base], [base], [4], [0], limit)


def test_workspaces_cover_the_largest():
    assert _lib.call("splahip_route_sort_workspace", 1 << 16, 2, 8) >= 32
    assert _lib.call("splahip_route_sort_workspace", (1 << 31) // 8 - 1, 8, 128) >= ((1 << 31) - 8) // 4096 * 128 * 4
    assert _lib.call("splahip_global_norm_workspace", 0, (C.c_uint64 * 1)()) >= 8
    assert _lib.call("splahip_global_norm_workspace", 2, (C.c_uint64 * 2)(0, 1)) >= 16
