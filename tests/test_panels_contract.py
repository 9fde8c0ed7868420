"""Refusals of the panel operators that their formulas do not show: calls whose results would be wrong or would lose something without a word."""
import ctypes as C
import subprocess
import sys
from pathlib import Path

import pytest
import torch
from torch.autograd import forward_ad

from spla_amd import _lib, kernels

INVALID = 6
BASE = 1 << 40  # addresses that nothing reads: the checks come first


def _clip(src, dst, lengths, types, norm, given=0):
    k, work = len(src), (C.c_uint64 * 4096)()
    with pytest.raises(_lib.SplaHipError) as e:
        _lib.call("splahip_clip_global_norm", k, (C.c_void_p * k)(*src), (C.c_void_p * k)(*dst), (C.c_uint64 * k)(*lengths), (C.c_int * k)(*types), 1.0, given,
                  C.cast(work, C.c_void_p), 4096 * 8, C.c_void_p(norm), None)
    return e.value.status


@pytest.mark.parametrize("at", [0, 4, 12])
def test_the_norm_may_not_be_written_into_an_array_that_is_still_to_be_scaled(at):
    """the results lie elsewhere, but the norm is written between the pass that sums and the one that scales"""
    assert _clip([BASE], [BASE + 4096], [4], [0], BASE + at) == INVALID
    assert _clip([BASE + 8192, BASE], [BASE + 16384, BASE + 4096], [4, 8], [0, 2], BASE + at) == INVALID


def test_the_workspace_is_no_array_and_no_norm():
    """partial sums are written while the arrays are read, and the norm in 64 bits is read while the results are written"""
    one, n, t = (C.c_void_p * 1), (C.c_uint64 * 1)(100), (C.c_int * 1)(0)
    need = _lib.call("splahip_global_norm_workspace", 1, n)

    def fails(name, *args):
        with pytest.raises(_lib.SplaHipError) as e:
            _lib.call(name, *args)
        assert e.value.status == INVALID, e.value

    far = C.c_void_p(BASE + (1 << 30))
    for array in (BASE, BASE + need - 4, BASE - 396):
        fails("splahip_global_norm", 1, one(array), n, t, C.c_void_p(BASE), need, far, None)
        fails("splahip_clip_global_norm", 1, one(BASE + (1 << 20)), one(array), n, t, 1.0, 0, C.c_void_p(BASE), need, far, None)
        fails("splahip_clip_global_norm", 1, one(array), one(array), n, t, 1.0, 0, C.c_void_p(BASE), need, far, None)
    for norm in (BASE, BASE + need - 4):
        fails("splahip_global_norm", 1, one(BASE + (1 << 20)), n, t, C.c_void_p(BASE), need, C.c_void_p(norm), None)


def _plan(rows=4, k=2, experts=3):
    plan = kernels.RoutePlan.__new__(kernels.RoutePlan)  # a plan of CPU tensors: what the checks look at, without a GPU
    return plan._set(torch.zeros(experts + 1, dtype=torch.int32), torch.zeros(rows * k, dtype=torch.int32), torch.zeros(rows, k, dtype=torch.int32))


# operands that have a gradient and are looked at first, with the call that they go into: call(plan, operand), the operand's shape
OPERANDS = [
    (lambda p, t: kernels.route_rows(p, t), (4, 8)),
    (lambda p, t: kernels.route_back(p, t), (8, 8)),
    (lambda p, t: kernels.route_back_grad(p, t, torch.ones(4, 2), torch.ones(4, 8)), (8, 8)),
    (lambda p, t: kernels.expert_product(p, torch.ones(8, 5), t), (3, 7, 5)),
    (lambda p, t: kernels.expert_product_grad(p, torch.ones(8, 5), t, torch.ones(8, 7)), (3, 7, 5)),
    (lambda p, t: kernels.global_norm([t, torch.ones(2)]), (6,)),
    (lambda p, t: kernels.clip_global_norm([t, torch.ones(2)], 1.0), (6,)),
]


@pytest.mark.parametrize("call,shape", OPERANDS)
def test_an_operand_whose_gradient_would_be_lost_is_refused(call, shape, monkeypatch):
    monkeypatch.setattr(kernels, "_launch", lambda *a: pytest.fail("launched"))
    with pytest.raises(ValueError, match="gradient"):
        call(_plan(), torch.ones(shape, requires_grad=True))
    with pytest.raises(ValueError, match="gradient"):
        call(_plan(), torch.nn.Parameter(torch.ones(shape)))
    with forward_ad.dual_level(), pytest.raises(ValueError, match="gradient"):
        call(_plan(), forward_ad.make_dual(torch.ones(shape), torch.ones(shape)))
    # with nothing to lose the next thing that is wrong here is said: these are not on the GPU
    with torch.no_grad(), pytest.raises(ValueError, match="on the GPU|on cpu"):
        call(_plan(), torch.ones(shape, requires_grad=True))
    with forward_ad.dual_level(), pytest.raises(ValueError, match="on the GPU|on cpu"):
        call(_plan(), torch.ones(shape))


NEGATED = OPERANDS[:5] + [
    (lambda p, t: kernels.clip_global_norm([t], 1.0, out=[torch.ones(6)]), (6,)),
]


@pytest.mark.parametrize("call,shape", NEGATED)
def test_a_tensor_that_negates_its_memory_is_refused(call, shape, monkeypatch):
    """the imaginary part of a conjugate, say: its values are its memory's with the other sign, which a call that takes the address would not see"""
    monkeypatch.setattr(kernels, "_launch", lambda *a: pytest.fail("launched"))
    with pytest.raises(ValueError, match="negat"):
        call(_plan(), torch._neg_view(torch.ones(shape)))
    one = torch.ones(1, 1, dtype=torch.complex64).conj().imag
    assert one.is_contiguous() and one.is_neg()


def test_the_module_loads_without_private_parts_of_torch():
    """the sparse operators of the same module need none of what the panel operators save time with"""
    program = """
import torch
for name in ("_cuda_getCurrentRawStream", "_cuda_getDevice", "_is_fwd_grad_enabled"):
    if hasattr(torch._C, name):
        delattr(torch._C, name)
if hasattr(torch.autograd.forward_ad, "_current_level"):
    del torch.autograd.forward_ad._current_level
from spla_amd import kernels
assert callable(kernels.mxv_masked) and callable(kernels.route_sort)
print("loaded")
"""
    run = subprocess.run([sys.executable, "-c", program], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "loaded" in run.stdout, run.stderr


@pytest.mark.parametrize("limit", [-1.0, -1e-45, float("inf"), float("nan"), 1e39])
def test_a_limit_that_is_no_largest_norm_is_a_value_error(limit, monkeypatch):
    """like every argument that the Python face can see to be wrong; before anything is allocated or launched"""
    monkeypatch.setattr(kernels, "_launch", lambda *a: pytest.fail("launched"))
    with pytest.raises(ValueError, match="limit"):
        kernels.clip_global_norm([torch.ones(3)], limit)


def test_a_tensor_in_host_memory_is_named_as_such():
    with pytest.raises(ValueError, match="on the GPU expected, not on cpu"):
        kernels.global_norm([torch.ones(3)])
    with pytest.raises(ValueError, match="on the GPU expected, not on cpu"):
        kernels.route_rows(_plan(), torch.ones(4, 8))
