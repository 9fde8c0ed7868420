"""What the documentation of the panel operators says beyond their formulas, on the GPU."""
import importlib.util

import pytest
import torch

from spla_amd import kernels

pytestmark = pytest.mark.gpu


def test_a_norm_beyond_fp32():
    """1000 values of 3e38: the norm, 9.5e39, reads as infinity in 32 bits.  Computed inside, it scales (by 64 bits); given as the 32-bit infinity, it does not, in place or into `out`."""
    values = torch.full((1000,), 3e38, device="cuda")
    norm = kernels.global_norm([values])
    assert float(norm) == float("inf")
    kept, out = values.clone(), [torch.zeros_like(values)]
    assert kernels.clip_global_norm([values], 1.0, out=out, norm=norm) is norm
    assert torch.equal(values, kept) and torch.equal(out[0], kept)
    kernels.clip_global_norm([values], 1.0, norm=norm)
    assert torch.equal(values, kept)
    assert float(kernels.clip_global_norm([values], 1.0, out=out)) == float("inf")
    # every value is 1000 ** -0.5 now: off by the factor's rounding, the product's and that of 3e38 to the input's type (which the factor takes out again)
    want = 1000 ** -0.5
    assert ((out[0].double() - want).abs() <= want * 3 * 2.0 ** -24).all()


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_a_given_norm_that_is_not_finite_scales_nothing(dtype, bad):
    t = [torch.arange(3001, device="cuda").to(dtype), torch.ones(5, device="cuda")]
    kept = [x.clone() for x in t]
    kernels.clip_global_norm(t, 0.25, norm=torch.tensor(bad, device="cuda"))
    assert all(torch.equal(a, b) for a, b in zip(t, kept))


def _layer():
    e = torch.tensor([[0, 1], [2, 0], [1, 1], [-1, 2]], dtype=torch.int32, device="cuda")
    plan = kernels.route_sort(e, 3)
    ones = lambda *shape: torch.ones(*shape, device="cuda")  # noqa: E731
    return plan, ones


CALLS = {  # every operand that has a gradient: (plan, operand, ones) -> call, shape
    "rows x": (lambda p, t, o: kernels.route_rows(p, t), (4, 8)),
    "rows weights": (lambda p, t, o: kernels.route_rows(p, o(4, 8), t), (4, 2)),
    "back y": (lambda p, t, o: kernels.route_back(p, t), (8, 8)),
    "back weights": (lambda p, t, o: kernels.route_back(p, o(8, 8), t), (4, 2)),
    "back_grad y": (lambda p, t, o: kernels.route_back_grad(p, t, o(4, 2), o(4, 8)), (8, 8)),
    "back_grad weights": (lambda p, t, o: kernels.route_back_grad(p, o(8, 8), t, o(4, 8)), (4, 2)),
    "back_grad dout": (lambda p, t, o: kernels.route_back_grad(p, o(8, 8), o(4, 2), t), (4, 8)),
    "product x": (lambda p, t, o: kernels.expert_product(p, t, o(3, 7, 5)), (8, 5)),
    "product w": (lambda p, t, o: kernels.expert_product(p, o(8, 5), t), (3, 7, 5)),
    "product_grad x": (lambda p, t, o: kernels.expert_product_grad(p, t, o(3, 7, 5), o(8, 7)), (8, 5)),
    "product_grad w": (lambda p, t, o: kernels.expert_product_grad(p, o(8, 5), t, o(8, 7)), (3, 7, 5)),
    "product_grad dy": (lambda p, t, o: kernels.expert_product_grad(p, o(8, 5), o(3, 7, 5), t), (8, 7)),
    "norm": (lambda p, t, o: kernels.global_norm([o(2), t]), (6,)),
    "clip": (lambda p, t, o: kernels.clip_global_norm([o(2), t], 1.0), (6,)),
    "clip out": (lambda p, t, o: kernels.clip_global_norm([o(2), o(6)], 1.0, out=[o(2), t]), (6,)),
    "clip norm": (lambda p, t, o: kernels.clip_global_norm([o(2)], 1.0, norm=t), ()),
}


@pytest.mark.parametrize("name", CALLS)
def test_an_operand_whose_gradient_would_be_lost_is_refused(name):
    call, shape = CALLS[name]
    plan, ones = _layer()
    tracked = torch.ones(shape, device="cuda", requires_grad=True)
    with pytest.raises(ValueError, match="gradient"):
        call(plan, tracked, ones)
    with pytest.raises(ValueError, match="gradient"):
        call(plan, tracked * 1, ones)
    with torch.autograd.forward_ad.dual_level(), pytest.raises(ValueError, match="gradient"):
        call(plan, torch.autograd.forward_ad.make_dual(torch.ones(shape, device="cuda"), torch.ones(shape, device="cuda")), ones)
    with pytest.raises(Exception):  # a batched tensor has no memory of its own
        torch.vmap(lambda t: call(plan, t, ones))(torch.ones(2, *shape, device="cuda"))
    # nothing to lose
    call(plan, tracked.detach(), ones)
    with torch.no_grad():
        call(plan, tracked, ones)
    with torch.autograd.forward_ad.dual_level():
        call(plan, torch.ones(shape, device="cuda"), ones)


def test_inside_an_autograd_function():
    """the way that a training program has the gradients: forward and backward call the operators, nothing is recorded inside"""
    class Product(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w, plan):
            ctx.plan = plan
            ctx.save_for_backward(x, w)
            return kernels.expert_product(plan, x, w)

        @staticmethod
        def backward(ctx, dy):
            return (*kernels.expert_product_grad(ctx.plan, *ctx.saved_tensors, dy.contiguous()), None)

    plan, ones = _layer()
    g = torch.Generator(device="cuda").manual_seed(3)
    x, w = (torch.randint(-3, 4, s, generator=g, device="cuda").float().requires_grad_() for s in ((8, 5), (3, 7, 5)))
    factor = torch.randint(-3, 4, (8, 7), generator=g, device="cuda").float()
    (Product.apply(x, w, plan) * factor).sum().backward()
    dx, dw = kernels.expert_product_grad(plan, x.detach(), w.detach(), factor)
    assert torch.equal(x.grad, dx) and torch.equal(w.grad, dw) and dx.any() and dw.any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_clipping_is_seen_by_a_graph_that_kept_the_tensor(dtype):
    """as any change in place: a backward pass over values that are no longer there raises instead of using the new ones"""
    w = torch.ones(9, device="cuda", dtype=dtype, requires_grad=True)
    kept, out = (torch.full((9,), 3.0, device="cuda", dtype=dtype) for _ in range(2))
    loss = (kept * w).sum()
    kernels.clip_global_norm([kept], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    bucket = torch.zeros(64, device="cuda", dtype=dtype)
    loss = (out * w).sum() + (bucket[32:41] * w).sum()
    before = [t._version for t in (kept, out, bucket)]
    kernels.clip_global_norm([kept, kept], 1.0, out=[out, bucket[32:41]])
    assert [t._version - b for t, b in zip((kept, out, bucket), before)] == [0, 1, 1]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    loss = (kept * w).sum()
    kernels.global_norm([kept])
    loss.backward()  # reading changes nothing


def test_clipping_tensors_of_inference_mode():
    with torch.inference_mode():
        t = torch.full((4,), 2.0, device="cuda")
        kernels.clip_global_norm([t], 1.0)
    kernels.clip_global_norm([t], 0.5)
    assert t.tolist() == [0.25] * 4


def test_tensors_that_negate_their_memory():
    """refused where the sign would be lost; the norm does not see it, and scaling in place keeps it"""
    plan, ones = _layer()
    negated = lambda *shape: torch._neg_view(ones(*shape))  # noqa: E731
    for call in (lambda: kernels.route_rows(plan, ones(4, 8), negated(4, 2)), lambda: kernels.route_back_grad(plan, ones(8, 8), ones(4, 2), negated(4, 8)),
                 lambda: kernels.expert_product(plan, negated(8, 5), ones(3, 7, 5)), lambda: kernels.clip_global_norm([negated(4)], 1.0, out=[ones(4)]),
                 lambda: kernels.clip_global_norm([ones(4)], 1.0, out=[negated(4)])):
        with pytest.raises(ValueError, match="negat"):
            call()
    t = negated(4)
    assert float(kernels.global_norm([t])) == 2.0
    kernels.clip_global_norm([t], 1.0)
    assert t.tolist() == [-0.5] * 4


def test_the_current_stream_by_public_calls(monkeypatch):
    """a copy of the module that found no private shortcuts: the same results, on a side stream and inside a graph"""
    spec = importlib.util.spec_from_file_location("spla_amd.kernels_without_shortcuts", kernels.__file__)
    copy = importlib.util.module_from_spec(spec)
    with monkeypatch.context() as m:
        for name in ("_cuda_getCurrentRawStream", "_cuda_getDevice"):
            m.delattr(torch._C, name)
        spec.loader.exec_module(copy)
    assert copy._raw_stream is not kernels._raw_stream and copy._current_device is not kernels._current_device
    e = torch.randint(-1, 5, (700, 2), dtype=torch.int32, device="cuda")
    x = torch.randn(700, 64, device="cuda")
    want = kernels.route_rows(kernels.route_sort(e, 5), x)
    side = torch.cuda.Stream()
    assert copy._raw_stream(0) == torch.cuda.current_stream().cuda_stream == kernels._raw_stream(0) and copy._current_device() == kernels._current_device()
    with torch.cuda.stream(side):
        assert copy._raw_stream(0) == side.cuda_stream == kernels._raw_stream(0)
        side.wait_stream(torch.cuda.default_stream())
        got = copy.route_rows(copy.route_sort(e, 5), x)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = copy.route_rows(copy.route_sort(e, 5), x)
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
