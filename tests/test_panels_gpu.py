"""The panel operators on the GPU against plain implementations in 64 bits: the sort of a router's choices, panels into expert order and back with weights, the
experts' products, their gradients, the global norm and clipping, and a training step that uses them together.

Tolerances.  u = 2^-24 is half a step of fp32, h(T) half a step of the panel's type relative to the value (bf16 2^-9 of the next power of two = at most 2^-8
of the value, torch.finfo(T).eps / 2).  A sum of n products in fp32 in any order is off by at most n u S, S the sum of the absolute products, and by n 2 u S where
the matrix cores' additions may drop bits instead of rounding; the result is rounded to T once.  fp16 results below 2^-14 have steps of 2^-24.
Panels of small whole numbers make every sum exact in fp32, so that results must be equal bit for bit."""
import pytest
import torch

from spla_amd import kernels

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
U = 2.0 ** -24


def _half(dtype):
    return torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0  # (an fp32 result is the sum itself: no rounding of its own)


def _floor(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -149


def _close(got, want, bound, dtype):
    """|got - want| <= bound (of the fp32 value) + the rounding to dtype"""
    got, want, bound = got.double().cpu(), want.cpu(), bound.cpu()
    limit = bound + (want.abs() + bound) * _half(dtype) + _floor(dtype)
    bad = ~((got - want).abs() <= limit)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} beyond the bound, first at {bad.nonzero()[0].tolist()}: {got[bad][0]} for {want[bad][0]} (limit {limit[bad][0]})"


def _router(rows, k, experts, seed=0, padding=0.0, strange=False):
    g = torch.Generator().manual_seed(seed)
    e = torch.randint(0, experts, (rows, k), generator=g, dtype=torch.int32)
    if padding:
        e[torch.rand(rows, k, generator=g) < padding] = -1
    if strange and rows:
        e.view(-1)[0] = experts
        e.view(-1)[-1] = -(2 ** 31)
        e.view(-1)[e.numel() // 2] = 2 ** 31 - 1
    return e


def _sorted(e, n_experts):
    flat = e.reshape(-1).tolist()
    order = sorted((i for i, x in enumerate(flat) if 0 <= x < n_experts), key=lambda i: flat[i])
    offsets = [0] * (n_experts + 1)
    for i in order:
        offsets[flat[i] + 1] += 1
    for x in range(n_experts):
        offsets[x + 1] += offsets[x]
    place = [-1] * len(flat)
    for p, i in enumerate(order):
        place[i] = p
    return offsets, order + [-1] * (len(flat) - len(order)), place


SORTS = [(0, 2, 4, 0, False), (1, 1, 1, 0, False), (1, 8, 8, 0, False), (5, 3, 7, 0.3, True), (64, 2, 8, 0, False), (63, 1, 2, 0, False), (2048, 1, 3, 0, False),
         (2049, 2, 65, 0.1, True), (5000, 8, 128, 0.1, False), (777, 5, 2048, 0, True), (300, 4, 16, 1.1, False), (1500, 7, 1, 0.5, False),
         (0, 1, 1500, 0, False), (8192, 1, 512, 0.1, True), (8193, 1, 512, 0.1, True), (4096, 3, 700, 0.2, True), (30011, 2, 128, 0.05, True), (9000, 1, 1, 0.5, False), (100003, 1, 500, 0.1, True), (400009, 1, 512, 0.1, True),
         (300007, 2, 5, 0.1, False)]


@pytest.mark.parametrize("rows,k,experts,padding,strange", SORTS)
def test_sort(rows, k, experts, padding, strange):
    e = _router(rows, k, experts, rows, padding, strange)
    plan = kernels.route_sort(e.cuda(), experts)
    offsets, order, place = _sorted(e, experts)
    assert plan.offsets.tolist() == offsets
    assert plan.order.tolist() == order
    assert plan.place.reshape(-1).tolist() == place


def test_sort_one_expert_takes_all():
    e = torch.full((9000, 2), 5, dtype=torch.int32, device="cuda")
    plan = kernels.route_sort(e, 9)
    assert torch.equal(plan.order.cpu(), torch.arange(18000, dtype=torch.int32)) and plan.offsets.tolist() == [0] * 6 + [18000] * 4


ROWS = [(1, 1, 1, 1), (1, 8, 8, 4104), (3, 2, 4, 7), (17, 3, 5, 8), (130, 4, 9, 333), (40, 2, 3, 1001), (257, 2, 8, 2048), (33, 5, 7, 64), (9, 2, 4, 20000)]


def _case(rows, k, experts, padding=0.2, seed=1):
    e = _router(rows, k, experts, seed, padding, strange=rows > 20)
    plan = kernels.route_sort(e.cuda(), experts)
    order = plan.order.cpu().long()
    place = plan.place.cpu().long()
    return plan, order, place, int(plan.offsets[-1])


def _panel(rows, width, dtype, seed, whole=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(-4, 5, (rows, width), generator=g).double() if whole else torch.randn(rows, width, generator=g, dtype=torch.float64)
    return x.to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,experts,width", ROWS)
def test_rows(rows, k, experts, width, dtype):
    plan, order, place, end = _case(rows, k, experts)
    x, w = _panel(rows, width, dtype, 2), _panel(rows, k, torch.float32, 3)
    w[place < 0] = float("nan")  # a weight of no entry does not count
    got = kernels.route_rows(plan, x.cuda())
    want = torch.zeros(rows * k, width, dtype=dtype)
    want[:end] = x[order[:end] // k]
    assert torch.equal(got.cpu(), want)
    got = kernels.route_rows(plan, x.cuda(), w.cuda())
    exact = torch.zeros(rows * k, width, dtype=torch.float64)
    exact[:end] = x.double()[order[:end] // k] * w.double().reshape(-1)[order[:end], None]
    _close(got, exact, exact.abs() * U, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,experts,width", ROWS)
def test_back(rows, k, experts, width, dtype):
    plan, order, place, end = _case(rows, k, experts)
    y, w = _panel(rows * k, width, dtype, 4), _panel(rows, k, torch.float32, 5)
    y[end:] = float("nan")  # rows behind the last entry and weights of no entry do not count
    w[place < 0] = float("nan")
    here = (place >= 0).double()[:, :, None]
    terms = torch.nan_to_num(y.double())[place.clamp(min=0)] * here
    _close(kernels.route_back(plan, y.cuda()), terms.sum(1), terms.abs().sum(1) * (k * U), dtype)
    terms = terms * torch.nan_to_num(w.double())[:, :, None]
    _close(kernels.route_back(plan, y.cuda(), w.cuda()), terms.sum(1), terms.abs().sum(1) * (k * U), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,experts,width", ROWS)
def test_back_grad(rows, k, experts, width, dtype):
    plan, order, place, end = _case(rows, k, experts)
    y, w, g = _panel(rows * k, width, dtype, 6), _panel(rows, k, torch.float32, 7), _panel(rows, width, dtype, 8)
    y[end:] = float("nan")
    w[place < 0] = float("nan")
    dy, dw = kernels.route_back_grad(plan, y.cuda(), w.cuda(), g.cuda())
    exact = torch.zeros(rows * k, width, dtype=torch.float64)
    exact[:end] = g.double()[order[:end] // k] * w.double().reshape(-1)[order[:end], None]
    _close(dy, exact, exact.abs() * U, dtype)
    terms = torch.nan_to_num(y.double())[place.clamp(min=0)] * g.double()[:, None, :] * (place >= 0).double()[:, :, None]
    _close(dw, terms.sum(2), terms.abs().sum(2) * (width * U), torch.float32)


def test_back_without_any_entry_is_zero():
    plan = kernels.route_sort(torch.full((6, 2), -1, dtype=torch.int32, device="cuda"), 4)
    y = torch.full((12, 33), float("nan"), device="cuda")
    assert torch.equal(kernels.route_back(plan, y).cpu(), torch.zeros(6, 33))
    dy, dw = kernels.route_back_grad(plan, y, torch.ones(6, 2, device="cuda"), torch.ones(6, 33, device="cuda"))
    assert torch.equal(dy.cpu(), torch.zeros(12, 33)) and torch.equal(dw.cpu(), torch.zeros(6, 2))
    assert torch.equal(kernels.route_rows(plan, torch.ones(6, 33, device="cuda")).cpu(), torch.zeros(12, 33))
    w = torch.ones(4, 7, 33, device="cuda")
    assert torch.equal(kernels.expert_product(plan, y, w).cpu(), torch.zeros(12, 7))
    dx, dw = kernels.expert_product_grad(plan, y, w, torch.full((12, 7), float("nan"), device="cuda"))
    assert torch.equal(dx.cpu(), torch.zeros(12, 33)) and torch.equal(dw.cpu(), torch.zeros(4, 7, 33))


# rows of tokens, entries a row, experts, n_in, n_out: one token, few rows an expert, ragged ranges around every tile's edge, odd and aligned sizes, more experts
# than a wavefront has lanes
PRODUCTS = [(1, 1, 1, 1, 1), (1, 2, 8, 64, 96), (1, 8, 8, 512, 256), (4, 2, 3, 33, 17), (16, 1, 1, 64, 64), (17, 1, 1, 128, 128), (64, 4, 32, 256, 192), (100, 3, 130, 40, 56),
            (255, 1, 1, 96, 64), (256, 1, 1, 256, 256), (257, 1, 1, 264, 520), (513, 2, 2, 128, 320), (333, 3, 5, 250, 333), (700, 2, 3, 512, 512), (1500, 2, 4, 1000, 264),
            (31, 2, 4, 2056, 72), (2000, 1, 300, 72, 136), (5000, 2, 2, 40, 56), (5000, 2, 3, 33, 65), (3001, 1, 1, 136, 72), (64, 4, 64, 128, 1024), (50, 8, 20, 2072, 24),
            (9, 2, 6, 1096, 1040)]


def _product_case(rows, k, experts, n_in, n_out, dtype, whole, seed=9):
    plan, order, place, end = _case(rows, k, experts, padding=0.1 if rows > 1 else 0.0, seed=seed)
    x, w = _panel(rows * k, n_in, dtype, 10, whole), _panel(experts * n_out, n_in, dtype, 11, whole).reshape(experts, n_out, n_in)
    dy = _panel(rows * k, n_out, dtype, 12, whole)
    x[end:] = float("nan")
    dy[end:] = float("nan")
    return plan, x, w, dy, plan.offsets.tolist()


def _products(x, w, dy, offsets):
    y, dx, dw = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64), torch.zeros(x.shape, dtype=torch.float64), torch.zeros(w.shape, dtype=torch.float64)
    for e, (a, b) in enumerate(zip(offsets, offsets[1:])):
        if a < b:
            y[a:b] = x[a:b].double() @ w[e].double().t()
            dx[a:b] = dy[a:b].double() @ w[e].double()
            dw[e] = dy[a:b].double().t() @ x[a:b].double()
    return y, dx, dw


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,experts,n_in,n_out", PRODUCTS)
def test_product_of_whole_numbers(rows, k, experts, n_in, n_out, dtype):
    """sums below 2^24: fp32 holds them exactly, only the rounding to the panel's type is left (fp16: below its largest value)"""
    plan, x, w, dy, offsets = _product_case(rows, k, experts, n_in, n_out, dtype, True)
    y, dx, dw = _products(x, w, dy, offsets)
    assert max(y.abs().max(), dx.abs().max(), dw.abs().max()) < (65504 if dtype == torch.float16 else 2 ** 24)
    assert torch.equal(kernels.expert_product(plan, x.cuda(), w.cuda()).cpu(), y.to(dtype))
    got_dx, got_dw = kernels.expert_product_grad(plan, x.cuda(), w.cuda(), dy.cuda())
    assert torch.equal(got_dx.cpu(), dx.to(dtype))
    assert torch.equal(got_dw.cpu(), dw.to(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,experts,n_in,n_out", [c for c in PRODUCTS if c[0] in (1, 64, 257, 333, 1500)])
def test_product_of_any_numbers(rows, k, experts, n_in, n_out, dtype):
    plan, x, w, dy, offsets = _product_case(rows, k, experts, n_in, n_out, dtype, False)
    y, dx, dw = _products(x, w, dy, offsets)
    sy, sdx, sdw = _products(x.abs(), w.abs(), dy.abs(), offsets)
    _close(kernels.expert_product(plan, x.cuda(), w.cuda()), y, sy * (n_in * 2 * U), dtype)
    got_dx, got_dw = kernels.expert_product_grad(plan, x.cuda(), w.cuda(), dy.cuda())
    _close(got_dx, dx, sdx * (n_out * 2 * U), dtype)
    _close(got_dw, dw, sdw * (rows * k * 2 * U), dtype)


# enough tiles that the card is full of large ones, with some left over that are cut in parts: ragged ranges, depths that end inside a slab, experts without rows, more experts than a wavefront has lanes
LARGE = [(6000, 2, 5, 328, 2056), (2600, 2, 70, 136, 2304), (700, 1, 200, 264, 520), (9000, 1, 2, 64, 2048), (3000, 2, 3, 2120, 1288), (4800, 2, 2, 2048, 264),
         (6000, 2, 3, 516, 768), (6000, 2, 3, 515, 769), (3000, 2, 20, 515, 769), (2600, 2, 30, 776, 1288)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,experts,n_in,n_out", LARGE)
def test_large_products_of_whole_numbers(rows, k, experts, n_in, n_out, dtype):
    """sums below 2^24 are exact in fp32 (and in the reference's fp32 product); values -1, 0, 1 keep fp16 results below its largest value"""
    plan, order, place, end = _case(rows, k, experts, padding=0.1, seed=13)
    g = torch.Generator(device="cuda").manual_seed(14)
    x, w, dy = (torch.randint(-1, 2, s, generator=g, device="cuda").to(dtype) for s in ((rows * k, n_in), (experts, n_out, n_in), (rows * k, n_out)))
    x[end:] = float("nan")
    dy[end:] = float("nan")
    y, dx, dw = torch.zeros(rows * k, n_out, device="cuda"), torch.zeros(rows * k, n_in, device="cuda"), torch.zeros(experts, n_out, n_in, device="cuda")
    offsets = plan.offsets.tolist()
    for e, (a, b) in enumerate(zip(offsets, offsets[1:])):
        if a < b:
            y[a:b] = x[a:b].float() @ w[e].float().t().contiguous()
            dx[a:b] = dy[a:b].float() @ w[e].float()
            dw[e] = dy[a:b].float().t().contiguous() @ x[a:b].float()
    assert max(float(t.abs().max()) for t in (y, dx, dw)) < 65504
    assert torch.equal(kernels.expert_product(plan, x, w), y.to(dtype))
    got_dx, got_dw = kernels.expert_product_grad(plan, x, w, dy)
    assert torch.equal(got_dx, dx.to(dtype)) and torch.equal(got_dw, dw.to(dtype))


def test_product_needs():
    plan, x, w, dy, _ = _product_case(20, 2, 3, 24, 40, torch.float32, True)
    x, w, dy = x.cuda(), w.cuda(), dy.cuda()
    both = kernels.expert_product_grad(plan, x, w, dy)
    dx, none = kernels.expert_product_grad(plan, x, w, dy, need=(True, False))
    assert none is None and torch.equal(dx, both[0])
    none, dw = kernels.expert_product_grad(plan, x, w, dy, need=(False, True))
    assert none is None and torch.equal(dw, both[1])


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,experts,n_in,n_out", [(70, 2, 3, 48, 40), (30, 2, 3, 72, 64), (70, 2, 3, 47, 41), (4000, 2, 3, 64, 2048), (4100, 1, 3, 250, 333)])
def test_product_keeps_bad_values_in_their_rows(rows, k, experts, n_in, n_out, dtype, bad):
    """an infinity or NaN of one expert's row reaches that row's results (and that expert's dw), nothing beside it"""
    plan, x, w, dy, offsets = _product_case(rows, k, experts, n_in, n_out, dtype, False)
    x, w, dy = x.cuda(), w.cuda(), dy.cuda()
    y = kernels.expert_product(plan, x, w)
    dx, dw = kernels.expert_product_grad(plan, x, w, dy)
    row = offsets[1]
    x[row, 7] = bad
    got = kernels.expert_product(plan, x, w)
    keep = torch.arange(x.shape[0]) != row
    assert torch.isfinite(y).all() and torch.equal(got[keep], y[keep]) and not torch.isfinite(got[row]).any()
    got_dx, got_dw = kernels.expert_product_grad(plan, x, w, dy)
    column = torch.arange(n_in) != 7
    assert torch.equal(got_dx, dx) and torch.equal(got_dw[[0, 2]], dw[[0, 2]]) and torch.equal(got_dw[1][:, column], dw[1][:, column])
    assert not torch.isfinite(got_dw[1, :, 7]).any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,experts,n_in,n_out", [(70, 2, 3, 48, 40), (30, 2, 3, 72, 64), (70, 2, 3, 47, 41), (4000, 2, 3, 64, 2048)])
def test_product_of_subnormal_numbers(rows, k, experts, n_in, n_out, dtype):
    """whole multiples of the type's smallest number times whole numbers: every sum is such a multiple, exactly"""
    plan, x, w, dy, offsets = _product_case(rows, k, experts, n_in, n_out, dtype, True)
    tiny = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}[dtype]
    scaled = (x.double() * tiny).to(dtype)
    assert torch.equal(torch.nan_to_num(scaled.double()), torch.nan_to_num(x.double()) * tiny)
    y, dx, dw = _products(x, w, dy, offsets)
    assert torch.equal(kernels.expert_product(plan, scaled.cuda(), w.cuda()).cpu(), (y * tiny).to(dtype))
    assert torch.equal(kernels.expert_product_grad(plan, scaled.cuda(), w.cuda(), dy.cuda())[1].cpu(), (dw * tiny).to(dtype))


def test_gradients_are_the_differences():
    """every operator is linear in each operand: with whole numbers, f(x + v) - f(x) paired with a direction equals the gradient paired with v, exactly"""
    plan, order, place, end = _case(40, 3, 5)
    n = 120
    x, v, w, dw_, g = (_panel(*s, torch.float32, i, True).cuda() for i, s in enumerate([(40, 24), (40, 24), (40, 3), (40, 3), (n, 24)]))
    pair = lambda a, b: float((a.double() * b.double()).sum())  # noqa: E731
    f = kernels.route_rows
    assert pair(f(plan, x + v, w) - f(plan, x, w), g) == pair(kernels.route_back(plan, g, w), v)
    assert pair(f(plan, x, w + dw_) - f(plan, x, w), g) == pair(kernels.route_back_grad(plan, g, w, x)[1], dw_)
    y, vy, out = (_panel(*s, torch.float32, 20 + i, True).cuda() for i, s in enumerate([(n, 24), (n, 24), (40, 24)]))
    b, (gy, gw) = kernels.route_back, kernels.route_back_grad(plan, y, w, out)
    assert pair(b(plan, y + vy, w) - b(plan, y, w), out) == pair(gy, vy)
    assert pair(b(plan, y, w + dw_) - b(plan, y, w), out) == pair(gw, dw_)
    m, vm, z = (_panel(*s, torch.float32, 30 + i, True).cuda() for i, s in enumerate([(5 * 16, 24), (5 * 16, 24), (n, 16)]))
    m, vm = m.reshape(5, 16, 24), vm.reshape(5, 16, 24)
    p, (gx, gm) = kernels.expert_product, kernels.expert_product_grad(plan, y, m, z)
    assert pair(p(plan, y + vy, m) - p(plan, y, m), z) == pair(gx, vy)
    assert pair(p(plan, y, m + vm) - p(plan, y, m), z) == pair(gm, vm)


def _tensors(sizes, dtypes, scale=1.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(s, generator=g, device="cuda") * scale).to(d) for s, d in zip(sizes, dtypes)]


def _norm(tensors):
    return torch.stack([t.double().square().sum() for t in tensors]).sum().sqrt().cpu()


LISTS = [([1], [torch.float32]), ([(3, 5), 0, 7], [torch.bfloat16, torch.float32, torch.float16]), ([2047, 2049, 1], DTYPES), ([70001] * 5, [torch.bfloat16] * 5),
         ([(i % 13) * 3 for i in range(300)], [DTYPES[i % 3] for i in range(300)]), ([5_000_003, 4096], [torch.float32, torch.bfloat16]), ([513] * 16, [DTYPES[i % 3] for i in range(16)]), ([513] * 17, [DTYPES[i % 3] for i in range(17)]), ([0, 0], [torch.float32] * 2)]


@pytest.mark.parametrize("sizes,dtypes", LISTS)
def test_norm_and_clip(sizes, dtypes):
    """64-bit sums, so one rounding of the norm; the factor, the product and the rounding to the type"""
    t = _tensors(sizes, dtypes)
    want = _norm(t)
    norm = kernels.global_norm(t)
    assert norm.shape == () and norm.dtype == torch.float32
    _close(norm, want, want * U, torch.float32)
    limit = float(want) / 3
    scale = limit / float(want) if float(want) else 1.0
    exact = [x.double().cpu() * scale for x in t]
    out = [torch.full_like(x, float("nan")) for x in t]
    assert torch.equal(kernels.clip_global_norm(t, limit, out=out), norm)
    for o, x in zip(out, exact):
        _close(o, x, x.abs() * (3 * U), o.dtype)  # (the limit's rounding to fp32 is the third)
    kernels.clip_global_norm(t, limit)
    for o, x in zip(out, t):
        assert torch.equal(o, x)
    before = [x.clone() for x in t]
    kernels.clip_global_norm(t, 1e9)  # below the limit: as they were
    kernels.clip_global_norm(t, 1e9, out=out)
    for b, x, o in zip(before, t, out):
        assert torch.equal(b, x) and torch.equal(b, o)


def test_norm_of_unaligned_and_strided_parts():
    base = _tensors([4099, 4099], [torch.bfloat16, torch.float32], seed=4)
    parts = [base[0][1:4001], base[1][3:3999], base[0][4002:4003]]
    want = _norm(parts)
    _close(kernels.global_norm(parts), want, want * U, torch.float32)
    kept = [base[0][:1].clone(), base[0][4001:4002].clone(), base[0][4003:].clone()]
    exact = [p.double().cpu() / float(want) for p in parts]
    kernels.clip_global_norm(parts, 1.0)
    for p, x in zip(parts, exact):
        _close(p, x, x.abs() * (2 * U), p.dtype)
    assert torch.equal(base[0][:1], kept[0]) and torch.equal(base[0][4001:4002], kept[1]) and torch.equal(base[0][4003:], kept[2])
    with pytest.raises(ValueError):
        kernels.global_norm([base[1][:4096].reshape(64, 64).t()])
    with pytest.raises(Exception):
        kernels.clip_global_norm([base[1], base[1]], 1.0)


def test_norm_of_extreme_values():
    big = torch.full((1000,), 3e38, device="cuda")           # squares beyond fp32
    small = torch.full((1000,), 1e-44, device="cuda")        # squares below fp32, the values themselves are subnormal
    want = _norm([small])
    _close(kernels.global_norm([small]), want, want * U, torch.float32)
    assert float(kernels.global_norm([big])) == float("inf")  # the norm itself leaves fp32 ...
    kernels.clip_global_norm([big], 1.0)                      # ... and still scales
    exact = torch.full((1000,), 1000 ** -0.5, dtype=torch.float64)
    _close(big, exact, exact * (2 * U), torch.float32)
    for bad in (float("inf"), float("nan")):
        t = [torch.ones(5000, device="cuda"), torch.ones(300, device="cuda", dtype=torch.bfloat16)]
        t[0][4321] = bad
        before = [x.clone() for x in t]
        n = float(kernels.clip_global_norm(t, 1.0))
        assert n == bad or (n != n and bad != bad)
        for b, x in zip(before, t):
            assert torch.equal(torch.nan_to_num(b), torch.nan_to_num(x))


def test_clip_with_a_given_norm():
    t = _tensors([1000, 37], [torch.float32, torch.float16], seed=6)
    exact = [x.double().cpu() * (0.5 / 64.0) for x in t]
    norm = torch.tensor(64.0, device="cuda")
    assert kernels.clip_global_norm(t, 0.5, norm=norm) is norm
    for x, e in zip(t, exact):
        _close(x, e, e.abs() * U, x.dtype)
    kernels.clip_global_norm(t, 0.0)
    assert all(not x.any() for x in t)


def _layer(x, experts, weights, w1, w2, g, n_experts, limit):
    """one training step of a layer of experts: forward, backward, clipped gradients"""
    plan = kernels.route_sort(experts, n_experts)
    s = kernels.route_rows(plan, x)
    h = kernels.expert_product(plan, s, w1)
    a = torch.relu(h)
    y = kernels.expert_product(plan, a, w2)
    out = kernels.route_back(plan, y, weights)
    dy, dweights = kernels.route_back_grad(plan, y, weights, g)
    da, dw2 = kernels.expert_product_grad(plan, a, w2, dy)
    dh = da * (h > 0)
    ds, dw1 = kernels.expert_product_grad(plan, s, w1, dh)
    dx = kernels.route_back(plan, ds)
    norm = kernels.clip_global_norm([dw1, dw2, dweights], limit)
    return out, dx, norm, dw1, dw2, dweights


def _layer_inputs(dtype, whole, rows=150, k=2, experts=6, n=64, hidden=96):
    e = _router(rows, k, experts, 3, 0.1)
    w = _panel(rows, k, torch.float32, 40, whole)
    return [t.cuda() for t in (_panel(rows, n, dtype, 41, whole), e, w, _panel(experts * hidden, n, dtype, 42, whole).reshape(experts, hidden, n),
                               _panel(experts * n, hidden, dtype, 43, whole).reshape(experts, n, hidden), _panel(rows, n, dtype, 44, whole))], experts


@pytest.mark.parametrize("dtype", DTYPES)
def test_training_step(dtype):
    """the operators of a step together, against the formulas in 64 bits on the same (rounded) intermediate values"""
    (x, e, w, w1, w2, g), experts = _layer_inputs(dtype, False)
    w1, w2 = (w1 * 0.125).contiguous(), (w2 * 0.125).contiguous()
    out, dx, norm, dw1, dw2, dweights = _layer(x, e, w, w1, w2, g, experts, 1.0)
    X, W, W1, W2 = (t.double().cpu().requires_grad_() for t in (x, w, w1, w2))
    E, ref = e.cpu(), []
    for t in range(x.shape[0]):
        row = torch.zeros(x.shape[1], dtype=torch.float64)
        for j in range(E.shape[1]):
            i = int(E[t, j])
            if i >= 0:
                row = row + W[t, j] * (W2[i] @ torch.relu(W1[i] @ X[t]))
        ref.append(row)
    ref = torch.stack(ref)
    ref.backward(g.double().cpu())
    total = torch.sqrt(sum(p.grad.square().sum() for p in (W1, W2, W)))
    # every intermediate panel is rounded to the type (6 of them in the longest chain) and every sum of n <= 300 terms stays below 2 n U: relative to the largest
    # value of the result (norm-wise, the roundings are independent of the values' signs) 6 h + 3 * 600 U, doubled for the relu's switch near 0
    tol = 2 * (6 * torch.finfo(dtype).eps / 2 + 1800 * U)
    for got, want in ((out, ref.detach()), (dx, X.grad), (dw1, W1.grad / total), (dw2, W2.grad / total), (dweights, W.grad / total)):
        got = got.double().cpu()
        assert (got - want).norm() <= tol * want.norm()
    assert abs(float(norm) - float(total)) <= tol * float(total)


def test_on_another_stream_and_in_a_graph():
    """two captured steps replayed in turn with eager work between: every replay equals the eager result bit for bit"""
    (x, e, w, w1, w2, g), experts = _layer_inputs(torch.bfloat16, True)
    eager = _layer(x, e, w, w1, w2, g, experts, 1.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = _layer(x, e, w, w1, w2, g, experts, 1.0)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(eager, other):
        assert torch.equal(a, b)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results = _layer(x, e, w, w1, w2, g, experts, 1.0)
        graphs.append((graph, results))
    for again in range(3):
        x.copy_(x.roll(1, 0))
        e.copy_(e.roll(1, 0))
        w.copy_(w.roll(1, 0))
        want = _layer(x, e, w, w1, w2, g, experts, 1.0)
        for graph, results in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, results in graphs:
            for a, b in zip(want, results):
                assert torch.equal(a, b)


def test_calls_on_two_streams_at_once():
    """two steps on different inputs under way together, each as it is alone"""
    sides = [torch.cuda.Stream() for _ in range(2)]
    inputs = [_layer_inputs(torch.bfloat16, True, rows=2000 + 700 * i, k=2, experts=6 + i, n=128, hidden=256) for i in range(2)]
    alone = [_layer(*args, experts, 1.0) for args, experts in inputs]
    torch.cuda.synchronize()
    for _ in range(3):
        together = []
        for side, (args, experts) in zip(sides, inputs):
            with torch.cuda.stream(side):
                together.append([_layer(*args, experts, 1.0) for _ in range(2)])
        torch.cuda.synchronize()
        for want, runs in zip(alone, together):
            for got in runs:
                assert all(torch.equal(torch.nan_to_num(a), torch.nan_to_num(b)) for a, b in zip(want, got))


def test_same_results_every_time():
    plan, x, w, dy, _ = _product_case(900, 2, 4, 512, 256, torch.bfloat16, False)
    x, w, dy = x.cuda(), w.cuda(), dy.cuda()
    first = [kernels.expert_product(plan, x, w), *kernels.expert_product_grad(plan, x, w, dy)]
    for _ in range(3):
        again = [kernels.expert_product(plan, x, w), *kernels.expert_product_grad(plan, x, w, dy)]
        assert all(torch.equal(torch.nan_to_num(a), torch.nan_to_num(b)) for a, b in zip(first, again))
    t = _tensors([1_000_001, 77], [torch.float32, torch.float16])
    norms = {float(kernels.global_norm(t)) for _ in range(4)}
    assert len(norms) == 1


def test_more_rows_than_a_launch_has_threads():
    """70 M rows: a wavefront each would be more than 2^32 threads"""
    rows = 70_000_000
    e = torch.arange(rows, dtype=torch.int32, device="cuda")[:, None] % 2
    plan = kernels.route_sort(e, 2)
    assert plan.offsets.tolist() == [0, rows // 2, rows]
    y = torch.ones(rows, 1, dtype=torch.bfloat16, device="cuda")
    g = (torch.arange(rows, device="cuda") % 128).bfloat16()[:, None]
    dy, dw = kernels.route_back_grad(plan, y, torch.ones(rows, 1, device="cuda"), g)
    assert torch.equal(dw, g.float()) and torch.equal(dy[:rows // 2], g[0::2]) and torch.equal(dy[rows // 2:], g[1::2])
    assert torch.equal(kernels.route_rows(plan, g), dy) and torch.equal(kernels.route_back(plan, dy), g)


def test_panels_of_no_columns_and_no_rows():
    plan = kernels.route_sort(torch.zeros(3, 2, dtype=torch.int32, device="cuda"), 2)
    empty = torch.empty(3, 0, device="cuda")
    assert kernels.route_rows(plan, empty).shape == (6, 0) and kernels.route_back(plan, torch.empty(6, 0, device="cuda")).shape == (3, 0)
    dy, dw = kernels.route_back_grad(plan, torch.empty(6, 0, device="cuda"), torch.ones(3, 2, device="cuda"), empty)
    assert dy.shape == (6, 0) and torch.equal(dw.cpu(), torch.zeros(3, 2))
    plan = kernels.route_sort(torch.empty(0, 2, dtype=torch.int32, device="cuda"), 2)
    x, w = torch.empty(0, 8, dtype=torch.bfloat16, device="cuda"), torch.ones(2, 16, 8, dtype=torch.bfloat16, device="cuda")
    assert kernels.route_rows(plan, x).shape == (0, 8) and kernels.route_back(plan, x).shape == (0, 8) and kernels.expert_product(plan, x, w).shape == (0, 16)
    dx, dw = kernels.expert_product_grad(plan, x, w, torch.empty(0, 16, dtype=torch.bfloat16, device="cuda"))
    assert dx.shape == (0, 8) and not dw.any() and dw.shape == w.shape


def test_panels_beyond_32_bit_offsets():
    """more than 2^31 elements and 2^32 bytes: the last rows and matrices are where they belong"""
    rows, width = 1_050_000, 2056
    e = torch.zeros(rows, 1, dtype=torch.int32, device="cuda")
    e[-3:] = torch.tensor([[1], [2], [1]], dtype=torch.int32, device="cuda")
    plan = kernels.route_sort(e, 3)
    x = torch.zeros(rows, width, dtype=torch.bfloat16, device="cuda")
    x[-3:] = torch.arange(1, 4, device="cuda")[:, None].to(torch.bfloat16)
    s = kernels.route_rows(plan, x)
    assert s[-4:, -1].tolist() == [0, 1, 3, 2] and s[-3:, 0].tolist() == [1, 3, 2]
    assert torch.equal(kernels.route_back(plan, s), x)
    w = torch.ones(3, 8, width, dtype=torch.bfloat16, device="cuda")
    w[2] *= 2
    y = kernels.expert_product(plan, s, w)
    near = lambda v: float(torch.tensor(float(v)).bfloat16())  # noqa: E731
    ys = [near(2056), near(3 * 2056), near(2 * 2 * 2056)]
    assert y[-4:, 5].tolist() == [0] + ys
    dx, dw = kernels.expert_product_grad(plan, s, w, y)
    assert dx[-3:, -1].tolist() == [near(8 * ys[0]), near(8 * ys[1]), near(8 * 2 * ys[2])]
    assert not dw[0].any() and dw[1, 0, 0] == near(ys[0] + 3 * ys[1]) and dw[2, 7, -1] == near(2 * ys[2])
    dy, dweights = kernels.route_back_grad(plan, s, torch.ones(rows, 1, device="cuda"), x)
    assert torch.equal(dy, s) and dweights[-3:, 0].tolist() == [2056, 4 * 2056, 9 * 2056]
    assert float(kernels.global_norm([x])) == pytest.approx((14 * 2056) ** 0.5, rel=2.0 ** -23)
