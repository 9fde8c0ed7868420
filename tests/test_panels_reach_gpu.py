"""The panel operators where a kernel is chosen by alignment, by a panel's size or by the average of the rows an expert has: experts far above that average, arrays
that start between two units, panels beyond the caches.  Whole numbers whose sums are exact in fp32: results must be equal bit for bit."""
import pytest
import torch

from spla_amd import kernels

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _whole(shape, dtype, seed, most=1, start=0):
    """whole numbers -most .. most, the first element `start` elements behind an address that is a multiple of 256 bytes"""
    n = 1
    for s in shape:
        n *= s
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.randint(-most, most + 1, (n + start,), generator=g, device="cuda").to(dtype)[start:].view(shape)
    assert t.is_contiguous() and t.data_ptr() % 256 == start * t.element_size()
    return t


def _products(x, w, dy, offsets):
    """in fp32, where these sums are exact"""
    y = torch.zeros(x.shape[0], w.shape[1], device="cuda")
    dx, dw = torch.zeros(x.shape, device="cuda"), torch.zeros(w.shape, device="cuda")
    for e, (a, b) in enumerate(zip(offsets, offsets[1:])):
        if a < b:
            y[a:b] = x[a:b].float() @ w[e].float().t().contiguous()
            dx[a:b] = dy[a:b].float() @ w[e].float()
            dw[e] = dy[a:b].float().t().contiguous() @ x[a:b].float()
    return y.to(x.dtype), dx.to(x.dtype), dw.to(x.dtype)


def _uneven(n_experts, n_places, rows, seed):
    """a plan of one entry a token in which expert e of `rows` has rows[e] entries, the others none; the rest of the tokens is padding, all in random order"""
    e = torch.full((n_places,), -1, dtype=torch.int32)
    flat = [i for i, n in rows.items() for _ in range(n)]
    assert len(flat) <= n_places
    e[:len(flat)] = torch.tensor(flat, dtype=torch.int32)
    plan = kernels.route_sort(e[torch.randperm(n_places, generator=torch.Generator().manual_seed(seed))][:, None].contiguous().cuda(), n_experts)
    return plan, plan.offsets.tolist()


# few rows an expert on the average (at most 24), so that the kernel without LDS serves them, but 31 .. 384 at some: one block of 32 rows, whole blocks, blocks and a rest, all rows at one.
# The widths reach its three forms: 16 columns a workgroup (experts x n / 32 below 192), 32, and 64 (experts x n / 64 from 1024 on).
UNEVEN = [(16, 384, {0: 33, 3: 200, 7: 64, 9: 65, 15: 1}), (16, 384, {5: 384}), (16, 380, {0: 96, 1: 31, 14: 32, 15: 129}), (2, 48, {1: 47})]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n_in,n_out", [(136, 72), (2056, 40), (72, 392), (328, 1000), (264, 4104)])
@pytest.mark.parametrize("n_experts,n_places,rows", UNEVEN)
def test_few_rows_on_the_average_but_many_at_one_expert(n_experts, n_places, rows, n_in, n_out, dtype):
    plan, offsets = _uneven(n_experts, n_places, rows, 3)
    assert n_places <= 24 * n_experts
    x, w, dy = _whole((n_places, n_in), dtype, 1), _whole((n_experts, n_out, n_in), dtype, 2), _whole((n_places, n_out), dtype, 3)
    x[offsets[-1]:] = float("nan")
    y, _, _ = _products(x, w, dy, offsets)
    assert torch.equal(kernels.expert_product(plan, x, w), y)


@pytest.mark.parametrize("dtype", DTYPES)
def test_few_rows_on_the_average_of_many_experts(dtype):
    """64 experts of 1024 columns: the form of 64 columns a workgroup"""
    rows = {e: 1 + e % 3 for e in range(64)}
    rows.update({0: 33, 31: 200, 40: 64, 63: 65})
    plan, offsets = _uneven(64, 1536, rows, 4)
    x, w, dy = _whole((1536, 520), dtype, 1), _whole((64, 1024, 520), dtype, 2), _whole((1536, 1024), dtype, 3)
    x[offsets[-1]:] = float("nan")
    assert torch.equal(kernels.expert_product(plan, x, w), _products(x, w, dy, offsets)[0])


def test_a_bad_value_stays_in_its_row_at_an_expert_of_many_rows():
    plan, offsets = _uneven(16, 384, {0: 33, 3: 200, 7: 64, 9: 65, 15: 1}, 5)
    x, w = _whole((384, 136), torch.bfloat16, 1), _whole((16, 1000, 136), torch.bfloat16, 2)
    y = kernels.expert_product(plan, x, w)
    for row in (offsets[3], offsets[3] + 31, offsets[3] + 32, offsets[4] - 1):
        bad = x.clone()
        bad[row, 7] = float("nan")
        got, keep = kernels.expert_product(plan, bad, w), torch.arange(384) != row
        assert got[row].isnan().all() and torch.equal(got[keep], y[keep])


# sizes in whole units, so that only the start decides: few rows; tiles; a matrix gradient in parts; enough tiles for the large kernels
STARTS = [(16, 300, {0: 33, 3: 200}, 136, 264), (3, 700, {0: 300, 1: 1, 2: 380}, 136, 264), (2, 9000, {0: 5000, 1: 3990}, 40, 56), (5, 5331, {0: 2000, 1: 500, 2: 1, 4: 2800}, 256, 336),
          (3, 9000, {0: 4000, 2: 4900}, 520, 2056), (30, 5200, {e: 170 for e in range(30)}, 776, 1288)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("late", ["x", "w", "dy", "all"])
@pytest.mark.parametrize("n_experts,n_places,rows,n_in,n_out", STARTS)
def test_panels_and_matrices_that_start_between_units(n_experts, n_places, rows, n_in, n_out, late, dtype):
    plan, offsets = _uneven(n_experts, n_places, rows, 6)
    start = {name: int(late in (name, "all")) for name in ("x", "w", "dy")}
    x, w = _whole((n_places, n_in), dtype, 1, start=start["x"]), _whole((n_experts, n_out, n_in), dtype, 2, start=start["w"])
    dy = _whole((n_places, n_out), dtype, 3, start=start["dy"])
    x[offsets[-1]:] = float("nan")
    dy[offsets[-1]:] = float("nan")
    y, dx, dw = _products(x, w, dy, offsets)
    assert torch.equal(kernels.expert_product(plan, x, w), y)
    got_dx, got_dw = kernels.expert_product_grad(plan, x, w, dy)
    assert torch.equal(got_dx, dx) and torch.equal(got_dw, dw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n_experts,n_places,rows,n_in,n_out", STARTS)
def test_results_that_start_between_units(n_experts, n_places, rows, n_in, n_out, dtype):
    """the entry points of the C interface take results of any start; the elements around them stay as they were"""
    plan, offsets = _uneven(n_experts, n_places, rows, 7)
    x, w, dy = _whole((n_places, n_in), dtype, 1), _whole((n_experts, n_out, n_in), dtype, 2), _whole((n_places, n_out), dtype, 3)
    t = kernels._panel_type("x", x)
    sizes = (t, n_places, n_experts, n_in, n_out)
    n_bytes = kernels._lib.load().splahip_expert_product_dw_workspace(*sizes)
    work = torch.empty(max(n_bytes, 16), dtype=torch.uint8, device="cuda")
    for name, operands, more, want in (("", (x, w), (), 0), ("_dx", (dy, w), (), 1), ("_dw", (dy, x), (work.data_ptr(), n_bytes), 2)):
        want = _products(x, w, dy, offsets)[want]
        around = torch.full((want.numel() + 2,), 77.0, dtype=dtype, device="cuda")
        out = around[1:-1].view(want.shape)
        kernels._launch(x.device, "splahip_expert_product" + name, *sizes, plan.offsets.data_ptr(), *(o.data_ptr() for o in operands), out.data_ptr(), *more)
        assert torch.equal(out, want) and around[0] == 77 and around[-1] == 77, name


# panels beyond 128 MB are streamed past the caches; a row's units a lane of back_grad's: 1, 2, 4, 8 and more
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [250, 500, 1001, 2047, 4001, 9000])
def test_streamed_panels(width, dtype):
    k, experts = 3, 7
    size = torch.empty(0, dtype=dtype).element_size()
    rows = (129 << 20) // (width * size * k) + 1
    assert rows * k * width * size > 128 << 20
    g = torch.Generator(device="cuda").manual_seed(width)
    e = torch.randint(-1, experts, (rows, k), generator=g, device="cuda", dtype=torch.int32)
    plan = kernels.route_sort(e, experts)
    end, order, place = int(plan.offsets[-1]), plan.order.long(), plan.place.long()
    weights = torch.randint(-2, 3, (rows, k), generator=g, device="cuda").float()
    x, y = _whole((rows, width), dtype, 1, 4), _whole((rows * k, width), dtype, 2, 4)
    y[end:] = float("nan")
    weights[place < 0] = float("nan")
    token, entry = order[:end] // k, order[:end]
    want = torch.zeros(rows * k, width, dtype=dtype, device="cuda")
    want[:end] = x[token]
    assert torch.equal(kernels.route_rows(plan, x), want)
    want[:end] = (x[token].float() * weights.reshape(-1)[entry, None]).to(dtype)
    assert torch.equal(kernels.route_rows(plan, x, weights), want)
    dy, dweights = kernels.route_back_grad(plan, y, weights, x)
    assert torch.equal(dy, want)
    plain, weighted, pairs = (torch.zeros(rows, width, device="cuda"), torch.zeros(rows, width, device="cuda"), torch.zeros(rows, k, device="cuda"))
    for j in range(k):
        here = place[:, j] >= 0
        mine = y[place[here, j]].float()
        plain[here] += mine
        weighted[here] += mine * weights[here, j, None]
        pairs[here, j] = (mine * x[here].float()).sum(1)
    assert torch.equal(dweights, pairs)
    assert torch.equal(kernels.route_back(plan, y), plain.to(dtype)) and torch.equal(kernels.route_back(plan, y, weights), weighted.to(dtype))
