"""Python face of the kernel-level C ABI for device-resident operands held in torch tensors.

PyTorch-ROCm is plumbing only (device memory, the current HIP stream, torch.distributed); every compute call goes
through libspla_amd.so.  Tensors are passed as raw device pointers (`tensor.data_ptr()`), int32 tensors stand in
for uint32 words where torch has no unsigned dtype.
"""
from __future__ import annotations

import ctypes as C
from array import array
from operator import attrgetter
from types import SimpleNamespace

import torch
from torch.autograd import forward_ad

from . import _lib
from .ops import binop_id, scalar_bits, selop_id, type_id

_TORCH_DTYPE = {0: torch.int32, 1: torch.int32, 2: torch.float32}  # uint32 words travel as int32 bit patterns


def torch_dtype(t):
    return _TORCH_DTYPE[type_id(t)]


def _ptr(t):
    if t is None:
        return None
    assert t.is_cuda and t.is_contiguous(), "device-resident contiguous tensor expected"
    return C.c_void_p(t.data_ptr())


def current_stream_ptr():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


class CsrPlan:
    """Wave-tile work decomposition of one device CSR matrix (splahip_csr_plan_*)."""

    def __init__(self, n_rows: int, nnz: int, Ap: torch.Tensor, n_cols: int = 0, Aj: torch.Tensor = None, Ax: torch.Tensor = None):
        """Ap alone gives the wave-tile decomposition of the CSR kernels.  With (n_cols, Aj, Ax) the plan also builds the
        sliced-ELL + hot-column copy that mxv uses for associative op_add (attach_sell)."""
        self.n_rows, self.nnz = int(n_rows), int(nnz)
        self.sell = None
        self.cob = None
        self._h = C.c_void_p()
        _lib.call("splahip_csr_plan_create", C.byref(self._h), self.n_rows, self.nnz, _ptr(Ap), current_stream_ptr())
        nb, nl = C.c_uint32(), C.c_uint32()
        _lib.call("splahip_csr_plan_info", self._h, C.byref(nb), C.byref(nl))
        self.n_items, self.n_long = nb.value, nl.value
        self.n_blocks = self.n_items  # work items (one per wavefront)
        if Aj is not None and Ax is not None and n_cols:
            self.attach_sell(n_cols, Ap, Aj, Ax)

    def attach_sell(self, n_cols: int, Ap: torch.Tensor, Aj: torch.Tensor, Ax: torch.Tensor):
        """sliced-ELL + hot-column copy of the matrix (values included: rebuild when the matrix changes)"""
        _lib.call("splahip_csr_plan_attach_sell", self._h, int(n_cols), _ptr(Ap), _ptr(Aj) if self.nnz else None, _ptr(Ax) if self.nnz else None,
                  current_stream_ptr())
        a, b, c, d = C.c_uint32(), C.c_uint32(), C.c_uint32(), C.c_uint32()
        _lib.call("splahip_csr_plan_sell_info", self._h, C.byref(a), C.byref(b), C.byref(c), C.byref(d))
        u, xb = C.c_int(), C.c_uint32()
        _lib.call("splahip_csr_plan_sell_values", self._h, C.byref(u), C.byref(xb))
        self.sell = {"slices": a.value, "slots": b.value, "hot_columns": c.value, "long_rows": d.value, "uniform_values": bool(u.value)} if a.value else None

    def attach_cob(self, n_cols: int, Ap: torch.Tensor, Aj: torch.Tensor, Ax: torch.Tensor, row_bits: int = 0, tile_chunks: int = 0):
        """column-ordered-blocks copy of the matrix (values included: rebuild when the matrix changes); mxv then uses it for every
        op_add with an LDS atomic.  row_bits / tile_chunks: 0 = the library's defaults."""
        _lib.call("splahip_csr_plan_attach_cob", self._h, int(n_cols), _ptr(Ap), _ptr(Aj) if self.nnz else None, _ptr(Ax) if self.nnz else None,
                  int(row_bits), int(tile_chunks), current_stream_ptr())
        a, b, c, d = C.c_uint32(), C.c_uint32(), C.c_uint32(), C.c_uint32()
        _lib.call("splahip_csr_plan_cob_info", self._h, C.byref(a), C.byref(b), C.byref(c), C.byref(d))
        nr, nh, hr, by = C.c_uint32(), C.c_uint32(), C.c_uint32(), C.c_uint64()
        _lib.call("splahip_csr_plan_cob_layout", self._h, C.byref(nr), C.byref(nh), C.byref(hr), C.byref(by))
        hs, ns = C.c_uint32(), C.c_uint32()
        _lib.call("splahip_csr_plan_cob_slots", self._h, C.byref(hs), C.byref(ns))
        hot = C.c_uint32()
        _lib.call("splahip_csr_plan_cob_relabel", self._h, C.byref(hot))
        self.cob = {"tiles": a.value, "chunks": b.value, "ranges_in_pieces": c.value, "slots_per_range": d.value, "natural_slots": ns.value, "ranges": nr.value,
                    "hub_ranges": nh.value, "hub_rows": hr.value, "bytes": by.value, "relabelled_hot_columns": hot.value} if a.value else None
        return self.cob

    def mask_probe(self):
        """what the last masked call over the blocks found when it probed its mask on the device (blocking): {"selected_entries", "served_by_rows"}"""
        se, by = C.c_uint64(), C.c_int()
        _lib.call("splahip_csr_plan_cob_probe", self._h, C.byref(se), C.byref(by))
        return {"selected_entries": se.value, "served_by_rows": bool(by.value)}

    def set_uniform_values(self, is_uniform: bool, value_bits: int = 0):
        """the owner of the value array says: every stored value is the word `value_bits` (or not)"""
        _lib.call("splahip_csr_plan_set_uniform_values", self._h, 1 if is_uniform else 0, int(value_bits) & 0xFFFFFFFF)

    def hint_products(self, products: int):
        """products of the next vxm_pull over this (transposed) plan (vxm_probe's count)"""
        _lib.call("splahip_csr_plan_hint_products", self._h, int(products))

    def first_hit(self):
        """what the plan's last BFS-like call did (mxv_first_hit.hpp): {"taken": ran on the first-hit kernel, "uniform": verdict of the last finished pass over
        v (None: none yet), "nonzeros": its non-zero count, "tail_pct": share of the sampled selected entries in rows the walk would enter past their fourth entry}"""
        t, u, n, p = C.c_int(), C.c_int(), C.c_uint32(), C.c_uint32()
        _lib.call("splahip_csr_plan_first_hit", self._h, C.byref(t), C.byref(u), C.byref(n), C.byref(p))
        return {"taken": bool(t.value), "uniform": None if u.value < 0 else bool(u.value), "nonzeros": n.value, "tail_pct": p.value}

    def footprint(self):
        """device bytes held for the matrix besides its CSR arrays: {"plan", "sliced_ell", "column_ordered_blocks"}"""
        a, b, c = C.c_uint64(), C.c_uint64(), C.c_uint64()
        _lib.call("splahip_csr_plan_footprint", self._h, C.byref(a), C.byref(b), C.byref(c))
        return {"plan": a.value, "sliced_ell": b.value, "column_ordered_blocks": c.value}

    @property
    def handle(self):
        return self._h

    def close(self):
        if self._h:
            _lib.call("splahip_csr_plan_destroy", self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def mxv_masked(plan: CsrPlan, t, n_cols, Ap, Aj, Ax, mask, v, r, op_mult, op_add, op_select, init, early_exit=False):
    """r = mask-selected rows of (M x v) over (op_mult, op_add), written for every row (splahip_mxv_masked)."""
    tid = type_id(t)
    _lib.call("splahip_mxv_masked", plan.handle, tid, plan.n_rows, int(n_cols), _ptr(Ap), _ptr(Aj), _ptr(Ax),
              _ptr(mask), _ptr(v), _ptr(r), binop_id(op_mult), binop_id(op_add), selop_id(op_select),
              scalar_bits(init, tid), 1 if early_exit else 0, current_stream_ptr())
    return r


def mxv_variant(t, op_mult, op_add, early_exit=False, plan: CsrPlan = None) -> str:
    """name of the kernel splahip_mxv_masked picks (with `plan`: its sliced-ELL copy taken into account)"""
    if plan is not None:
        return _lib.call("splahip_mxv_variant_of", plan.handle, type_id(t), binop_id(op_mult), binop_id(op_add), 1 if early_exit else 0).decode()
    return _lib.call("splahip_mxv_variant", type_id(t), binop_id(op_mult), binop_id(op_add), 1 if early_exit else 0).decode()


def csr_transpose(n_rows, n_cols, Ap, Aj, Ax):
    """Device CSR of the transpose (rows ascending inside every column): returns (Tp, Tj, Tx)."""
    nnz = int(Aj.numel())
    Tp = torch.empty(n_cols + 1, dtype=torch.int32, device=Ap.device)
    Tj = torch.empty(max(nnz, 1), dtype=torch.int32, device=Ap.device)[:nnz]
    Tx = torch.empty(max(nnz, 1), dtype=Ax.dtype, device=Ap.device)[:nnz]
    _lib.call("splahip_csr_transpose", int(n_rows), int(n_cols), nnz, _ptr(Ap), _ptr(Aj) if nnz else None, _ptr(Ax) if nnz else None,
              _ptr(Tp), _ptr(Tj) if nnz else None, _ptr(Tx) if nnz else None, current_stream_ptr())
    return Tp, Tj, Tx


def vxm_probe(vi, Ap):
    prod, srt = C.c_uint64(), C.c_int()
    _lib.call("splahip_vxm_probe", int(vi.numel()), _ptr(vi) if vi.numel() else None, _ptr(Ap), C.byref(prod), C.byref(srt), current_stream_ptr())
    return prod.value, bool(srt.value)


def vxm_pull(plan_T: CsrPlan, t, n_rows, n_cols, Tp, Tj, Tx, mask, vi, vx, op_mult, op_add, op_select, identity=False):
    """Pull form of vxm over the transposed CSR; returns (ri, rx) index-sorted COO tensors."""
    tid = type_id(t)
    ri = torch.empty(max(n_cols, 1), dtype=torch.int32, device=mask.device)
    rx = torch.empty(max(n_cols, 1), dtype=torch_dtype(t), device=mask.device)
    cnt = C.c_uint32()
    _lib.call("splahip_vxm_pull", plan_T.handle, tid, int(n_rows), int(n_cols), _ptr(Tp), _ptr(Tj), _ptr(Tx), _ptr(mask),
              int(vi.numel()), _ptr(vi), _ptr(vx), 1 if identity else 0, _ptr(ri), _ptr(rx), C.byref(cnt),
              binop_id(op_mult), binop_id(op_add), selop_id(op_select), current_stream_ptr())
    return ri[:cnt.value], rx[:cnt.value]


def vxm_push(t, n_rows, n_cols, Ap, Aj, Ax, mask, vi, vx, op_mult, op_add, op_select):
    """Push form of vxm (expand / stable sort / fold); returns (ri, rx) index-sorted COO tensors."""
    tid = type_id(t)
    ri = torch.empty(max(n_cols, 1), dtype=torch.int32, device=mask.device)
    rx = torch.empty(max(n_cols, 1), dtype=torch_dtype(t), device=mask.device)
    cnt = C.c_uint32()
    _lib.call("splahip_vxm_push", tid, int(n_rows), int(n_cols), _ptr(Ap), _ptr(Aj), _ptr(Ax), _ptr(mask),
              int(vi.numel()), _ptr(vi) if vi.numel() else None, _ptr(vx) if vi.numel() else None, _ptr(ri), _ptr(rx), C.byref(cnt),
              binop_id(op_mult), binop_id(op_add), selop_id(op_select), current_stream_ptr())
    return ri[:cnt.value], rx[:cnt.value]


def vxm_push_small(t, n_rows, n_cols, Ap, Aj, Ax, mask, vi, vx, op_mult, op_add, op_select, max_products):
    """Single-synchronisation push for small frontiers: returns (done, products, sorted, ri, rx); when the device-side product count
    exceeds max_products nothing is computed (done = False) and the caller falls back to vxm_push / vxm_pull."""
    tid = type_id(t)
    ri = torch.empty(max(n_cols, 1), dtype=torch.int32, device=mask.device)
    rx = torch.empty(max(n_cols, 1), dtype=torch_dtype(t), device=mask.device)
    cnt, products, srt, done = C.c_uint32(), C.c_uint64(), C.c_int(), C.c_int()
    _lib.call("splahip_vxm_push_small", tid, int(n_rows), int(n_cols), _ptr(Ap), _ptr(Aj), _ptr(Ax), _ptr(mask),
              int(vi.numel()), _ptr(vi) if vi.numel() else None, _ptr(vx) if vi.numel() else None, _ptr(ri), _ptr(rx), int(max_products), C.byref(cnt),
              C.byref(products), C.byref(srt), C.byref(done), binop_id(op_mult), binop_id(op_add), selop_id(op_select), current_stream_ptr())
    return bool(done.value), int(products.value), bool(srt.value), ri[:cnt.value], rx[:cnt.value]


def _adopt(ptr, n, dtype):
    """Copy a library-allocated device array of n words into a torch tensor and release the original."""
    out = torch.empty(max(n, 1), dtype=dtype, device="cuda")[:n]
    if n:
        _lib.call("splahip_memcpy_d2d", _ptr(out), ptr, n * 4, current_stream_ptr())
        torch.cuda.current_stream().synchronize()
    if ptr:
        _lib.call("splahip_free", ptr)
    return out


def mxmT_masked(t, n_rows, M, A, B, op_mult, op_add, op_select, init):
    """R = (A x B^T) .mask; M, A, B are (Ap, Aj, Ax) device CSR triples; returns the CSR triple of R."""
    tid = type_id(t)
    Rp = torch.empty(n_rows + 1, dtype=torch.int32, device="cuda")
    pj, px, nnz = C.c_void_p(), C.c_void_p(), C.c_uint32()
    mask_nnz = int(M[1].numel())
    args = []
    for (p_, j_, x_) in (M, A, B):
        args += [_ptr(p_), _ptr(j_) if j_.numel() else None, _ptr(x_) if x_.numel() else None]
    _lib.call("splahip_mxmT_masked", tid, int(n_rows), mask_nnz, *args, _ptr(Rp), C.byref(pj), C.byref(px), C.byref(nnz),
              binop_id(op_mult), binop_id(op_add), selop_id(op_select), scalar_bits(init, tid), current_stream_ptr())
    return Rp, _adopt(pj, nnz.value, torch.int32), _adopt(px, nnz.value, torch_dtype(t))


class LibraryCsr:
    """A CSR result whose column / value arrays are still the library's allocations (no copy): `.nnz`, `.Rp` (tensor), raw
    device pointers `.pj / .px`; `.adopt(t)` copies them into torch tensors, `.free()` releases them (splahip_free)."""

    def __init__(self, Rp, pj, px, nnz):
        self.Rp, self.pj, self.px, self.nnz = Rp, pj, px, int(nnz)

    def adopt(self, t):
        out = (self.Rp, _adopt(self.pj, self.nnz, torch.int32), _adopt(self.px, self.nnz, torch_dtype(t)))
        self.pj = self.px = None
        return out

    def free(self):
        for q in (self.pj, self.px):
            if q:
                _lib.call("splahip_free", q)
        self.pj = self.px = None


def mxm(t, a_rows, b_cols, A, B, op_mult, op_add, init, block_products=0, adopt=True):
    """R = A x B (ESC); returns ((Rp, Rj, Rx), products), or (LibraryCsr, products) with adopt=False (what a C host sees:
    the call itself, without this wrapper's copy of the result into torch tensors)."""
    tid = type_id(t)
    Rp = torch.empty(a_rows + 1, dtype=torch.int32, device="cuda")
    pj, px, nnz, prod = C.c_void_p(), C.c_void_p(), C.c_uint32(), C.c_uint64()
    args = []
    for (p_, j_, x_) in (A, B):
        args += [_ptr(p_), _ptr(j_) if j_.numel() else None, _ptr(x_) if x_.numel() else None]
    _lib.call("splahip_mxm", tid, int(a_rows), int(b_cols), *args, _ptr(Rp), C.byref(pj), C.byref(px), C.byref(nnz), C.byref(prod),
              binop_id(op_mult), binop_id(op_add), scalar_bits(init, tid), int(block_products), current_stream_ptr())
    raw = LibraryCsr(Rp, pj, px, nnz.value)
    return (raw.adopt(t) if adopt else raw), prod.value


# ---- panels: products with a routing matrix, the experts' products, the norm over many tensors --------------------------------------------------------------
# A panel is a contiguous 2-D tensor [rows, width] of float32, float16 or bfloat16.  The calls are asynchronous on the current stream of the tensors' device,
# record no autograd graph (the gradients have calls of their own) and can be captured into a graph.  An operand whose gradient would be lost by that (it requires
# one while gradients are recorded, or carries a forward-mode tangent) is refused: such calls belong under torch.no_grad() or into an autograd.Function.

_LARGEST = torch.finfo(torch.float32).max
_PANEL_TYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


_entries = {}
# the current stream's handle and device without the Python objects and checks around them (a fifth of a small call's time; the tensors have initialised the GPU), where
# torch has these
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _launch(device, name, *args):
    """call an entry point of the panel operators on the current stream of `device` (they read no environment knobs)"""
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(_lib.load(), name)
    index = device.index
    if index == _current_device():
        status = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            status = fn(*args, _raw_stream(index))
    if status:
        raise _lib.SplaHipError(status, _lib.load().splahip_last_error().decode(errors="replace"))


_requires_grad, _is_neg = attrgetter("requires_grad"), torch.Tensor.is_neg
_forward_recorded = getattr(torch._C, "_is_fwd_grad_enabled", lambda: True)
_forward = forward_ad if hasattr(forward_ad, "_current_level") else SimpleNamespace(_current_level=0)  # (below 0: no tangents anywhere; saves the look at each tensor)


def _has_tangent(t):
    return _forward_recorded() and forward_ad.unpack_dual(t).tangent is not None


def _differentiated(t):
    return t.requires_grad and torch.is_grad_enabled() or _forward._current_level >= 0 and _has_tangent(t)


def _checked(name, t, dtype, shape, device=None):
    """t is a contiguous tensor on the GPU of this type, shape and device, and no gradient of it is asked for, else ValueError; returns its address"""
    if (isinstance(t, torch.Tensor) and t.dtype == dtype and t.shape == shape and t.is_cuda and (device is None or t.device == device) and t.is_contiguous()
            and not t.is_neg() and not (t.requires_grad and _differentiated(t)) and (_forward._current_level < 0 or not _has_tangent(t))):
        return t.data_ptr()
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name}: a tensor expected, not {type(t).__name__}")
    if _differentiated(t):
        raise ValueError(f"{name}: its gradient would be lost, since the call records no autograd graph: call it under torch.no_grad() or in an autograd.Function, or detach the tensor")
    if t.is_neg():
        raise ValueError(f"{name}: its values are those of its memory negated: resolve_neg() expected")
    if t.dtype != dtype or t.shape != shape:
        raise ValueError(f"{name}: {dtype} of shape {tuple(shape)} expected, not {t.dtype} of {tuple(t.shape)}")
    if not t.is_cuda or (device is not None and t.device != device):
        raise ValueError(f"{name}: a tensor on {device if t.is_cuda else 'the GPU'} expected, not on {t.device}")
    raise ValueError(f"{name}: a contiguous tensor expected, not one of strides {t.stride()}")


def _panel_type(name, t):
    if not isinstance(t, torch.Tensor) or t.dtype not in _PANEL_TYPE:
        raise ValueError(f"{name}: a tensor of float32, float16 or bfloat16 expected, not {t.dtype if isinstance(t, torch.Tensor) else type(t).__name__}")
    return _PANEL_TYPE[t.dtype]


def _width(name, t, rows):
    if t.dim() != 2 or t.shape[0] != rows:
        raise ValueError(f"{name}: a panel of {rows} rows expected, not shape {tuple(t.shape)}")
    return t.shape[1]


class RoutePlan:
    """The entries of a routing matrix (n_rows tokens x n_experts, per_row entries a row) sorted by expert (route_sort).

    offsets  int32 [n_experts + 1]     the places of expert e are offsets[e] .. offsets[e + 1]
    order    int32 [n_rows * per_row]  the entry (row * per_row + choice) at each place, -1 behind the last entry
    place    int32 [n_rows, per_row]   the place of each entry, -1 for no entry
    """

    __slots__ = ("offsets", "order", "place", "n_rows", "per_row", "n_places", "n_experts", "device")

    def __init__(self, offsets: torch.Tensor, order: torch.Tensor, place: torch.Tensor):
        if not isinstance(offsets, torch.Tensor) or offsets.dim() != 1 or not isinstance(place, torch.Tensor) or place.dim() != 2:
            raise ValueError("a plan's offsets are an int32 tensor [n_experts + 1], its places one of [n_rows, per_row]")
        self._set(offsets, order, place)
        _checked("offsets", offsets, torch.int32, (self.n_experts + 1,))
        _checked("order", order, torch.int32, (self.n_places,), self.device)
        _checked("place", place, torch.int32, (self.n_rows, self.per_row), self.device)

    def _set(self, offsets, order, place):
        self.offsets, self.order, self.place, self.device = offsets, order, place, offsets.device
        self.n_rows, self.per_row = place.shape
        self.n_places, self.n_experts = self.n_rows * self.per_row, offsets.shape[0] - 1
        return self


def route_sort(experts: torch.Tensor, n_experts: int) -> RoutePlan:
    """Sort a router's choices by expert, stable: experts int32 [n_rows, per_row], any number outside [0, n_experts) meaning no entry (padding)."""
    if not isinstance(experts, torch.Tensor) or experts.dim() != 2:
        raise ValueError("experts: an int32 tensor [n_rows, per_row] expected")
    n_rows, per_row = experts.shape
    src = _checked("experts", experts, torch.int32, (n_rows, per_row))
    n_experts, device = int(n_experts), experts.device
    if not 1 <= n_experts <= 2048 or per_row < 1 or n_rows * per_row >= 1 << 31:
        raise ValueError(f"route_sort serves 1 .. 2048 experts, at least one entry a row and fewer than 2^31 entries, not {n_experts}, {per_row}, {n_rows * per_row}")
    offsets = torch.empty(n_experts + 1, dtype=torch.int32, device=device)
    order = torch.empty(n_rows * per_row, dtype=torch.int32, device=device)
    place = torch.empty_like(experts)
    n_bytes = _lib.load().splahip_route_sort_workspace(n_rows, per_row, n_experts)
    work = torch.empty(n_bytes, dtype=torch.uint8, device=device) if n_bytes else None
    _launch(device, "splahip_route_sort", n_rows, per_row, n_experts, src, offsets.data_ptr(), order.data_ptr(), place.data_ptr(),
            work.data_ptr() if n_bytes else None, n_bytes)
    return RoutePlan.__new__(RoutePlan)._set(offsets, order, place)


def _weights(plan, weights):
    return None if weights is None else _checked("weights", weights, torch.float32, (plan.n_rows, plan.per_row), plan.device)


def route_rows(plan: RoutePlan, x: torch.Tensor, weights: torch.Tensor = None) -> torch.Tensor:
    """The rows of x [n_rows, width] in expert order: out[p] = w * x[row of the entry at p], 0 behind the last entry; weights float32 [n_rows, per_row] or None
    for 1.  Gradients: dx = route_back(plan, dout, weights), dweights = route_back_grad(plan, dout, weights, x)[1]."""
    t = _panel_type("x", x)
    width = _width("x", x, plan.n_rows)
    src, w = _checked("x", x, x.dtype, (plan.n_rows, width), plan.device), _weights(plan, weights)
    out = torch.empty(plan.n_places, width, dtype=x.dtype, device=plan.device)
    _launch(plan.device, "splahip_route_rows", t, plan.n_rows, plan.per_row, plan.n_experts, width, plan.offsets.data_ptr(), plan.place.data_ptr(), w, src, out.data_ptr())
    return out


def route_back(plan: RoutePlan, y: torch.Tensor, weights: torch.Tensor = None) -> torch.Tensor:
    """The rows of y [n_places, width], in expert order, summed back: out[row] = sum of w * y[place] over the row's entries, 0 for a row without any."""
    t = _panel_type("y", y)
    width = _width("y", y, plan.n_places)
    src, w = _checked("y", y, y.dtype, (plan.n_places, width), plan.device), _weights(plan, weights)
    out = torch.empty(plan.n_rows, width, dtype=y.dtype, device=plan.device)
    _launch(plan.device, "splahip_route_back", t, plan.n_rows, plan.per_row, width, plan.place.data_ptr(), w, src, out.data_ptr())
    return out


def route_back_grad(plan: RoutePlan, y: torch.Tensor, weights: torch.Tensor, dout: torch.Tensor):
    """The gradients (dy, dweights) of route_back(plan, y, weights): dy[p] = w * dout[row] (0 behind the last entry), dweights = <dout[row], y[place]>."""
    t = _panel_type("y", y)
    width = _width("y", y, plan.n_places)
    src = _checked("y", y, y.dtype, (plan.n_places, width), plan.device)
    w = _checked("weights", weights, torch.float32, (plan.n_rows, plan.per_row), plan.device)
    g = _checked("dout", dout, y.dtype, (plan.n_rows, width), plan.device)
    dy, dweights = torch.empty_like(y), torch.empty_like(weights)
    _launch(plan.device, "splahip_route_back_grad", t, plan.n_rows, plan.per_row, plan.n_experts, width, plan.offsets.data_ptr(), plan.place.data_ptr(), w, src, g,
            dy.data_ptr(), dweights.data_ptr())
    return dy, dweights


def _matrices(plan, w, dtype):
    """the address of w [n_experts, n_out, n_in], n_out and n_in"""
    shape = w.shape if isinstance(w, torch.Tensor) else ()
    if len(shape) != 3 or shape[0] != plan.n_experts or shape[1] < 1 or shape[2] < 1:
        raise ValueError(f"w: matrices [{plan.n_experts}, n_out, n_in] expected, not {tuple(shape) if isinstance(w, torch.Tensor) else type(w).__name__}")
    return _checked("w", w, dtype, shape, plan.device), shape[1], shape[2]


def expert_product(plan: RoutePlan, x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    """y[p] = w[e] @ x[p] for the places p of expert e: x [n_places, n_in] in expert order, w [n_experts, n_out, n_in] of the same type.  Rows behind the last
    entry become 0, whatever x holds there."""
    t = _panel_type("x", x)
    src_w, n_out, n_in = _matrices(plan, w, x.dtype)
    src = _checked("x", x, x.dtype, (plan.n_places, n_in), plan.device)
    y = torch.empty(plan.n_places, n_out, dtype=x.dtype, device=plan.device)
    _launch(plan.device, "splahip_expert_product", t, plan.n_places, plan.n_experts, n_in, n_out, plan.offsets.data_ptr(), src, src_w, y.data_ptr())
    return y


def expert_product_grad(plan: RoutePlan, x: torch.Tensor, w: torch.Tensor, dy: torch.Tensor, need=(True, True)):
    """The gradients (dx, dw) of expert_product(plan, x, w): dx[p] = w[e]^T @ dy[p] (0 behind the last entry), dw[e] = sum of dy[p] x[p]^T over the expert's
    places (0 for an expert without any).  need: which of the two to compute, None stands in the place of the other."""
    t = _panel_type("x", x)
    src_w, n_out, n_in = _matrices(plan, w, x.dtype)
    src = _checked("x", x, x.dtype, (plan.n_places, n_in), plan.device)
    src_dy = _checked("dy", dy, x.dtype, (plan.n_places, n_out), plan.device)
    dx = dw = None
    args, offsets = (t, plan.n_places, plan.n_experts, n_in, n_out), plan.offsets.data_ptr()
    if need[0]:
        dx = torch.empty_like(x)
        _launch(plan.device, "splahip_expert_product_dx", *args, offsets, src_dy, src_w, dx.data_ptr())
    if need[1]:
        dw = torch.empty_like(w)
        n_bytes = _lib.load().splahip_expert_product_dw_workspace(*args)
        work = torch.empty(n_bytes, dtype=torch.uint8, device=plan.device) if n_bytes else None
        _launch(plan.device, "splahip_expert_product_dw", *args, offsets, src_dy, src, dw.data_ptr(), work.data_ptr() if n_bytes else None, n_bytes)
    return dx, dw


class _Words:
    """a list of numbers as an array that an entry point reads"""

    __slots__ = ("words", "ptr")

    def __init__(self, code, numbers):
        self.words = array(code, numbers)
        self.ptr = self.words.buffer_info()[0]


def _arrays(name, tensors):
    """address, length and type arrays of the tensors, all on one device, and the device"""
    try:
        types = _Words("i", [_PANEL_TYPE[t.dtype] for t in tensors])
        places = set(map(torch.Tensor.get_device, tensors))
        fits = len(places) == 1 and places.pop() >= 0 and all(map(torch.Tensor.is_contiguous, tensors))
        fits = fits and not (torch.is_grad_enabled() and any(map(_requires_grad, tensors))) and not (_forward._current_level >= 0 and any(map(_has_tangent, tensors)))
    except (AttributeError, KeyError, TypeError):
        fits = False
    if not fits:  # say which
        for i, t in enumerate(tensors):
            _panel_type(f"{name}[{i}]", t)
            _checked(f"{name}[{i}]", t, t.dtype, t.shape, tensors[0].device)
    return _Words("Q", list(map(torch.Tensor.data_ptr, tensors))), _Words("Q", list(map(torch.Tensor.numel, tensors))), types, tensors[0].device


def global_norm(tensors) -> torch.Tensor:
    """The 2-norm over all elements of all tensors (a list of contiguous float32 / float16 / bfloat16 tensors of any shapes on one device), a float32 scalar on
    that device (infinity for a norm beyond float32).  Squares and sums in 64 bits; the order of the sum is fixed."""
    tensors = list(tensors)
    if not tensors:
        raise ValueError("tensors: at least one expected")
    ptrs, lengths, types, device = _arrays("tensors", tensors)
    norm = torch.empty((), dtype=torch.float32, device=device)
    n_bytes = _lib.load().splahip_global_norm_workspace(len(tensors), lengths.ptr)
    work = torch.empty(n_bytes, dtype=torch.uint8, device=device)
    _launch(device, "splahip_global_norm", len(tensors), ptrs.ptr, lengths.ptr, types.ptr, work.data_ptr(), n_bytes, norm.data_ptr())
    return norm


def clip_global_norm(tensors, limit: float, out=None, norm: torch.Tensor = None) -> torch.Tensor:
    """Scale the tensors by min(1, limit / norm), in place or into the list `out` (same lengths and types), and return the norm before.  A NaN or infinity among the
    values scales nothing, and the result is NaN or infinity.  Finite values are scaled whatever their norm (it is used in 64 bits): the result is infinity for one
    beyond float32 too.  norm: a float32 scalar on the device to use instead (the norm over several devices' tensors, say); NaN or infinity there scales nothing."""
    tensors, limit = list(tensors), float(limit)
    if not tensors:
        raise ValueError("tensors: at least one expected")
    if not 0.0 <= limit <= _LARGEST:
        raise ValueError(f"limit: a largest norm of 0 or more that float32 holds expected, not {limit}")
    ptrs, lengths, types, device = _arrays("tensors", tensors)
    out_ptrs = ptrs
    if out is not None:
        out = list(out)
        for name, list_ in (("tensors", tensors), ("out", out)):  # (in place the sign stays with the tensor, and the norm does not see it)
            if any(map(_is_neg, list_)):
                raise ValueError(f"{name}: the values of one are those of its memory negated: resolve_neg() expected")
        if len(out) != len(tensors):
            raise ValueError(f"out: {len(tensors)} tensors expected, not {len(out)}")
        out_ptrs, out_lengths, out_types, out_device = _arrays("out", out)
        if out_device != device or out_types.words != types.words or out_lengths.words != lengths.words:
            raise ValueError("out: tensors of the same lengths, types and device as the tensors expected")
    if norm is not None:
        _checked("norm", norm, torch.float32, (), device)
        work, n_bytes, given = None, 0, 1
    else:
        norm = torch.empty((), dtype=torch.float32, device=device)
        n_bytes, given = _lib.load().splahip_global_norm_workspace(len(tensors), lengths.ptr), 0
        work = torch.empty(n_bytes, dtype=torch.uint8, device=device)
    _launch(device, "splahip_clip_global_norm", len(tensors), ptrs.ptr, out_ptrs.ptr, lengths.ptr, types.ptr, limit, given, work.data_ptr() if work is not None else None,
            n_bytes, norm.data_ptr())
    torch.autograd.graph.increment_version(tensors if out is None else out)  # (a graph that kept one of them for its backward pass notices)
    return norm
