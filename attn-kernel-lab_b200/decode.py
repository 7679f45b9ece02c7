"""Decode attention over the pool that `prefill_extend` reads: one new token per request.

`paged_decode` takes a page table (one row of slots per request, position order, as an engine's
request-to-token table holds them) with lengths and rows in device memory, so a captured CUDA graph
follows them from step to step.  K and V are read once, in the pool's own type; long requests are
split over the whole GPU and joined by log-sum-exp.  With `weights` the call also records what the new
tokens attended to, which is what `eviction.evict_lightest` judges a cache by.

The reference covers the extend alone; validation order, error types, workspace and stream semantics
are those of `ops.prefill_extend`.  Nothing here loads the native library before validation passed.
"""
from __future__ import annotations

import ctypes

import torch

from . import kernel
from .capability import DECODE_CAPABILITY, CapabilityError, OperatorCapability, check_supported
from .ops import _dtype_name, _reject, _same_device

__all__ = ["DecodeWorkspace", "check_decode", "paged_decode", "plan_decode_workspace"]

_INDEX = {torch.int64: 0, torch.int32: 1}          # AKL_IDX_*
_KV = {torch.bfloat16: 0, torch.float16: 1}        # AKL_KV_*
_SCALES = 2.0 ** -126, 2.0 ** 127                  # sm_scale and sm_scale log2e are normal 32-bit numbers
_CHUNK = 64                                        # positions per chunk of recorded scores


class _Scratch:
    """One device allocation with a status word at its start, 1024-byte aligned."""

    def __init__(self, device, layout):
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.layout = layout
        self._bytes = int(layout.total_bytes)
        self._buf = torch.empty(self._bytes + 1024, dtype=torch.uint8, device=self.device)
        self._ptr = self._buf.data_ptr() + (-self._buf.data_ptr()) % 1024
        at = self._ptr - self._buf.data_ptr() + int(layout.off_status)
        self._status = self._buf[at:at + 256].view(torch.int32)
        self._status.zero_()
        self.device_index = -1 if self.device.type != "cuda" else self.device.index

    def base_ptr(self) -> int:
        return self._ptr

    def nbytes(self) -> int:
        return self._bytes

    def status(self) -> int:
        """First device-side error code recorded since allocation or the last reset (synchronises)."""
        return int(self._status[0].item())

    def reset_status(self) -> None:
        self._status.zero_()


def _check_sizes(**sizes) -> None:
    """Within the fields that carry them: ctypes would cut a larger number to its low bits without a word."""
    for name, value in sizes.items():
        low, high = (0, 1 << 40) if name == "max_weight_tokens" else (1, 1 << 31)
        if isinstance(value, bool) or not isinstance(value, int) or not low <= value < high:
            raise ValueError(f"{name} must be an int >= {low} and below 2^{high.bit_length() - 1}, got {value!r}")


class DecodeWorkspace(_Scratch):
    """Capacity-reserved scratch of `paged_decode`; one call at a time (stream order) may use it.

    `max_weight_tokens` bounds the positions of a batch whose weights are recorded: the sum of the
    lengths, each rounded up to 64.  0 reserves nothing for weights."""

    def __init__(self, device, *, max_requests: int, q_heads: int, kv_heads: int, max_weight_tokens: int = 0):
        _check_sizes(max_requests=max_requests, q_heads=q_heads, kv_heads=kv_heads,
                     max_weight_tokens=max_weight_tokens)
        self.plan = kernel.DecodePlan(max_requests, q_heads, kv_heads, 0, max_weight_tokens)
        layout = kernel.DecodeLayout()
        kernel.check(kernel.load().akl_decode_layout(ctypes.byref(self.plan), ctypes.byref(layout)),
                     "akl_decode_layout")
        super().__init__(device, layout)
        self._plan_fields = (max_requests, q_heads, kv_heads, 0, max_weight_tokens)
        self._declared = _declares(q_heads, kv_heads, "decode")


def _declares(q_heads: int, kv_heads: int, mode: str) -> bool:
    """Whether the default surface has these heads."""
    try:
        _check_heads(q_heads, kv_heads, 256, "bfloat16", mode, False, DECODE_CAPABILITY)
    except CapabilityError:
        return False
    return True


def _check_heads(q_heads: int, kv_heads: int, head_dim: int, kv_dtype: str, mode: str, return_lse: bool,
                 capability: OperatorCapability) -> None:
    check_supported(head_dim=head_dim, q_heads=q_heads, kv_heads=kv_heads, page_size=1, mode=mode,
                    mask="bottom_right_causal", kv_dtype=kv_dtype, return_lse=return_lse, capability=capability)
    if q_heads > 8 * kv_heads:
        _reject(f"q_heads={q_heads} over kv_heads={kv_heads}: at most 8 query heads may share a kv head",
                field="q_heads", value=q_heads, supported=f"<= {8 * kv_heads}")


def plan_decode_workspace(device, *, max_requests: int, q_heads: int | None = None, kv_heads: int | None = None,
                          max_weight_tokens: int = 0, capability: OperatorCapability = DECODE_CAPABILITY):
    """A `DecodeWorkspace` for batches of up to `max_requests`; heads default to 32:4 and are validated
    against the declared surface."""
    q_heads = 32 if q_heads is None else int(q_heads)
    kv_heads = 4 if kv_heads is None else int(kv_heads)
    _check_heads(q_heads, kv_heads, max(capability.head_dim), capability.kv_dtypes[0], "decode", False, capability)
    return DecodeWorkspace(device, max_requests=max_requests, q_heads=q_heads, kv_heads=kv_heads,
                           max_weight_tokens=max_weight_tokens)


def _need(name, t, dtypes, dims, device, what) -> None:
    """Type, rank, dtype and device of one tensor argument."""
    if not isinstance(t, torch.Tensor):
        _reject(f"{name} must be a torch.Tensor, got {type(t).__name__}", field=name, value=type(t).__name__,
                supported="torch.Tensor")
    if t.dim() != dims:
        _reject(f"{name} must be {dims}-D {what}, got {t.dim()}-D with shape {tuple(t.shape)}", field=name,
                value=tuple(t.shape), supported=what)
    if t.dtype not in dtypes:
        names = tuple(_dtype_name(d) for d in dtypes)
        _reject(f"{name} dtype must be {' or '.join(names)}, got {_dtype_name(t.dtype)}", field=name,
                value=_dtype_name(t.dtype), supported=names)
    if t.device != device and not _same_device(t.device, device):
        _reject(f"{name} is on {t.device} but q is on {device}: every operand of one call must live on one device",
                field=name, value=str(t.device), supported=str(device))


def _check_rows(name, t, heads) -> None:
    """[rows, heads, 256] with dense heads and channels; rows may lie further apart (a slice of a fused
    projection, some heads of a pool), a multiple of 16 bytes."""
    s = t.stride()
    if (s[2] != 1 or (heads > 1 and s[1] != 256)
            or (t.shape[0] > 1 and (s[0] % 8 or s[0] < heads * 256))):
        _reject(f"{name} strides {tuple(s)}: heads and channels must be dense and rows a multiple of 8 elements "
                f"apart, without overlap", field=name, value=tuple(s), supported="(multiple of 8, 256, 1)")
    if t.data_ptr() & 15 and t.device.type != "meta":
        _reject(f"{name} must start on a 16-byte boundary", field=name, value=t.data_ptr() & 15, supported=0)


def _check_scale(sm_scale) -> None:
    if isinstance(sm_scale, bool) or not isinstance(sm_scale, (int, float)):
        _reject(f"sm_scale must be a real number or None, got {type(sm_scale).__name__}", field="sm_scale",
                value=type(sm_scale).__name__, supported="float | None")
    if not _SCALES[0] <= sm_scale <= _SCALES[1]:
        _reject(f"sm_scale must be positive, finite and within 32 bits, got {sm_scale!r}", field="sm_scale", value=sm_scale,
                supported=_SCALES)


def _check_decay(weight_decay) -> None:
    if isinstance(weight_decay, bool) or not isinstance(weight_decay, (int, float)) or not 0.0 <= weight_decay <= 1.0:
        _reject(f"weight_decay must be a number in [0, 1], got {weight_decay!r}", field="weight_decay",
                value=weight_decay, supported="[0, 1]")


def _overlap(a, b) -> bool:
    """Whether two tensors share memory, or may: rows side by side in one buffer are told apart, other mixtures
    of rows are not (as the C entries look at it)."""
    if a.device.type == "meta" or b.device.type == "meta" or not a.numel() or not b.numel():
        return False

    def span(t):                       # address, rows, bytes of one, bytes from row to row
        item = t.element_size()
        rows = t.shape[0] if t.dim() > 1 else 1
        inner = list(zip(t.shape, t.stride()))[t.dim() > 1:]
        return t.data_ptr(), rows, (sum((n - 1) * s for n, s in inner) + 1) * item, (t.stride(0) if rows > 1 else 0) * item

    (a0, a_rows, a_bytes, a_pitch), (b0, b_rows, b_bytes, b_pitch) = span(a), span(b)
    if a0 + (a_rows - 1) * a_pitch + a_bytes <= b0 or b0 + (b_rows - 1) * b_pitch + b_bytes <= a0:
        return False
    pitch = a_pitch or b_pitch
    if not pitch or (a_pitch and b_pitch and a_pitch != b_pitch):
        return True
    apart = (b0 - a0) % pitch
    return apart < a_bytes or apart + b_bytes > pitch


def _check_apart(outputs, inputs) -> None:
    """Every output has memory of its own: lists of (name, tensor or None)."""
    outputs = [(name, t) for name, t in outputs if t is not None]
    for i, (name, t) in enumerate(outputs):
        for other, u in inputs + outputs[:i]:
            if u is not None and _overlap(t, u):
                _reject(f"{name} must not overlap {other}", field=name, value=f"overlaps {other}",
                        supported="memory of its own")


def _row_stride(t) -> int:
    """Elements from row to row of a 2-D tensor (of one row: its width, so that a stride of no meaning
    does not travel)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _check_table(name, t) -> None:
    if t.shape[0] < 1 or t.shape[1] < 1:
        _reject(f"{name} must have at least one row and one column, got {tuple(t.shape)}", field=name,
                value=tuple(t.shape), supported=">= [1, 1]")
    if (t.stride(1) != 1 and t.shape[1] > 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        _reject(f"{name} strides {tuple(t.stride())}: a row must be dense and rows must not overlap", field=name,
                value=tuple(t.stride()), supported="(>= width, 1)")
    if max(t.shape) >= 1 << 31:
        _reject(f"{name} shape {tuple(t.shape)} exceeds 32 bits", field=name, value=tuple(t.shape), supported="< 2^31")


def _check_width(table) -> None:
    """Positions are 32-bit in the kernels, and loops over them run past the end."""
    if table.shape[1] >= 1 << 30:
        _reject(f"page_table rows of {table.shape[1]} entries: at most 2^30 - 1", field="page_table",
                value=int(table.shape[1]), supported="< 2^30")


def _check_batch_vector(name, t, batch, device) -> None:
    _need(name, t, _INDEX, 1, device, "[batch]")
    if t.shape[0] != batch:
        _reject(f"{name} has {t.shape[0]} entries for a batch of {batch}", field=name, value=int(t.shape[0]),
                supported=batch)
    if batch > 1 and t.stride(0) != 1:
        _reject(f"{name} must be contiguous", field=name, value=tuple(t.stride()), supported="contiguous")


def check_decode(q, k_pool, v_pool, page_table, kv_lens, *, rows=None, workspace=None, out=None, lse_out=None,
                 weights=None, weight_decay: float = 1.0, sm_scale=None, return_lse: bool = False,
                 capability: OperatorCapability = DECODE_CAPABILITY) -> tuple:
    """Validate one decode call without touching device memory; returns (batch, q_heads, kv_heads).

    Raises `CapabilityError` naming the field; order: ranks, dtypes and devices, the declared surface,
    strides, lengths and rows, options, outputs, weights, workspace."""
    device = q.device if isinstance(q, torch.Tensor) else None
    _need("q", q, (torch.bfloat16,), 3, device, "[batch, q_heads, head_dim]")
    if not isinstance(k_pool, torch.Tensor) or k_pool.dim() != 3:
        _need("k_pool", k_pool, _KV, 3, device, "[pool, kv_heads, head_dim]")
    batch, q_heads, head_dim = q.shape
    kv_heads = k_pool.shape[1]
    _check_heads(q_heads, kv_heads, head_dim, _dtype_name(k_pool.dtype), "decode", return_lse, capability)
    _need("k_pool", k_pool, _KV, 3, device, "[pool, kv_heads, head_dim]")
    _need("v_pool", v_pool, (k_pool.dtype,), 3, device, "[pool, kv_heads, head_dim]")
    if k_pool.shape[2] != head_dim:
        _reject(f"k_pool head_dim {k_pool.shape[2]} must equal q head_dim {head_dim}", field="k_pool",
                value=int(k_pool.shape[2]), supported=head_dim)
    if v_pool.shape != k_pool.shape:
        _reject(f"v_pool shape {tuple(v_pool.shape)} must equal k_pool shape {tuple(k_pool.shape)}: one pool "
                "geometry, two planes", field="v_pool", value=tuple(v_pool.shape), supported=tuple(k_pool.shape))
    if batch < 1:
        _reject("q must hold at least one request: an empty batch must be skipped by the caller", field="q",
                value=batch, supported=">= 1")
    if not 1 <= k_pool.shape[0] < 1 << 31:
        _reject(f"k_pool must hold 1 to 2^31 - 1 slots, got {k_pool.shape[0]}", field="k_pool",
                value=tuple(k_pool.shape), supported="1 .. 2^31 - 1")
    _check_rows("q", q, q_heads)
    _check_rows("k_pool", k_pool, kv_heads)
    _check_rows("v_pool", v_pool, kv_heads)
    _need("page_table", page_table, _INDEX, 2, device, "[rows, width]")
    _check_table("page_table", page_table)
    _check_width(page_table)
    _check_batch_vector("kv_lens", kv_lens, batch, device)
    if rows is not None:
        _check_batch_vector("rows", rows, batch, device)
    elif page_table.shape[0] < batch:
        _reject(f"page_table has {page_table.shape[0]} rows for a batch of {batch}", field="page_table",
                value=int(page_table.shape[0]), supported=f">= {batch}")
    if sm_scale is not None:
        _check_scale(sm_scale)
    if out is not None:
        _need("out", out, (torch.bfloat16,), 3, device, "[batch, q_heads, head_dim]")
        if out.shape != q.shape or not out.is_contiguous():
            _reject(f"out must be contiguous {tuple(q.shape)}, got {tuple(out.shape)} with strides "
                    f"{tuple(out.stride())}", field="out", value=tuple(out.shape), supported=tuple(q.shape))
        if out.data_ptr() & 15:
            _reject("out must start on a 16-byte boundary", field="out", value=out.data_ptr() & 15, supported=0)
        if _overlap(out, q):
            _reject("out must not overlap q", field="out", value="aliases q", supported="memory of its own")
    if lse_out is not None:
        if not return_lse:
            _reject("lse_out was supplied but return_lse=False: a destination for an output that will not be "
                    "produced is a caller mistake", field="lse_out", value="supplied", supported="return_lse=True")
        _need("lse_out", lse_out, (torch.float32,), 2, device, "[batch, q_heads]")
        if lse_out.shape != q.shape[:2] or not lse_out.is_contiguous():
            _reject(f"lse_out must be contiguous {(batch, q_heads)}, got {tuple(lse_out.shape)}", field="lse_out",
                    value=tuple(lse_out.shape), supported=(batch, q_heads))
    if weights is not None:
        _need("weights", weights, (torch.float32,), 2, device, "[table rows, >= width]")
        _check_table("weights", weights)
        if weights.shape[0] != page_table.shape[0] or weights.shape[1] < page_table.shape[1]:
            _reject(f"weights shape {tuple(weights.shape)} must cover the page table's {tuple(page_table.shape)}",
                    field="weights", value=tuple(weights.shape), supported=tuple(page_table.shape))
        _check_decay(weight_decay)
    _check_apart([("out", out), ("lse_out", lse_out), ("weights", weights)],
                 [("q", q), ("k_pool", k_pool), ("v_pool", v_pool), ("page_table", page_table), ("kv_lens", kv_lens),
                  ("rows", rows)])
    if workspace is not None:
        if not isinstance(workspace, DecodeWorkspace):
            _reject(f"workspace must be a DecodeWorkspace or None, got {type(workspace).__name__}",
                    field="workspace", value=type(workspace).__name__, supported="DecodeWorkspace | None")
        if not _same_device(workspace.device, device):
            _reject(f"workspace is on {workspace.device} but q is on {device}", field="workspace",
                    value=str(workspace.device), supported=str(device))
    return batch, q_heads, kv_heads


def _admit(ws: DecodeWorkspace, batch: int, q_heads: int, kv_heads: int, weights: bool) -> None:
    p = ws.plan
    if batch > p.max_requests or (q_heads, kv_heads) != (p.q_heads, p.kv_heads) or (weights and not p.max_weight_tokens):
        from .quant import WorkspaceCapacityError

        raise WorkspaceCapacityError(
            f"decode of {batch} requests at {q_heads}:{kv_heads} heads{' with weights' if weights else ''} is outside "
            f"the workspace plan (max_requests={p.max_requests}, heads {p.q_heads}:{p.kv_heads}, "
            f"max_weight_tokens={p.max_weight_tokens}); the allocation never changes")


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def _call(index: int, fn, name: str, packed: bytes) -> None:
    """One native call on CUDA device `index` and its current stream."""
    if index == torch.cuda.current_device():
        code = fn(packed, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            code = fn(packed, _raw_stream(index))
    if code:
        kernel.check(code, name)


def _need_cuda(name, device) -> None:
    if device.type != "cuda":
        raise RuntimeError(f"{name} needs CUDA tensors, got q on {device}: this operator has no CPU path")


def paged_decode(q, k_pool, v_pool, page_table, kv_lens, *, rows=None, workspace=None, out=None, lse_out=None,
                 weights=None, weight_decay: float = 1.0, sm_scale=None, return_lse: bool = False,
                 capability: OperatorCapability = DECODE_CAPABILITY, check_status: bool = False):
    """Attention of one new token per request over its cached positions, its own among them.

    `q` [batch, q_heads, 256] BF16; `k_pool`, `v_pool` [pool, kv_heads, 256] BF16 or FP16; `page_table`
    [rows, width] int32 or int64 pool slots in position order; `kv_lens` [batch] and `rows` [batch] (the
    table row of each request, default its own index) int32 or int64, read on the device.  A length is
    cut to the table's width; a request of length 0 (or less), or with a row outside the table, gives
    zeros and an LSE of -inf; a slot outside the pool is skipped.  Rows of `q`, pool rows and table rows
    may be strided.  `out`, `lse_out` and `weights` share no memory with each other or with an input.

    `weights` [rows, >= width] FP32: position i of each request's row becomes `weight_decay` times itself
    plus the sum over the q heads of what they put on it (the sum over i of that is q_heads); 0
    overwrites.  Requests of one call must then name distinct rows, except those of length 0.

    `workspace` from `plan_decode_workspace`; without one the call allocates its own (with `weights`
    sized by the table's width).  Enqueues on the current stream and does not synchronise, unless
    `check_status` (a debugging aid): then it waits and raises `NativeError` when a bounded device-side
    wait ran out, or when the lengths exceed the plan's `max_weight_tokens` (the outputs are whole then;
    from the first request on that does not fit, rows of `weights` are left as they were).

    Returns `out` [batch, q_heads, 256] BF16, or `(out, lse)` with the base-2 `lse` [batch, q_heads]."""
    if workspace is not None and out is not None and capability is DECODE_CAPABILITY:
        packed = _ordinary(q, k_pool, v_pool, page_table, kv_lens, rows, workspace, out, lse_out, weights, weight_decay,
                           sm_scale, return_lse)
        if packed is not None:
            try:
                _call(workspace.device_index, kernel.load().akl_paged_decode, "akl_paged_decode", packed)
            except kernel.NativeError as e:
                if e.code == kernel.AKL_ERR_INVALID:       # tensors that share memory: say which
                    check_decode(q, k_pool, v_pool, page_table, kv_lens, rows=rows, workspace=workspace, out=out,
                                 lse_out=lse_out, weights=weights, weight_decay=weight_decay, sm_scale=sm_scale,
                                 return_lse=return_lse, capability=capability)
                raise
            if check_status:
                _raise_on_status(workspace, "akl_paged_decode")
            return (out, lse_out) if return_lse else out
    batch, q_heads, kv_heads = check_decode(
        q, k_pool, v_pool, page_table, kv_lens, rows=rows, workspace=workspace, out=out, lse_out=lse_out,
        weights=weights, weight_decay=weight_decay, sm_scale=sm_scale, return_lse=return_lse, capability=capability)
    device = q.device
    _need_cuda("paged_decode", device)
    lib = kernel.load()
    table_rows, width = page_table.shape
    if workspace is None:
        workspace = DecodeWorkspace(device, max_requests=batch, q_heads=q_heads, kv_heads=kv_heads,
                                    max_weight_tokens=0 if weights is None else batch * (-(-width // _CHUNK) * _CHUNK))
    else:
        _admit(workspace, batch, q_heads, kv_heads, weights is not None)
    if out is None:
        out = torch.empty((batch, q_heads, 256), dtype=torch.bfloat16, device=device)
    if return_lse and lse_out is None:
        lse_out = torch.empty((batch, q_heads), dtype=torch.float32, device=device)
    packed = kernel.pack_decode(
        q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), page_table.data_ptr(),
        0 if rows is None else rows.data_ptr(), kv_lens.data_ptr(), out.data_ptr(),
        lse_out.data_ptr() if return_lse else 0, 0 if weights is None else weights.data_ptr(),
        workspace._ptr, workspace._bytes, *workspace._plan_fields, k_pool.shape[0],
        q.stride(0) if batch > 1 else q_heads * 256, _pool_stride(k_pool), _pool_stride(v_pool),
        _row_stride(page_table), 0 if weights is None else _row_stride(weights),
        batch, q_heads, kv_heads, table_rows, width, _KV[k_pool.dtype], _INDEX[page_table.dtype],
        0 if rows is None else _INDEX[rows.dtype], _INDEX[kv_lens.dtype],
        0.0625 if sm_scale is None else sm_scale, 1.0 if weights is None else weight_decay)
    _call(workspace.device_index, lib.akl_paged_decode, "akl_paged_decode", packed)
    if check_status:
        _raise_on_status(workspace, "akl_paged_decode")
    return (out, lse_out) if return_lse else out


def _ordinary(q, k_pool, v_pool, page_table, kv_lens, rows, ws, out, lse_out, weights, weight_decay, sm_scale,
              return_lse):
    """The packed call when every argument has its ordinary form -- contiguous tensors of the expected
    types on one GPU, a plan that admits them -- or None: `check_decode` then looks closer, and either
    accepts or says what is wrong.  A single step is short enough for the checks to show (they were 15
    of 26 us a call), and these few comparisons are the same ones; that outputs share no memory with
    anything else is left to the C entry, which refuses before it launches."""
    try:
        if type(ws) is not DecodeWorkspace or not ws._declared:
            return None
        index = ws.device_index
        max_requests, q_heads, kv_heads, _, max_tokens = ws._plan_fields
        q_shape, pool_shape = q.shape, k_pool.shape
        batch, heads, dim = q_shape
        pool, kv, kv_dim = pool_shape
        table_shape = page_table.shape
        table_rows, width = table_shape
        kv_type, idx_type, lens_type = _KV[k_pool.dtype], _INDEX[page_table.dtype], _INDEX[kv_lens.dtype]
        if (index < 0 or heads != q_heads or kv != kv_heads or dim != 256 or kv_dim != 256
                or not 1 <= batch <= max_requests or not 1 <= pool < 1 << 31 or not 1 <= table_rows < 1 << 31
                or not 1 <= width < 1 << 30 or v_pool.shape != pool_shape or v_pool.dtype is not k_pool.dtype
                or q.dtype is not torch.bfloat16 or out.dtype is not torch.bfloat16 or out.shape != q_shape
                or kv_lens.shape != (batch,)
                or not (q.is_contiguous() and k_pool.is_contiguous() and v_pool.is_contiguous()
                        and page_table.is_contiguous() and kv_lens.is_contiguous() and out.is_contiguous())
                or not (q.get_device() == k_pool.get_device() == v_pool.get_device() == page_table.get_device()
                        == kv_lens.get_device() == out.get_device() == index)):
            return None
        rows_ptr = rows_type = lse_ptr = weights_ptr = 0
        if rows is not None:
            rows_type = _INDEX[rows.dtype]
            if rows.shape != (batch,) or not rows.is_contiguous() or rows.get_device() != index:
                return None
            rows_ptr = rows.data_ptr()
        elif table_rows < batch:
            return None
        if return_lse:
            if (lse_out.dtype is not torch.float32 or lse_out.shape != (batch, heads) or not lse_out.is_contiguous()
                    or lse_out.get_device() != index):
                return None
            lse_ptr = lse_out.data_ptr()
        elif lse_out is not None:
            return None
        if weights is None:
            weight_decay = 1.0
        else:
            if (not max_tokens or weights.dtype is not torch.float32 or weights.shape != table_shape
                    or not weights.is_contiguous() or weights.get_device() != index
                    or type(weight_decay) is not float or not 0.0 <= weight_decay <= 1.0):
                return None
            weights_ptr = weights.data_ptr()
        if sm_scale is None:
            sm_scale = 0.0625
        elif type(sm_scale) is not float or not 2.0 ** -126 <= sm_scale <= 2.0 ** 127:
            return None
        q_ptr, k_ptr, v_ptr, out_ptr = q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), out.data_ptr()
        row = heads * 256
        if (q_ptr | k_ptr | v_ptr | out_ptr) & 15 or abs(out_ptr - q_ptr) < batch * row * 2:
            return None
    except (AttributeError, TypeError, ValueError, KeyError):
        return None
    return kernel.pack_decode(
        q_ptr, k_ptr, v_ptr, page_table.data_ptr(), rows_ptr, kv_lens.data_ptr(), out_ptr, lse_ptr, weights_ptr, ws._ptr,
        ws._bytes, *ws._plan_fields, pool, row, kv * 256, kv * 256, width, width if weights_ptr else 0, batch, heads, kv, table_rows, width,
        kv_type, idx_type, rows_type, lens_type, sm_scale, weight_decay)


def _pool_stride(t) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1] * 256


def _raise_on_status(ws, where: str) -> None:
    from .ops import _raise_on_status as raise_on_status

    raise_on_status(ws, kernel, where)
