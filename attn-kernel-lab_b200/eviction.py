"""Bounding a request's cache by what its tokens were attended to.

`extend_weights` adds up what the query rows of an extend (all of them, or the last ones as a window)
put on every cached position, from the log-sum-exp that `prefill_extend` returns with `pool_lse`; `paged_decode` with
`weights` goes on with the same accumulator token by token.  `evict_lightest` then shortens page-table
rows to the heaviest positions, in place, and lists the slots that became free.  The pool itself is
never moved: a slot is a page.

The reference has no counterpart; validation, errors, workspaces and streams are those of `ops`.
"""
from __future__ import annotations

import ctypes

import torch

from . import kernel
from .capability import DECODE_CAPABILITY, OperatorCapability
from .decode import (_INDEX, _KV, _Scratch, _call, _check_apart, _check_batch_vector, _check_decay, _check_heads, _check_rows,
                     _check_scale, _check_sizes, _check_table, _check_width, _declares, _need, _need_cuda, _overlap,
                     _pool_stride, _raise_on_status, _row_stride)
from .ops import _dtype_name, _reject, _same_device

__all__ = ["WeightsWorkspace", "evict_lightest", "extend_weights", "plan_weights_workspace"]


class WeightsWorkspace(_Scratch):
    """Capacity-reserved scratch of `extend_weights`; one call at a time (stream order) may use it."""

    def __init__(self, device, *, max_kv_len: int, max_q_len: int, q_heads: int, kv_heads: int):
        _check_sizes(max_kv_len=max_kv_len, max_q_len=max_q_len, q_heads=q_heads, kv_heads=kv_heads)
        self.plan = kernel.WeightsPlan(max_kv_len, max_q_len, q_heads, kv_heads)
        layout = kernel.WeightsLayout()
        kernel.check(kernel.load().akl_weights_layout(ctypes.byref(self.plan), ctypes.byref(layout)),
                     "akl_weights_layout")
        super().__init__(device, layout)
        self._plan_fields = (max_kv_len, max_q_len, q_heads, kv_heads)
        self._declared = _declares(q_heads, kv_heads, "extend_weights")


def plan_weights_workspace(device, *, max_kv_len: int, max_q_len: int, q_heads: int | None = None,
                           kv_heads: int | None = None, capability: OperatorCapability = DECODE_CAPABILITY):
    """A `WeightsWorkspace` for extends within the two maxima; heads default to 32:4 and are validated
    against the declared surface."""
    q_heads = 32 if q_heads is None else int(q_heads)
    kv_heads = 4 if kv_heads is None else int(kv_heads)
    _check_heads(q_heads, kv_heads, max(capability.head_dim), capability.kv_dtypes[0], "extend_weights", False,
                 capability)
    return WeightsWorkspace(device, max_kv_len=max_kv_len, max_q_len=max_q_len, q_heads=q_heads, kv_heads=kv_heads)


def _check_extend(q, k_pool, idx, prefix, lse, weights, weight_decay, workspace, sm_scale, capability) -> None:
    device = q.device if isinstance(q, torch.Tensor) else None
    _need("q", q, (torch.bfloat16,), 3, device, "[q_len, q_heads, head_dim]")
    if not isinstance(k_pool, torch.Tensor) or k_pool.dim() != 3:
        _need("k_pool", k_pool, _KV, 3, device, "[pool, kv_heads, head_dim]")
    q_len, q_heads, head_dim = q.shape
    kv_heads = k_pool.shape[1]
    _check_heads(q_heads, kv_heads, head_dim, _dtype_name(k_pool.dtype), "extend_weights", False, capability)
    _need("k_pool", k_pool, _KV, 3, device, "[pool, kv_heads, head_dim]")
    if k_pool.shape[2] != head_dim:
        _reject(f"k_pool head_dim {k_pool.shape[2]} must equal q head_dim {head_dim}", field="k_pool",
                value=int(k_pool.shape[2]), supported=head_dim)
    if q_len < 1 or k_pool.shape[0] < 1:
        _reject(f"q_len must be >= 1 and the pool must hold a slot, got {q_len} and {k_pool.shape[0]}", field="q_len",
                value=q_len, supported=">= 1")
    _check_rows("q", q, q_heads)
    _check_rows("k_pool", k_pool, kv_heads)
    _need("idx", idx, _INDEX, 1, device, "[kv_len]")
    kv_len = idx.shape[0]
    if kv_len < 1 or not idx.is_contiguous():
        _reject(f"idx must be contiguous and name at least one position, got {kv_len} with stride {idx.stride()}",
                field="idx", value=kv_len, supported=">= 1, contiguous")
    if kv_len >= 1 << 30 or q_len >= 1 << 27:
        _reject(f"{q_len} rows over {kv_len} positions: at most 2^27 - 1 over 2^30 - 1", field="idx", value=(q_len, kv_len),
                supported="< 2^27 rows, < 2^30 positions")
    if isinstance(prefix, bool) or not isinstance(prefix, int):
        _reject(f"prefix must be a Python int, got {type(prefix).__name__}", field="prefix",
                value=type(prefix).__name__, supported="int")
    if not 0 <= prefix <= kv_len - q_len:
        _reject(f"prefix={prefix} is outside [0, kv_len - q_len] = [0, {kv_len - q_len}] for kv_len={kv_len}, "
                f"q_len={q_len}", field="prefix", value=prefix, supported=(0, kv_len - q_len))
    _need("lse", lse, (torch.float32,), 2, device, "[q_len, q_heads]")
    if lse.shape != q.shape[:2] or not lse.is_contiguous():
        _reject(f"lse must be contiguous {(q_len, q_heads)}, got {tuple(lse.shape)} with strides "
                f"{tuple(lse.stride())}", field="lse", value=tuple(lse.shape), supported=(q_len, q_heads))
    _need("weights", weights, (torch.float32,), 1, device, "[kv_len]")
    if weights.shape[0] != kv_len or not weights.is_contiguous():
        _reject(f"weights must be contiguous [{kv_len}], got {tuple(weights.shape)} with stride {weights.stride()}",
                field="weights", value=tuple(weights.shape), supported=(kv_len,))
    _check_apart([("weights", weights)], [("q", q), ("k_pool", k_pool), ("idx", idx), ("lse", lse)])
    _check_decay(weight_decay)
    if sm_scale is not None:
        _check_scale(sm_scale)
    if workspace is not None:
        if not isinstance(workspace, WeightsWorkspace):
            _reject(f"workspace must be a WeightsWorkspace or None, got {type(workspace).__name__}",
                    field="workspace", value=type(workspace).__name__, supported="WeightsWorkspace | None")
        if not _same_device(workspace.device, device):
            _reject(f"workspace is on {workspace.device} but q is on {device}", field="workspace",
                    value=str(workspace.device), supported=str(device))


def extend_weights(q, k_pool, idx, prefix, lse, weights, *, weight_decay: float = 1.0, workspace=None, sm_scale=None,
                   capability: OperatorCapability = DECODE_CAPABILITY, check_status: bool = False):
    """Attention weight of every cached position under the query rows of an extend, in place.

    `q` [q_len, q_heads, 256] BF16, `k_pool` [pool, kv_heads, 256] BF16 or FP16, `idx` [kv_len] int32 or
    int64 and `prefix` as in `prefill_extend`: row t sees the positions 0 .. prefix + t.  `lse` [q_len,
    q_heads] FP32 base 2 is the log-sum-exp of the scores of the pool's own keys: what that call returned
    with `pool_lse=True` (or with `center_k=False`; the default's is over centred keys, and would put every row
    off by a factor of its own).  `weights` [kv_len] FP32 becomes `weight_decay` times itself plus

        sum over t, h with i <= prefix + t of 2^(sm_scale log2e <q[t, h], k_i> - lse[t, h]).

    A row whose `lse` is infinite adds nothing, whatever its `q` holds (it saw no key); a key that is not finite
    can make its own position's weight NaN, and no other's; a slot outside the pool gets no weight.
    `weights` shares no memory with an input.
    To judge by a window of w rows pass `q[-w:]`, `lse[-w:]` and `prefix + q_len - w`.  The sum has a
    fixed order: equal inputs give equal bits.

    Enqueues on the current stream and does not synchronise unless `check_status` (a debugging aid).
    Returns `weights`."""
    if workspace is not None and capability is DECODE_CAPABILITY:
        packed = _ordinary_extend(q, k_pool, idx, prefix, lse, weights, weight_decay, workspace, sm_scale)
        if packed is not None:
            try:
                _call(workspace.device_index, kernel.load().akl_extend_weights, "akl_extend_weights", packed)
            except kernel.NativeError as e:
                if e.code == kernel.AKL_ERR_INVALID:       # tensors that share memory: say which
                    _check_extend(q, k_pool, idx, prefix, lse, weights, weight_decay, workspace, sm_scale, capability)
                raise
            if check_status:
                _raise_on_status(workspace, "akl_extend_weights")
            return weights
    _check_extend(q, k_pool, idx, prefix, lse, weights, weight_decay, workspace, sm_scale, capability)
    device = q.device
    _need_cuda("extend_weights", device)
    lib = kernel.load()
    q_len, q_heads = q.shape[:2]
    kv_heads, kv_len = k_pool.shape[1], idx.shape[0]
    if workspace is None:
        workspace = WeightsWorkspace(device, max_kv_len=kv_len, max_q_len=q_len, q_heads=q_heads, kv_heads=kv_heads)
    else:
        p = workspace.plan
        if kv_len > p.max_kv_len or q_len > p.max_q_len or (q_heads, kv_heads) != (p.q_heads, p.kv_heads):
            from .quant import WorkspaceCapacityError

            raise WorkspaceCapacityError(
                f"extend of {q_len} rows over {kv_len} positions at {q_heads}:{kv_heads} heads is outside the "
                f"workspace plan (max_q_len={p.max_q_len}, max_kv_len={p.max_kv_len}, heads "
                f"{p.q_heads}:{p.kv_heads}); the allocation never changes")
    packed = kernel.pack_weights(
        q.data_ptr(), k_pool.data_ptr(), idx.data_ptr(), lse.data_ptr(), weights.data_ptr(), workspace._ptr,
        workspace._bytes, *workspace._plan_fields, k_pool.shape[0], q.stride(0) if q_len > 1 else q_heads * 256,
        _pool_stride(k_pool), q_len, kv_len, prefix, q_heads, kv_heads, _KV[k_pool.dtype], _INDEX[idx.dtype],
        0.0625 if sm_scale is None else sm_scale, weight_decay)
    _call(workspace.device_index, lib.akl_extend_weights, "akl_extend_weights", packed)
    if check_status:
        _raise_on_status(workspace, "akl_extend_weights")
    return weights


def _ordinary_extend(q, k_pool, idx, prefix, lse, weights, weight_decay, ws, sm_scale):
    """The packed call when every argument has its ordinary form, or None: the full checks then decide
    (as `decode._ordinary`)."""
    try:
        if type(ws) is not WeightsWorkspace or not ws._declared:
            return None
        index = ws.device_index
        max_kv_len, max_q_len, q_heads, kv_heads = ws._plan_fields
        q_len, heads, dim = q.shape
        pool, kv, kv_dim = k_pool.shape
        kv_len, = idx.shape
        kv_type, idx_type = _KV[k_pool.dtype], _INDEX[idx.dtype]
        if sm_scale is None:
            sm_scale = 0.0625
        if (index < 0 or heads != q_heads or kv != kv_heads or dim != 256 or kv_dim != 256 or not 1 <= q_len <= max_q_len
                or not 1 <= kv_len <= max_kv_len or pool < 1 or type(prefix) is not int or not 0 <= prefix <= kv_len - q_len
                or q.dtype is not torch.bfloat16 or lse.dtype is not torch.float32 or lse.shape != (q_len, heads)
                or weights.dtype is not torch.float32 or weights.shape != (kv_len,)
                or type(sm_scale) is not float or not 2.0 ** -126 <= sm_scale <= 2.0 ** 127
                or type(weight_decay) is not float or not 0.0 <= weight_decay <= 1.0
                or not (q.is_contiguous() and k_pool.is_contiguous() and idx.is_contiguous() and lse.is_contiguous()
                        and weights.is_contiguous())
                or not (q.get_device() == k_pool.get_device() == idx.get_device() == lse.get_device()
                        == weights.get_device() == index)):
            return None
        q_ptr, k_ptr, lse_ptr, weights_ptr = q.data_ptr(), k_pool.data_ptr(), lse.data_ptr(), weights.data_ptr()
        if (q_ptr | k_ptr) & 15 or (weights_ptr < lse_ptr + q_len * heads * 4 and lse_ptr < weights_ptr + kv_len * 4):
            return None
    except (AttributeError, TypeError, ValueError, KeyError):
        return None
    return kernel.pack_weights(q_ptr, k_ptr, idx.data_ptr(), lse_ptr, weights_ptr, ws._ptr, ws._bytes, *ws._plan_fields,
                               pool, heads * 256, kv * 256, q_len, kv_len, prefix, heads, kv, kv_type, idx_type, sm_scale,
                               weight_decay)


def _check_out(name, t, like, source_name) -> None:
    """An output table: the input itself, or a tensor of its shape that shares nothing with it."""
    if t is like:
        return
    _need(name, t, (like.dtype,), 2, like.device, "[rows, width]")
    if t.shape != like.shape:
        _reject(f"{name} shape {tuple(t.shape)} must equal {source_name}'s {tuple(like.shape)}", field=name,
                value=tuple(t.shape), supported=tuple(like.shape))
    _check_table(name, t)
    if _overlap(t, like) and (t.data_ptr() != like.data_ptr() or _row_stride(t) != _row_stride(like)):
        _reject(f"{name} overlaps {source_name} at another address: it must be {source_name} itself or a distinct "
                "allocation", field=name, value="overlaps", supported=f"{source_name} or a distinct allocation")


def _check_evict(page_table, weights, kv_lens, keep, first, last, rows, table_out, weights_out, lens_out, freed,
                 freed_lens) -> None:
    device = page_table.device if isinstance(page_table, torch.Tensor) else None
    _need("page_table", page_table, _INDEX, 2, device, "[rows, width]")
    _check_table("page_table", page_table)
    _need("weights", weights, (torch.float32,), 2, device, "[rows, >= width]")
    _check_table("weights", weights)
    width = page_table.shape[1]
    _check_width(page_table)
    if weights.shape[0] != page_table.shape[0] or weights.shape[1] < width:
        _reject(f"weights shape {tuple(weights.shape)} must cover the page table's {tuple(page_table.shape)}",
                field="weights", value=tuple(weights.shape), supported=tuple(page_table.shape))
    _need("kv_lens", kv_lens, _INDEX, 1, device, "[batch]")
    batch = kv_lens.shape[0]
    if batch < 1:
        _reject("kv_lens must hold at least one request", field="kv_lens", value=0, supported=">= 1")
    _check_batch_vector("kv_lens", kv_lens, batch, device)
    if rows is not None:
        _check_batch_vector("rows", rows, batch, device)
    elif page_table.shape[0] < batch:
        _reject(f"page_table has {page_table.shape[0]} rows for a batch of {batch}", field="page_table",
                value=int(page_table.shape[0]), supported=f">= {batch}")
    for name, value, low in (("keep", keep, 1), ("protect_first", first, 0), ("protect_last", last, 0)):
        if isinstance(value, bool) or not isinstance(value, int) or not low <= value < 1 << 31:
            _reject(f"{name} must be an int >= {low}, got {value!r}", field=name, value=value, supported=f">= {low}")
    if first + last > keep:
        _reject(f"protect_first={first} and protect_last={last} exceed keep={keep}", field="keep", value=keep,
                supported=f">= {first + last}")
    _check_out("page_table_out", table_out, page_table, "page_table")
    _check_out("weights_out", weights_out, weights, "weights")
    if lens_out is not kv_lens:
        _check_batch_vector("kv_lens_out", lens_out, batch, device)
        if lens_out.dtype != kv_lens.dtype:
            _reject(f"kv_lens_out dtype {_dtype_name(lens_out.dtype)} must equal kv_lens dtype "
                    f"{_dtype_name(kv_lens.dtype)}", field="kv_lens_out", value=_dtype_name(lens_out.dtype),
                    supported=_dtype_name(kv_lens.dtype))
        if _overlap(lens_out, kv_lens) and lens_out.data_ptr() != kv_lens.data_ptr():
            _reject("kv_lens_out overlaps kv_lens at another address", field="kv_lens_out", value="overlaps",
                    supported="kv_lens or a distinct allocation")
    if freed is not None:
        _need("freed", freed, (page_table.dtype,), 2, device, "[batch, >= width - keep]")
        if freed.shape[0] != batch or freed.shape[1] < max(1, width - keep):
            _reject(f"freed shape {tuple(freed.shape)} must be at least {(batch, max(1, width - keep))}", field="freed",
                    value=tuple(freed.shape), supported=(batch, max(1, width - keep)))
        _check_table("freed", freed)
    if freed_lens is not None:
        _need("freed_lens", freed_lens, (torch.int32,), 1, device, "[batch]")
        _check_batch_vector("freed_lens", freed_lens, batch, device)
    # an output in place of its input is the one thing they may share (the checks above)
    for name, t, own in (("page_table_out", table_out, page_table), ("weights_out", weights_out, weights),
                         ("kv_lens_out", lens_out, kv_lens)):
        _check_apart([(name, t)], [(other, u) for other, u in (("page_table", page_table), ("weights", weights),
                                                               ("kv_lens", kv_lens), ("rows", rows)) if u is not own])
    _check_apart([("page_table_out", table_out), ("weights_out", weights_out), ("kv_lens_out", lens_out), ("freed", freed),
                  ("freed_lens", freed_lens)], [])
    _check_apart([("freed", freed), ("freed_lens", freed_lens)],
                 [("page_table", page_table), ("weights", weights), ("kv_lens", kv_lens), ("rows", rows)])


def evict_lightest(page_table, weights, kv_lens, *, keep: int, protect_first: int = 0, protect_last: int = 0, rows=None,
                   page_table_out=None, weights_out=None, kv_lens_out=None, freed=None, freed_lens=None):
    """Shorten every request of more than `keep` positions to `keep`, by accumulated weight.

    `page_table` [rows, width] int32 or int64, `weights` [rows, >= width] FP32, `kv_lens` [batch] and
    `rows` [batch] int32 or int64 as in `paged_decode`.  The first `protect_first` and the last
    `protect_last` positions of a request stay; of the others the heaviest stay (NaN counts as -inf; of
    equal weights the lowest positions stay).  What stays moves to the front of its row in position
    order, slots and weights alike; the weights behind it, up to the old length, become 0; table entries
    behind it are left as they were.  A shorter request keeps its row.  Requests must name distinct rows.
    A length is cut to the table's width, and what comes back for it is at most that; for a length below 0 or
    a row outside the table it is 0.

    By default `page_table`, `weights` and `kv_lens` are changed in place; `page_table_out`,
    `weights_out` and `kv_lens_out` of the same shapes take the result instead (other rows, and what lies
    behind a request's old length, stay as they are).  But for that, no output shares memory with an input or
    another output; a table and its weights may lie side by side in one buffer.
    `freed` [batch, >= width - keep] receives the
    slots that go, in position order, and `freed_lens` [batch] int32 their number; both are allocated
    when not given.  Enqueues on the current stream and does not synchronise.

    Returns (page_table_out, weights_out, kv_lens_out, freed, freed_lens)."""
    table_out = page_table if page_table_out is None else page_table_out
    acc_out = weights if weights_out is None else weights_out
    lens_out = kv_lens if kv_lens_out is None else kv_lens_out
    index, packed = _ordinary_evict(page_table, weights, kv_lens, keep, protect_first, protect_last, rows, table_out,
                                    acc_out, lens_out, freed, freed_lens)
    if packed is None:
        _check_evict(page_table, weights, kv_lens, keep, protect_first, protect_last, rows, table_out, acc_out, lens_out,
                     freed, freed_lens)
        device = page_table.device
        _need_cuda("evict_lightest", device)
        index = device.index if device.index is not None else torch.cuda.current_device()
        batch, (table_rows, width) = kv_lens.shape[0], page_table.shape
        if freed is None:
            freed = torch.empty((batch, max(1, width - keep)), dtype=page_table.dtype, device=device)
        if freed_lens is None:
            freed_lens = torch.empty(batch, dtype=torch.int32, device=device)
        packed = kernel.pack_evict(
            page_table.data_ptr(), weights.data_ptr(), 0 if rows is None else rows.data_ptr(), kv_lens.data_ptr(),
            table_out.data_ptr(), acc_out.data_ptr(), lens_out.data_ptr(), freed.data_ptr(), freed_lens.data_ptr(),
            _row_stride(page_table), _row_stride(weights), _row_stride(table_out), _row_stride(acc_out),
            _row_stride(freed), batch, table_rows, width, freed.shape[1], keep, protect_first, protect_last,
            _INDEX[page_table.dtype], 0 if rows is None else _INDEX[rows.dtype], _INDEX[kv_lens.dtype])
    try:
        _call(index, kernel.load().akl_evict_lightest, "akl_evict_lightest", packed)
    except kernel.NativeError as e:
        if e.code == kernel.AKL_ERR_INVALID:               # tensors that share memory: say which
            _check_evict(page_table, weights, kv_lens, keep, protect_first, protect_last, rows, table_out, acc_out, lens_out,
                         freed, freed_lens)
        raise
    return table_out, acc_out, lens_out, freed, freed_lens


def _ordinary_evict(page_table, weights, kv_lens, keep, first, last, rows, table_out, acc_out, lens_out, freed,
                    freed_lens):
    """(device index, packed call) when every argument has its ordinary form, or (None, None): the full checks
    then decide (as `decode._ordinary`)."""
    no = None, None
    try:
        index = page_table.get_device()
        shape = page_table.shape
        table_rows, width = shape
        batch, = kv_lens.shape
        idx_type, lens_type = _INDEX[page_table.dtype], _INDEX[kv_lens.dtype]
        freed_rows, freed_width = freed.shape
        if (index < 0 or table_rows < 1 or not 1 <= width < 1 << 30 or table_rows >= 1 << 31 or batch < 1
                or weights.shape != shape or weights.dtype is not torch.float32
                or type(keep) is not int or type(first) is not int or type(last) is not int
                or first < 0 or last < 0 or not max(1, first + last) <= keep < 1 << 31
                or freed_rows != batch or not max(1, width - keep) <= freed_width < 1 << 31 or freed.dtype is not page_table.dtype
                or freed_lens.shape != (batch,) or freed_lens.dtype is not torch.int32
                or not (page_table.is_contiguous() and weights.is_contiguous() and kv_lens.is_contiguous()
                        and freed.is_contiguous() and freed_lens.is_contiguous())
                or not (weights.get_device() == kv_lens.get_device() == freed.get_device() == freed_lens.get_device()
                        == index)):
            return no
        table_ptr, weights_ptr, lens_ptr = page_table.data_ptr(), weights.data_ptr(), kv_lens.data_ptr()
        freed_ptr, count_ptr = freed.data_ptr(), freed_lens.data_ptr()
        table_out_ptr, acc_out_ptr, lens_out_ptr = table_ptr, weights_ptr, lens_ptr
        item = 8 if idx_type == 0 else 4
        table_bytes, acc_bytes = table_rows * width * item, table_rows * width * 4
        lens_bytes = batch * (8 if lens_type == 0 else 4)
        for out, src in ((table_out, page_table), (acc_out, weights), (lens_out, kv_lens)):
            if out is not src and (out.dtype is not src.dtype or out.shape != src.shape or not out.is_contiguous()
                                   or out.get_device() != index):
                return no
        if table_out is not page_table:
            table_out_ptr = table_out.data_ptr()
            if 0 < abs(table_out_ptr - table_ptr) < table_bytes:
                return no
        if acc_out is not weights:
            acc_out_ptr = acc_out.data_ptr()
            if 0 < abs(acc_out_ptr - weights_ptr) < acc_bytes:
                return no
        if lens_out is not kv_lens:
            lens_out_ptr = lens_out.data_ptr()
            if 0 < abs(lens_out_ptr - lens_ptr) < lens_bytes:
                return no
        rows_ptr = rows_type = rows_bytes = 0
        if rows is not None:
            rows_type = _INDEX[rows.dtype]
            if rows.shape != (batch,) or not rows.is_contiguous() or rows.get_device() != index:
                return no
            rows_ptr = rows.data_ptr()
            rows_bytes = batch * (8 if rows_type == 0 else 4)
            if lens_out_ptr < rows_ptr + rows_bytes and rows_ptr < lens_out_ptr + lens_bytes:
                return no
        elif table_rows < batch:
            return no
        freed_end, count_end = freed_ptr + batch * freed_width * item, count_ptr + batch * 4
        if freed_ptr < count_end and count_ptr < freed_end:
            return no
        for at, end in ((table_ptr, table_ptr + table_bytes), (table_out_ptr, table_out_ptr + table_bytes),
                        (weights_ptr, weights_ptr + acc_bytes), (acc_out_ptr, acc_out_ptr + acc_bytes),
                        (lens_ptr, lens_ptr + lens_bytes), (lens_out_ptr, lens_out_ptr + lens_bytes),
                        (rows_ptr, rows_ptr + rows_bytes)):
            if freed_ptr < end and at < freed_end or count_ptr < end and at < count_end:
                return no
    except (AttributeError, TypeError, ValueError, KeyError):
        return no
    return index, kernel.pack_evict(table_ptr, weights_ptr, rows_ptr, lens_ptr, table_out_ptr, acc_out_ptr, lens_out_ptr,
                                    freed_ptr, count_ptr, width, width, width, width, freed_width, batch, table_rows, width,
                                    freed_width, keep, first, last, idx_type, rows_type, lens_type)
