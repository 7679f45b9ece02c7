"""Sizes, addresses and numbers at the edge of what decode, attention weights and eviction take, on the host."""
import ctypes

import pytest
import torch

import decode_ref
from test_decode_rejection import _c_decode, _evict, short  # noqa: F401 - a fixture


@pytest.fixture(scope="module")
def K(pkg):
    from attn_kernel_lab_b200 import kernel

    return kernel


def _wide(width, rows=1):
    """A table of that width without its memory."""
    return torch.empty((rows, width), dtype=torch.int32, device="meta")


def _on_meta(**over):
    return {k: v.to("meta") if isinstance(v, torch.Tensor) else v for k, v in dict(decode_ref.case([5], 24, 4, device="cpu"), **over).items()}


def test_page_tables_of_2_30_columns_are_refused(pkg, K):
    for width, fits in (((1 << 30) - 1, True), (1 << 30, False), ((1 << 31) - 1, False)):
        kw = _on_meta(page_table=_wide(width), rows=None)
        if fits:
            assert pkg.check_decode(**kw) == (1, 24, 4)
        else:
            with pytest.raises(pkg.CapabilityError) as e:
                pkg.paged_decode(**kw)
            assert e.value.field == "page_table"
            with pytest.raises(pkg.CapabilityError) as e:
                pkg.evict_lightest(**_evict(page_table=_wide(width), weights=torch.empty((1, width), device="meta"),
                                            kv_lens=torch.empty(1, dtype=torch.int64, device="meta")))
            assert e.value.field == "page_table"
    # in C the check comes before any CUDA call (a case that passes it would launch)
    c = _c_decode(K, table_width=1 << 30, table_stride=1 << 30)
    assert K.load().akl_paged_decode(ctypes.byref(c), None) == -2


def test_the_short_form_leaves_wide_tables_alone(pkg, short):      # noqa: F811
    decode, _, seen = short
    ws = pkg.plan_decode_workspace("cpu", max_requests=1, q_heads=24, kv_heads=4)
    ws.device_index = 0
    host = decode_ref.case([5], 24, 4, device="cpu")
    host_out = torch.zeros((1, 24, 256), dtype=torch.bfloat16)

    class Table:
        """A page table of any width, as far as the short form looks."""
        dtype = torch.int32

        def __init__(self, width):
            self.shape = torch.Size((1, width))

        def is_contiguous(self):
            return True

        def get_device(self):
            return 0

        def data_ptr(self):
            return 4096

    def packed(width):
        return decode._ordinary(host["q"], host["k_pool"], host["v_pool"], Table(width), host["kv_lens"], None, ws, host_out, None,
                                None, 1.0, None, False)

    assert packed((1 << 30) - 1) is not None and packed(1 << 30) is None and packed((1 << 31) - 1) is None


def test_plans_refuse_sizes_that_their_fields_cut(pkg, K):
    """2^32 + 5 requests would be planned for as 5, and 2^60 tokens take a workspace of nearly nothing."""
    for over in (dict(max_requests=1 << 31), dict(max_requests=(1 << 32) + 5), dict(max_weight_tokens=1 << 40),
                 dict(max_weight_tokens=1 << 60), dict(max_weight_tokens=1 << 64), dict(q_heads=(1 << 32) + 24)):
        with pytest.raises(ValueError):
            pkg.DecodeWorkspace("meta", **dict(dict(max_requests=1, q_heads=24, kv_heads=4), **over))
    for over in (dict(max_kv_len=(1 << 32) + 64), dict(max_q_len=(1 << 32) + 1)):
        with pytest.raises(ValueError):
            pkg.WeightsWorkspace("meta", **dict(dict(max_kv_len=64, max_q_len=1, q_heads=24, kv_heads=4), **over))
    lib, L = K.load(), K.DecodeLayout()
    for tokens, code in (((1 << 40) - 1, 0), (1 << 40, -2), (1 << 60, -2), ((1 << 63) - 1, -2), (-1, -1)):
        assert lib.akl_decode_layout(ctypes.byref(K.DecodePlan(4, 64, 8, 0, tokens)), ctypes.byref(L)) == code
        if code == 0:
            assert L.total_bytes - L.off_scores >= tokens * 64 * 4


def test_extends_beyond_32_bit_positions_are_refused(pkg):
    n = 1 << 30
    kw = dict(k_pool=torch.empty((4, 4, 256), dtype=torch.bfloat16, device="meta"), prefix=0)
    for rows, size in ((1, n), (1 << 27, 1 << 28), (1, (1 << 32) + 3)):
        q = torch.empty((rows, 24, 256), dtype=torch.bfloat16, device="meta")
        with pytest.raises(pkg.CapabilityError) as e:
            pkg.extend_weights(q=q, idx=torch.empty(size, dtype=torch.int32, device="meta"),
                               lse=torch.empty((rows, 24), device="meta"), weights=torch.empty(size, device="meta"), **kw)
        assert e.value.field == "idx"


# ---- outputs have memory of their own -----------------------------------------------------------
def _bytes_of(t):
    return t.numel() * t.element_size()


def _sharing(args, output, other, at):
    """The call with `output` moved so that its first byte is byte `at` of `other`'s memory (both 16-byte aligned)."""
    u, t = args[other], args[output]
    buf = torch.zeros(-(-_bytes_of(u) // 16) * 16 + _bytes_of(t) + 32, dtype=torch.uint8)
    base = -buf.data_ptr() % 16
    a, b = (buf[base + o:base + o + _bytes_of(x)].view(x.dtype).view(x.shape) for o, x in ((0, u), (at, t)))
    a.copy_(u)
    return dict(args, **{other: a, output: b})


def _decode_args():
    c = decode_ref.case([5, 9], 24, 4, device="cpu")
    c["page_table"] = c["page_table"].contiguous()
    return dict(c, out=torch.zeros(2, 24, 256, dtype=torch.bfloat16), lse_out=torch.zeros(2, 24), return_lse=True,
                weights=torch.zeros(c["page_table"].shape))


_DECODE_PAIRS = [(o, i) for o in ("out", "lse_out", "weights") for i in ("q", "k_pool", "v_pool", "page_table", "kv_lens", "rows")]
_DECODE_PAIRS += [("lse_out", "out"), ("weights", "out"), ("weights", "lse_out")]


@pytest.mark.parametrize("output,other", _DECODE_PAIRS)
def test_decode_outputs_share_no_memory(pkg, output, other):
    args = _decode_args()
    assert pkg.check_decode(**args) == (2, 24, 4)
    last = (_bytes_of(args[other]) - 1) // 16 * 16
    for at in (0, last):
        with pytest.raises(pkg.CapabilityError) as e:
            pkg.paged_decode(**_sharing(args, output, other, at))
        assert e.value.field == output
    assert pkg.check_decode(**_sharing(args, output, other, last + 16)) == (2, 24, 4)


@pytest.mark.parametrize("other", ["q", "k_pool", "idx", "lse"])
def test_extend_weights_output_shares_no_memory(pkg, other):
    args = dict(q=torch.zeros(4, 24, 256, dtype=torch.bfloat16), k_pool=torch.zeros(40, 4, 256, dtype=torch.float16),
                idx=torch.arange(20), lse=torch.zeros(4, 24), weights=torch.zeros(20))
    last = (_bytes_of(args[other]) - 1) // 16 * 16
    for at in (0, last):
        with pytest.raises(pkg.CapabilityError) as e:
            pkg.extend_weights(**_sharing(args, "weights", other, at), prefix=16)
        assert e.value.field == "weights"
    with pytest.raises(RuntimeError, match="no CPU path"):
        pkg.extend_weights(**_sharing(args, "weights", other, last + 16), prefix=16)


_EVICT_PAIRS = [(o, i) for o in ("page_table_out", "weights_out", "kv_lens_out") for i in ("page_table", "weights", "kv_lens", "rows")
                if o != i + "_out"] + [("weights_out", "page_table_out"), ("kv_lens_out", "page_table_out"), ("kv_lens_out", "weights_out")]


def _evict_args(in_place):
    args = dict(page_table=torch.zeros(4, 12, dtype=torch.int32), weights=torch.zeros(4, 12), kv_lens=torch.zeros(2, dtype=torch.int32),
                rows=torch.zeros(2, dtype=torch.int32), keep=8, freed=torch.zeros(2, 4, dtype=torch.int32),
                freed_lens=torch.zeros(2, dtype=torch.int32))
    outs = dict(page_table_out=torch.zeros(4, 12, dtype=torch.int32), weights_out=torch.zeros(4, 12),
                kv_lens_out=torch.zeros(2, dtype=torch.int32))
    return args if in_place else dict(args, **outs)


@pytest.mark.parametrize("output,other", _EVICT_PAIRS)
def test_eviction_results_share_no_memory_with_other_arguments(pkg, output, other):
    args = _evict_args(False)
    last = (_bytes_of(args[other]) - 1) // 16 * 16
    for at in (0, last):
        with pytest.raises(pkg.CapabilityError) as e:
            pkg.evict_lightest(**_sharing(args, output, other, at))
        assert e.value.field in (output, output.removesuffix("_out"))
    with pytest.raises(RuntimeError, match="no CPU path"):
        pkg.evict_lightest(**_sharing(args, output, other, last + 16))


def test_eviction_in_place_still_minds_the_other_arguments(pkg):
    with pytest.raises(RuntimeError, match="no CPU path"):
        pkg.evict_lightest(**_evict_args(True))
    same = _evict_args(True)                               # in place by another view of the same memory
    with pytest.raises(RuntimeError, match="no CPU path"):
        pkg.evict_lightest(**same, page_table_out=same["page_table"].view(4, 12), weights_out=same["weights"][:], kv_lens_out=same["kv_lens"][:])
    for output, other in (("weights", "page_table"), ("kv_lens", "page_table"), ("kv_lens", "weights")):
        with pytest.raises(pkg.CapabilityError):
            pkg.evict_lightest(**_sharing(_evict_args(True), output, other, 0))


def test_rows_side_by_side_in_one_buffer_are_apart(pkg):
    from attn_kernel_lab_b200.decode import _overlap

    buf = torch.zeros(6, 40, dtype=torch.int32)
    left, right = buf[:, :16], buf[:, 16:36].view(torch.float32)
    assert not _overlap(left, right) and not _overlap(right, left)
    assert _overlap(left, buf[:, 15:20]) and _overlap(buf[:, 15:20], left) and _overlap(left, buf[2:4, 3:5])
    assert not _overlap(left[2:], buf[:3, 16:]) and not _overlap(left, buf[3, 16:40]) and _overlap(left, buf[3, 10:20])
    assert not _overlap(buf[0, 36:], left) and not _overlap(right, buf[5, 36:])
    assert _overlap(left, buf.view(-1)[5:200]) and _overlap(left, buf.view(-1)[0:239].as_strided((5, 3), (47, 1)))
    table, weights = buf[:, :16], buf[:, 16:36].view(torch.float32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        pkg.evict_lightest(table, weights, torch.zeros(2, dtype=torch.int32), keep=8)


def _shared_pointers(K, c, pairs):
    """Addresses far apart for every pointer; then each pair, where the second is moved onto the last bytes of the first."""
    for i, name in enumerate(n for n, t in c._fields_ if t is ctypes.c_void_p):
        setattr(c, name, (i + 2) << 32)
    for first, size, second in pairs:
        copy = type(c).from_buffer_copy(c)
        setattr(copy, second, getattr(c, first) + (size - 1) // 16 * 16)
        yield first, second, copy


def test_c_entries_refuse_shared_memory(K):
    """Every call here is refused on the host, so no pointer is followed."""
    lib = K.load()
    c = _c_decode(K, lse_out=1, weights=1, weights_stride=32, rows=1)
    c.plan.max_weight_tokens = 64
    L = K.DecodeLayout()
    K.check(lib.akl_decode_layout(ctypes.byref(c.plan), ctypes.byref(L)), "layout")
    c.workspace_bytes = int(L.total_bytes)
    q, pool, table, vec = 2 * 24 * 512, 64 * 2048, 4 * 32 * 8, 16
    pairs = [(i, n, o) for i, n in (("q", q), ("k_pool", pool), ("v_pool", pool), ("page_table", table), ("rows", vec), ("kv_lens", vec))
             for o in ("out", "lse_out", "weights")] + [("out", q, "lse_out"), ("out", q, "weights"), ("lse_out", 192, "weights")]
    for first, second, call in _shared_pointers(K, c, pairs):
        assert lib.akl_paged_decode(ctypes.byref(call), None) == -1, (first, second)
    w = K.Weights()
    plan, M = K.WeightsPlan(64, 8, 24, 4), K.WeightsLayout()
    K.check(lib.akl_weights_layout(ctypes.byref(plan), ctypes.byref(M)), "layout")
    w.workspace_bytes, w.plan = int(M.total_bytes), plan
    w.pool_rows, w.q_stride, w.k_stride, w.T, w.N, w.prefix, w.q_heads, w.kv_heads = 64, 6144, 1024, 4, 20, 16, 24, 4
    w.sm_scale = 0.0625
    for first, second, call in _shared_pointers(K, w, [("q", 4 * 24 * 512, "weights"), ("k_pool", pool, "weights"), ("idx", 160, "weights"),
                                                       ("lse", 4 * 24 * 4, "weights")]):
        assert lib.akl_extend_weights(ctypes.byref(call), None) == -1, (first, second)
    e = K.Evict()
    e.table_stride = e.table_out_stride = e.weights_stride = e.weights_out_stride = e.freed_stride = 16
    e.batch, e.table_rows, e.table_width, e.freed_width, e.keep = 2, 4, 16, 16, 8
    sizes = dict(page_table=512, weights=256, rows=16, kv_lens=16, page_table_out=512, weights_out=256, kv_lens_out=16, freed=256, freed_lens=8)
    outputs = ["page_table_out", "weights_out", "kv_lens_out", "freed", "freed_lens"]
    pairs = [(i, sizes[i], o) for i in sizes for o in outputs if i != o and (i not in outputs or outputs.index(i) < outputs.index(o))]
    for first, second, call in _shared_pointers(K, e, pairs):
        if (first, second) == ("kv_lens", "kv_lens_out"):
            call.kv_lens_out = call.kv_lens + 8            # at its first byte it would be in place
        assert lib.akl_evict_lightest(ctypes.byref(call), None) == -1, (first, second)


@pytest.mark.parametrize("sm_scale,fits", [(2.0 ** -126, True), (2.0 ** 127, True), (1, True), (2.0 ** -127, False), (1e300, False),
                                           (1e-300, False), (10 ** 400, False), (float("inf"), False)])
def test_scales_are_refused_where_32_bits_do_not_hold_them(pkg, short, monkeypatch, sm_scale, fits):      # noqa: F811
    decode, eviction, seen = short
    c = decode_ref.case([5, 9], 24, 4, device="cpu")
    ws = pkg.plan_decode_workspace("cpu", max_requests=2, q_heads=24, kv_heads=4)
    wws = pkg.plan_weights_workspace("cpu", max_kv_len=20, max_q_len=4, q_heads=24, kv_heads=4)
    ws.device_index = wws.device_index = 0
    extend = dict(q=torch.zeros(4, 24, 256, dtype=torch.bfloat16), k_pool=torch.zeros(40, 4, 256, dtype=torch.float16),
                  idx=torch.arange(20), prefix=16, lse=torch.zeros(4, 24), weights=torch.zeros(20), workspace=wws)
    for call in (lambda: pkg.paged_decode(**c, workspace=ws, out=torch.zeros(2, 24, 256, dtype=torch.bfloat16), sm_scale=sm_scale),
                 lambda: pkg.extend_weights(**extend, sm_scale=sm_scale)):
        if fits:
            call()
        else:
            with pytest.raises(pkg.CapabilityError) as e:
                call()
            assert e.value.field == "sm_scale"
    assert len(seen) == (2 if fits else 0)


def test_a_call_whose_second_launch_does_not_fit_is_refused_before_the_first(K):
    batch = 1 << 26
    c = _c_decode(K, batch=batch, rows=1, weights=1, table_width=1 << 14, table_stride=1 << 14, weights_stride=1 << 14)
    c.plan = K.DecodePlan(batch, 24, 4, 0, 64)
    L = K.DecodeLayout()
    K.check(K.load().akl_decode_layout(ctypes.byref(c.plan), ctypes.byref(L)), "layout")
    c.workspace_bytes = int(L.total_bytes)
    for i, name in enumerate(n for n, t in c._fields_ if t is ctypes.c_void_p):
        setattr(c, name, (i + 2) << 48)
    assert K.load().akl_paged_decode(ctypes.byref(c), None) == -2
