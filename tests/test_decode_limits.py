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
