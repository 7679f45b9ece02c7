"""`pool_lse` on the host: refusals, and the flag that every entry hands down."""
import re

import pytest
import torch

from conftest import ROOT


def _request(**over):
    r = dict(q=torch.zeros(2, 24, 256, dtype=torch.bfloat16), k_pool=torch.zeros(9, 4, 256, dtype=torch.bfloat16),
             v_pool=torch.zeros(9, 4, 256, dtype=torch.bfloat16), idx=torch.arange(9), prefix=7)
    r.update(over)
    return r


def test_pool_lse_belongs_to_a_returned_lse(pkg):
    for call in (lambda **kw: pkg.prefill_extend(**_request(), **kw),
                 lambda **kw: pkg.prefill_extend_batch([_request()], workspace=None, **kw)):
        with pytest.raises(pkg.CapabilityError) as e:
            call(pool_lse=True)
        assert e.value.field == "pool_lse"
        with pytest.raises(TypeError, match="pool_lse"):
            call(pool_lse=1, return_lse=True)
        with pytest.raises(RuntimeError, match="no CPU path"):
            call(pool_lse=True, return_lse=True)
    r = _request()
    paged = (r["q"], r["k_pool"][:, None], r["v_pool"][:, None], r["idx"])
    with pytest.raises(pkg.CapabilityError) as e:
        pkg.fp8_paged_prefill(*paged, pool_lse=True)
    assert e.value.field == "pool_lse"
    with pytest.raises(RuntimeError, match="no CPU path"):
        pkg.fp8_paged_prefill(*paged, pool_lse=True, return_lse=True)


def test_flag_matches_the_header_and_travels(pkg):
    from attn_kernel_lab_b200 import kernel as K, quant
    from attn_kernel_lab_b200.dist import kv_split_local

    value = re.search(r"#define AKL_FLAG_POOL_LSE (\d+)u", (ROOT / "include" / "akl.h").read_text())
    assert int(value.group(1)) == K.AKL_FLAG_POOL_LSE
    ws = quant.FP8PrefillWorkspace("cpu")
    r = _request()
    for asked in (False, True):
        seen = []
        kv_split_local(ws, r["q"], r["k_pool"], r["v_pool"], r["idx"], 7, n_total=9, kv_lo=0, sm_scale=0.0625,
                       phases=lambda name, call: seen.append(call.flags), pool_lse=asked)
        assert seen and all(bool(f & K.AKL_FLAG_POOL_LSE) == asked for f in seen)
    bw = pkg.plan_batch_workspace("cpu", max_requests=1, max_total_kv_len=64, max_total_q_len=8, q_heads=24, kv_heads=4)
    r.update(out=torch.zeros_like(r["q"]))
    for asked in (False, True):
        plan = bw.plan([r], sm_scale=0.0625, pool_lse=asked)
        assert bool(plan.batch.flags & K.AKL_FLAG_POOL_LSE) == asked
