"""Decode, attention weights and eviction, host side: what is refused and how, before any device work,
and the argument checks of the C entry points."""
import ctypes

import pytest
import torch

import decode_ref


@pytest.fixture(scope="module")
def K(pkg):
    from attn_kernel_lab_b200 import kernel

    return kernel


def _decode(**over):
    args = decode_ref.case([5, 9], 24, 4, device="cpu")
    kw = dict(args)
    kw.update(over)
    return kw


def _refused(pkg, field, **over):
    with pytest.raises(pkg.CapabilityError) as e:
        pkg.paged_decode(**_decode(**over))
    assert e.value.field == field, e.value


def test_decode_accepts_the_geometry_then_needs_a_gpu(pkg):
    assert pkg.check_decode(**_decode()) == (2, 24, 4)
    with pytest.raises(RuntimeError, match="no CPU path"):
        pkg.paged_decode(**_decode())


DECODE_REFUSALS = [
    ("q", dict(q=None)), ("q", dict(q=torch.zeros(2, 24 * 256, dtype=torch.bfloat16))),
    ("q", dict(q=torch.zeros(2, 24, 256))), ("q", dict(q=torch.zeros(0, 24, 256, dtype=torch.bfloat16))),
    ("q", dict(q=torch.zeros(24, 2, 256, dtype=torch.bfloat16).transpose(0, 1))),
    ("q", dict(q=torch.zeros(1, 24, 256, dtype=torch.bfloat16).expand(2, 24, 256))),
    ("q", dict(q=torch.zeros(2 * 24 * 256 + 1, dtype=torch.bfloat16)[1:].view(2, 24, 256))),
    ("head_dim", dict(q=torch.zeros(2, 24, 128, dtype=torch.bfloat16))),
    ("q_heads", dict(q=torch.zeros(2, 64, 256, dtype=torch.bfloat16))),
    ("q_heads", dict(q=torch.zeros(2, 36, 256, dtype=torch.bfloat16))),
    ("k_pool", dict(k_pool=torch.zeros(4, 256, dtype=torch.bfloat16))),
    ("kv_heads", dict(k_pool=torch.zeros(4, 3, 256, dtype=torch.bfloat16))),
    ("kv_dtype", dict(k_pool=torch.zeros(4, 4, 256, dtype=torch.float8_e4m3fn))),
    ("v_pool", dict(v_pool=torch.zeros(35, 4, 256, dtype=torch.float16))),
    ("v_pool", dict(v_pool=torch.zeros(34, 4, 256, dtype=torch.bfloat16))),
    ("page_table", dict(page_table=torch.zeros(4, 12))),
    ("page_table", dict(page_table=torch.zeros(4, 0, dtype=torch.int32))),
    ("page_table", dict(page_table=torch.zeros(12, 4, dtype=torch.int32).T)),
    ("page_table", dict(rows=None, page_table=torch.zeros(1, 12, dtype=torch.int32))),
    ("kv_lens", dict(kv_lens=torch.zeros(3, dtype=torch.int32))), ("kv_lens", dict(kv_lens=[1, 2])),
    ("rows", dict(rows=torch.zeros(2))), ("rows", dict(rows=torch.zeros(4, dtype=torch.int32)[::2])),
    ("sm_scale", dict(sm_scale=0.0)), ("sm_scale", dict(sm_scale=float("nan"))), ("sm_scale", dict(sm_scale="1")),
    ("out", dict(out=torch.zeros(2, 24, 256))), ("out", dict(out=torch.zeros(1, 24, 256, dtype=torch.bfloat16))),
    ("lse_out", dict(lse_out=torch.zeros(2, 24))), ("lse_out", dict(lse_out=torch.zeros(24, 2), return_lse=True)),
    ("weights", dict(weights=torch.zeros(4, 11))), ("weights", dict(weights=torch.zeros(4, 12, dtype=torch.float64))),
    ("weight_decay", dict(weights=torch.zeros(4, 12), weight_decay=1.5)),
    ("weight_decay", dict(weights=torch.zeros(4, 12), weight_decay=float("nan"))),
    ("workspace", dict(workspace=object())),
    ("kv_lens", dict(kv_lens=torch.zeros(2, dtype=torch.int32, device="meta"))),
]
_IDS = lambda v: v if isinstance(v, str) else ",".join(v)      # noqa: E731


@pytest.mark.parametrize("field,over", DECODE_REFUSALS, ids=_IDS)
def test_decode_refusals(pkg, field, over):
    _refused(pkg, field, **over)


def test_decode_output_may_not_alias_the_query(pkg):
    kw = _decode()
    _refused(pkg, "out", q=kw["q"], out=kw["q"])


def test_plans_validate_their_heads(pkg):
    with pytest.raises(pkg.CapabilityError):
        pkg.plan_decode_workspace("cpu", max_requests=4, q_heads=64, kv_heads=4)
    with pytest.raises(ValueError, match="max_requests"):
        pkg.plan_decode_workspace("cpu", max_requests=0)
    with pytest.raises(pkg.CapabilityError):
        pkg.plan_weights_workspace("cpu", max_kv_len=64, max_q_len=4, q_heads=20, kv_heads=3)
    with pytest.raises(ValueError, match="max_kv_len"):
        pkg.plan_weights_workspace("cpu", max_kv_len=0, max_q_len=4)


def _extend(**over):
    kw = dict(q=torch.zeros(4, 24, 256, dtype=torch.bfloat16), k_pool=torch.zeros(40, 4, 256, dtype=torch.float16),
              idx=torch.arange(20), prefix=16, lse=torch.zeros(4, 24), weights=torch.zeros(20))
    kw.update(over)
    return kw


EXTEND_REFUSALS = [
    ("q", dict(q=torch.zeros(4, 24, 256))), ("q_len", dict(q=torch.zeros(0, 24, 256, dtype=torch.bfloat16))),
    ("kv_heads", dict(k_pool=torch.zeros(40, 6, 256, dtype=torch.float16))),
    ("idx", dict(idx=torch.zeros(0, dtype=torch.int64))), ("idx", dict(idx=torch.zeros(20))),
    ("prefix", dict(prefix=17)), ("prefix", dict(prefix=-1)), ("prefix", dict(prefix=torch.tensor(3))),
    ("lse", dict(lse=torch.zeros(24, 4).T)), ("lse", dict(lse=torch.zeros(4, 24, dtype=torch.float64))),
    ("weights", dict(weights=torch.zeros(21))), ("weights", dict(weights=torch.zeros(40)[::2])),
    ("weight_decay", dict(weight_decay=-0.5)), ("sm_scale", dict(sm_scale=-1.0)), ("workspace", dict(workspace=3)),
]


@pytest.mark.parametrize("field,over", EXTEND_REFUSALS, ids=_IDS)
def test_extend_weights_refusals(pkg, field, over):
    with pytest.raises(pkg.CapabilityError) as e:
        pkg.extend_weights(**_extend(**over))
    assert e.value.field == field, e.value


def test_extend_weights_needs_a_gpu(pkg):
    with pytest.raises(RuntimeError, match="no CPU path"):
        pkg.extend_weights(**_extend())


def _evict(**over):
    kw = dict(page_table=torch.zeros(4, 12, dtype=torch.int32), weights=torch.zeros(4, 14),
              kv_lens=torch.zeros(2, dtype=torch.int64), keep=8, protect_first=2, protect_last=3)
    kw.update(over)
    return kw


_TABLE = torch.zeros(5, 12, dtype=torch.int32)


EVICT_REFUSALS = [
    ("page_table", dict(page_table=torch.zeros(4, 12))), ("weights", dict(weights=torch.zeros(4, 11))),
    ("weights", dict(weights=torch.zeros(3, 12))), ("kv_lens", dict(kv_lens=torch.zeros(0, dtype=torch.int64))),
    ("page_table", dict(kv_lens=torch.zeros(5, dtype=torch.int64))), ("rows", dict(rows=torch.zeros(3, dtype=torch.int32))),
    ("keep", dict(keep=0)), ("keep", dict(keep=4)), ("keep", dict(keep=True)), ("protect_first", dict(protect_first=-1)),
    ("protect_last", dict(protect_last=1.0)),
    ("page_table_out", dict(page_table_out=torch.zeros(4, 12, dtype=torch.int64))),
    ("page_table_out", dict(page_table_out=torch.zeros(3, 12, dtype=torch.int32))),
    ("page_table_out", dict(page_table=_TABLE[:4], page_table_out=_TABLE[1:])),
    ("weights_out", dict(weights_out=torch.zeros(4, 12))),
    ("kv_lens_out", dict(kv_lens_out=torch.zeros(2, dtype=torch.int32))),
    ("freed", dict(freed=torch.zeros(2, 3, dtype=torch.int32))), ("freed", dict(freed=torch.zeros(2, 4, dtype=torch.int64))),
    ("freed_lens", dict(freed_lens=torch.zeros(2, dtype=torch.int64))),
]


@pytest.mark.parametrize("field,over", EVICT_REFUSALS, ids=_IDS)
def test_eviction_refusals(pkg, field, over):
    with pytest.raises(pkg.CapabilityError) as e:
        pkg.evict_lightest(**_evict(**over))
    assert e.value.field == field, e.value


def test_eviction_needs_a_gpu(pkg):
    with pytest.raises(RuntimeError, match="no CPU path"):
        pkg.evict_lightest(**_evict())


# ---- the short form of the checks: what it takes it packs as the full form does, the rest it leaves alone
@pytest.fixture()
def short(pkg, monkeypatch):
    """CPU tensors stand for those of GPU 0 (nothing is launched); calls are recorded, not made."""
    from attn_kernel_lab_b200 import decode, eviction

    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 0)
    monkeypatch.setattr(decode, "_need_cuda", lambda *a: None)
    monkeypatch.setattr(eviction, "_need_cuda", lambda *a: None)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    seen = []
    for module in (decode, eviction):
        monkeypatch.setattr(module, "_call", lambda index, fn, name, packed: seen.append((index, name, packed)))
    return decode, eviction, seen


def _on_gpu0(ws):
    ws.device_index = 0
    return ws


@pytest.mark.parametrize("rows", [True, False])
@pytest.mark.parametrize("weights", [None, 0.5])
@pytest.mark.parametrize("lse", [True, False])
def test_short_decode_packs_what_the_full_form_packs(pkg, short, monkeypatch, rows, weights, lse):
    decode, _, seen = short
    ws = _on_gpu0(pkg.plan_decode_workspace("cpu", max_requests=3, q_heads=24, kv_heads=4, max_weight_tokens=640))
    kw = _decode(workspace=ws, out=torch.zeros(2, 24, 256, dtype=torch.bfloat16), sm_scale=0.125)
    if not rows:
        kw["rows"] = None
    if weights is not None:
        kw.update(weights=torch.zeros(kw["page_table"].shape), weight_decay=weights)
    if lse:
        kw.update(return_lse=True, lse_out=torch.zeros(2, 24))
    pkg.paged_decode(**kw)
    monkeypatch.setattr(decode, "_ordinary", lambda *a: None)
    pkg.paged_decode(**kw)
    assert len(seen) == 2 and seen[0] == seen[1]


@pytest.mark.parametrize("field,over", DECODE_REFUSALS, ids=_IDS)
def test_short_decode_leaves_refusals_to_the_full_form(pkg, short, field, over):
    decode, _, seen = short
    kw = dict(return_lse=False)
    kw.update(_decode(workspace=_on_gpu0(pkg.plan_decode_workspace("cpu", max_requests=3, q_heads=24, kv_heads=4,
                                                                   max_weight_tokens=640)),
                      out=torch.zeros(2, 24, 256, dtype=torch.bfloat16)))
    kw.update(over)
    if any(isinstance(v, torch.Tensor) and v.device.type == "meta" for v in over.values()):
        pytest.skip("every tensor is on GPU 0 here")
    with pytest.raises(pkg.CapabilityError) as e:
        pkg.paged_decode(**kw)
    assert e.value.field == field and not seen


def test_short_extend_and_eviction_pack_what_the_full_forms_pack(pkg, short, monkeypatch):
    _, eviction, seen = short
    ws = _on_gpu0(pkg.plan_weights_workspace("cpu", max_kv_len=64, max_q_len=8, q_heads=24, kv_heads=4))
    kw = _extend(workspace=ws, weight_decay=0.25)
    outs = dict(freed=torch.zeros(2, 6, dtype=torch.int32), freed_lens=torch.zeros(2, dtype=torch.int32))
    ev = [dict(_evict(weights=torch.zeros(4, 12)), **outs),
          dict(_evict(weights=torch.zeros(4, 12), rows=torch.zeros(2, dtype=torch.int32)), **outs,
               page_table_out=torch.zeros(4, 12, dtype=torch.int32), weights_out=torch.zeros(4, 12),
               kv_lens_out=torch.zeros(2, dtype=torch.int64))]
    for _ in range(2):
        pkg.extend_weights(**kw)
        for e in ev:
            pkg.evict_lightest(**e)
        monkeypatch.setattr(eviction, "_ordinary_extend", lambda *a: None)
        monkeypatch.setattr(eviction, "_ordinary_evict", lambda *a: (None, None))
    # (the full form names the device of the tensors, which the stand-ins do not have)
    assert [s[1:] for s in seen[:3]] == [s[1:] for s in seen[3:]] and len({s[2] for s in seen[:3]}) == 3


@pytest.mark.parametrize("field,over", EXTEND_REFUSALS, ids=_IDS)
def test_short_extend_leaves_refusals_to_the_full_form(pkg, short, field, over):
    ws = _on_gpu0(pkg.plan_weights_workspace("cpu", max_kv_len=64, max_q_len=8, q_heads=24, kv_heads=4))
    with pytest.raises(pkg.CapabilityError) as e:
        pkg.extend_weights(**dict(_extend(workspace=ws), **over))
    assert e.value.field == field and not short[2]


_SHARED = [("freed", "rows"), ("freed", "kv_lens"), ("freed", "weights"), ("freed", "weights_out"), ("freed", "page_table_out"),
           ("freed_lens", "freed"), ("freed_lens", "rows"), ("freed_lens", "page_table"), ("freed_lens", "weights_out"),
           ("freed_lens", "kv_lens_out"), ("kv_lens_out", "rows")]


@pytest.mark.parametrize("quick", [False, True])
@pytest.mark.parametrize("field,other", _SHARED)
def test_eviction_outputs_share_no_memory(pkg, short, field, other, quick, monkeypatch):
    """Refused wherever the shared entry lies; the same tensors one entry apart are taken."""
    _, eviction, seen = short
    if not quick:
        monkeypatch.setattr(eviction, "_ordinary_evict", lambda *a: (None, None))
    shapes = dict(freed=(2, 6), freed_lens=(2,), rows=(2,), kv_lens=(2,), kv_lens_out=(2,), page_table=(4, 12),
                  page_table_out=(4, 12), weights=(4, 12), weights_out=(4, 12))
    size = {k: torch.Size(v).numel() for k, v in shapes.items()}
    for at, refused in ((0, True), (size[other] - 1, True), (size[other], False)):
        buf = torch.zeros(size[other] + size[field], dtype=torch.int32)
        kw = {k: torch.zeros(v, dtype=torch.float32 if k.startswith("weights") else torch.int32)
              for k, v in shapes.items()}
        kw[field] = buf[at:at + size[field]].view(shapes[field])
        kw[other] = buf[:size[other]].view(kw[other].dtype).view(shapes[other])
        kw.update(keep=8)
        if refused:
            with pytest.raises(pkg.CapabilityError) as e:
                pkg.evict_lightest(**kw)
            assert e.value.field == field and not seen
        else:
            pkg.evict_lightest(**kw)
            assert len(seen) == 1


@pytest.mark.parametrize("field,over", EVICT_REFUSALS, ids=_IDS)
def test_short_eviction_leaves_refusals_to_the_full_form(pkg, short, field, over):
    base = dict(_evict(weights=torch.zeros(4, 12)), freed=torch.zeros(2, 6, dtype=torch.int32),
                freed_lens=torch.zeros(2, dtype=torch.int32))
    if field == "weights_out":
        over = dict(weights_out=torch.zeros(4, 13))
    with pytest.raises(pkg.CapabilityError) as e:
        pkg.evict_lightest(**dict(base, **over))
    assert e.value.field == field and not short[2]


# ---- C entry points: every case fails host validation, so no pointer is followed -----------------
def test_struct_sizes_match_the_header(K):
    assert ctypes.sizeof(K.DecodePlan) == 24 and ctypes.sizeof(K.DecodeLayout) == 40
    assert ctypes.sizeof(K.Decode) == 10 * 8 + 8 + 24 + 6 * 8 + 9 * 4 + 2 * 4 + 4
    assert ctypes.sizeof(K.Weights) == 6 * 8 + 8 + 16 + 3 * 8 + 7 * 4 + 2 * 4 + 4
    assert ctypes.sizeof(K.Evict) == 9 * 8 + 5 * 8 + 10 * 4


def _c_decode(K, **over):
    plan = K.DecodePlan(4, 24, 4, 0, 0)
    L = K.DecodeLayout()
    K.check(K.load().akl_decode_layout(ctypes.byref(plan), ctypes.byref(L)), "layout")
    c = K.Decode()
    c.q = c.k_pool = c.v_pool = c.page_table = c.kv_lens = c.out = 4096
    c.workspace, c.workspace_bytes, c.plan = 1 << 20, int(L.total_bytes), plan
    c.pool_rows, c.q_stride, c.k_stride, c.v_stride, c.table_stride = 64, 24 * 256, 1024, 1024, 32
    c.batch, c.q_heads, c.kv_heads, c.table_rows, c.table_width = 2, 24, 4, 4, 32
    c.sm_scale = 0.0625
    for k, v in over.items():
        setattr(c, k, v)
    return c


@pytest.mark.parametrize("over,code", [
    (dict(q=None), -1), (dict(kv_lens=None), -1), (dict(workspace=None), -1), (dict(batch=0), -1), (dict(pool_rows=0), -1),
    (dict(kv_dtype=2), -1), (dict(idx_dtype=2), -1), (dict(lens_dtype=-1), -1), (dict(sm_scale=0.0), -1),
    (dict(sm_scale=float("nan")), -1), (dict(weight_decay=2.0), -1), (dict(table_rows=1), -1), (dict(k_stride=1016), -1),
    (dict(table_stride=31), -1), (dict(weights=4096, weights_stride=16), -1), (dict(q_heads=26), -2),
    (dict(q_heads=36), -2), (dict(batch=5, table_rows=5), -3), (dict(workspace_bytes=512), -3), (dict(kv_heads=8, k_stride=2048, v_stride=2048), -3),
    (dict(weights=4096, weights_stride=32), -3), (dict(q=4104), -5), (dict(k_stride=1028), -5),
    (dict(workspace=(1 << 20) + 16), -5),
], ids=lambda v: str(v))
def test_c_decode_checks(K, over, code):
    lib = K.load()
    assert lib.akl_paged_decode(ctypes.byref(_c_decode(K, **over)), None) == code
    assert lib.akl_paged_decode(None, None) == K.AKL_ERR_INVALID


def test_c_layouts(K):
    lib = K.load()
    L, W = K.DecodeLayout(), K.WeightsLayout()
    assert lib.akl_decode_layout(ctypes.byref(K.DecodePlan(0, 24, 4, 0, 0)), ctypes.byref(L)) == -1
    assert lib.akl_decode_layout(ctypes.byref(K.DecodePlan(1, 36, 4, 0, 0)), ctypes.byref(L)) == -2
    assert lib.akl_weights_layout(ctypes.byref(K.WeightsPlan(1, 1, 24, 0)), ctypes.byref(W)) == -1
    sizes = []
    for tokens in (0, 64, 6400):
        K.check(lib.akl_decode_layout(ctypes.byref(K.DecodePlan(8, 24, 4, 0, tokens)), ctypes.byref(L)), "layout")
        assert all(getattr(L, f) % 1024 == 0 for f in ("total_bytes", "off_parts", "off_lse", "off_scores"))
        sizes.append(int(L.total_bytes))
    assert sizes == sorted(sizes)


@pytest.mark.parametrize("over,code", [
    (dict(q=None), -1), (dict(T=0), -1), (dict(prefix=17), -1), (dict(kv_dtype=3), -1), (dict(sm_scale=0.0), -1),
    (dict(k_stride=512), -1), (dict(q_heads=25), -2), (dict(N=65, prefix=0), -3), (dict(q_heads=16), -3),
    (dict(k_pool=4100), -5),
], ids=lambda v: str(v))
def test_c_weights_checks(K, over, code):
    lib = K.load()
    plan = K.WeightsPlan(64, 8, 24, 4)
    L = K.WeightsLayout()
    K.check(lib.akl_weights_layout(ctypes.byref(plan), ctypes.byref(L)), "layout")
    c = K.Weights()
    c.q = c.k_pool = c.idx = c.lse = c.weights = 4096
    c.workspace, c.workspace_bytes, c.plan = 1 << 20, int(L.total_bytes), plan
    c.pool_rows, c.q_stride, c.k_stride, c.T, c.N, c.prefix, c.q_heads, c.kv_heads = 64, 6144, 1024, 4, 20, 16, 24, 4
    c.sm_scale = 0.0625
    for k, v in over.items():
        setattr(c, k, v)
    assert lib.akl_extend_weights(ctypes.byref(c), None) == code
    assert lib.akl_extend_weights(None, None) == K.AKL_ERR_INVALID


@pytest.mark.parametrize("over,code", [
    (dict(weights=None), -1), (dict(batch=0), -1), (dict(keep=0), -1), (dict(first=-1), -1), (dict(first=6, last=6), -1),
    (dict(idx_dtype=9), -1), (dict(table_rows=1), -1), (dict(weights_stride=8), -1), (dict(freed_width=5, freed_stride=5), -3),
], ids=lambda v: str(v))
def test_c_evict_checks(K, over, code):
    lib = K.load()
    c = K.Evict()
    for name in ("page_table", "weights", "kv_lens", "page_table_out", "weights_out", "kv_lens_out", "freed", "freed_lens"):
        setattr(c, name, 4096)
    c.table_stride = c.table_out_stride = c.weights_stride = c.weights_out_stride = c.freed_stride = 16
    c.batch, c.table_rows, c.table_width, c.freed_width, c.keep, c.first, c.last = 2, 4, 16, 16, 8, 2, 2
    for k, v in over.items():
        setattr(c, k, v)
    assert lib.akl_evict_lightest(ctypes.byref(c), None) == code
    assert lib.akl_evict_lightest(None, None) == K.AKL_ERR_INVALID
