"""Decode attention, the attention weights of an extend and eviction on the GPU, against 64 bits."""
import pytest
import torch

import decode_ref as R

pytestmark = pytest.mark.gpu

BF16, FP16, I32, I64 = torch.bfloat16, torch.float16, torch.int32, torch.int64


def run_decode(pkg, c, *, decay=None, workspace=None, **kw):
    """Call and compare: out, lse and (with `decay`) weights, whose untouched entries must stay."""
    weights = before = None
    if decay is not None:
        g = torch.Generator(device=c["q"].device).manual_seed(5)
        weights = torch.rand(c["page_table"].shape, generator=g, device=c["q"].device)
        before = weights.clone()
    out, lse = pkg.paged_decode(**c, weights=weights, weight_decay=1.0 if decay is None else decay,
                                workspace=workspace, return_lse=True, check_status=True, **kw)
    ref = R.decode(c["q"], c["k_pool"], c["v_pool"], c["page_table"], c["kv_lens"], c.get("rows"), weights=before,
                   decay=1.0 if decay is None else decay, sm_scale=kw.get("sm_scale", 1 / 16))
    R.within(out, ref["out"], ref["out_tol"])
    R.within(lse, ref["lse"], ref["lse_tol"])
    if decay is not None:
        R.within(weights, ref["weights"], ref["weights_tol"])      # a bound of zero where nothing is written
    return out, lse, weights


@pytest.mark.parametrize("lens,heads,dtype,idx,decay", [
    ([1], (24, 4), BF16, I32, None),
    ([1, 0, 3, 2], (24, 4), BF16, I64, 1.0),
    ([15, 16, 17, 31, 32, 33], (16, 4), FP16, I32, 0.0),
    ([63, 64, 65, 0, 127, 128, 129], (32, 4), BF16, I32, 0.5),
    ([1000], (24, 4), BF16, I32, 1.0),
    ([5003], (32, 4), FP16, I64, 1.0),
    ([2047, 1, 700], (8, 2), BF16, I32, 1.0),
    ([777, 3000], (6, 1), FP16, I32, 1.0),
    ([777, 3000, 0, 1], (1, 1), BF16, I32, 1.0),
    ([500, 1234], (40, 8), BF16, I32, 1.0),
    ([0, 300, 5], (64, 8), FP16, I64, 0.0),
    ([321, 100], (6, 2), BF16, I64, None),
    ([0], (24, 4), BF16, I32, 0.0),
    ([0, 0, 0], (24, 4), FP16, I32, 1.0),
    ([(37 * i) % 53 for i in range(300)], (24, 4), BF16, I32, 1.0),
    ([20000] + [3] * 40, (24, 4), BF16, I32, 1.0),
    ([40001], (32, 4), BF16, I32, 1.0),
], ids=lambda v: (f"{len(v)}x{max(v)}" if isinstance(v, list) else str(v)))
def test_decode_matches_64_bits(pkg, cuda, lens, heads, dtype, idx, decay):
    run_decode(pkg, R.case(lens, *heads, dtype=dtype, idx=idx, seed=len(lens) + max(lens)), decay=decay)


def test_decode_with_a_planned_workspace_allocates_nothing_and_repeats_its_bits(pkg, cuda):
    c = R.case([3000, 17, 900], 24, 4, seed=3)
    ws = pkg.plan_decode_workspace(cuda, max_requests=3, q_heads=24, kv_heads=4, max_weight_tokens=4096)
    out, lse = torch.empty_like(c["q"]), torch.empty((3, 24), device=cuda)
    weights = torch.zeros(c["page_table"].shape, device=cuda)
    kw = dict(workspace=ws, out=out, lse_out=lse, weights=weights, weight_decay=0.0, return_lse=True)
    pkg.paged_decode(**c, **kw)
    first = [t.clone() for t in (out, lse, weights)]
    torch.cuda.synchronize()
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    got = pkg.paged_decode(**c, **kw)
    assert torch.cuda.memory_stats()["allocation.all.allocated"] == before
    assert got[0] is out and got[1] is lse
    assert all(torch.equal(a, b) for a, b in zip(first, (out, lse, weights)))
    other = R.case([70], 32, 4, seed=1)
    with pytest.raises(pkg.WorkspaceCapacityError):
        pkg.paged_decode(**other, workspace=ws)
    with pytest.raises(pkg.WorkspaceCapacityError):
        pkg.paged_decode(**R.case([1] * 4, 24, 4), workspace=ws)
    plain = pkg.plan_decode_workspace(cuda, max_requests=3, q_heads=24, kv_heads=4)
    with pytest.raises(pkg.WorkspaceCapacityError):
        pkg.paged_decode(**c, workspace=plain, weights=weights)


def test_decode_reads_strided_operands(pkg, cuda):
    c = R.case([100, 333], 12, 2, seed=9)
    fused = torch.full((2, 20, 256), float("nan"), dtype=BF16, device=cuda)
    fused[:, 4:16] = c["q"]
    both = torch.full((c["k_pool"].shape[0], 2, 3, 256), float("nan"), dtype=BF16, device=cuda)
    both[:, 0, 1:], both[:, 1, :2] = c["k_pool"], c["v_pool"]
    wide = torch.full((c["page_table"].shape[0], 500), -7, dtype=I32, device=cuda)
    wide[:, 11:11 + c["page_table"].shape[1]] = c["page_table"]
    c.update(q=fused[:, 4:16], k_pool=both[:, 0, 1:], v_pool=both[:, 1, :2],
             page_table=wide[:, 11:11 + c["page_table"].shape[1]])
    assert not c["q"].is_contiguous() and not c["k_pool"].is_contiguous()
    run_decode(pkg, c, decay=1.0)
    # one kv head with its group, as a view of the whole pool
    j = 1
    part = dict(c, q=fused[:, 10:16], k_pool=both[:, 0, 2:3], v_pool=both[:, 1, 1:2])
    run_decode(pkg, part)


@pytest.mark.parametrize("index", [I32, I64])
def test_decode_survives_lengths_rows_and_slots_out_of_range(pkg, cuda, index):
    c = R.case([40, 200, 64, 10, 90, 16], 24, 4, idx=index, seed=11, poison=True)
    pool = c["k_pool"].shape[0]
    r = c["rows"].long()
    c["page_table"][r[0], 3] = -1
    c["page_table"][r[0], 39] = pool
    c["page_table"][r[1], 64:80] = torch.iinfo(index).max
    c["page_table"][r[2], :] = torch.iinfo(index).min            # no slot at all
    c["page_table"][r[5], 1:] = pool + 5
    c["kv_lens"] = c["kv_lens"].to(index)
    c["rows"] = c["rows"].to(index)
    c["kv_lens"][3] = -5
    c["rows"][4] = c["page_table"].shape[0]
    ref = run_decode(pkg, c, decay=1.0)
    assert torch.isinf(ref[1][2]).all() and not ref[0][2:5].any()
    c["kv_lens"][1] = torch.iinfo(index).max                     # cut to the table's width
    c["page_table"][r[1], 200:] = -3
    run_decode(pkg, c, decay=0.0)


def test_decode_without_rows_takes_the_first_rows(pkg, cuda):
    c = R.case([100, 7], 16, 4, seed=2)
    c["page_table"] = c["page_table"][c.pop("rows").long()].contiguous()
    run_decode(pkg, c, decay=1.0)


def test_decode_slots_may_repeat(pkg, cuda):
    c = R.case([50, 60], 24, 4, seed=4)
    r = c["rows"].long()
    c["page_table"][r[0], 10:50] = c["page_table"][r[0], 3]      # one key forty times
    c["page_table"][r[1], :20] = c["page_table"][r[0], :20]      # a shared prefix
    run_decode(pkg, c, decay=1.0)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_decode_holds_its_range(pkg, cuda, dtype):
    c = R.case([600, 33], 24, 4, dtype=dtype, seed=6)
    c["q"] *= 500                                                # one-hot softmax, |x| in the thousands
    run_decode(pkg, c, decay=1.0)
    c["q"] *= 2.0 ** -40                                         # uniform softmax, q far below 16-bit range
    run_decode(pkg, c, decay=1.0)
    c["q"].zero_()
    _, lse, w = run_decode(pkg, c, decay=0.0)
    # a score of -inf in a valid place weighs nothing; NaN reaches the request that reads it, no other
    slot = int(c["page_table"][c["rows"][1].long(), 5])
    c["v_pool"][slot] = float("nan")
    out = pkg.paged_decode(**c)
    assert torch.isnan(out[1]).all() and torch.isfinite(out[0]).all()


def test_decode_offsets_beyond_32_bits(pkg, cuda):
    slots = (1 << 23) + 1000                                     # x 256 channels: past 2^31 elements
    k = torch.empty((slots, 1, 256), dtype=BF16, device=cuda)
    v = torch.empty((slots, 1, 256), dtype=BF16, device=cuda)
    n = 500
    at = slots - 1 - 2 * torch.arange(n, device=cuda)
    k[at] = torch.randn((n, 1, 256), device=cuda).to(BF16)
    v[at] = torch.randn((n, 1, 256), device=cuda).to(BF16)
    q = torch.randn((1, 8, 256), device=cuda).to(BF16)
    run_decode(pkg, dict(q=q, k_pool=k, v_pool=v, page_table=at[None].contiguous(),
                         kv_lens=torch.tensor([n], device=cuda)))


def test_decode_reports_weights_beyond_the_plan(pkg, cuda):
    c = R.case([100, 100], 24, 4, seed=8)
    ws = pkg.plan_decode_workspace(cuda, max_requests=2, q_heads=24, kv_heads=4, max_weight_tokens=128)
    weights = torch.zeros(c["page_table"].shape, device=cuda)
    out, lse = torch.empty_like(c["q"]), torch.empty((2, 24), device=cuda)
    with pytest.raises(pkg.NativeError) as e:
        pkg.paged_decode(**c, workspace=ws, out=out, lse_out=lse, weights=weights, return_lse=True, check_status=True)
    assert e.value.code == -3
    ref = R.decode(c["q"], c["k_pool"], c["v_pool"], c["page_table"], c["kv_lens"], c["rows"], weights=weights * 0)
    R.within(out, ref["out"], ref["out_tol"])
    R.within(lse, ref["lse"], ref["lse_tol"])
    first = c["rows"][0].long()
    R.within(weights[first], ref["weights"][first], ref["weights_tol"][first])
    assert not weights[c["rows"][1].long()].any()
    pkg.paged_decode(**c, workspace=ws, check_status=True)       # the workspace goes on working


def test_decode_in_a_graph_follows_lengths_and_rows(pkg, cuda):
    c = R.case([700, 90, 5], 24, 4, seed=12)
    long = R.case([2000, 1500, 600], 24, 4, seed=13, width=c["page_table"].shape[1] + 1297)
    # one pool, the longer table first
    n0 = long["k_pool"].shape[0]
    table = torch.cat([long["page_table"], torch.nn.functional.pad(c["page_table"] + n0, (0, 1297))])
    c = dict(c, k_pool=torch.cat([long["k_pool"], c["k_pool"]]), v_pool=torch.cat([long["v_pool"], c["v_pool"]]),
             page_table=table, rows=c["rows"] + long["page_table"].shape[0])
    ws = pkg.plan_decode_workspace(cuda, max_requests=3, q_heads=24, kv_heads=4, max_weight_tokens=8192)
    out, lse = torch.empty_like(c["q"]), torch.empty((3, 24), device=cuda)
    weights = torch.zeros(table.shape, device=cuda)
    kw = dict(workspace=ws, out=out, lse_out=lse, weights=weights, return_lse=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pkg.paged_decode(**c, **kw)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pkg.paged_decode(**c, **kw)
    for lens, rows in (([700, 90, 5], c["rows"].tolist()), ([2000, 0, 600], long["rows"].tolist()),
                       ([1, 1500, 0], long["rows"].tolist())):
        c["kv_lens"].copy_(torch.tensor(lens)), c["rows"].copy_(torch.tensor(rows))
        before = weights.clone()
        out.fill_(float("nan")), lse.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        ref = R.decode(c["q"], c["k_pool"], c["v_pool"], table, lens, rows, weights=before)
        R.within(out, ref["out"], ref["out_tol"])
        R.within(lse, ref["lse"], ref["lse_tol"])
        R.within(weights, ref["weights"], ref["weights_tol"])
    assert ws.status() == 0


def test_decode_on_two_streams_with_two_workspaces(pkg, cuda):
    cases = [R.case([3000, 40], 24, 4, seed=20), R.case([100, 2500], 24, 4, seed=21)]
    spaces = [pkg.plan_decode_workspace(cuda, max_requests=2, q_heads=24, kv_heads=4) for _ in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(10):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                outs[i].append(pkg.paged_decode(**cases[i], workspace=spaces[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        alone = pkg.paged_decode(**cases[i], workspace=spaces[i])
        assert all(torch.equal(alone, o) for o in outs[i])


def test_decode_of_thousands_of_short_requests(pkg, cuda):
    lens = [(31 * i) % 43 for i in range(2500)]
    run_decode(pkg, R.case(lens, 1, 1, seed=40), decay=1.0)
    # more requests than a warp's window of lengths, nearly all of them empty
    lens = [0] * 700 + [300] + [0] * 500 + [5, 0, 17]
    run_decode(pkg, R.case(lens, 2, 2, dtype=FP16, seed=41), decay=0.0)


def test_decode_rows_may_repeat_without_weights(pkg, cuda):
    c = R.case([500, 80], 24, 4, seed=42)
    c["rows"] = c["rows"][:1].repeat(3)
    c["kv_lens"] = torch.tensor([500, 500, 123], dtype=I32, device=cuda)
    c["q"] = torch.cat([c["q"][:1], c["q"]])
    run_decode(pkg, c)


# ---- attention weights of an extend ---------------------------------------------------------------
def extend_case(rows, prefix, q_heads, kv_heads, *, dtype=BF16, idx=I32, extra=0, seed=0, gain=1.0):
    """`extra` positions lie behind the last row's diagonal: nobody sees them, and their keys are NaN."""
    n = prefix + rows + extra
    c = R.case([n], q_heads, kv_heads, dtype=dtype, idx=idx, seed=seed)
    g = torch.Generator().manual_seed(seed + 1)
    q = (torch.randn((rows, q_heads, 256), generator=g) * gain).to(BF16).to(c["q"].device)
    at = c["page_table"][c["rows"][0].long(), :n].contiguous()
    k = c["k_pool"]
    kf = k[at.long()].double()
    lse = torch.empty((rows, q_heads), device=q.device)
    seen = torch.arange(n, device=q.device)[None] <= prefix + torch.arange(rows, device=q.device)[:, None]
    for h in range(q_heads):
        x = (q[:, h].double() @ kf[:, h // (q_heads // kv_heads)].T) / 16
        lse[:, h] = torch.logsumexp(x.masked_fill(~seen, -float("inf")), 1) * R.LOG2E
    if extra:
        k[at[prefix + rows:].long()] = float("nan")
    return dict(q=q, k_pool=k, idx=at, prefix=prefix, lse=lse)


def run_extend(pkg, c, decay=1.0, **kw):
    n = c["idx"].shape[0]
    weights = torch.rand(n, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    ref, tol = R.extend_weights(c["q"], c["k_pool"], c["idx"], c["prefix"], c["lse"], weights, decay)
    if decay == 0.0:
        weights.fill_(float("nan"))
    got = pkg.extend_weights(**c, weights=weights, weight_decay=decay, check_status=True, **kw)
    assert got is weights
    R.within(weights, ref, tol)
    return weights


@pytest.mark.parametrize("rows,prefix,heads,dtype,idx,extra,decay", [
    (1, 0, (24, 4), BF16, I32, 0, 1.0),
    (1, 63, (24, 4), BF16, I64, 0, 0.0),
    (5, 7, (32, 4), FP16, I32, 3, 0.5),
    (32, 1000, (24, 4), BF16, I32, 0, 1.0),
    (33, 480, (16, 4), FP16, I64, 130, 1.0),
    (128, 0, (24, 4), BF16, I32, 0, 0.0),
    (129, 127, (24, 4), BF16, I32, 1, 1.0),
    (300, 700, (8, 2), BF16, I32, 0, 1.0),
    (257, 255, (6, 1), FP16, I32, 513, 1.0),
    (200, 3000, (1, 1), BF16, I32, 0, 1.0),
    (64, 300, (56, 8), FP16, I32, 0, 1.0),
    (1000, 24, (10, 2), BF16, I64, 0, 0.0),
    (700, 5000, (24, 4), FP16, I32, 40, 1.0),
], ids=str)
def test_extend_weights_match_64_bits(pkg, cuda, rows, prefix, heads, dtype, idx, extra, decay):
    c = extend_case(rows, prefix, *heads, dtype=dtype, idx=idx, extra=extra, seed=rows)
    weights = run_extend(pkg, c, decay)
    if decay == 0.0:                       # what a row gives sums to one, over every head and row
        assert abs(float(weights.double().sum()) / (rows * heads[0]) - 1) < 1e-4
        if extra:
            assert not weights[prefix + rows:].any()


def test_extend_weights_skip_blind_rows_and_bad_slots(pkg, cuda):
    c = extend_case(70, 200, 24, 4, seed=5)
    c["lse"][3, 5], c["lse"][60] = -float("inf"), float("inf")
    c["idx"][10], c["idx"][130], c["idx"][269] = -1, c["k_pool"].shape[0], 1 << 30
    weights = run_extend(pkg, c, 0.0)
    assert not weights[[10, 130, 269]].any()
    c["k_pool"][c["idx"][250].long()] = float("nan")           # seen by rows 50 and later only
    got = pkg.extend_weights(**c, weights=torch.zeros(270, device=cuda))
    assert torch.isnan(got[250]) and torch.isfinite(got[:250]).all() and torch.isfinite(got[251:]).all()


def test_extend_weights_range_strides_window_and_repeats(pkg, cuda):
    c = extend_case(150, 333, 24, 4, dtype=FP16, seed=7, gain=200.0)       # one-hot rows
    run_extend(pkg, c)
    c = extend_case(150, 333, 24, 4, dtype=FP16, seed=8, gain=2.0 ** -40)
    run_extend(pkg, c)
    c = extend_case(90, 200, 12, 4, seed=9)
    fused = torch.full((90, 20, 256), float("nan"), dtype=BF16, device=cuda)
    fused[:, 4:16] = c["q"]
    both = torch.full((c["k_pool"].shape[0], 2, 4, 256), float("nan"), dtype=BF16, device=cuda)
    both[:, 1] = c["k_pool"]
    c.update(q=fused[:, 4:16], k_pool=both[:, 1])
    full = run_extend(pkg, c)
    assert torch.equal(full, run_extend(pkg, c))               # a fixed order of addition
    window = dict(c, q=c["q"][-17:], lse=c["lse"][-17:], prefix=200 + 90 - 17)
    run_extend(pkg, window)
    ws = pkg.plan_weights_workspace(cuda, max_kv_len=400, max_q_len=90, q_heads=12, kv_heads=4)
    assert torch.equal(full, run_extend(pkg, c, workspace=ws))
    run_extend(pkg, window, workspace=ws)
    with pytest.raises(pkg.WorkspaceCapacityError):
        pkg.extend_weights(**extend_case(91, 5, 12, 4), weights=torch.zeros(96, device=cuda), workspace=ws)


def test_extend_weights_in_a_graph(pkg, cuda):
    c = extend_case(100, 900, 24, 4, seed=10)
    ws = pkg.plan_weights_workspace(cuda, max_kv_len=1000, max_q_len=100, q_heads=24, kv_heads=4)
    weights = torch.zeros(1000, device=cuda)
    pkg.extend_weights(**c, weights=weights, weight_decay=0.0, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pkg.extend_weights(**c, weights=weights, weight_decay=0.0, workspace=ws)
    c["q"].copy_(torch.randn(c["q"].shape, device=cuda))
    c["idx"].copy_(c["idx"].flip(0))
    graph.replay()
    torch.cuda.synchronize()
    ref, tol = R.extend_weights(c["q"], c["k_pool"], c["idx"], 900, c["lse"], weights, 0.0)
    R.within(weights, ref, tol)


# ---- eviction ---------------------------------------------------------------------------------------
def run_evict(pkg, table, weights, lens, rows=None, in_place=False, lens_dtype=I32, **kw):
    dev = torch.device("cuda")
    t, w = table.to(dev), weights.to(dev)
    n = torch.tensor(lens, dtype=lens_dtype, device=dev)
    r = None if rows is None else torch.tensor(rows, dtype=lens_dtype, device=dev)
    want = R.evict(table, weights, lens, kw["keep"], kw.get("protect_first", 0), kw.get("protect_last", 0), rows)
    outs = {}
    if not in_place:
        # what is not written shows through: start from the expected rows' untouched entries
        outs = dict(page_table_out=t.clone(), weights_out=w.clone(), kv_lens_out=torch.full_like(n, -9))
    freed = torch.full((len(lens), max(1, table.shape[1] - kw["keep"]) + 2), -5, dtype=t.dtype, device=dev)
    got = pkg.evict_lightest(t, w, n, rows=r, freed=freed, **outs, **kw)
    assert (got[0] is t) == in_place and (got[2] is n) == in_place and got[3] is freed
    assert got[2].tolist() == want[2]
    assert got[4].tolist() == [len(f) for f in want[3]]
    for b, f in enumerate(want[3]):
        assert freed[b, :len(f)].tolist() == f and bool((freed[b, len(f):] == -5).all())
    assert torch.equal(got[0].cpu(), want[0])
    assert torch.equal(got[1].cpu().view(torch.int32), want[1].view(torch.int32))
    if not in_place:
        assert torch.equal(t.cpu(), table) and n.tolist() == list(lens)
    return got


def evict_case(lens, width, *, rows=None, idx=I32, seed=0, kind="heavy"):
    g = torch.Generator().manual_seed(seed)
    shape = (rows or len(lens), width)
    table = torch.randint(0, 1 << 30, shape, generator=g).to(idx)
    w = torch.exp(2 * torch.randn(shape, generator=g))
    if kind == "ties":
        w = torch.randint(0, 4, shape, generator=g).float() - 1
    elif kind == "same":
        w = torch.full(shape, 0.25)
    elif kind == "odd":
        pick = torch.tensor([float("nan"), float("inf"), -float("inf"), -0.0, 0.0, 1e-45, -1e-45, 3e38, -3e38, 1.0])
        w = pick[torch.randint(0, len(pick), shape, generator=g)]
    return table, w


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("lens,width,keep,first,last,idx,kind", [
    ([1], 1, 1, 0, 0, I32, "heavy"),
    ([2, 0, 1, 3], 3, 1, 0, 0, I64, "heavy"),
    ([2, 0, 1, 3], 5, 2, 1, 1, I32, "heavy"),
    ([100, 31, 32, 33, 64, 65], 100, 32, 4, 8, I32, "heavy"),
    ([100, 50, 99], 103, 40, 0, 0, I64, "ties"),
    ([1025, 1024, 1023, 2049], 2050, 512, 16, 100, I32, "ties"),
    ([5000, 1], 5001, 4999, 0, 0, I32, "same"),
    ([5000, 4097], 5000, 64, 0, 64, I64, "heavy"),
    ([3000, 777], 3000, 300, 3, 17, I32, "odd"),
    ([33333], 33333, 1, 0, 0, I32, "heavy"),
    ([70001], 70003, 30011, 5, 999, I64, "heavy"),
    ([150000, 40], 150001, 20000, 4, 128, I32, "ties"),
    ([400, 90], 400, 200, 200, 0, I32, "heavy"),
], ids=str)
def test_eviction_is_exact(pkg, cuda, lens, width, keep, first, last, idx, kind, in_place):
    table, w = evict_case(lens, width, idx=idx, kind=kind, seed=width)
    run_evict(pkg, table, w, lens, in_place=in_place, keep=keep, protect_first=first, protect_last=last)


@pytest.mark.parametrize("in_place", [False, True])
def test_eviction_rows_strides_and_lengths_out_of_range(pkg, cuda, in_place):
    table, w = evict_case([0] * 9, 80, idx=I64, seed=2)
    run_evict(pkg, table, w, [80, 200, -4, 30, 10, 60], rows=[3, 8, 0, 5, 9, -1], lens_dtype=I64, in_place=in_place,
              keep=20, protect_first=2, protect_last=5)
    many, wm = evict_case([300] * 200, 300, seed=4)
    run_evict(pkg, many, wm, [(7 * i) % 301 for i in range(200)], in_place=in_place, keep=100, protect_last=10)
    # more requests than SMs, nearly all of them shortened: nobody may go by a length that another one wrote
    crowd, wc = evict_case([300] * 400, 300, seed=5)
    run_evict(pkg, crowd, wc, [90 + (37 * i) % 211 for i in range(400)], in_place=in_place, keep=100, protect_first=3)
    run_evict(pkg, torch.cat([crowd] * 3), torch.cat([wc] * 3), [300 - (i % 7) for i in range(1200)], in_place=in_place, keep=64)
    # rows of larger tables
    big = torch.zeros((9, 200), dtype=I64, device=cuda)
    acc = torch.full((9, 130), 7.0, device=cuda)
    t, a = big[:, 60:140], acc[:, 21:101]
    t.copy_(table), a.copy_(w)
    n = torch.full((9,), 77, dtype=I32, device=cuda)
    want = R.evict(table, w, [77] * 9, 33, 1, 2)
    _, _, _, freed, counts = pkg.evict_lightest(t, a, n, keep=33, protect_first=1, protect_last=2)
    assert torch.equal(t.cpu(), want[0]) and torch.equal(a.cpu(), want[1]) and counts.tolist() == [44] * 9
    assert [r[:44] for r in freed.tolist()] == want[3]
    assert not big[:, :60].any() and not big[:, 140:].any() and bool((acc[:, :21] == 7).all() and (acc[:, 101:] == 7).all())


@pytest.mark.parametrize("part", ["table", "weights"])
def test_eviction_with_one_output_in_place(pkg, cuda, part):
    """The table alone, or the weights alone, in place; weights that are read a second time (NaN, -0) among them."""
    for lens, width, keep in (([30000, 777, 9000], 30003, 4000), ([70001], 70001, 30000)):
        table, w = evict_case(lens, width, kind="odd", seed=width)
        want = R.evict(table, w, lens, keep, 5, 70)
        for _ in range(3):
            t, a, n = table.to(cuda), w.to(cuda), torch.tensor(lens, dtype=I32, device=cuda)
            outs = dict(weights_out=a.clone()) if part == "table" else dict(page_table_out=t.clone())
            got = pkg.evict_lightest(t, a, n, keep=keep, protect_first=5, protect_last=70, **outs)
            assert torch.equal(got[0].cpu(), want[0]) and n.tolist() == want[2]
            assert torch.equal(got[1].cpu().view(torch.int32), want[1].view(torch.int32))
            assert (got[0] is t) == (part == "table") and (got[1] is a) == (part == "weights")


def test_eviction_in_a_graph_reads_lengths_at_replay(pkg, cuda):
    table, w = evict_case([500, 400], 512, seed=6)
    t, a, n = table.to(cuda), w.to(cuda), torch.tensor([500, 400], dtype=I32, device=cuda)
    freed, counts = torch.zeros((2, 512), dtype=I32, device=cuda), torch.zeros(2, dtype=I32, device=cuda)
    outs = dict(page_table_out=t.clone(), weights_out=a.clone(), kv_lens_out=n.clone(), freed=freed, freed_lens=counts)
    pkg.evict_lightest(t, a, n, keep=128, **outs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pkg.evict_lightest(t, a, n, keep=128, protect_first=3, **outs)
    for lens in ([500, 400], [130, 512], [128, 0]):
        n.copy_(torch.tensor(lens))
        outs["page_table_out"].copy_(t), outs["weights_out"].copy_(a)
        graph.replay()
        want = R.evict(table, w, lens, 128, 3, 0)
        assert torch.equal(outs["page_table_out"].cpu(), want[0]) and torch.equal(outs["weights_out"].cpu(), want[1])
        assert outs["kv_lens_out"].tolist() == want[2] and counts.tolist() == [len(f) for f in want[3]]


def test_extend_weights_and_eviction_on_two_streams(pkg, cuda):
    """Their own workspaces, or none: nothing is shared between streams, and clusters of both fit side by side."""
    extends = [extend_case(90, 700, 24, 4, seed=50), extend_case(40, 1500, 24, 4, dtype=FP16, seed=51)]
    spaces = [pkg.plan_weights_workspace(cuda, max_kv_len=1600, max_q_len=90, q_heads=24, kv_heads=4) for _ in extends]
    evicts = [evict_case([40000], 40000, seed=52), evict_case([9000, 8000], 9000, seed=53)]
    tables = [[t.to(cuda) for t in e] for e in evicts]
    lens = [torch.tensor(n, dtype=I32, device=cuda) for n in ([40000], [9000, 8000])]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                w = torch.zeros(extends[i]["idx"].shape[0], device=cuda)
                pkg.extend_weights(**extends[i], weights=w, workspace=spaces[i])
                t, a, n = tables[i][0].clone(), tables[i][1].clone(), lens[i].clone()
                pkg.evict_lightest(t, a, n, keep=700, protect_last=9)
                got[i].append((w, t, a, n))
    torch.cuda.synchronize()
    for i in (0, 1):
        ref, tol = R.extend_weights(*(extends[i][k] for k in ("q", "k_pool", "idx", "prefix", "lse")), torch.zeros_like(got[i][0][0]))
        want = R.evict(*evicts[i], lens[i].tolist(), 700, 0, 9)
        for w, t, a, n in got[i]:
            R.within(w, ref, tol)
            assert torch.equal(w, got[i][0][0])
            assert torch.equal(t.cpu(), want[0]) and torch.equal(a.cpu(), want[1]) and n.tolist() == want[2]


def test_eviction_of_long_rows_in_a_graph(pkg, cuda):
    """Clusters of CTAs, in place, replayed: the second replay finds short rows and leaves them."""
    table, w = evict_case([60000, 20000], 60000, seed=60)
    t, a, n = table.to(cuda), w.to(cuda), torch.tensor([60000, 20000], dtype=I64, device=cuda)
    freed, counts = torch.zeros((2, 60000), dtype=I32, device=cuda), torch.zeros(2, dtype=I32, device=cuda)
    scratch = (t.clone(), a.clone(), n.clone())
    pkg.evict_lightest(*scratch, keep=5000, protect_first=1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pkg.evict_lightest(t, a, n, keep=5000, protect_first=1, freed=freed, freed_lens=counts)
    want = R.evict(table, w, [60000, 20000], 5000, 1, 0)
    graph.replay()
    assert counts.tolist() == [55000, 15000] and freed[0, :55000].tolist() == want[3][0]
    for _ in range(2):
        assert torch.equal(t.cpu(), want[0]) and torch.equal(a.cpu(), want[1]) and n.tolist() == [5000, 5000]
        graph.replay()
        assert counts.tolist() == [0, 0]


def test_eviction_of_a_row_named_again_stays_in_bounds(pkg, cuda):
    """Distinct rows are the caller's part; where two requests change one row at once, longer than shared
    memory holds, its result is anybody's, but nothing outside it and the requests' own entries is written."""
    batch, width, keep = 80, 40000, 3000
    g = torch.Generator().manual_seed(61)
    table = torch.randint(0, 1 << 30, (3, width + 64), generator=g, dtype=I32).to(cuda)
    w = torch.rand((3, width + 64), generator=g).to(cuda)
    kept = table.clone(), w.clone()
    rows, lens = torch.ones(batch, dtype=I32, device=cuda), torch.full((batch,), width, dtype=I32, device=cuda)
    freed = torch.full((batch + 2, width - keep + 8), -5, dtype=I32, device=cuda)
    counts = torch.zeros(batch, dtype=I32, device=cuda)
    for _ in range(3):
        w[1] = kept[1][1]
        lens.fill_(width)
        pkg.evict_lightest(table[:, :width], w[:, :width], lens, keep=keep, rows=rows, freed=freed[1:-1, :width - keep], freed_lens=counts)
        torch.cuda.synchronize()
        assert bool((freed[0] == -5).all()) and bool((freed[-1] == -5).all()) and bool((freed[:, width - keep:] == -5).all())
        for got, before in zip((table, w), kept):
            assert torch.equal(got[0], before[0]) and torch.equal(got[2], before[2]) and torch.equal(got[1, width:], before[1, width:])
        assert bool(((lens >= 0) & (lens <= width) & (lens + counts == width)).all())


# ---- together --------------------------------------------------------------------------------------
def test_prefill_judge_decode_evict_decode(pkg, cuda):
    """One request's life: prefill, the prompt's weights, decode steps that go on with them, an eviction,
    and decoding over what is left."""
    heads, kv, prompt, steps, keep = 24, 4, 300, 5, 200
    g = torch.Generator().manual_seed(31)
    pool = 1024
    k = torch.randn((pool, kv, 256), generator=g).to(BF16).to(cuda)
    v = torch.randn((pool, kv, 256), generator=g).to(BF16).to(cuda)
    free = torch.randperm(pool, generator=g).to(cuda)
    table = torch.zeros((3, 512), dtype=I32, device=cuda)
    acc = torch.zeros((3, 512), device=cuda)
    row = torch.tensor([1], dtype=I32, device=cuda)
    table[1, :prompt] = free[:prompt].to(I32)
    q = torch.randn((prompt, heads, 256), generator=g).to(BF16).to(cuda)
    idx = table[1, :prompt]
    _, lse = pkg.prefill_extend(q, k, v, idx, 0, sm_scale=1 / 16, qk_i8=False, return_lse=True)
    want, tol = R.extend_weights(q, k, idx, 0, lse, acc[1, :prompt])
    pkg.extend_weights(q, k, idx, 0, lse, acc[1, :prompt], check_status=True)
    R.within(acc[1, :prompt], want, tol)
    lens = torch.tensor([prompt], dtype=I32, device=cuda)
    ws = pkg.plan_decode_workspace(cuda, max_requests=1, q_heads=heads, kv_heads=kv, max_weight_tokens=512)

    def step(i):
        lens.add_(1)
        table[1, int(lens) - 1] = free[prompt + i].to(I32)
        qs = torch.randn((1, heads, 256), generator=g).to(BF16).to(cuda)
        before = acc.clone()
        out, one = pkg.paged_decode(qs, k, v, table, lens, rows=row, workspace=ws, weights=acc, return_lse=True,
                                    check_status=True)
        ref = R.decode(qs, k, v, table, lens, row, weights=before)
        R.within(out, ref["out"], ref["out_tol"])
        R.within(acc, ref["weights"], ref["weights_tol"])

    for i in range(steps):
        step(i)
    total = float(acc.sum())
    t0, a0 = table.cpu().clone(), acc.cpu().clone()
    want = R.evict(t0, a0, lens.tolist(), keep, 4, 32, row.tolist())
    _, _, _, freed, gone = pkg.evict_lightest(table, acc, lens, keep=keep, protect_first=4, protect_last=32, rows=row)
    assert torch.equal(table.cpu(), want[0]) and torch.equal(acc.cpu(), want[1]) and lens.tolist() == [keep]
    assert freed[0, :int(gone[0])].tolist() == want[3][0] and int(gone[0]) == prompt + steps - keep
    assert float(acc.sum()) < total and not acc[1, keep:].any()
    for i in range(steps, steps + 3):
        step(i)
