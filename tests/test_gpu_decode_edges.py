"""Decode attention where its sums, masks and limits can go wrong."""
import math

import pytest
import torch

import decode_ref as R

pytestmark = pytest.mark.gpu

BF16, FP16, I32, I64 = torch.bfloat16, torch.float16, torch.int32, torch.int64


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_decode_sums_over_positions_are_rounded_not_truncated(pkg, cuda, dtype):
    """Position n and position n + half have one key and opposite values, so every output is exactly 0 and
    what comes out is what the sum over the positions lost on its way up and down again.

    With a request per SM a warp adds `tiles` = 2 half / 16 tile sums, one rounding each: off by at most
    half a step of the running sum |o| <= l / 2 (values are at most 1, and the two halves weigh l / 2), of
    standard deviation step / sqrt(12) with a step of 2^-23 |o| at most.  Six standard deviations of
    `tiles` of them, divided by l, are the bound.  Tile sums themselves cancel: equal probabilities (the largest
    score comes first, so no maximum moves later) and mirrored values, in the same places of their tiles.
    A sum that is cut off at 32 bits twice a tile loses 2 tiles x 0.36 steps of l / 4 x 0.75, three to five bounds."""
    half, heads, kv = 8192, 24, 4
    batch = torch.cuda.get_device_properties(cuda).multi_processor_count
    g = torch.Generator().manual_seed(1)
    k = torch.randn((half, kv, 256), generator=g)
    k[:, :, 0] = 0.0
    k[0, :, 0] = 8.0
    v = torch.rand((half, kv, 256), generator=g) * 0.5 + 0.5
    q = torch.randn((batch, heads, 256), generator=g) * 0.5
    q[:, :, 0] = 8.0                                             # scores of +-0.7, and 5.8 more for the first key
    pool = dict(k_pool=torch.cat([k, k]).to(dtype).to(cuda), v_pool=torch.cat([v, -v]).to(dtype).to(cuda))
    out = pkg.paged_decode(q.to(BF16).to(cuda), **pool, page_table=torch.arange(2 * half, device=cuda)[None],
                           kv_lens=torch.full((batch,), 2 * half, device=cuda), rows=torch.zeros(batch, dtype=I32, device=cuda))
    bound = 6 * math.sqrt(2 * half / 16) * 2.0 ** -23 / math.sqrt(12) / 2
    worst = float(out.float().abs().max())
    assert worst <= bound, f"{worst:.3g}, bound {bound:.3g}"


@pytest.mark.parametrize("tokens,fit", [(64, 0), (128, 1), (320, 1), (384, 2), (448, 3)])
def test_weights_beyond_the_plan_leave_whole_rows_alone(pkg, cuda, tokens, fit):
    """A limit that falls inside a request: its row is neither decayed nor added to, in any of its places."""
    c = R.case([100, 250, 30], 24, 4, seed=18)                   # 2, 4 and 1 chunks of 64 positions
    ws = pkg.plan_decode_workspace(cuda, max_requests=3, q_heads=24, kv_heads=4, max_weight_tokens=tokens)
    before = torch.rand(c["page_table"].shape, generator=torch.Generator().manual_seed(2)).to(cuda)
    weights = before.clone()
    out, lse = pkg.paged_decode(**c, workspace=ws, weights=weights, weight_decay=0.5, return_lse=True)
    ref = R.decode(c["q"], c["k_pool"], c["v_pool"], c["page_table"], c["kv_lens"], c["rows"], weights=before, decay=0.5)
    R.within(out, ref["out"], ref["out_tol"])
    R.within(lse, ref["lse"], ref["lse_tol"])
    done = c["rows"][:fit].long()
    R.within(weights[done], ref["weights"][done], ref["weights_tol"][done])
    before[done] = weights[done]
    assert torch.equal(weights, before)
    assert ws.status() == (0 if fit == 3 else -3)


def test_outputs_in_other_memory_are_refused_and_neighbours_are_not(pkg, cuda):
    """With a workspace and outputs of its own, as an engine calls it."""
    c = R.case([100, 40], 24, 4, seed=30)
    ws = pkg.plan_decode_workspace(cuda, max_requests=2, q_heads=24, kv_heads=4, max_weight_tokens=256)
    out, lse = torch.empty_like(c["q"]), torch.empty((2, 24), device=cuda)
    weights = torch.zeros(c["page_table"].shape, device=cuda)
    kw = dict(workspace=ws, lse_out=lse, return_lse=True)
    for field, over in (("out", dict(out=c["k_pool"].view(-1)[:2 * 24 * 256].view(2, 24, 256))), ("lse_out", dict(out=out, lse_out=out.view(-1).view(torch.float32)[:48].view(2, 24))),
                        ("weights", dict(out=out, weights=c["page_table"].view(torch.float32)))):
        with pytest.raises(pkg.CapabilityError) as e:
            pkg.paged_decode(**c, **dict(kw, **over))
        assert e.value.field == field
    # table and weights side by side in one buffer, the outputs one behind the other in another
    rows, width = c["page_table"].shape
    both = torch.zeros((rows, 2 * width), dtype=I32, device=cuda)
    both[:, :width] = c["page_table"]
    flat = torch.zeros(2 * 24 * 256 + 96, dtype=BF16, device=cuda)
    got = pkg.paged_decode(**dict(c, page_table=both[:, :width]), workspace=ws, out=flat[:-96].view(2, 24, 256),
                           lse_out=flat[-96:].view(torch.float32).view(2, 24), return_lse=True, weights=both[:, width:].view(torch.float32))
    want = pkg.paged_decode(**c, **kw, out=out, weights=weights)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(both[:, width:].view(torch.float32), weights)
    assert torch.equal(both[:, :width], c["page_table"])
    lens = c["kv_lens"].clone()
    pkg.evict_lightest(both[:, :width], both[:, width:].view(torch.float32), lens, keep=30, rows=c["rows"])
    want = R.evict(c["page_table"].cpu(), weights.cpu(), [100, 40], 30, rows=c["rows"].tolist())
    assert torch.equal(both[:, :width].cpu(), want[0]) and torch.equal(both[:, width:].view(torch.float32).cpu(), want[1])
    # eviction and the extend's weights, in their short forms
    t, n = c["page_table"].clone(), c["kv_lens"].clone()
    freed, counts = torch.zeros((2, max(1, width - 30)), dtype=I32, device=cuda), torch.zeros(2, dtype=I32, device=cuda)
    with pytest.raises(pkg.CapabilityError) as e:
        pkg.evict_lightest(t, weights, n, keep=30, rows=c["rows"], freed=freed, freed_lens=counts, page_table_out=torch.zeros_like(t),
                           weights_out=t.view(torch.float32))
    assert e.value.field == "weights_out"
    q = c["q"][:2].contiguous()
    idx = c["page_table"][c["rows"][0].long(), :100].contiguous()
    wws = pkg.plan_weights_workspace(cuda, max_kv_len=128, max_q_len=2, q_heads=24, kv_heads=4)
    with pytest.raises(pkg.CapabilityError) as e:
        pkg.extend_weights(q, c["k_pool"], idx, 98, lse, idx.view(torch.float32), workspace=wws)
    assert e.value.field == "weights"


@pytest.mark.parametrize("batch", [8, 9, 10, 17, 18, 19, 37, 74, 75, 149])
def test_eviction_whatever_clusters_the_device_holds_at_once(pkg, cuda, batch):
    """Requests just below and above what fits the GPU in clusters of sixteen, eight, four, two and one."""
    width, keep = 33000, 900
    g = torch.Generator().manual_seed(batch)
    table = torch.randint(0, 1 << 30, (batch, width), generator=g).to(I32)
    w = torch.exp(2 * torch.randn((batch, width), generator=g))
    lens = [width - 17 * i for i in range(batch)]
    t, a, n = table.to(cuda), w.to(cuda), torch.tensor(lens, dtype=I32, device=cuda)
    _, _, _, freed, counts = pkg.evict_lightest(t, a, n, keep=keep, protect_first=2, protect_last=30)
    for b, length in enumerate(lens):
        middle = torch.arange(2, length - 30)
        order = middle[torch.sort(w[b, 2:length - 30], descending=True, stable=True).indices[:keep - 32]]
        stays = torch.zeros(length, dtype=torch.bool)
        stays[:2] = stays[length - 30:] = stays[order] = True
        assert torch.equal(t[b, :keep].cpu(), table[b, :length][stays]) and torch.equal(a[b, :keep].cpu(), w[b, :length][stays])
        assert torch.equal(freed[b, :length - keep].cpu(), table[b, :length][~stays]) and not a[b, keep:length].any()
    assert n.tolist() == [keep] * batch and counts.tolist() == [x - keep for x in lens]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("blind", [math.inf, -math.inf])
def test_rows_without_a_finite_lse_add_nothing_whatever_they_hold(pkg, cuda, dtype, blind):
    from test_gpu_decode import extend_case

    c = extend_case(70, 200, 24, 4, dtype=dtype, seed=25)
    for row, head, value in ((3, 5, math.nan), (40, 0, math.inf), (41, 23, -math.inf), (69, 7, 3e38)):
        c["q"][row, head], c["lse"][row, head] = value, blind
    c["q"][12, 8, 17], c["lse"][12, 8] = math.nan, blind
    kept = c["q"].nan_to_num(0.0, 0.0, 0.0)
    want, tol = R.extend_weights(kept, c["k_pool"], c["idx"], 200, c["lse"], torch.zeros(270, device=cuda), 0.0)
    got = pkg.extend_weights(**c, weights=torch.zeros(270, device=cuda), weight_decay=0.0)
    R.within(got, want, tol)
    c["k_pool"][c["idx"][100].long(), 1, 3] = math.inf          # one position's key: seen by every row
    got = pkg.extend_weights(**c, weights=torch.zeros(270, device=cuda), weight_decay=0.0)
    others = torch.arange(270, device=cuda) != 100
    R.within(got[others], want[others], tol[others])


def test_extend_weights_with_millions_of_positions_that_no_row_sees(pkg, cuda):
    """They lie behind the last row's diagonal: their weights decay, and no more.  (A call takes 0.12 ms; with a
    walk over all tiles of positions before each of them it took 33, and minutes at the largest lengths.)"""
    n, rows, prefix = 1 << 23, 3, 300
    k = torch.randn((512, 4, 256), device=cuda).to(BF16)
    q = torch.randn((rows, 24, 256), device=cuda).to(BF16)
    idx = torch.randint(0, 512, (n,), device=cuda)
    seen = prefix + rows
    x = torch.einsum("tjgd,njd->tjgn", q.view(rows, 4, 6, 256).double(), k[idx[:seen]].double()).reshape(rows, 24, seen) / 16
    hidden = torch.arange(seen, device=cuda) > prefix + torch.arange(rows, device=cuda)[:, None, None]
    lse = (torch.logsumexp(x.masked_fill(hidden, -math.inf), -1) * R.LOG2E).float()
    before = torch.rand(n, device=cuda)
    ws = pkg.plan_weights_workspace(cuda, max_kv_len=n, max_q_len=rows, q_heads=24, kv_heads=4)
    weights = before.clone()
    pkg.extend_weights(q, k, idx, prefix, lse, weights, weight_decay=0.5, workspace=ws, check_status=True)
    want, tol = R.extend_weights(q, k, idx[:seen], prefix, lse, before[:seen], 0.5)
    R.within(weights[:seen], want, tol)
    assert torch.equal(weights[seen:], before[seen:] * 0.5)
    start, stop = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    pkg.extend_weights(q, k, idx, prefix, lse, weights, workspace=ws)
    stop.record()
    stop.synchronize()
    assert start.elapsed_time(stop) < 5.0


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("heads", [(24, 4), (6, 1), (10, 2)])
@pytest.mark.parametrize("where", ["some", "tiles", "part", "all"])
def test_scores_of_minus_infinity_weigh_nothing(pkg, cuda, dtype, heads, where):
    """Keys of -inf under positive queries, at scattered positions, over whole tiles, over more than a CTA's part of a
    request, at every position: as if their slots were not there."""
    c = R.case([700, 5000, 40], *heads, dtype=dtype, seed=33)
    c["q"] = c["q"].abs().clamp(min=0.01)
    r = c["rows"].long()
    gone = torch.zeros(c["page_table"].shape, dtype=torch.bool, device=cuda)
    if where == "some":
        gone[r] = torch.rand((3, gone.shape[1]), generator=torch.Generator().manual_seed(4)).to(cuda) < 0.2
    elif where == "tiles":
        gone[r[0], 64:192] = gone[r[1], 4992:] = gone[r[2], :16] = True
    elif where == "part":
        gone[r[1], :2500] = gone[r[0], 300:] = True
    else:
        gone[r[0]] = gone[r[2]] = True
    for b, n in enumerate((700, 5000, 40)):
        c["k_pool"][c["page_table"][r[b], :n][gone[r[b], :n]].long()] = -math.inf
    before = torch.rand(c["page_table"].shape, generator=torch.Generator().manual_seed(5)).to(cuda)
    weights = before.clone()
    out, lse = pkg.paged_decode(**c, weights=weights, weight_decay=0.5, return_lse=True, check_status=True)
    ref = R.decode(c["q"], c["k_pool"], c["v_pool"], torch.where(gone, -1, c["page_table"]), c["kv_lens"], c["rows"], weights=before,
                   decay=0.5)
    R.within(out, ref["out"], ref["out_tol"])
    R.within(lse, ref["lse"], ref["lse_tol"])
    R.within(weights, ref["weights"], ref["weights_tol"])
    if where == "all":
        assert not out[0].any() and bool((lse[2] == -math.inf).all())


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_weights_of_rows_whose_products_are_exact(pkg, cuda, dtype):
    """Queries of a few channels: nothing is cut off their scores, of up to some thousands, and little may be added."""
    g = torch.Generator().manual_seed(6)
    rows, prefix, n = 40, 260, 300
    q = torch.zeros((rows, 24, 256))
    for at in (0, 77, 200):
        q[:, :, at] = torch.randint(-64, 65, (rows, 24), generator=g) * 4.0
    k = torch.randint(-16, 17, (n, 4, 256), generator=g).float() * 8
    q, k = q.to(BF16).to(cuda), k.to(dtype).to(cuda)
    x = torch.einsum("tjgd,njd->tjgn", q.view(rows, 4, 6, 256).double(), k.double()).reshape(rows, 24, n) / 16
    hidden = torch.arange(n, device=cuda) > prefix + torch.arange(rows, device=cuda)[:, None, None]
    x = x.masked_fill(hidden, -math.inf)
    assert float(x.amax(-1).median()) > 1000
    lse = (torch.logsumexp(x, -1) * R.LOG2E).float()
    got = pkg.extend_weights(q, k, torch.arange(n, device=cuda), prefix, lse, torch.zeros(n, device=cuda), weight_decay=0.0)
    want, tol = R.extend_weights(q, k, torch.arange(n, device=cuda), prefix, lse, torch.zeros(n, device=cuda), 0.0)
    # (an exponential below 2^-126 may come out as 0: 32 bits hold no normal number there)
    R.within(got, want, tol + rows * 24 * 2.0 ** -126)
    # per row and head: half a step of the score and of the LSE, and the 2^-22 that the factor adds on average to make up for
    # what longer products lose; three roundings of the factor and the exponent's argument besides
    size = float(x.amax()) * R.LOG2E
    assert float(((got.double() - want).abs() / want.clamp(min=1e-3)).max()) <= math.log(2) * size * (2.0 ** -22 + 5 * 2.0 ** -24) + 1e-5


@pytest.mark.parametrize("lens,heads,dtype", [
    ([30000] + [3] * 12, (24, 4), BF16), ([2] * 30 + [9000, 1, 7000, 0] + [5] * 20 + [20000], (24, 4), FP16),
    ([4000] * 12 + [1] * 300, (6, 1), BF16), ([1] * 40 + [33000], (64, 8), BF16), ([12000] + [0] * 200 + [300] * 3, (8, 2), FP16),
], ids=lambda v: f"{len(v)}x{max(v)}" if isinstance(v, list) else str(v))
def test_long_requests_among_many_short_ones(pkg, cuda, lens, heads, dtype):
    """Parts of one request in nearly every CTA, and more (request, head) pairs than the wide join takes."""
    c = R.case(lens, *heads, dtype=dtype, seed=len(lens))
    weights = torch.zeros(c["page_table"].shape, device=cuda)
    ws = pkg.plan_decode_workspace(cuda, max_requests=len(lens), q_heads=heads[0], kv_heads=heads[1],
                                   max_weight_tokens=sum(lens) + 64 * len(lens))
    got = [pkg.paged_decode(**c, workspace=ws, return_lse=True, weights=weights, weight_decay=0.0, check_status=True) for _ in range(2)]
    ref = R.decode(c["q"], c["k_pool"], c["v_pool"], c["page_table"], c["kv_lens"], c["rows"], weights=torch.zeros_like(weights))
    R.within(got[0][0], ref["out"], ref["out_tol"])
    R.within(got[0][1], ref["lse"], ref["lse_tol"])
    R.within(weights, ref["weights"], ref["weights_tol"])
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_probabilities_keep_their_32_bits_in_the_second_product(pkg, cuda, dtype):
    """Three positions with the values 0, 1 and -1, so an output is (p1 - p2) / l, a difference of nearly equal numbers.

    p1 and p2 lie about 0.53 to 0.73 and 2^-13 apart.  Their exponentials are off by 2^-22 of themselves, their scores
    (of one product and a small one, so next to exact) by two roundings of 2^-25; l is at least 2.  So the output, below
    2^-13 and rounded to 2^-9 of itself, is off by 2 * 0.73 / 2 * (2^-22 + 2^-24) and 2^-22 at most: by 2^-21.  In two numbers of
    eight bits a probability would be off by up to 2^-18."""
    g = torch.Generator().manual_seed(9)
    batch, heads, kv = 200, 24, 4
    q = torch.zeros((batch, heads, 256))
    q[:, :, 0] = 1 + torch.randint(0, 128, (batch, heads), generator=g) / 128
    q[:, :, 1] = 2.0 ** -12 * torch.randint(-128, 129, (batch, heads), generator=g) / 128
    k = torch.zeros((batch, 3, kv, 256))
    k[:, 0, :, 0], k[:, 1:, :, 0] = 8.0, 3.0
    k[:, 1, :, 1] = torch.randint(1, 9, (batch, kv), generator=g).float()
    k[:, 2, :, 1] = -torch.randint(1, 9, (batch, kv), generator=g).float()
    v = torch.tensor([0.0, 1.0, -1.0])[None, :, None, None].expand(batch, 3, kv, 256)
    pool = [t.reshape(3 * batch, kv, 256).to(dtype).to(cuda) for t in (k, v)]
    table = torch.arange(3 * batch, device=cuda).view(batch, 3)
    out = pkg.paged_decode(q.to(BF16).to(cuda), *pool, table, torch.full((batch,), 3, device=cuda))
    x = torch.einsum("bjgd,bnjd->bjgn", q.double().view(batch, kv, heads // kv, 256), k.double()).reshape(batch, heads, 3) / 16
    p = torch.softmax(x, -1)
    want = (p[:, :, 1] - p[:, :, 2]).to(cuda)
    assert float(want.abs().max()) < 2.0 ** -13 and float(p[:, :, 0].max()) < 0.5
    worst = float((out.double() - want[:, :, None]).abs().max())
    assert worst <= 2.0 ** -21, f"2^{math.log2(worst):.2f}"
