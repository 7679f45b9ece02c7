"""The extend's log-sum-exp over the pool's own keys (`pool_lse`), and what is built on it: attention weights,
eviction by them, and merging with a decode step.  Keys have a mean per channel, as those of models do."""
import math

import pytest
import torch

import decode_ref as R

pytestmark = pytest.mark.gpu

BF16, FP16, I32, I64 = torch.bfloat16, torch.float16, torch.int32, torch.int64
C = R.LOG2E / 16                      # sm_scale 1/16 and base 2
HEADS, KV = 24, 4


def case(rows, prefix, mean, dtype, *, idx=I32, seed=0):
    """A request whose keys are unit normal plus a constant per head and channel of standard deviation `mean`."""
    g = torch.Generator().manual_seed(seed)
    n = prefix + rows
    pool = n + 40
    k = torch.randn((pool, KV, 256), generator=g) + mean * torch.randn((1, KV, 256), generator=g)
    v = torch.randn((pool, KV, 256), generator=g)
    at = torch.randperm(pool, generator=g)[:n].to(idx)
    q = torch.randn((rows, HEADS, 256), generator=g).to(BF16)
    return dict(q=q.cuda(), k_pool=k.to(dtype).cuda(), v_pool=v.to(dtype).cuda(), idx=at.cuda(), prefix=prefix)


def exact(c):
    """(keys [n, KV, 256], scores [HEADS, rows, n] in base 2 with -inf where nothing is seen), in 64 bits."""
    k = c["k_pool"][c["idx"].long()].double()
    rows, n = c["q"].shape[0], k.shape[0]
    qg = c["q"].double().view(rows, KV, HEADS // KV, 256)
    x = C * torch.einsum("tjgd,njd->jgtn", qg, k).reshape(HEADS, rows, n)
    seen = torch.arange(n, device="cuda") <= c["prefix"] + torch.arange(rows, device="cuda")[:, None]
    return k, x.masked_fill(~seen, -math.inf)


def quantised_score_bound(c, k, qk_i8):
    """[HEADS] six standard deviations of what quantising Q and K does to a score, at its worst row and key.

    The extend quantises the rotated Q rows and the rotated, centred K.  A rounding to INT8 is off by at most half of
    amax / 127 (of the row, of the 64-key tile), to E4M3 by 2^-4 of the value; evenly spread that is a standard
    deviation of step / sqrt(12) and of 2^-4 |x| / sqrt(3).  A score adds up 256 of them for K and 256 for Q."""
    h = torch.ones((1, 1), dtype=torch.float64, device="cuda")
    for _ in range(8):
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
    h /= 16
    qr, kr = c["q"].double() @ h, (k - k.mean(0)) @ h
    out = []
    for head in range(HEADS):
        qh, kh = qr[:, head], kr[:, head // (HEADS // KV)]
        if qk_i8:
            sq = qh.abs().amax(1) / 127
            sk = torch.cat([t.abs().max().expand(len(t)) for t in kh.split(64)]) / 127
            var = (sq[:, None] ** 2 * (kh ** 2).sum(1) + (qh ** 2).sum(1)[:, None] * sk ** 2) / 12
        else:
            var = 2 * (qh ** 2 @ (kh ** 2).T) * 2.0 ** -8 / 3
        out.append(6 * C * float(var.max().sqrt()))
    return torch.tensor(out, dtype=torch.float64, device="cuda")


def extend(pkg, c, entry, **kw):
    args = dict(sm_scale=1 / 16, return_lse=True, **kw)
    if entry == "single":
        return pkg.prefill_extend(c["q"], c["k_pool"], c["v_pool"], c["idx"], c["prefix"], **args)
    other = case(9, 70, 3.0, c["k_pool"].dtype, idx=c["idx"].dtype, seed=99)        # in front of it in the batch
    ws = pkg.plan_batch_workspace(c["q"].device, max_requests=2, max_total_kv_len=c["idx"].shape[0] + 79,
                                  max_total_q_len=c["q"].shape[0] + 9, q_heads=HEADS, kv_heads=KV)
    return pkg.prefill_extend_batch([other, c], workspace=ws, **args)[1]


@pytest.mark.parametrize("entry", ["single", "batch"])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("qk_i8", [True, False])
@pytest.mark.parametrize("rows,prefix,mean,idx", [(33, 480, 1.0, I32), (1, 0, 1.0, I64), (130, 2500, 0.0, I64)])
def test_the_term_of_the_mean(pkg, cuda, entry, dtype, qk_i8, rows, prefix, mean, idx):
    """`out` keeps its bits; the LSE grows by c <q, mean>.  The mean is a 32-bit sum at most 64 + tiles roundings
    deep (u = 2^-24 of sum |k| each), the product one of 16, and the sum with the LSE one more."""
    c = case(rows, prefix, mean, dtype, idx=idx, seed=rows)
    out0, lse0 = extend(pkg, c, entry, qk_i8=qk_i8)
    out1, lse1 = extend(pkg, c, entry, qk_i8=qk_i8, pool_lse=True)
    assert torch.equal(out0, out1)
    k, _ = exact(c)
    kbar, kabs = (t.repeat_interleave(HEADS // KV, 0) for t in (k.mean(0), k.abs().mean(0)))
    q = c["q"].double()
    term = C * (q * kbar).sum(-1)
    u = 2.0 ** -24
    tol = u * (C * (q.abs() * ((66 + k.shape[0] / 64) * kabs + 18 * kbar.abs())).sum(-1) + lse0.double().abs() + 2 * term.abs())
    R.within(lse1, lse0.double() + term, tol)
    plain = extend(pkg, c, entry, qk_i8=qk_i8, center_k=False)
    same = extend(pkg, c, entry, qk_i8=qk_i8, center_k=False, pool_lse=True)
    assert torch.equal(plain[1], same[1]) and torch.equal(plain[0], same[0])


@pytest.mark.parametrize("entry", ["single", "batch"])
@pytest.mark.parametrize("mean", [0.5, 1.0, 2.0])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("qk_i8", [True, False])
def test_weights_and_eviction_after_an_extend(pkg, cuda, entry, mean, dtype, qk_i8):
    """The weights are those of the pool's 64-bit softmax.  The scores of `extend_weights` are exact to 32 bits; the LSE
    carries the extend's quantisation, and as a mean over a row's scores it is off by no more than the worst of
    them, so a row's weights are off by one factor within 2^+-bound."""
    rows, prefix, keep, first, last = 32, 480, 128, 4, 16
    c = case(rows, prefix, mean, dtype, seed=int(10 * mean))
    n = rows + prefix
    _, lse = extend(pkg, c, entry, qk_i8=qk_i8, pool_lse=True)
    weights = torch.full((1, n), float("nan"), device=cuda)
    pkg.extend_weights(c["q"], c["k_pool"], c["idx"], prefix, lse, weights[0], weight_decay=0.0, check_status=True)
    k, x = exact(c)
    bound = quantised_score_bound(c, k, qk_i8)
    true_lse = torch.logsumexp(x * math.log(2), -1) / math.log(2)
    assert bool(((lse.double().T - true_lse).abs() <= bound[:, None]).all())
    p = torch.softmax(x * math.log(2), -1)
    want = p.sum((0, 1))
    tol = (p.sum(1) * (torch.exp2(bound) - 1)[:, None]).sum(0) + 1e-4 * want
    R.within(weights[0], want, tol)
    # the positions that stay are the heaviest, up to weights that the bound cannot tell apart
    table = torch.arange(n, dtype=I32, device=cuda)[None]
    pkg.evict_lightest(table, weights, torch.tensor([n], dtype=I32, device=cuda), keep=keep, protect_first=first,
                       protect_last=last)
    stays = torch.zeros(n, dtype=torch.bool, device=cuda)
    stays[table[0, :keep].long()] = True
    assert int(stays.sum()) == keep and bool(stays[:first].all()) and bool(stays[n - last:].all())
    middle = torch.arange(n, device=cuda)
    middle = (middle >= first) & (middle < n - last)
    assert float((want + tol)[middle & stays].min()) >= float((want - tol)[middle & ~stays].max())


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_a_decode_step_merges_with_an_extend(pkg, cuda, dtype):
    """One query over two parts of its cache, one part by each operator: the parts' shares are those of the whole."""
    from attn_kernel_lab_b200.dist import merge_states

    n, cut = 900, 500
    c = case(1, n - 1, 2.0, dtype, seed=5)
    k, x = exact(c)
    o1, l1 = pkg.paged_decode(c["q"], c["k_pool"], c["v_pool"], c["idx"][None], torch.tensor([cut], device=cuda), return_lse=True)
    rest = dict(c, idx=c["idx"][cut:].contiguous(), prefix=n - cut - 1)
    o2, l2 = pkg.prefill_extend(**rest, sm_scale=1 / 16, return_lse=True, pool_lse=True)
    out, lse = merge_states([o1, o2], [l1, l2])
    bound = quantised_score_bound(rest, k[cut:], True)
    true = torch.logsumexp(x[:, 0] * math.log(2), -1) / math.log(2)
    assert bool(((lse[0].double() - true).abs() <= bound + 1e-5).all())
    share = torch.softmax(x[:, 0] * math.log(2), -1)[:, :cut].sum(-1)[:, None]
    want = share * o1[0].double() + (1 - share) * o2[0].double()
    tol = (torch.exp2(bound) - 1)[:, None] * (o1[0].double() - o2[0].double()).abs() + 2.0 ** -8 * want.abs() + 1e-5
    R.within(out[0], want, tol)


def test_graphs_and_phases_carry_it(pkg, cuda):
    c = case(40, 300, 1.0, BF16, seed=7)
    from attn_kernel_lab_b200.dist import kv_split_local
    from attn_kernel_lab_b200.quant import FP8PrefillWorkspace

    ws = pkg.plan_workspace(cuda, max_kv_len=400, max_q_len=64, q_heads=HEADS, kv_heads=KV)
    out, lse = torch.empty_like(c["q"]), torch.empty((40, HEADS), device=cuda)
    kw = dict(workspace=ws, out=out, lse_out=lse, sm_scale=1 / 16, return_lse=True, pool_lse=True)
    pkg.prefill_extend(**c, **kw)
    want = lse.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pkg.prefill_extend(**c, **kw)
    lse.zero_()
    graph.replay()
    assert torch.equal(lse, want)
    c["k_pool"] += 1.0
    graph.replay()
    assert torch.equal(lse, pkg.prefill_extend(**c, sm_scale=1 / 16, return_lse=True, pool_lse=True)[1])
    # the phases, with the statistics between them as a split request has them
    single = FP8PrefillWorkspace(cuda)
    _, split = kv_split_local(single, c["q"], c["k_pool"], c["v_pool"], c["idx"], 300, n_total=340, kv_lo=0, sm_scale=1 / 16,
                              qk_i8=True, pool_lse=True)
    assert torch.equal(split, lse)
    # a batch whose requests do not all want an LSE, replanned
    bw = pkg.plan_batch_workspace(cuda, max_requests=3, max_total_kv_len=2000, max_total_q_len=400, q_heads=HEADS, kv_heads=KV)
    reqs = [dict(case(t, p, 2.0, BF16, seed=t)) for t, p in ((200, 64), (3, 900), (70, 11))]
    for r in reqs:
        r.update(out=torch.empty_like(r["q"]), lse_out=torch.full(r["q"].shape[:2], -7.0, device=cuda))
    reqs[1]["lse_out"] = None
    plan = bw.plan(reqs, sm_scale=1 / 16, qk_i8=True, pool_lse=True)
    bw.launch(plan)
    for r in (reqs[0], reqs[2]):
        one = pkg.prefill_extend(*(r[k] for k in ("q", "k_pool", "v_pool", "idx", "prefix")), sm_scale=1 / 16, return_lse=True, pool_lse=True)
        assert torch.equal(r["lse_out"], one[1]) and torch.equal(r["out"], one[0])
    reqs[2]["lse_out"].fill_(-7.0)
    bw.replan(plan, reqs[2:])
    bw.launch(plan)
    assert torch.equal(reqs[2]["lse_out"], one[1]) and bw.status() == 0
