"""What the paged decode attention, the attention weights of an extend and the eviction by
accumulated weight cost, case by case.

`run` makes one pass: with `own` the framework's entry points, without it the same operators in
elementary torch operations.  `exact` gives a pass's outputs from the definitions in 64 bits.

The operators, over a token-granular pool `k_pool`, `v_pool` [slots, kv_heads, 256] and a page table
[rows, width] that lists each request's slots in position order (c = sm_scale * log2 e):

  paged_decode     x[h, n] = c <q_h, k_n>, n < len;  lse_h = log2 sum_n 2^x;
                   out_h = sum_n 2^(x - lse_h) v_n;  weights[n] = decay weights[n] + sum_h 2^(x - lse_h)
  extend_weights   weights[n] = decay weights[n] + sum_{t, h: n <= prefix + t} 2^(c <q_th, k_n> - lse_th)
  evict_lightest   keeps the first and the last positions of a request and the heaviest of the
                   others (of equal ones the lowest positions), in position order
"""
import math
import random

import numpy as np
import torch

own = False

D = 256
LOG2E = 1.4426950408889634
SM_SCALE = 0.0625


def listed():
    return [
        # one short conversation: latency of a single step
        dict(name="decode one short", op="decode", batch=1, shortest=1000, longest=1000, lengths=1, q_heads=24,
             kv_heads=4, dtype="bfloat16", idx="int32", weights=False),
        # the requests of the main prefill profile (prefix 1024 to 8192 and 2048 new tokens), now decoding
        dict(name="decode profile batch", op="decode", batch=8, shortest=1025, longest=10240, lengths=2, q_heads=24,
             kv_heads=4, dtype="bfloat16", idx="int64", weights=False),
        # a serving step over ragged requests with an FP16 pool, an empty padding entry among them
        dict(name="decode ragged fp16", op="decode", batch=64, shortest=0, longest=16384, lengths=3, q_heads=32,
             kv_heads=4, dtype="float16", idx="int32", weights=False),
        # the long single request (131072 cached and 8192 extended positions)
        dict(name="decode one long", op="decode", batch=1, shortest=139264, longest=139264, lengths=4, q_heads=32,
             kv_heads=4, dtype="bfloat16", idx="int32", weights=False),
        # one key/value head with its group: a rank's part of a batch that is split by heads
        dict(name="decode head shard", op="decode", batch=17, shortest=1, longest=16385, lengths=5, q_heads=6,
             kv_heads=1, dtype="bfloat16", idx="int32", weights=False),
        # a serving step that also records what the new tokens attend to
        dict(name="decode weights serving", op="decode", batch=128, shortest=0, longest=8192, lengths=6, q_heads=24,
             kv_heads=4, dtype="bfloat16", idx="int32", weights=True),
        # the same for a few requests of moderate length
        dict(name="decode weights few", op="decode", batch=4, shortest=300, longest=4097, lengths=7, q_heads=16,
             kv_heads=4, dtype="float16", idx="int64", weights=True),
        # the last rows of a prompt as the window that judges its cache
        dict(name="weights window", op="weights", rows=32, prefix=4065, q_heads=24, kv_heads=4, dtype="bfloat16",
             idx="int32"),
        # every row of a chunk of the main profile at its longest prefix
        dict(name="weights profile", op="weights", rows=2048, prefix=8192, q_heads=24, kv_heads=4, dtype="bfloat16",
             idx="int64"),
        # a ragged chunk of the head sweep, FP16 pool, lengths that divide by nothing
        dict(name="weights ragged fp16", op="weights", rows=511, prefix=14981, q_heads=32, kv_heads=4,
             dtype="float16", idx="int32"),
        # bounding the cache of a serving batch
        dict(name="evict serving", op="evict", batch=256, shortest=0, longest=32768, lengths=8, keep=4096, first=4,
             last=512, idx="int32"),
        # bounding the cache of the long request
        dict(name="evict one long", op="evict", batch=1, shortest=139264, longest=139264, lengths=9, keep=16384,
             first=4, last=1024, idx="int64"),
    ]


def draw(rng):
    def spread(low, high):
        return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))

    op = rng.choice(["decode", "decode", "weights", "evict"])
    idx = rng.choice(["int32", "int64"])
    q_heads, kv_heads = rng.choice([(16, 4), (24, 4), (32, 4), (8, 2), (12, 2), (6, 1), (8, 1)])
    dtype = rng.choice(["bfloat16", "float16"])
    if op == "weights":
        rows = spread(1, 2048)
        return dict(op=op, rows=rows, prefix=spread(64, 8192), q_heads=min(q_heads, 24), kv_heads=kv_heads,
                    dtype=dtype, idx=idx)
    batch = spread(1, 128 if op == "decode" else 256)
    longest = spread(17, max(17, min(131072, (524288 if op == "decode" else 4194304) // batch)))
    shortest = rng.choice([0, 1, longest // 2, longest])
    case = dict(op=op, batch=batch, shortest=shortest, longest=longest, lengths=rng.randrange(1 << 30), idx=idx)
    if op == "decode":
        return dict(case, q_heads=q_heads, kv_heads=kv_heads, dtype=dtype, weights=rng.random() < 0.4)
    keep = spread(8, max(8, longest))
    first, last = rng.randrange(0, keep // 4 + 1), rng.randrange(0, keep // 2 + 1)
    return dict(case, keep=keep, first=first, last=last)


def lengths_of(case):
    r = random.Random(case["lengths"])
    return [r.randint(case["shortest"], case["longest"]) for _ in range(case["batch"])]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"decode": prepare_decode, "weights": prepare_weights, "evict": prepare_evict}[case["op"]](case, g)


def pool_of(slots, case, g):
    """Keys and values as a projection leaves them: unit normal, a token's norm varying by four."""
    dtype = getattr(torch, case["dtype"])

    def rows():
        x = torch.randn((slots, case["kv_heads"], D), generator=g, device="cuda", dtype=torch.float32)
        return (x * (torch.rand((slots, 1, 1), generator=g, device="cuda") * 1.5 + 0.5)).to(dtype)

    return rows(), rows()


def table_of(lens, width, slots, idx, g):
    """A page table whose rows hold disjoint slots in shuffled order; requests sit in shuffled rows."""
    batch = len(lens)
    n = torch.tensor(lens, device="cuda")
    order = torch.randperm(slots, generator=g, device="cuda")
    start = torch.cumsum(n, 0) - n
    at = torch.arange(width, device="cuda")
    inside = at < n[:, None]
    rows = torch.randperm(batch, generator=g, device="cuda")
    table = torch.zeros((batch, width), dtype=getattr(torch, idx), device="cuda")
    table[rows] = torch.where(inside, order[(start[:, None] + at).clamp(max=slots - 1)], 0).to(table.dtype)
    return table, rows.to(torch.int32), n.to(torch.int32)


def prepare_decode(case, g):
    lens = lengths_of(case)
    slots = sum(lens) + 64
    width = max(max(lens), 1) + 16
    k_pool, v_pool = pool_of(slots, case, g)
    table, rows, n = table_of(lens, width, slots, case["idx"], g)
    q = torch.randn((case["batch"], case["q_heads"], D), generator=g, device="cuda").to(torch.bfloat16)
    s = dict(case, q=q, k_pool=k_pool, v_pool=v_pool, table=table, table_rows=rows, lens=n, out=torch.empty_like(q),
             lse=torch.empty(q.shape[:2], device="cuda"))
    s["acc"] = torch.zeros(table.shape, device="cuda") if case["weights"] else None
    if own:
        import attn_kernel_lab_b200 as akl

        s["workspace"] = akl.plan_decode_workspace(
            q.device, max_requests=case["batch"], q_heads=case["q_heads"], kv_heads=case["kv_heads"],
            max_weight_tokens=sum(lens) + 64 * case["batch"] if case["weights"] else 0)
    return s


def prepare_weights(case, g):
    n = case["prefix"] + case["rows"]
    slots = n + 64
    k_pool, _ = pool_of(slots, case, g)
    idx = torch.randperm(slots, generator=g, device="cuda")[:n].to(getattr(torch, case["idx"])).contiguous()
    q = torch.randn((case["rows"], case["q_heads"], D), generator=g, device="cuda").to(torch.bfloat16)
    s = dict(case, q=q, k_pool=k_pool, idx_list=idx, acc=torch.zeros(n, device="cuda"))
    x = extend_logits(s)          # the log-sum-exp that the chunk's attention returned
    s["lse"] = (torch.logsumexp(x / LOG2E, dim=1) * LOG2E).reshape(case["q_heads"], case["rows"]).T.contiguous()
    if own:
        import attn_kernel_lab_b200 as akl

        s["workspace"] = akl.plan_weights_workspace(q.device, max_kv_len=n, max_q_len=case["rows"],
                                                    q_heads=case["q_heads"], kv_heads=case["kv_heads"])
    return s


def prepare_evict(case, g):
    lens = lengths_of(case)
    width = max(max(lens), 1) + 16
    table, rows, n = table_of(lens, width, sum(lens) + 64, case["idx"], g)
    # accumulated attention: heavy-tailed, and nothing at all on many positions
    acc = torch.exp(2 * torch.randn(table.shape, generator=g, device="cuda"))
    acc = torch.where(torch.rand(table.shape, generator=g, device="cuda") < 0.1, 0.0, acc)
    return dict(case, table=table, table_rows=rows, lens=n, acc=acc, table_out=torch.zeros_like(table),
                acc_out=torch.zeros_like(acc), lens_out=torch.zeros_like(n),
                freed=torch.zeros((case["batch"], max(1, width - case["keep"])), dtype=table.dtype, device="cuda"),
                freed_lens=torch.zeros_like(n))


def run(state):
    return {"decode": run_decode, "weights": run_weights, "evict": run_evict}[state["op"]](state)


def run_decode(s):
    if own:
        import attn_kernel_lab_b200 as akl

        out, lse = akl.paged_decode(s["q"], s["k_pool"], s["v_pool"], s["table"], s["lens"], rows=s["table_rows"],
                                    workspace=s["workspace"], out=s["out"], lse_out=s["lse"], weights=s["acc"],
                                    weight_decay=0.0, sm_scale=SM_SCALE, return_lse=True)
    else:
        out, lse = decode_plain(s)
    return {"out": out, "lse": lse} if s["acc"] is None else {"out": out, "lse": lse, "weights": s["acc"]}


def decode_plain(s):
    q, k_pool, lens, rows = s["q"], s["k_pool"], s["lens"], s["table_rows"].long()
    batch, heads, kv_heads = q.shape[0], q.shape[1], k_pool.shape[1]
    slots = s["table"][rows].long()
    valid = torch.arange(slots.shape[1], device=q.device) < lens[:, None]
    slots = torch.where(valid, slots, 0)
    k = k_pool[slots].float()                                      # [batch, width, kv_heads, 256]
    qf = q.float().reshape(batch, kv_heads, heads // kv_heads, D)
    x = torch.einsum("bjgd,bnjd->bjgn", qf, k) * (SM_SCALE * LOG2E)
    del k
    x = torch.where(valid[:, None, None, :], x, -math.inf)
    top = x.amax(dim=-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp2(x - top)
    total = p.sum(dim=-1, keepdim=True)
    p = torch.where(total > 0, p / total, 0.0)
    v = torch.where(valid[:, :, None, None], s["v_pool"][slots].float(), 0.0)
    out = torch.einsum("bjgn,bnjd->bjgd", p, v).reshape(batch, heads, D).to(q.dtype)
    if s["acc"] is not None:
        s["acc"][rows] = torch.where(valid, p.sum(dim=(1, 2)), s["acc"][rows])
    return out, (top + torch.log2(total)).reshape(batch, heads)


def extend_logits(s):
    """c <q, k> as [kv_heads, group * rows, positions] in 32 bits; -inf above the diagonal."""
    q, k_pool = s["q"], s["k_pool"]
    rows, heads, kv_heads = q.shape[0], q.shape[1], k_pool.shape[1]
    k = k_pool[s["idx_list"].long()].float()
    qf = q.float().permute(1, 0, 2).reshape(kv_heads, heads // kv_heads * rows, D)
    x = torch.einsum("jrd,njd->jrn", qf, k).mul_(SM_SCALE * LOG2E).reshape(heads, rows, -1)
    hidden = torch.arange(k.shape[0], device=q.device) > s["prefix"] + torch.arange(rows, device=q.device)[:, None]
    return x.masked_fill_(hidden, -math.inf).reshape(heads * rows, -1)


def run_weights(s):
    if own:
        import attn_kernel_lab_b200 as akl

        return akl.extend_weights(s["q"], s["k_pool"], s["idx_list"], s["prefix"], s["lse"], s["acc"],
                                  weight_decay=0.0, workspace=s["workspace"], sm_scale=SM_SCALE)
    x = extend_logits(s)
    s["acc"].copy_(x.sub_(s["lse"].T.reshape(-1, 1)).exp2_().sum(dim=0))
    return s["acc"]


def run_evict(s):
    if own:
        import attn_kernel_lab_b200 as akl

        return akl.evict_lightest(s["table"], s["acc"], s["lens"], keep=s["keep"], protect_first=s["first"],
                                  protect_last=s["last"], rows=s["table_rows"], page_table_out=s["table_out"],
                                  weights_out=s["acc_out"], kv_lens_out=s["lens_out"], freed=s["freed"],
                                  freed_lens=s["freed_lens"])
    return evict_plain(s)


def evict_plain(s):
    rows, keep = s["table_rows"].long(), s["keep"]
    n = s["lens"].long()[:, None]
    slots, acc = s["table"][rows], s["acc"][rows]
    at = torch.arange(slots.shape[1], device=acc.device)
    valid = at < n
    guarded = valid & ((at < s["first"]) | (at >= n - s["last"]))
    full = n > keep
    # heaviest first, equal ones by position: a stable sort of the weights of the positions that compete
    weight = torch.where(acc.isnan(), -math.inf, acc).double().clamp(min=-1e300)
    weight = torch.where(valid & ~guarded, weight, -math.inf)
    order = torch.sort(weight, dim=1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(1, order, at.expand_as(order).contiguous())
    stays = valid & (~full | guarded | (rank < keep - s["first"] - s["last"]))
    goes = valid & ~stays
    put(s["table_out"], rows, stays, slots)
    left = torch.where(valid, 0.0, s["acc_out"][rows])
    s["acc_out"][rows] = left
    put(s["acc_out"], rows, stays, acc)
    put(s["freed"], torch.arange(len(rows), device=acc.device), goes, slots)
    s["lens_out"].copy_(stays.sum(dim=1))
    s["freed_lens"].copy_(goes.sum(dim=1))
    return s["table_out"], s["acc_out"], s["lens_out"], s["freed"], s["freed_lens"]


def put(to, rows, chosen, values):
    """The chosen values of each row, moved together to the row's front."""
    row = rows[:, None].expand_as(chosen)[chosen]
    to[row, (chosen.cumsum(dim=1) - 1)[chosen]] = values[chosen]


def work(case):
    item = 2
    index = 4 if case["idx"] == "int32" else 8
    if case["op"] == "decode":
        n, rows = sum(lengths_of(case)), case["batch"] * case["q_heads"]
        moved = n * (case["kv_heads"] * D * item * 2 + index + (4 if case["weights"] else 0)) + rows * (4 * D + 4)
        return {"bytes": moved + 8 * case["batch"], "flops": 4.0 * case["q_heads"] * D * n}
    if case["op"] == "weights":
        t, n = case["rows"], case["prefix"] + case["rows"]
        moved = n * (case["kv_heads"] * D * item + index + 4) + t * case["q_heads"] * (D * 2 + 4)
        return {"bytes": moved, "flops": 2.0 * case["q_heads"] * D * t * (case["prefix"] + (t + 1) / 2)}
    moved = 0
    for n in lengths_of(case):
        kept = min(n, case["keep"])
        moved += n * (4 + index) + n * 4 + kept * index + (n - kept) * index
    return {"bytes": moved + 16 * case["batch"], "flops": 0}


def exact(case, seed):
    s = prepare(case, seed)
    return {"decode": exact_decode, "weights": exact_weights, "evict": exact_evict}[case["op"]](s)


def exact_decode(s):
    """Request by request, head by head, in 64 bits."""
    q, heads, kv_heads = s["q"].double(), s["q"].shape[1], s["k_pool"].shape[1]
    group = heads // kv_heads
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    acc = None if s["acc"] is None else s["acc"].double()
    for b, (row, n) in enumerate(zip(s["table_rows"].tolist(), s["lens"].tolist())):
        if n == 0:
            continue
        at = s["table"][row, :n].long()
        share = torch.zeros(n, dtype=torch.float64, device=q.device)
        for j in range(kv_heads):
            k, v = s["k_pool"][at, j].double(), s["v_pool"][at, j].double()
            for h in range(j * group, (j + 1) * group):
                z = (k @ q[b, h]) * SM_SCALE
                total = torch.logsumexp(z, 0)
                p = torch.exp(z - total)
                out[b, h] = p @ v
                lse[b, h] = total / math.log(2.0)
                share += p
        if acc is not None:
            acc[row, :n] = share
    return {"out": out, "lse": lse} if acc is None else {"out": out, "lse": lse, "weights": acc}


def exact_weights(s):
    q, heads, kv_heads = s["q"].double(), s["q"].shape[1], s["k_pool"].shape[1]
    rows, n = q.shape[0], s["idx_list"].numel()
    total = torch.zeros(n, dtype=torch.float64, device=q.device)
    at = s["idx_list"].long()
    seen = torch.ones((rows, n), dtype=torch.float64, device=q.device).tril(s["prefix"])
    for h in range(heads):
        k = s["k_pool"][at, h // (heads // kv_heads)].double()
        p = torch.exp((q[:, h] @ k.T) * SM_SCALE - (s["lse"][:, h].double() * math.log(2.0))[:, None])
        total += (p * seen).sum(0)
    return total


def exact_evict(s):
    table, acc = s["table"].cpu().numpy(), s["acc"].cpu().numpy().astype(np.float64)
    table_out, acc_out = s["table_out"].cpu().numpy(), s["acc_out"].cpu().numpy().astype(np.float64)
    freed, lens = s["freed"].cpu().numpy(), s["lens"].tolist()
    lens_out, freed_lens = np.zeros(len(lens), np.int32), np.zeros(len(lens), np.int32)
    for b, (row, n) in enumerate(zip(s["table_rows"].tolist(), lens)):
        stays = np.arange(n)
        if n > s["keep"]:
            middle = np.arange(s["first"], n - s["last"])
            w = np.where(np.isnan(acc[row, middle]), -np.inf, acc[row, middle])
            best = middle[np.lexsort((middle, -w))][:s["keep"] - s["first"] - s["last"]]
            stays = np.sort(np.concatenate([stays[:s["first"]], best, stays[n - s["last"]:]]))
        goes = np.setdiff1d(np.arange(n), stays)
        acc_out[row, :n] = 0
        table_out[row, :len(stays)], acc_out[row, :len(stays)] = table[row, stays], acc[row, stays]
        freed[b, :len(goes)] = table[row, goes]
        lens_out[b], freed_lens[b] = len(stays), len(goes)
    return tuple(torch.from_numpy(x) for x in (table_out, acc_out, lens_out, freed, freed_lens))
