"""The decode-side operators in 64 bits, with bounds on what 32-bit kernels may differ by.

Bounds.  u = 2^-23 is one rounding of a 32-bit operation, truncating ones included.  A score is the sum
of 256 products, added at most 32 roundings deep (blocks of 16 products, and at most 16 inside one), so
it is off by 32 u S with S = c sum |q_d k_d|; scaling, subtracting the maximum and the exponential (2 u
relative, 4 u to be safe) add 4 u (|x| + |m|).  A probability is therefore off by the factor 1 + 2 ln2 dx at
most (its own score and the normaliser's).  Sums over the positions go through blocks of 16 and then
at most n / 16 + 64 further roundings; probabilities enter the second product as two 16-bit parts, off by 2^-16.
The BF16 output is off by eps / 2 = 2^-8 of itself.
"""
import math

import torch

U = 2.0 ** -23
LOG2E = 1.4426950408889634


def decode(q, k_pool, v_pool, table, lens, rows=None, sm_scale=1 / 16, weights=None, decay=1.0):
    """{out, lse, weights} in 64 bits and {out_tol, lse_tol, weights_tol}; on the tensors' device."""
    dev = q.device
    batch, heads, _ = q.shape
    pool, kv_heads = k_pool.shape[:2]
    group = heads // kv_heads
    out = torch.zeros(q.shape, dtype=torch.float64, device=dev)
    out_tol = torch.zeros_like(out)
    lse = torch.full((batch, heads), -math.inf, dtype=torch.float64, device=dev)
    lse_tol = torch.zeros_like(lse)
    acc = None if weights is None else weights.double().clone()
    acc_tol = None if weights is None else torch.zeros_like(acc)
    c = sm_scale * LOG2E
    for b in range(batch):
        row = b if rows is None else int(rows[b])
        n = min(max(int(lens[b]), 0), table.shape[1])
        if row < 0 or row >= table.shape[0] or n == 0:
            continue
        slots = table[row, :n].long()
        good = (slots >= 0) & (slots < pool)
        at = torch.nonzero(good)[:, 0]
        share = torch.zeros(n, dtype=torch.float64, device=dev)
        share_tol = torch.zeros_like(share)
        if len(at):
            k, v = k_pool[slots[at]].double(), v_pool[slots[at]].double()
            for h in range(heads):
                j = h // group
                x = c * (k[:, j] @ q[b, h].double())
                top = float(x.max())
                size = c * (k[:, j].abs() @ q[b, h].double().abs())
                dx = float((32 * U * size + 4 * U * (x.abs() + abs(top))).max())
                p = torch.exp2(x - top)
                total = float(p.sum())
                p = p / total
                steps = (n / 16 + 64) * U
                rel = 2 * math.log(2) * dx + 2.0 ** -16 + 2 * steps
                out[b, h] = p @ v[:, j]
                out_tol[b, h] = out[b, h].abs() * 2.0 ** -8 + rel * (p @ v[:, j].abs()) + 2.0 ** -126
                lse[b, h] = top + math.log2(total)
                lse_tol[b, h] = dx + LOG2E * steps + 4 * U * (abs(float(lse[b, h])) + abs(top))
                share[at] += p
                share_tol[at] += p * (math.log(2) * (2 * dx + float(lse_tol[b, h])) + 16 * U)
        if acc is not None:
            old = acc[row, :n] * decay if decay != 0 else torch.zeros_like(share)
            acc[row, :n] = old + share
            acc_tol[row, :n] = share_tol + 8 * U * (old.abs() + share)
    got = {"out": out, "lse": lse, "out_tol": out_tol, "lse_tol": lse_tol}
    return got if acc is None else dict(got, weights=acc, weights_tol=acc_tol)


def extend_weights(q, k_pool, idx, prefix, lse, weights, decay=1.0, sm_scale=1 / 16):
    """(weights, tolerance) in 64 bits; sums over rows and heads may be 2 (T / 64 + 256) roundings deep."""
    rows, heads, _ = q.shape
    pool, kv_heads = k_pool.shape[:2]
    n = idx.shape[0]
    c = sm_scale * LOG2E
    slots = idx.long()
    good = (slots >= 0) & (slots < pool)
    k = k_pool[torch.where(good, slots, 0)].double()
    seen = (torch.arange(n, device=q.device)[None, :] <= prefix + torch.arange(rows, device=q.device)[:, None]) & good
    total = torch.zeros(n, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(total)
    for h in range(heads):
        kj, qh, row = k[:, h // (heads // kv_heads)], q[:, h].double(), lse[:, h].double()[:, None]
        x = c * (qh @ kj.T)
        size = c * (qh.abs() @ kj.abs().T)
        live = seen & ~torch.isinf(row)
        p = torch.where(live, torch.exp2(x - row), 0.0)
        dx = torch.where(live, 32 * U * size + 4 * U * (x.abs() + row.abs()), 0.0)
        total += p.sum(0)
        tol += (p * (math.log(2) * dx + 4 * U + 2 * (rows / 64 + 256) * U)).sum(0)
    old = weights.double() * decay if decay != 0 else torch.zeros_like(total)
    return old + total, tol + 8 * U * (old.abs() + total)


def evict(table, weights, lens, keep, first=0, last=0, rows=None):
    """What stays and goes, one position after the other: (table, weights, lens, freed lists)."""
    table, weights = table.clone(), weights.clone()
    new_lens, freed = [], []
    for b in range(len(lens)):
        row = b if rows is None else int(rows[b])
        n = min(max(int(lens[b]), 0), table.shape[1])
        if not 0 <= row < table.shape[0]:
            new_lens.append(0), freed.append([])
            continue
        slots, w = table[row, :n].tolist(), weights[row, :n].tolist()
        stays = set(range(n))
        if n > keep:
            middle = sorted(range(first, n - last), key=lambda i: (-(w[i] if w[i] == w[i] else -math.inf), i))
            stays = set(range(first)) | set(range(n - last, n)) | set(middle[:keep - first - last])
        kept = [i for i in range(n) if i in stays]
        freed.append([slots[i] for i in range(n) if i not in stays])
        weights[row, :n] = 0
        table[row, :len(kept)] = torch.tensor([slots[i] for i in kept], dtype=table.dtype)
        weights[row, :len(kept)] = torch.tensor([w[i] for i in kept], dtype=weights.dtype)
        new_lens.append(len(kept))
    return table, weights, new_lens, freed


def within(got, ref, tol):
    """Both finite and inside the bound, or both the same infinity."""
    got = got.double()
    same = (got == ref) & torch.isinf(ref)
    ok = same | ((got - ref).abs() <= tol)
    worst = torch.where(same, 0.0, (got - ref).abs() / tol.clamp(min=1e-300))
    assert bool(ok.all()), f"{int((~ok).sum())} of {ok.numel()} outside, worst {float(worst.nan_to_num(1e9).max()):.3g} x bound"


def case(lens, q_heads, kv_heads, *, dtype=torch.bfloat16, idx=torch.int32, device="cuda", seed=0, width=None,
         poison=True, table_rows=None):
    """Pools whose unused slots are NaN, a table whose unused entries name them, requests in shuffled rows."""
    g = torch.Generator().manual_seed(seed)
    batch, total = len(lens), sum(lens)
    width = max(max(lens), 1) + 3 if width is None else width
    table_rows = batch + 2 if table_rows is None else table_rows
    pool = 2 * total + 7
    fill = float("nan") if poison else 0.0
    k = torch.full((pool, kv_heads, 256), fill, dtype=dtype)
    v = torch.full((pool, kv_heads, 256), fill, dtype=dtype)
    order = torch.randperm(pool, generator=g)
    used, unused = order[:total], order[total:]
    jitter = torch.rand((total, 1, 1), generator=g) * 1.5 + 0.5
    k[used] = (torch.randn((total, kv_heads, 256), generator=g) * jitter).to(dtype)
    v[used] = torch.randn((total, kv_heads, 256), generator=g).to(dtype)
    table = unused[torch.randint(0, len(unused), (table_rows, width), generator=g)].to(idx)
    rows = torch.randperm(table_rows, generator=g)[:batch]
    at = 0
    for b, n in enumerate(lens):
        table[rows[b], :n] = used[at:at + n].to(idx)
        at += n
    q = torch.randn((batch, q_heads, 256), generator=g).to(torch.bfloat16)
    d = torch.device(device)
    return dict(q=q.to(d), k_pool=k.to(d), v_pool=v.to(d), page_table=table.to(d),
                kv_lens=torch.tensor(lens, dtype=torch.int32, device=d), rows=rows.to(torch.int32).to(d))
