"""Plain 64-bit attention with a learned relative position bias, its gradients, and how far a bf16 kernel may be from them (test code only).

Bounds, per element, u = 2^-8 (half a step of bf16, relative): o: the probabilities are rounded to bf16 for the second product (u sum p |v|), the result once (u |o|).
delta = dO.o is formed from the rounded o: off by dd = sum_d |dO| tol_o.  ds = p (dp - delta) is off by p dd before and u |ds| more after its rounding for the last two
products.  fp32 arithmetic (sums of up to a few thousand terms, exp2 of arguments below 2^7) adds at most c = 2^-13 of the terms' absolute values."""
import torch

U, FP = 2.0 ** -8, 2.0 ** -13


def first_distances(num_buckets, max_distance, causal):
    """bucket -> its first distance within one sign, in whole numbers: distance n >= e belongs to step j where (n / e)^L >= (max_distance / e)^j"""
    half = num_buckets if causal else num_buckets // 2
    e = half // 2
    L = half - e
    out = list(range(e + 1))
    n = e
    for j in range(1, L):
        while n ** L * e ** j < max_distance ** j * e ** L:
            n += 1
        out.append(n)
    return out[:half]


def bucket_index(S, num_buckets, max_distance, causal, device):
    """[S, S] bucket of (query, key)"""
    first = torch.tensor(first_distances(num_buckets, max_distance, causal), device=device)
    half = first.numel()
    pos = torch.arange(S, device=device)
    rel = pos[None, :] - pos[:, None]
    n = (-rel).clamp(min=0) if causal else rel.abs()
    j = torch.searchsorted(first, n.contiguous(), right=True) - 1
    return j if causal else j + (rel > 0).long() * half


def attention(q, k, v, table, *, B, H, S, scale, key_mask, max_distance, causal, do=None, delta_from_o=True):
    """dict of float64 results and tolerances ([B*S, H*64] layout); `do` adds the gradients; delta_from_o=False: delta is not formed from the rounded o"""
    split = lambda t: t.double().reshape(B, S, H, 64).transpose(1, 2).contiguous()  # noqa: E731
    join = lambda t: t.transpose(1, 2).reshape(B * S, H * 64)  # noqa: E731
    q, k, v = split(q), split(k), split(v)
    dev = q.device
    keep = torch.ones(B, 1, S, S, dtype=torch.bool, device=dev)
    if key_mask is not None:
        keep = keep & (key_mask != 0)[:, None, None, :]
        dead = (key_mask == 0)[:, None, :, None]
        k, v = k.masked_fill(dead, 0.0), v.masked_fill(dead, 0.0)  # what masked keys hold does not count
    if causal:
        keep = keep & torch.ones(S, S, dtype=torch.bool, device=dev).tril()
    s = torch.matmul(q, k.transpose(2, 3).contiguous()) * scale
    if table is not None:
        idx = bucket_index(S, table.shape[0], max_distance, causal, dev)
        s = s + table.double()[idx].permute(2, 0, 1)
    s = s.masked_fill(~keep, float("-inf"))
    m = s.amax(3, keepdim=True)
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    p = torch.exp(s - m)
    l = p.sum(3, keepdim=True)
    lse2 = torch.log2(l) + m / torch.log(torch.tensor(2.0, dtype=torch.float64))
    p = p / torch.where(l > 0, l, torch.ones_like(l))
    o = torch.matmul(p, v)
    tol_o = (U + FP) * torch.matmul(p, v.abs()) + U * o.abs()
    r = {"o": join(o), "tol_o": join(tol_o), "lse": lse2[..., 0]}
    if do is None:
        return r
    do = split(do)
    pt = p.transpose(2, 3).contiguous()
    dv = torch.matmul(pt, do)
    r["dv"], r["tol_dv"] = join(dv), join((U + FP) * torch.matmul(pt, do.abs()) + U * dv.abs())
    vt = v.transpose(2, 3).contiguous()
    dp, delta = torch.matmul(do, vt), (do * o).sum(3, keepdim=True)
    ds = p * (dp - delta)
    raw = p * (float(delta_from_o) * (do.abs() * tol_o).sum(3, keepdim=True) + FP * (torch.matmul(do.abs(), vt.abs()) + (do * o).abs().sum(3, keepdim=True)))
    err = raw + U * ds.abs()
    dq, dk = torch.matmul(ds, k) * scale, torch.matmul(ds.transpose(2, 3).contiguous(), q) * scale
    r["dq"], r["tol_dq"] = join(dq), join(torch.matmul(err, k.abs()) * scale + (U + FP) * dq.abs())
    r["dk"], r["tol_dk"] = join(dk), join(torch.matmul(err.transpose(2, 3).contiguous(), q.abs()) * scale + (U + FP) * dk.abs())
    if table is not None:
        nb = table.shape[0]
        sum_by = lambda t: torch.stack([torch.bincount(idx.view(-1), weights=t[h].reshape(-1), minlength=nb) for h in range(H)], 1)  # noqa: E731
        r["dtable"], r["tol_dtable"] = sum_by(ds.sum(0)), sum_by(raw.sum(0))
    return r
