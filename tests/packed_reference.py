"""Attention over packed sequences and its gradients written out in 64 bits, with a bound of what a kernel that follows
the type's roundings may be off by, element by element."""
import math

import torch


def bucket_by_logarithms(apart, num, far, two_sided):
    m = num // 2 if two_sided else num
    e = m // 2
    n = apart.abs().double() if two_sided else (-apart).clamp_min(0).double()
    wide = e + torch.floor((m - e) * torch.log(n.clamp_min(1) / e) / math.log(far / e) + 1e-9)
    b = torch.where(n < e, n, wide.clamp_max(m - 1))
    return (b + m * (apart > 0) if two_sided else b).long()


def reference(q, k, v, cu_q, cu_k=None, len_k=None, causal=False, scale=None, table=None, buckets=None, pos_q=None,
              pos_k=None, dout=None):
    """-> {name: (value, bound)} for out, dq, dk, dv, dtable.  Hidden pairs are taken out, not multiplied by zero.

    The bounds count, with u half a step of the type (0 for the probabilities' rounding in fp32) and w = 2^-24:
    a score's products and sums (D + 8 roundings of at most the sum of magnitudes), the exponential's argument and value,
    the rounding of a probability and of ds to the type, the sums' own roundings, and the result's."""
    dt, dim = q.dtype, q.shape[2]
    u = torch.finfo(dt).eps / 2
    up = 0.0 if dt == torch.float32 else u
    w = 2.0**-24
    scale = dim**-0.5 if scale is None else scale
    cu_k = cu_q if cu_k is None else cu_k
    pos_k = pos_q if pos_k is None else pos_k
    heads, group = q.shape[1], q.shape[1] // k.shape[1]
    Q, K, V = q.double(), k.double(), v.double()
    got = {"out": torch.zeros_like(Q)}
    err = {"out": torch.zeros_like(Q)}
    if dout is not None:
        dO = dout.double()
        for n, t in (("dq", Q), ("dk", K), ("dv", V)):
            got[n], err[n] = torch.zeros_like(t), torch.zeros_like(t)
        if table is not None:
            got["dtable"] = torch.zeros(table.shape, dtype=torch.float64, device=q.device)
            err["dtable"] = torch.zeros_like(got["dtable"])
    for b in range(len(cu_q) - 1):
        lq, lk = cu_q[b + 1] - cu_q[b], cu_k[b + 1] - cu_k[b]
        if len_k is not None:
            lk = min(lk, len_k[b])
        if lq <= 0 or lk <= 0:
            continue
        rq, rk = slice(cu_q[b], cu_q[b] + lq), slice(cu_k[b], cu_k[b] + lk)
        i, j = torch.arange(lq, device=q.device), torch.arange(lk, device=q.device)
        open_ = torch.ones(lq, lk, dtype=torch.bool, device=q.device)
        if causal:
            open_ = j[None, :] <= i[:, None] + lk - lq
        if table is not None:
            pq = i + lk - lq if pos_q is None else pos_q[rq].long()
            pk = j if pos_k is None else pos_k[rk].long()
            bucket = bucket_by_logarithms(pk[None, :] - pq[:, None], buckets.num_buckets, buckets.max_distance,
                                          buckets.bidirectional)
        for h in range(heads):
            g = h // group
            qh, kh, vh = Q[rq, h], K[rk, g], V[rk, g]
            s = qh @ kh.T * scale
            mag = qh.abs() @ kh.abs().T * abs(scale)
            see = open_
            if table is not None:
                t = table[h].double()[bucket]
                see = see & (t != -math.inf)
                # a table value beyond 2^100 absorbs the product below it, in 32 bits as in 64: such scores are the table
                # value itself on both sides, differences of equal ones are exactly 0, of others exp() makes exactly 0
                s, mag = s + t, torch.where(t.abs() > 2.0**100, 0.0, mag + t.abs())
            s = torch.where(see, s, -math.inf)
            mag = torch.where(see, mag, 0.0)
            m = s.amax(-1, keepdim=True)
            p = torch.where(see, torch.exp(s - torch.where(m == -math.inf, 0.0, m)), 0.0)
            p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
            top = mag.amax(-1, keepdim=True)
            ep = torch.expm1(2 * (dim + 8) * w * top) + (16 + lk**0.5) * w  # a probability's relative error
            # value by value: a masked pair's NaN must not meet a zero
            dead = ~see.any(0)
            vz = torch.where(dead[:, None], 0.0, vh)
            sel = not bool(torch.isfinite(vz).all())
            o = _safe_mm(p, vz, see) if sel else p @ vz
            A = _safe_mm(p, vz.abs(), see) if sel else p @ vz.abs()
            got["out"][rq, h] = o
            err["out"][rq, h] = (u * o.abs() + (up + ep + lk * w) * A * (1 + u)) * 1.01 + 1e-30
            if dout is None:
                continue
            do = dO[rq, h]
            dp = torch.where(see, do @ vz.T, 0.0)
            delta = (do * o).sum(-1, keepdim=True)
            ds = p * (dp - delta)
            edelta = (do.abs() * (A * (up + ep + lk * w) + dim * w * o.abs())).sum(-1, keepdim=True)
            eds = (ep + 4 * w) * ds.abs() + p * (1 + ep) * ((dim + 4) * w * (do.abs() @ vz.abs().T) + edelta)
            kz = torch.where(dead[:, None], 0.0, kh)
            got["dq"][rq, h] = ds @ kz * scale
            err["dq"][rq, h] = (eds + (up + lk * w) * ds.abs()) @ kz.abs() * abs(scale)
            got["dk"][rk, g] += ds.T @ qh * scale
            err["dk"][rk, g] += (eds + (up + lq * group * w) * ds.abs()).T @ qh.abs() * abs(scale)
            got["dv"][rk, g] += p.T @ do
            err["dv"][rk, g] += ((up + ep + lq * group * w) * p).T @ do.abs()
            if table is not None:
                got["dtable"][h].index_add_(0, bucket.reshape(-1), torch.where(see, ds, 0.0).reshape(-1))
                # the sums' own roundings: lanes, tiles and parts, each of at most 2^11 terms in a row
                err["dtable"][h].index_add_(0, bucket.reshape(-1), (eds + 2.0**11 * w * ds.abs()).reshape(-1))
    for n in ("dq", "dk", "dv", "dtable"):
        if n in got:
            un = u if n != "dtable" else w
            # values below the type's normal range round to a whole number of its smallest steps
            err[n] = err[n] * 1.01 + un * got[n].abs() + torch.finfo(dt).smallest_normal * u + 1e-30
    err["out"] = err["out"] + torch.finfo(dt).smallest_normal * u
    return {n: (got[n], err[n]) for n in got}


def _safe_mm(p, v, see):
    """p @ v over the pairs that are seen only."""
    out = torch.zeros(p.shape[0], v.shape[1], dtype=p.dtype, device=p.device)
    for r in range(p.shape[0]):
        out[r] = p[r][see[r]] @ v[see[r]]
    return out


def check(name, got, want, bound):
    got = got.double()
    off = (got - want).abs()
    wrong = ~((off <= bound) | (torch.isnan(got) & torch.isnan(want)) | (got == want))
    if bool(wrong.any()):
        at = tuple(wrong.nonzero()[0].tolist())
        raise AssertionError(f"{name}: {int(wrong.sum())} of {wrong.numel()} outside their bounds, first at {at}: "
                             f"{got[at].item()} for {want[at].item()} (bound {bound[at].item():.3e})")
