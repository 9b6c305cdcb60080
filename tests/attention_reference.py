"""Plain 64-bit attention over another set of states, its gradients, and how far a kernel may be from them.

Error bounds, entry by entry, u = half a step of the operands' type (2^-24, 2^-8, 2^-11):
  * a score: operands enter exactly (16-bit types) or as two fp16 terms (2^-22 of the value, the product of the second
    terms left out: another 2^-22); sums of at most 3 * 8 matrix instructions in fp32 and the scaling lose at most 2^-19 of
    sum |q k| in all.  A change d of all scores changes a probability by at most a factor exp(2 d): 2.5 d for small d.
  * a sum over keys (or queries) of probabilities times x: each probability is rounded to the operands' type (u; fp32: two
    terms, inside the 2^-19), so it is off by (u + 2.5 d + 2^-19) of sum p |x|, and the result is rounded: u times the
    computed result, which is at most |result| plus what it is off already, or half a subnormal step of the type.
  * dS = p (dP - delta): p as above; dP off by 2^-19 of sum |g v|, delta by 2^-19 of sum |g o| and, where the outputs were
    rounded to 16 bits, by u times that, plus what o is off.  dS is rounded (u) before the products with k and q.
"""
import math

import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}     # half a subnormal step
SUMS = 2.0 ** -19


def buckets(q_pos, k_pos, lut):
    """Bucket of every (query, key) pair from whole numbers alone."""
    d = k_pos.long()[None] - q_pos.long()[:, None]
    if q_pos.shape[1] == 1:
        reach = lut.shape[0] // 2
        return lut.long()[d[..., 0].clamp(-reach, reach) + reach]
    reach = lut.shape[0] - 1
    d2 = (d * d).sum(-1)
    at = torch.tensor([math.isqrt(int(v)) for v in d2.flatten()]).reshape(d2.shape) if d2.numel() < 4096 else d2.double().sqrt().long()
    return lut.long()[at.clamp(max=reach)]


def reference(q, k, v, g=None, q_ptr=None, k_ptr=None, key_mask=None, bias_table=None, bucket_lut=None, q_pos=None, k_pos=None, scale=None):
    """dict of 64-bit values and, under the same name with ``_tol``, bounds; rows outside all segments are NaN."""
    u, tiny = HALF_STEP[q.dtype], TINY[q.dtype]
    u16 = 0.0 if q.dtype is torch.float32 else u
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    heads, kvh, dim = q.shape[1], k.shape[1], q.shape[2]
    rep, scale = heads // kvh, dim ** -0.5 if scale is None else scale
    qp = [0, q.shape[0]] if q_ptr is None else q_ptr.tolist()
    kp = [0, k.shape[0]] if k_ptr is None else k_ptr.tolist()
    names = ["o"] if g is None else ["o", "dq", "dk", "dv"]
    out = {}
    for n in names:
        like, ptr = (q, qp) if n in ("o", "dq") else (k, kp)
        for s in (n, n + "_tol"):
            out[s] = torch.full(like.shape, math.nan, dtype=torch.float64)
            out[s][ptr[0]:ptr[-1]] = 0.0
    if g is not None:
        g = g.detach().cpu().double()
        if bias_table is not None:
            out["dtable"], out["dtable_tol"] = (torch.zeros(bias_table.shape, dtype=torch.float64) for _ in range(2))
    for b in range(len(qp) - 1):
        rows = slice(qp[b], qp[b + 1])
        keys = torch.arange(kp[b], kp[b + 1])
        if key_mask is not None:
            keys = keys[key_mask.detach().cpu().bool()[keys]]
        if not keys.numel() or qp[b] == qp[b + 1]:
            continue
        bk = None if bias_table is None else buckets(q_pos.cpu()[rows], k_pos.cpu()[keys], bucket_lut.cpu())
        for h in range(heads):
            qh, kh, vh = q[rows, h], k[keys, h // rep], v[keys, h // rep]
            s = qh @ kh.T * scale
            d = SUMS * scale * (qh.abs() @ kh.abs().T).amax(1, keepdim=True)
            if bk is not None:
                bias = bias_table.detach().cpu().double()[h][bk]
                s = s + bias
                d = d + 2.0 ** -22 * bias.abs().masked_fill(bias.abs() > 1e30, 0.0).amax(1, keepdim=True)
            m = s.amax(1, keepdim=True)
            p = torch.exp(s - m.masked_fill(m == -math.inf, 0.0))
            total = p.sum(1, keepdim=True)
            p = p / total.masked_fill(total == 0, 1.0)
            o = p @ vh
            loss = u16 + 2.5 * d + SUMS
            o_loss = loss * (p @ vh.abs())
            out["o"][rows, h] = o
            o_loss = o_loss + u * (o.abs() + o_loss) + tiny
            out["o_tol"][rows, h] = o_loss
            if g is None:
                continue
            gh = g[rows, h]
            dp = gh @ vh.T
            delta = (gh * o).sum(1, keepdim=True)
            ds = p * (dp - delta)
            d_loss = SUMS * (gh.abs() @ vh.abs().T + (gh * o).abs().sum(1, keepdim=True)) + (gh.abs() * o_loss).sum(1, keepdim=True)
            ds_loss = p * ((dp - delta).abs() * loss + d_loss)
            out["dq"][rows, h] = ds @ kh * scale
            off = (ds_loss + SUMS * ds.abs()) @ kh.abs() * scale
            out["dq_tol"][rows, h] = off + u * (out["dq"][rows, h].abs() + off) + tiny
            for name, x, y in (("dk", ds.T @ qh * scale, (ds_loss + SUMS * ds.abs()).T @ qh.abs() * scale), ("dv", p.T @ gh, (p * loss).T @ gh.abs())):
                out[name][keys, h // rep] += x
                out[name + "_tol"][keys, h // rep] += y
            if bk is not None:
                out["dtable"][h].index_add_(0, bk.flatten(), ds.flatten())
                # fp32 dS, unrounded outputs (16 bits of the probabilities for bf16): no u, 2^-17 for what the outputs are off
                t_loss = p * ((dp - delta).abs() * (2.5 * d + SUMS) + SUMS * (gh.abs() @ vh.abs().T) + (gh.abs() * (2.0 ** -16 * (p @ vh.abs()))).sum(1, keepdim=True))
                out["dtable_tol"][h].index_add_(0, bk.flatten(), t_loss.flatten())
    for name in ("dk", "dv"):
        if name in out:
            out[name + "_tol"] += u * (out[name].abs() + out[name + "_tol"]) + tiny
    return out


def assert_close(got, ref, name, outside_kept=None):
    """``got`` within the reference's bound; rows outside all segments hold ``outside_kept`` (default: zeros)."""
    got, want, tol = got.detach().cpu().double(), ref[name], ref[name + "_tol"]
    outside = torch.isnan(want)
    assert not torch.isnan(got[~outside]).any(), f"{name}: NaN"
    assert (got[outside] == (0.0 if outside_kept is None else outside_kept)).all(), f"{name}: a row outside all segments was written"
    off = ((got - want).abs() - tol)[~outside]
    tiny = 1e-30                                    # denormal results
    assert not off.numel() or float(off.max()) <= tiny, f"{name}: {float(off.max()):.3e} over its bound, error {float((got - want).abs()[~outside].max()):.3e}"
