"""What is measured of the attention and 8-bit activation operators: their cases, inputs, plain forms and exact values.

Three operators, each forwards and backwards:

* ``attention``: queries of one set of states (the nodes of a mesh, a probe point, a sequence) read the keys and values of
  another set of another length (the coarse graph's nodes, a mesh's states), in ragged batches:
  ``o_i = sum_j softmax_j(scale * <q_i, k_j> + bias) v_j`` over the keys of the query's own segment that are not masked.
* the learned bias by buckets (cases with ``bias`` > 0): ``bias = table[head, lut[distance(i, j)]]`` with a signed distance
  on a line (``bias`` 1) or the whole part of the Euclidean distance between integer lattice points (``bias`` 2), and the
  gradient of the table.
* ``q8``: rows of activations kept in 8 bits with a scale per row for the backward pass, and a Linear layer's backward
  pass that reads them (input gradient behind a ReLU, weight and bias gradients).
"""
import math

import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
H = 128                                     # latent width of the repository's models


# ------------------------------------------------------------------------------------------------------------- cases
def _att(name, dtype, batch, queries, keys, heads, kv_heads, dim, train=False, bias=0, buckets=32, reach=128, mask=False):
    return {"name": name, "op": "attention", "dtype": dtype, "batch": batch, "queries": queries, "keys": keys, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "train": train, "bias": bias, "buckets": buckets, "reach": reach, "mask": mask}


def listed():
    return [
        # one frame of the bending mesh (33 x 17 nodes) reading its coarse half: the latency of a rollout step
        _att("readout_bending", "f32", 1, 561, 280, 4, 4, 32),
        # eight bending trajectories of a batched rollout, distances in lattice cells
        _att("readout_bias_batch", "f32", 8, 561, 140, 4, 4, 32, bias=2, reach=64),
        # the 100k-node mesh reading a coarse graph of 2000 nodes
        _att("readout_bias_100k", "f32", 1, 100000, 2000, 4, 4, 32, bias=2, reach=512),
        # a training step's readout on a mesh of 20k nodes
        _att("readout_bias_train", "f32", 1, 20000, 2501, 4, 4, 32, train=True, bias=2, reach=256),
        # training on a ragged padded batch with shared key heads, in bf16
        _att("cross_train_bf16", "bf16", 16, 1536, 1100, 8, 2, 64, train=True, mask=True),
        # a long set of states read by as many queries
        _att("cross_long_bf16", "bf16", 1, 8192, 8192, 8, 8, 128),
        # sequences with the signed bias on a line, in training, fp16
        _att("line_bias_train_f16", "f16", 4, 1800, 1800, 8, 8, 64, train=True, bias=1, reach=128),
        # serving: one query each of 64 streams over long ragged states
        _att("probe_bf16", "bf16", 64, 1, 8000, 16, 4, 128),
        # one probe point reading all states of the 100k-node mesh with the distance bias
        _att("probe_bias_100k", "f32", 1, 1, 100000, 4, 4, 32, bias=2, reach=1000),
        # the edge latents of a 250k-node mesh kept for the backward pass and taken back
        {"name": "q8_keep_edges", "op": "q8_keep", "dtype": "f32", "rows": 1498001, "width": H},
        # a node-level tensor of the bending mesh: latency
        {"name": "q8_linear_small", "op": "q8_linear", "dtype": "f32", "rows": 561, "width": H},
        # edge-level Linear backward of the 250k-node training step
        {"name": "q8_linear_edges", "op": "q8_linear", "dtype": "f32", "rows": 1498001, "width": H},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("readout", "cross", "line", "probe", "keep", "linear"))
    if kind == "readout":                   # meshes reading coarse graphs
        batch = rng.choice((1, 1, 2, 5))
        return _strip(_att("", "f32", batch, _log(rng, 300, 40000 // batch), _log(rng, 40, 3000), *rng.choice(((4, 4, 32), (8, 8, 16), (2, 2, 64), (1, 1, 128))),
                           train=rng.random() < 0.4, bias=rng.choice((0, 2)), buckets=rng.choice((16, 32, 48)), reach=rng.randint(20, 900)))
    if kind == "cross":
        batch = rng.randint(1, 12)
        kv, rep = rng.choice((1, 2, 4)), rng.choice((1, 2, 4))
        return _strip(_att("", rng.choice(("bf16", "f16", "f32")), batch, _log(rng, 40, 6000 // batch + 40), _log(rng, 30, 6000 // batch + 30), kv * rep, kv,
                           rng.choice((24, 32, 64, 80, 128)), train=rng.random() < 0.5, mask=rng.random() < 0.5))
    if kind == "line":
        batch = rng.randint(1, 6)
        n = _log(rng, 50, 2000)
        return _strip(_att("", rng.choice(("bf16", "f16", "f32")), batch, n, n, rng.choice((2, 4, 8)), 2, rng.choice((32, 64)), train=rng.random() < 0.6,
                           bias=1, buckets=rng.choice((8, 32, 64)), reach=rng.randint(16, 500), mask=rng.random() < 0.3))
    if kind == "probe":
        batch = _log(rng, 1, 64)
        return _strip(_att("", rng.choice(("bf16", "f16", "f32")), batch, rng.randint(1, 3), _log(rng, 100, 400000 // batch), rng.choice((4, 8, 16)),
                           rng.choice((2, 4)), rng.choice((32, 64, 128)), bias=rng.choice((0, 0, 1, 2)), reach=rng.randint(20, 900), mask=rng.random() < 0.3))
    if kind == "keep":
        return {"op": "q8_keep", "dtype": rng.choice(("f32", "bf16", "f16")), "rows": _log(rng, 200, 1400000), "width": rng.choice((H, H, 64, 200))}
    return {"op": "q8_linear", "dtype": "f32", "rows": _log(rng, 200, 1400000), "width": H}


def _strip(c):
    return {k: v for k, v in c.items() if k != "name"}


def _lengths(batch, most):
    """Ragged lengths of a batch: between 40 and 100 per cent of the longest, the first one the longest."""
    return [max(1, int(round(most * (1.0 - 0.6 * ((0.618034 * b) % 1.0))))) for b in range(batch)]


def bucket_lut(buckets, reach, signed):
    """Bucket of every distance: the first half of the buckets one distance each, the others spaced evenly in the logarithm
    up to ``reach``; whole-number comparisons throughout, so no border depends on a rounding.  ``signed``: entries for
    -reach .. reach, the buckets shared out half and half; otherwise 0 .. reach."""
    n = buckets // 2 if signed else buckets
    exact = max(1, n // 2)

    def of(d):
        if d < exact:
            return d
        b = exact                            # the last b with (d / exact)^(n - exact) >= (reach / exact)^(b - exact)
        while b + 1 < n and reach > exact and d ** (n - exact) * exact ** (b + 1 - exact) >= reach ** (b + 1 - exact) * exact ** (n - exact):
            b += 1
        return b
    line = [of(d) for d in range(reach + 1)]
    return [line[-r] for r in range(-reach, 0)] + [line[0]] + [n + b for b in line[1:]] if signed else line


# ------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    dt = DT[case["dtype"]]

    def normal(*shape, dtype=dt, by=1.0):
        return (torch.randn(*shape, generator=gen, device=dev) * by).to(dtype)

    s = {"case": case}
    if case["op"] == "q8_keep":
        # latents behind a LayerNorm and residuals: rows of different sizes
        s["x"] = (normal(case["rows"], case["width"], dtype=torch.float32) * torch.exp(normal(case["rows"], 1, dtype=torch.float32))).to(dt)
        return s
    if case["op"] == "q8_linear":
        x = normal(case["rows"], H, dtype=torch.float32).clamp_min_(0.0) * torch.exp(0.5 * normal(case["rows"], 1, dtype=torch.float32))
        s["codes"], s["scale"] = _codes(x, True)
        s["g"] = normal(case["rows"], H, by=1e-3)
        s["w"] = normal(H, H, by=H ** -0.5)
        if own:
            from gnn_amd import ops
            s["scratch"] = torch.empty(ops.train_scratch_bytes(), dtype=torch.uint8, device=dev)
        return s
    nq, nk = _lengths(case["batch"], case["queries"]), _lengths(case["batch"], case["keys"])
    if case["queries"] <= 3:                # probes: the same few queries in every stream
        nq = [case["queries"]] * case["batch"]
    tq, tk = sum(nq), sum(nk)
    s["max_q"], s["max_k"] = max(nq), max(nk)
    s["q"] = normal(tq, case["heads"], case["dim"])
    s["k"] = normal(tk, case["kv_heads"], case["dim"])
    s["v"] = normal(tk, case["kv_heads"], case["dim"])
    s["q_ptr"] = torch.tensor([sum(nq[:i]) for i in range(len(nq) + 1)], dtype=torch.int32, device=dev)
    s["k_ptr"] = torch.tensor([sum(nk[:i]) for i in range(len(nk) + 1)], dtype=torch.int32, device=dev)
    s["g"] = normal(tq, case["heads"], case["dim"]) if case["train"] else None
    s["mask"] = None
    if case["mask"]:                        # a tenth of the keys left out, and all keys of the last segment of a batch
        s["mask"] = torch.rand(tk, generator=gen, device=dev) > 0.1
        if case["batch"] > 1:
            s["mask"][tk - nk[-1]:] = False
    s["table"] = s["lut"] = s["q_pos"] = s["k_pos"] = None
    if case["bias"]:
        s["table"] = normal(case["heads"], case["buckets"], dtype=torch.float32, by=0.5)
        s["lut"] = torch.tensor(bucket_lut(case["buckets"], case["reach"], case["bias"] == 1), dtype=torch.int32, device=dev)
        if case["bias"] == 1:               # places on a line, the queries at the end of their keys
            s["k_pos"] = torch.cat([torch.arange(n, device=dev) for n in nk]).to(torch.int32)[:, None].contiguous()
            s["q_pos"] = torch.cat([torch.arange(n, device=dev) + max(0, m - n) for n, m in zip(nq, nk)]).to(torch.int32)[:, None].contiguous()
        else:                               # lattice cells of a mesh twice as long as high
            def cells(n):
                u = torch.rand(n, 2, generator=gen, device=dev)
                return (u * torch.tensor([1.6 * case["reach"], 0.8 * case["reach"]], device=dev)).to(torch.int32)
            s["q_pos"], s["k_pos"] = cells(tq), cells(tk)
    return s


# ------------------------------------------------------------------------------------------------------------- plain form
def _codes(x, keep_nonzero):
    """Whole codes -127 .. 127 and the scale of every row, nearest code with ties to even; with ``keep_nonzero`` a value
    other than zero keeps a code other than zero (the pattern of a ReLU)."""
    x = x.double()
    most = x.abs().amax(dim=-1, keepdim=True)
    by = torch.where(most > 0, 127.0 / most, 0.0).float()       # the factor and the scale are 32-bit values, rounded once
    codes = (x * by.double()).round().clamp(-127, 127)
    if keep_nonzero:
        codes = torch.where((codes == 0) & (x != 0), torch.sign(x), codes)
    return codes.to(torch.int8), (most / 127.0)[:, 0].float().contiguous()


def _places(ptr, most, total):
    """Row index [batch, most] of a ragged set laid out as a padded one, and which places hold a row."""
    at = ptr[:-1, None].long() + torch.arange(most, device=ptr.device)
    return at.clamp(max=total - 1), at < ptr[1:, None]


def _buckets(s, qi, ki):
    a, b = s["q_pos"].long()[qi][:, :, None], s["k_pos"].long()[ki][:, None]
    reach = s["case"]["reach"]
    if s["case"]["bias"] == 1:
        at = (b - a)[..., 0].clamp(-reach, reach) + reach
    else:
        at = (a - b).square().sum(-1).clamp(max=reach * reach).double().sqrt().long()
    return s["lut"].long()[at]


def _plain_attention(s):
    c = s["case"]
    rep, scale = c["heads"] // c["kv_heads"], c["dim"] ** -0.5
    qi, qv = _places(s["q_ptr"], s["max_q"], s["q"].shape[0])
    ki, kv = _places(s["k_ptr"], s["max_k"], s["k"].shape[0])
    if s["mask"] is not None:
        kv = kv & s["mask"][ki]
    q = s["q"].float()[qi].permute(0, 2, 1, 3).contiguous()
    k = torch.where(kv[..., None, None], s["k"].float()[ki], 0.0).repeat_interleave(rep, dim=2).permute(0, 2, 1, 3).contiguous()
    v = torch.where(kv[..., None, None], s["v"].float()[ki], 0.0).repeat_interleave(rep, dim=2).permute(0, 2, 1, 3).contiguous()
    p = torch.matmul(q, k.transpose(2, 3).contiguous()) * scale
    bucket = None
    if c["bias"]:
        bucket = _buckets(s, qi, ki)
        p += s["table"][:, bucket].transpose(0, 1)
    p = p.masked_fill_(~kv[:, None, None, :], -math.inf)
    p = torch.exp(p - p.amax(dim=-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min))
    total = p.sum(dim=-1, keepdim=True)
    p /= torch.where(total > 0, total, 1.0)
    o = torch.matmul(p, v)
    out = [o.permute(0, 2, 1, 3)[qv].to(s["q"].dtype)]
    if s["g"] is None:
        return out
    g = torch.where(qv[..., None, None], s["g"].float()[qi], 0.0).permute(0, 2, 1, 3).contiguous()
    dv = torch.matmul(p.transpose(2, 3).contiguous(), g)
    ds = torch.matmul(g, v.transpose(2, 3).contiguous())
    ds = p * (ds - (o * g).sum(dim=-1, keepdim=True))
    dq = torch.matmul(ds, k) * scale
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q) * scale
    out.append(dq.permute(0, 2, 1, 3)[qv].to(s["q"].dtype))
    for d in (dk, dv):
        d = d.reshape(c["batch"], c["kv_heads"], rep, s["max_k"], c["dim"]).sum(dim=2).permute(0, 2, 1, 3)
        out.append(d[_places(s["k_ptr"], s["max_k"], s["k"].shape[0])[1]].to(s["k"].dtype))
    if c["bias"]:
        by_row = torch.zeros(*ds.shape[:3], c["buckets"], device=ds.device)
        by_row.scatter_add_(3, bucket[:, None].expand_as(ds), ds)
        out.append(by_row.double().sum(dim=(0, 2)).float())
    return out


def _plain_q8_linear(s):
    x = s["codes"].float() * s["scale"][:, None]
    ga = torch.where(x > 0, torch.matmul(s["g"], s["w"]), 0.0)
    return [ga, torch.matmul(s["g"].t().contiguous(), x), s["g"].sum(dim=0)]


def run(state):
    s, c = state, state["case"]
    if own:
        return _own(s, c)
    if c["op"] == "q8_keep":
        codes, scale = _codes(s["x"], False)
        return [(codes.float() * scale[:, None]).to(s["x"].dtype), scale]
    if c["op"] == "q8_linear":
        return _plain_q8_linear(s)
    return _plain_attention(s)


def _own(s, c):
    from gnn_amd import attention, ops
    if c["op"] == "q8_keep":
        kept = ops.q8_rows(s["x"])
        return [ops.q8_restore(kept, s["x"].dtype), kept.scale]
    if c["op"] == "q8_linear":
        kept = ops.Q8Rows(s["codes"], s["scale"])
        ga, dw, db = torch.empty_like(s["g"]), torch.empty_like(s["w"]), torch.empty_like(s["w"][0])
        ops.train_linear_bwd(s["g"], s["scratch"], a=kept, w=s["w"], mask=kept, ga=ga, dw=dw, db=db)
        return [ga, dw, db]
    q, k, v, table = s["q"], s["k"], s["v"], s["table"]
    if s["g"] is not None:
        q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
        table = table.detach().requires_grad_() if table is not None else None
    bias = dict(bias_table=table, bucket_lut=s["lut"], q_pos=s["q_pos"], k_pos=s["k_pos"]) if c["bias"] else {}
    o = attention.cross_attention(q, k, v, q_ptr=s["q_ptr"], k_ptr=s["k_ptr"], key_mask=s["mask"], **bias)
    if s["g"] is None:
        return [o]
    return [o.detach(), *torch.autograd.grad(o, (q, k, v) + ((table,) if table is not None else ()), s["g"])]


# ------------------------------------------------------------------------------------------------------------- work
def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}[case["dtype"]]
    if case["op"] == "q8_keep":             # rows read, codes and scales written and read, rows written
        n = case["rows"]
        return {"bytes": n * (2 * size * case["width"] + 2 * (case["width"] + 4)), "flops": 4 * n * case["width"]}
    if case["op"] == "q8_linear":           # gradient and codes read, input gradient written, two products
        n = case["rows"]
        return {"bytes": n * (4 * H + H + 4 + 4 * H) + 8 * H * H, "flops": 4 * n * H * H}
    nq, nk = _lengths(case["batch"], case["queries"]), _lengths(case["batch"], case["keys"])
    if case["queries"] <= 3:
        nq = [case["queries"]] * case["batch"]
    pairs = sum(a * b for a, b in zip(nq, nk)) * case["heads"]
    q, k = sum(nq) * case["heads"] * case["dim"] * size, sum(nk) * case["kv_heads"] * case["dim"] * size
    if case["train"]:                       # two products forwards, five backwards
        return {"bytes": 4 * q + 4 * k, "flops": 14 * pairs * case["dim"]}
    return {"bytes": 2 * q + 2 * k, "flops": 4 * pairs * case["dim"]}


# ------------------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "q8_keep":
        x = s["x"].double()
        top = x.abs().max(dim=1).values
        # the factor onto the codes is part of the definition: 127 / (largest magnitude), rounded to 32 bits
        factor = (127.0 / top).float().double().masked_fill(top == 0, 0.0)
        scale = (top / 127.0).float().double()
        return [torch.round(x * factor[:, None]).clamp(-127, 127) * scale[:, None], scale]
    if case["op"] == "q8_linear":
        g, w = s["g"].double(), s["w"].double()
        x = s["codes"].double() * s["scale"].double()[:, None]
        return [(g @ w) * (s["codes"] > 0), (x.t().contiguous() @ g).t(), g.sum(0)]
    return _exact_attention(s, case)


def _exact_attention(s, c):
    rep, scale = c["heads"] // c["kv_heads"], 1.0 / math.sqrt(c["dim"])
    qp, kp = s["q_ptr"].tolist(), s["k_ptr"].tolist()
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    dq = torch.zeros_like(o)
    dk, dv = (torch.zeros(s["k"].shape, dtype=torch.float64, device=o.device) for _ in range(2))
    dt = torch.zeros(c["heads"], c["buckets"], dtype=torch.float64, device=o.device)
    for b in range(c["batch"]):
        keys = torch.arange(kp[b], kp[b + 1], device=o.device)
        if s["mask"] is not None:
            keys = keys[s["mask"][keys]]
        if keys.numel() == 0:
            continue
        step = max(1, 60_000_000 // keys.numel())
        for q0 in range(qp[b], qp[b + 1], step):
            rows = slice(q0, min(q0 + step, qp[b + 1]))
            bucket = None
            if c["bias"]:
                d = [s["k_pos"][keys, a].double()[None] - s["q_pos"][rows, a].double()[:, None] for a in range(s["q_pos"].shape[1])]
                if c["bias"] == 1:
                    at = d[0].clamp(-c["reach"], c["reach"]) + c["reach"]
                else:
                    at = torch.floor(torch.sqrt(d[0] * d[0] + d[1] * d[1])).clamp(max=c["reach"])
                bucket = s["lut"][at.long()]
            for h in range(c["heads"]):
                k, v = s["k"][keys, h // rep].double(), s["v"][keys, h // rep].double()
                q = s["q"][rows, h].double()
                e = torch.einsum("id,jd->ij", q, k) * scale
                if bucket is not None:
                    e = e + s["table"][h].double()[bucket.long()]
                w = torch.softmax(e, dim=1)
                o[rows, h] = w @ v
                if s["g"] is None:
                    continue
                g = s["g"][rows, h].double()
                u = torch.einsum("id,jd->ij", g, v)
                u = w * (u - (w * u).sum(1, keepdim=True))
                dq[rows, h] = u @ k * scale
                dk.index_add_(0, keys, _one_head(torch.einsum("ij,id->jd", u, q) * scale, h // rep, c))
                dv.index_add_(0, keys, _one_head(torch.einsum("ij,id->jd", w, g), h // rep, c))
                if bucket is not None:
                    for n in range(c["buckets"]):
                        dt[h, n] += torch.where(bucket == n, u, 0.0).sum()
    return [o] + ([dq, dk, dv] if s["g"] is not None else []) + ([dt] if c["bias"] and s["g"] is not None else [])


def _one_head(x, head, c):
    full = torch.zeros(x.shape[0], c["kv_heads"], x.shape[1], dtype=x.dtype, device=x.device)
    full[:, head] = x
    return full
