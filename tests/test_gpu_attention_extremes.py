"""Attention on operands of very different sizes: blocks that are zero, tiny or masked beside ordinary ones, rows far larger or
smaller than their neighbours, NaN and infinities.  Values and gradients against tests/attention_reference.py, whose bounds are
relative to the sums of magnitudes of each result's own row."""
import math

import pytest
import torch

from attention_reference import assert_close, buckets, reference
from test_gpu_attention import BF16, DEV, F16, F32, bias_args, check, make, ptr

pytestmark = pytest.mark.gpu

def run(q, k, v, g, **kw):
    """Outputs and gradients of the public entry point."""
    from gnn_amd import attention
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    if kw.get("bias_table") is not None:
        leaves.append(kw["bias_table"].detach().requires_grad_())
        kw = dict(kw, bias_table=leaves[3])
    o = attention.cross_attention(*leaves[:3], **kw)
    return dict(zip(("o", "dq", "dk", "dv", "dtable"), (o.detach(),) + torch.autograd.grad(o, leaves, g)))


def sized_rows(x):
    """Size a row is scaled by: its own largest magnitude, or that of its 32 neighbours where it is within 2^14 of it (or zero)."""
    out = x.abs().amax(-1)
    for at in range(0, x.shape[0], 32):
        rows = out[at:at + 32]
        most = rows.amax(0, keepdim=True)
        out[at:at + 32] = torch.where((rows == 0) | (rows * 2.0 ** 14 >= most), most.expand_as(rows), rows)
    return out.clamp_min(2.0 ** -126)


def smallest_digits(ref, q, k, v, g, bias_table=None, bucket_lut=None, q_pos=None, k_pos=None):
    """Adds to the bounds what the smallest number of fp16 takes from a sum of addends of very different sizes.

    An addend w x of a sum enters as (w 2^(ex - unit)) (x 2^-ex) with 2^ex the size of x's row and the sum's unit such that the
    largest w 2^ex so far was at least 2^11 in it (raised to 2^11 .. 2^12, forwards to 2^11).  The two terms of the first factor
    leave at most half the smallest number of fp16, 2^-25: 2^-36 of the largest w 2^ex.  So the sum is off by at most 2^-36 of
    max(|w| X) sum(|x| / X), X the rows' sizes, 1 or 2 times 2^ex each (2^-34)."""
    q, k, v, g = (t.detach().cpu().double() for t in (q, k, v, g))
    rep, scale = q.shape[1] // k.shape[1], q.shape[2] ** -0.5
    xq, xk, xv, xg = (sized_rows(t) for t in (q, k, v, g))
    bk = None if bias_table is None else buckets(q_pos.cpu(), k_pos.cpu(), bucket_lut.cpu())
    for h in range(q.shape[1]):
        c = h // rep
        s = q[:, h] @ k[:, c].T * scale
        if bk is not None:
            s = s + bias_table.detach().cpu().double()[h][bk]
        p = torch.softmax(s, 1)
        o = p @ v[:, c]
        ds = p * (g[:, h] @ v[:, c].T - (g[:, h] * o).sum(1, keepdim=True))
        for name, w, x, size, col, by in (("o", p, v[:, c], xv[:, c], h, 1.0), ("dq", ds, k[:, c], xk[:, c], h, scale),
                                          ("dk", ds.T, q[:, h], xq[:, h], c, scale), ("dv", p.T, g[:, h], xg[:, h], c, 1.0)):
            ref[name + "_tol"][:, col] += 2.0 ** -34 * by * (w.abs() * size).amax(1, keepdim=True) * (x.abs() / size[:, None]).sum(0)


def check_sizes(q, k, v, g, **kw):
    got, ref = run(q, k, v, g, **kw), reference(q, k, v, g, **kw)
    smallest_digits(ref, q, k, v, g, **kw)
    for name, t in got.items():
        assert_close(t, ref, name)


# small problems, the tiled kernel, the tiled kernel with two heads per wave (with a lattice bias), split key ranges
SHAPES = [(60, 200, 4, 32), (300, 1500, 8, 64), (1100, 300, 64, 32), (700, 2500, 4, 24), (130, 2200, 2, 128)]


def bias(nq, nk, heads, axes):
    return bias_args(nq, nk, heads, axes, 30) if axes else {}


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("axes", [0, 1, 2])
@pytest.mark.parametrize("nq,nk,heads,dim", SHAPES)
def test_zero_and_tiny_queries_beside_masked_keys(nq, nk, heads, dim, axes, dtype):
    """A padded batch: queries of zero and of 1e-3 beside whole blocks of masked keys and a masked end."""
    q, k, v, g = make(nq, nk, heads, heads, dim, dtype)
    q[:40] = 0
    q[40:50] *= 1e-3
    mask = torch.ones(nk, dtype=torch.bool, device=DEV)
    mask[32:100] = False
    mask[nk - 45:] = False
    check(q, k, v, g, key_mask=mask, **bias(nq, nk, heads, axes))
    check(torch.zeros_like(q), k * 1e-3, v, g, key_mask=mask, **bias(nq, nk, heads, axes))


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("axes", [0, 2])
@pytest.mark.parametrize("nq,nk,heads,dim", SHAPES)
def test_blocks_of_zero_or_tiny_values(nq, nk, heads, dim, axes, dtype):
    """Every key has a gradient of its own even where its value is zero: <g, o> holds the values of all the others."""
    nk = nk // 32 * 32 + 1                                                  # a last subtile of one key
    for size in (0.0, 1e-6 if dtype is F32 else 2.0 ** -13):
        q, k, v, g = make(nq, nk, heads, heads, dim, dtype)
        v[32:64] *= size
        v[-1] *= size
        check(q, k, v, g, **bias(nq, nk, heads, axes))


@pytest.mark.parametrize("axes", [0, 2])
@pytest.mark.parametrize("nq,nk,heads,dim", SHAPES)
def test_fp32_gradient_rows_beside_larger_ones(nq, nk, heads, dim, axes):
    for size in (1e4, 1e6, 1e10):
        q, k, v, g = make(nq, nk, heads, heads, dim, F32)
        g[5::32] *= size
        check_sizes(q, k, v, g, **bias(nq, nk, heads, axes))


@pytest.mark.parametrize("dim", [32, 64])
@pytest.mark.parametrize("apart", [10, 14])
def test_fp16_gradient_rows_beside_larger_ones(apart, dim):
    """Rows 2^apart smaller than a neighbour at thousands of keys: no gradient sinks into the smallest numbers of fp16."""
    q, k, v, g = make(96, 5000, 2, 2, dim, F16)
    g *= 2.0 ** (10 - apart)
    g[5::32] *= 2.0 ** apart
    check(q, k, v, g)


@pytest.mark.parametrize("axes", [0, 1, 2])
@pytest.mark.parametrize("nq,nk,heads,dim", SHAPES + [(2, 3000, 4, 32)])
def test_large_values_that_weigh_nothing(nq, nk, heads, dim, axes):
    """A value 1e3 .. 1e10 times the others at a weight near e^-60, in a block of its own and among ordinary rows, first or last."""
    for size in (1e3, 1e6, 1e10):
        for where in (slice(0, 32), slice(64, 65), slice(nk - 3, nk)):
            q, k, v, g = make(nq, nk, heads, heads, dim, F32)
            q[..., 0] = 4.0
            k[..., 0] = 0.0
            k[where, :, 0] = -15.0 * dim ** 0.5
            v[where] *= size
            check_sizes(q, k, v, g, **bias(nq, nk, heads, axes))


@pytest.mark.parametrize("nq,nk,heads,dim", SHAPES)
def test_fp16_large_values_that_weigh_nothing(nq, nk, heads, dim):
    q, k, v, g = make(nq, nk, heads, heads, dim, F16)
    q[..., 0] = 4.0
    k[..., 0] = 0.0
    k[64:96, :, 0] = -5.0 * dim ** 0.5
    v *= 2.0 ** -6
    v[64:96] = v[64:96] * 2.0 ** 18
    check(q, k, v, g)


@pytest.mark.parametrize("nq,nk,heads,dim", SHAPES)
def test_rows_of_every_size_side_by_side(nq, nk, heads, dim):
    """Neighbouring values and gradients sixteen orders of magnitude apart; keys and queries six."""
    gen = torch.Generator().manual_seed(4)
    spread = lambda n, by: (10.0 ** (by * (2 * torch.rand(n, generator=gen) - 1)))[:, None, None].to(DEV)  # noqa: E731
    q, k, v, g = make(nq, nk, heads, heads, dim, F32)
    check_sizes(q, k, v * spread(nk, 8), g * spread(nq, 8))
    check_sizes(q * spread(nq, 3) * 1e-3, k * spread(nk, 3) * 1e-3, v, g)


def test_keys_of_little_weight_keep_their_gradients():
    """Keys that a bias of -20 holds down for every query: their own gradients keep their digits."""
    q, k, v, g = make(200, 300)
    kw = bias_args(200, 300, 4, 1, 1)
    kw["q_pos"], kw["k_pos"] = torch.zeros(200, 1, dtype=torch.int32, device=DEV), (torch.arange(300, device=DEV)[:, None] // 60 % 2).int()
    kw["bias_table"] = torch.where(torch.arange(16, device=DEV) == kw["bucket_lut"][2], -20.0, 0.0).expand(4, 16).contiguous()
    check(q, k, v, g, **kw)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("axes", [0, 2])
@pytest.mark.parametrize("nq,nk,heads,dim", SHAPES + [(2, 3000, 4, 32)])
def test_an_infinite_value_spoils_its_column_only(nq, nk, heads, dim, axes, dtype):
    from gnn_amd import ops
    q, k, v, _ = make(nq, nk, heads, heads, dim, dtype)
    kw = bias(nq, nk, heads, axes)
    v[37, 1, 3] = 0
    ref = reference(q, k, v, **kw)
    v[37, 1, 3] = math.inf
    o = ops.cross_attention(q, k, v, **kw)
    assert not torch.isfinite(o[:, 1, 3]).any()
    o[:, 1, 3] = ref["o"][:, 1, 3].to(o)
    assert_close(o, ref, "o")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("nq,nk,heads,dim", [(60, 90, 4, 32), (700, 1500, 8, 64), (500, 300, 2, 128)])
@pytest.mark.parametrize("axes", [0, 1, 2])
def test_nan_reaches_the_gradients_it_belongs_to(nq, nk, heads, dim, dtype, axes):
    """A NaN in a query, key, value or bias, and a score that overflows: every gradient that plain arithmetic makes NaN is NaN, the
    other segment's and the other heads' are finite.  None hides as the zero of a row without keys."""
    kw = bias(nq, 2 * nk, heads, axes)
    kw.update(q_ptr=ptr([nq // 2, nq - nq // 2]), k_ptr=ptr([nk, nk]))
    first, head = slice(0, nq // 2), 1
    cases = ["query", "key", "value", "overflow"] + ["bias"] * (axes > 0)
    for case in cases:
        q, k, v, g = make(nq, 2 * nk, heads, heads, dim, dtype)
        args = dict(kw)
        if case == "query":
            q[3, head, 5] = math.nan
        elif case == "key":
            k[40, head, 5] = math.nan
        elif case == "value":
            v[40, head, 5] = math.nan
        elif case == "overflow":
            args["scale"] = 3e38
            q[:, [h for h in range(heads) if h != head]] = 0
        else:
            args["bias_table"] = kw["bias_table"].clone()
            args["bias_table"][head] = math.nan
        got = run(q, k, v, g, **args)
        seg = (slice(0, nk),) if case in ("query", "key", "value") else (slice(0, 2 * nk),)
        rows = {"query": slice(3, 4), "key": first, "value": first}.get(case, slice(0, nq))
        hit = {n: torch.zeros_like(got[n], dtype=torch.bool) for n in got}
        hit["o"][rows, head] = case != "value"
        if case == "value":
            hit["o"][rows, head, 5] = True
        hit["dq"][rows, head] = True
        hit["dk"][seg[0], head] = True
        hit["dv"][seg[0], head] = case != "value"
        if axes:
            hit["dtable"][head] = True
        for name, t in got.items():
            if name == "dtable":                                    # buckets without a pair of that row stay finite
                assert torch.isnan(t[head]).any() and torch.isfinite(t[hit[name].logical_not()]).all(), (case, name)
                continue
            assert torch.isnan(t[hit[name]]).all(), (case, name)
            if case == "overflow" and name == "dq":
                continue                    # the other heads' dq, scale dS K at a scale of 3e38, overflows itself
            assert torch.isfinite(t[~hit[name]]).all(), (case, name)


def test_tiny_gradients_and_weights_beside_large_operands():
    """Factors that do not fit one power of two: gradients of 1e-34 that meet keys (queries) of 1e9, and keys at a weight of e^-80 whose
    queries have gradients of 1e30."""
    q, k, v, g = make(200, 300)
    check(q * 1e-9, k * 1e9, v, g * 1e-34)
    check(q * 1e9, k * 1e-9, v, g * 1e-34)
    check(q, k, v, g * 1e-36)
    kw = bias_args(200, 300, 4, 1, 1)
    kw["q_pos"], kw["k_pos"] = torch.zeros(200, 1, dtype=torch.int32, device=DEV), (torch.arange(300, device=DEV)[:, None] // 60 % 2).int()
    kw["bias_table"] = torch.where(torch.arange(16, device=DEV) == kw["bucket_lut"][2], -80.0, 0.0).expand(4, 16).contiguous()
    for q, k, v, g in ((q, k, v, g * 1e30), (q * 1e9, k * 1e-9, v * 1e-15, g * 1e30)):
        got, ref = run(q, k, v, g, **kw), reference(q, k, v, g, **kw)
        # e^-80 is 2^-115.4, and a weight below 2^-126 is zero: the exponential gives no smaller number.  Each pair may lose that much.
        for h in range(4):
            qh, vh, gh = (t[:, h].double().cpu().abs() for t in (q, v, g))
            ref["dv_tol"][:, h] += 2.0 ** -126 * gh.sum(0)
            d_p = gh @ vh.T + (gh * ref["o"][:, h].abs()).sum(1, keepdim=True)
            ref["dk_tol"][:, h] += 2.0 ** -126 * 32 ** -0.5 * (d_p.T @ qh)
        for name, t in got.items():
            assert_close(t, ref, name)
