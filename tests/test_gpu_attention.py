"""Attention over another set of states on the GPU: values, gradients and refusals, against tests/attention_reference.py
(64 bits, bounds derived there)."""
import math

import pytest
import torch

from attention_reference import assert_close, reference

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def ptr(lengths, first=0):
    at = [first]
    for n in lengths:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device=DEV)


def make(nq, nk, heads=4, kv_heads=4, dim=32, dtype=F32, seed=0, size=1.0):
    gen = torch.Generator().manual_seed(seed)
    q, k, v, g = (torch.randn(n, h, dim, generator=gen) * size for n, h in ((nq, heads), (nk, kv_heads), (nk, kv_heads), (nq, heads)))
    return tuple(t.to(DEV, dtype) for t in (q, k, v, g))


def bias_args(nq, nk, heads, axes, reach, n_buckets=16, seed=1, spread=1.5):
    from gnn_amd.attention import RelativeBuckets
    gen = torch.Generator().manual_seed(seed)
    b = RelativeBuckets(n_buckets, reach, axes)
    hi = max(2, int(spread * reach))
    return dict(bias_table=(torch.randn(heads, n_buckets, generator=gen) * 0.7).to(DEV), bucket_lut=b.lut(DEV),
                q_pos=torch.randint(-hi, hi, (nq, axes), generator=gen, dtype=torch.int32).to(DEV),
                k_pos=torch.randint(-hi, hi, (nk, axes), generator=gen, dtype=torch.int32).to(DEV))


def check(q, k, v, g=None, **kw):
    """Runs the public entry point (with gradients if ``g``) and compares everything with the reference."""
    from gnn_amd import attention
    if g is None:
        got = {"o": attention.cross_attention(q, k, v, **kw)}
    else:
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        table = kw.get("bias_table")
        if table is not None:
            kw = dict(kw, bias_table=table.detach().requires_grad_())
            leaves.append(kw["bias_table"])
        o = attention.cross_attention(*leaves[:3], **kw)
        grads = torch.autograd.grad(o, leaves, g)
        got = dict(zip(("o", "dq", "dk", "dv", "dtable"), (o.detach(),) + grads))
    ref = reference(q, k, v, g, **kw)
    for name, t in got.items():
        assert_close(t, ref, name)
    return got


SIZES = [(1, 1), (1, 33), (5, 1), (31, 32), (33, 65), (128, 64), (129, 200), (300, 97)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("nq,nk", SIZES)
def test_sizes(nq, nk, dtype):
    check(*make(nq, nk, dtype=dtype))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("dim", [8, 16, 24, 40, 64, 72, 128])
def test_head_widths(dim, dtype):
    check(*make(150, 90, heads=2, kv_heads=2, dim=dim, dtype=dtype))
    check(*make(2, 700, heads=2, kv_heads=2, dim=dim, dtype=dtype)[:3])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 1), (6, 2), (8, 8), (16, 2), (12, 1)])
def test_shared_key_heads(heads, kv_heads, dtype):
    check(*make(140, 75, heads, kv_heads, 32, dtype))
    check(*make(3, 600, heads, kv_heads, 32, dtype)[:3])


@pytest.mark.parametrize("dtype", [F32, F16])
def test_ragged_segments_and_rows_outside(dtype):
    """Empty query and key segments, segments that end inside a tile, rows in front of the first and behind the last."""
    nq, nk = [33, 0, 1, 128, 50], [64, 7, 0, 31, 200]
    q, k, v, g = make(sum(nq) + 9, sum(nk) + 12, dtype=dtype)
    check(q, k, v, g, q_ptr=ptr(nq, 4), k_ptr=ptr(nk, 5))


@pytest.mark.parametrize("few", [False, True])
def test_rows_outside_all_segments_are_left_as_they_were(few):
    from gnn_amd import ops
    nq, nk = ([3, 2], [300, 90]) if few else ([40, 70], [30, 90])
    q, k, v, _ = make(sum(nq) + 20, sum(nk) + 5)
    out = torch.full_like(q, 7.0)
    args = dict(q_ptr=ptr(nq, 6), k_ptr=ptr(nk, 5))
    ops.cross_attention(q, k, v, out=out, **args)
    assert_close(out, reference(q, k, v, **args), "o", outside_kept=7.0)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("nq", [2, 150])
def test_masked_keys(nq, dtype):
    """A segment whose keys are all masked, NaN and infinities in masked rows."""
    nqs, nks = [nq, nq, nq], [100, 65, 70]
    q, k, v, g = make(3 * nq, sum(nks), dtype=dtype)
    gen = torch.Generator().manual_seed(3)
    mask = (torch.rand(sum(nks), generator=gen) > 0.4).to(DEV)
    mask[100:165] = False
    k, v = k.clone(), v.clone()
    k[~mask] = math.nan
    v[~mask] = math.inf
    clean = [torch.where(mask[:, None, None], t, torch.zeros_like(t)) for t in (k, v)]
    from gnn_amd import attention
    kw = dict(q_ptr=ptr(nqs), k_ptr=ptr(nks), key_mask=mask)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = attention.cross_attention(*leaves, **kw)
    grads = torch.autograd.grad(o, leaves, g)
    ref = reference(q, *clean, g, **kw)
    for name, t in zip(("o", "dq", "dk", "dv"), (o, *grads)):
        assert_close(t, ref, name)
    assert (o[nq:2 * nq] == 0).all() and (grads[0][nq:2 * nq] == 0).all() and (grads[1][~mask] == 0).all()


@pytest.mark.parametrize("nq", [1, 90])
def test_no_keys_at_all(nq):
    from gnn_amd import attention
    q, k, v, g = make(nq, 0)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = attention.cross_attention(*leaves)
    dq, dk, dv = torch.autograd.grad(o, leaves, g)
    assert (o == 0).all() and (dq == 0).all() and dk.shape == k.shape and dv.shape == v.shape


def test_no_queries():
    from gnn_amd import attention
    q, k, v, g = make(0, 40)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = attention.cross_attention(*leaves)
    dq, dk, dv = torch.autograd.grad(o, leaves, g)
    assert o.shape == q.shape and dq.shape == q.shape and (dk == 0).all() and (dv == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("axes,reach", [(1, 7), (1, 1024), (2, 1), (2, 60), (3, 1024)])
def test_bias_by_buckets(axes, reach, dtype):
    q, k, v, g = make(170, 130, dtype=dtype)
    check(q, k, v, g, **bias_args(170, 130, 4, axes, reach))
    q, k, v, _ = make(3, 500, heads=8, kv_heads=2, dtype=dtype)
    check(q, k, v, **bias_args(3, 500, 8, axes, reach))


@pytest.mark.parametrize("n_buckets", [2, 33, 64])
def test_bucket_counts(n_buckets):
    for dim, dtype in ((32, F32), (128, F32), (128, BF16)):
        q, k, v, g = make(140, 100, heads=2, kv_heads=1, dim=dim, dtype=dtype)
        check(q, k, v, g, **bias_args(140, 100, 2, 2, 90, n_buckets))


def test_places_at_every_border_and_far_away():
    """One query at the origin, keys at every whole distance around each border of the buckets and at the ends of the range."""
    reach = 1024
    edge = [(r, 0) for r in range(0, 1030)] + [(0, -r) for r in range(0, 1030)] + [(3 * r, 4 * r) for r in range(0, 210)]
    edge += [(724, 724), (725, 724), (2 ** 30, 2 ** 30), (-2 ** 30, 5), (70000, 70000)]
    k_pos = torch.tensor(edge, dtype=torch.int32)
    for nq in (1, 40):
        kw = bias_args(nq, len(edge), 4, 2, reach, 64)
        kw["k_pos"], kw["q_pos"] = k_pos.to(DEV), torch.zeros(nq, 2, dtype=torch.int32, device=DEV)
        kw["bias_table"] = torch.arange(256, dtype=F32, device=DEV).reshape(4, 64) / 16
        q, k, v, _ = make(nq, len(edge))
        check(q, k, v, **kw)


@pytest.mark.parametrize("nq", [2, 64])
@pytest.mark.parametrize("axes", [1, 2])
def test_bias_at_the_ends_of_its_type(nq, axes):
    """Minus infinity takes a bucket out (all of them: a row of zeros); the lowest finite value everywhere is a uniform softmax."""
    q, k, v, g = make(nq, 90)
    kw = bias_args(nq, 90, 4, axes, 20)
    kw["bias_table"][:, ::3] = -math.inf
    check(q, k, v, g, **kw)
    kw["bias_table"][:] = -math.inf
    got = check(q, k, v, g, **kw)
    assert all((got[n] == 0).all() for n in ("o", "dq", "dk", "dv", "dtable"))
    from gnn_amd import attention
    kw["bias_table"][:] = torch.finfo(F32).min
    o = attention.cross_attention(q, k, v, **kw)
    mean = v.double().mean(0, keepdim=True).expand_as(o)
    tol = 2.0 ** -19 * v.double().abs().mean(0, keepdim=True) + 2.0 ** -24 * mean.abs()
    assert ((o.double() - mean).abs() <= tol).all()
    leaf = v.detach().requires_grad_()
    dv, = torch.autograd.grad(attention.cross_attention(q, k, leaf, **kw), leaf, g)
    want = g.double().sum(0, keepdim=True) / 90
    assert ((dv.double() - want).abs() <= 2.0 ** -19 * g.double().abs().sum(0, keepdim=True) / 90 + 2.0 ** -24 * want.abs()).all()


@pytest.mark.parametrize("size", [1e-18, 1e-4, 30.0, 1e15])
def test_fp32_operands_of_any_size(size):
    """Values and gradients far from one (the two fp16 terms are scaled per subtile), rows of very different sizes."""
    q, k, v, g = make(100, 140)
    rows = torch.logspace(-2, 2, 140, device=DEV)[:, None, None]
    check(q, k, v * size * rows, g)
    check(q, k, v, g * size)
    check(q * size, k / size, v, g)


def test_strided_operands_of_a_packed_projection():
    gen = torch.Generator().manual_seed(5)
    packed = torch.randn(90, 3, 4, 32, generator=gen).to(DEV, BF16)
    g = torch.randn(90, 4, 32, generator=gen).to(DEV, BF16)
    check(packed[:, 0], packed[:, 1], packed[:, 2], g)
    by_head = torch.randn(4, 90, 32, generator=gen).to(DEV).transpose(0, 1)        # heads outermost
    check(by_head, by_head.flip(0), by_head * 2, torch.ones(1, 1, 1, device=DEV).expand(90, 4, 32))


@pytest.mark.parametrize("nq,nk", [(1, 40000), (3, 5000), (40, 9000)])
def test_long_key_ranges_are_split_and_joined(nq, nk):
    for dtype in (F32, BF16):
        check(*make(nq, nk, heads=2, kv_heads=1, dtype=dtype)[:3])


def test_offsets_beyond_32_bits():
    """The last segment of keys lies beyond 2^31 elements (and 2^32 bytes) of its tensor."""
    heads, dim, n = 8, 128, (2 ** 31) // (8 * 128) + 500
    k = torch.zeros(n, heads, dim, dtype=BF16, device=DEV)
    gen = torch.Generator().manual_seed(2)
    tail = torch.randn(300, heads, dim, generator=gen).to(DEV, BF16)
    k[n - 300:] = tail
    kp = torch.tensor([0, n - 300, n], dtype=torch.int32, device=DEV)
    for nq in (2, 90):
        q = torch.randn(nq + 1, heads, dim, generator=gen).to(DEV, BF16)
        from gnn_amd import ops
        o = ops.cross_attention(q, k, k, q_ptr=torch.tensor([0, 1, nq + 1], dtype=torch.int32, device=DEV), k_ptr=kp)
        assert_close(o[1:], reference(q[1:], tail, tail), "o")
    del k


def test_two_runs_agree_bit_for_bit():
    from gnn_amd import attention
    q, k, v, g = make(700, 900, dtype=F32)
    kw = bias_args(700, 900, 4, 2, 50)

    def run():
        leaves = [t.detach().requires_grad_() for t in (q, k, v, kw["bias_table"])]
        o = attention.cross_attention(*leaves[:3], **dict(kw, bias_table=leaves[3]))
        return (o.detach(),) + torch.autograd.grad(o, leaves, g)
    first = run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, run()))


def test_another_stream_and_two_calls_at_once():
    from gnn_amd import ops
    q, k, v, _ = make(400, 500)
    want = ops.cross_attention(q, k, v)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(5):
                outs.append(ops.cross_attention(q, k, v))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_captured_forward_and_backward_replay():
    """Forward and backward recorded into HIP graphs through the raw entry points, replayed with new inputs between eager calls."""
    from gnn_amd import ops
    q, k, v, g = make(200, 300)
    kw = bias_args(200, 300, 4, 2, 40)
    st = torch.empty(2, 4, 200, device=DEV)

    def step():
        o = ops.cross_attention(q, k, v, stats=st, **kw)
        return (o,) + ops.cross_attention_bwd(g, q, k, v, o, st, **kw)
    step()
    torch.cuda.synchronize()
    graphs, held = [], []
    for _ in range(2):                              # two graphs alive at once, each with its own workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(step())
        graphs.append(graph)
    for i in range(4):
        fresh = make(200, 300, seed=10 + i)
        for a, b in zip((q, k, v, g), fresh):
            a.copy_(b)
        for graph, out in zip(graphs, held):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_capture_beside_a_live_eager_graph_is_refused():
    """The backward of a captured forward would accumulate into leaves held by an eager graph, outside the capture."""
    from gnn_amd import attention
    q, k, v, g = make(64, 64)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    eager = attention.cross_attention(*leaves)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    raised = False
    with torch.cuda.stream(stream):
        graph.capture_begin()
        try:
            attention.cross_attention(*leaves)
        except RuntimeError as e:
            raised = "still alive" in str(e)
        graph.capture_end()
    assert raised
    del eager
    torch.cuda.synchronize()


def test_gradient_against_differences():
    """Central differences of a weighted sum along random directions.  For a step e along a unit direction, truncation is of
    order e^2 and the fp32 output errors (measured by the forward bound) enter divided by 2 e."""
    from gnn_amd import attention
    q, k, v, g = make(40, 50, heads=2, kv_heads=1, dim=16)
    kw = bias_args(40, 50, 2, 2, 12)
    table = kw.pop("bias_table")
    leaves = [t.detach().requires_grad_() for t in (q, k, v, table)]
    f = lambda a, b, c, t: attention.cross_attention(a, b, c, bias_table=t, **kw)  # noqa: E731
    grads = torch.autograd.grad(f(*leaves), leaves, g)
    gen = torch.Generator().manual_seed(9)
    step = 2.0 ** -7
    for i in range(4):
        d = torch.randn(leaves[i].shape, generator=gen).to(DEV)
        d /= d.norm()
        up, dn = ([t.detach() + (s * step * d if n == i else 0) for n, t in enumerate(leaves)] for s in (1, -1))
        diff = ((f(*up).double() - f(*dn).double()) * g.double()).sum() / (2 * step)
        ref = reference(q, k, v, g, bias_table=table, **kw)
        noise = 2 * float((ref["o_tol"] * g.cpu().double().abs()).sum()) / (2 * step)
        # third derivatives of softmax averages of unit-size values along a unit direction stay below |g| |v| sums
        slack = step ** 2 * float(g.double().abs().sum() * v.double().abs().max())
        assert abs(float(diff) - float((grads[i].double() * d.double()).sum())) <= noise + slack


def test_only_the_wanted_gradients():
    from gnn_amd import attention
    q, k, v, g = make(64, 64)
    kw = bias_args(64, 64, 4, 1, 10)
    leaf = k.detach().requires_grad_()
    o = attention.cross_attention(q, leaf, v, **kw)
    o.backward(g)
    assert_close(leaf.grad, reference(q, k, v, g, **kw), "dk")
    assert not attention.cross_attention(q, k, v, **kw).requires_grad


# The kernels chosen for many workgroups, reached by many heads and segments instead of long inputs.
@pytest.mark.parametrize("dtype,dim", [(F32, 32), (F32, 24), (F16, 64), (BF16, 40)])
@pytest.mark.parametrize("axes", [2, 3])
def test_two_heads_that_share_places(axes, dtype, dim):
    nq, nk = [9, 0, 33, 1, 5, 130, 2, 7, 40, 3, 8, 6, 64, 4, 11, 31], [70, 33, 0, 5, 64, 90, 31, 1, 65, 40, 2, 8, 100, 7, 32, 20]
    q, k, v, g = make(sum(nq) + 5, sum(nk) + 6, heads=64, kv_heads=16, dim=dim, dtype=dtype)
    gen = torch.Generator().manual_seed(8)
    mask = (torch.rand(k.shape[0], generator=gen) > 0.2).to(DEV)
    mask[70:103] = False
    check(q, k, v, g, q_ptr=ptr(nq, 2), k_ptr=ptr(nk, 3), key_mask=mask, **bias_args(q.shape[0], k.shape[0], 64, axes, 40))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_wide_heads_in_workgroups_of_eight_waves(dtype):
    nq, nk = [300, 1, 0, 256, 40], [129, 0, 64, 300, 31]
    q, k, v, g = make(sum(nq) + 3, sum(nk) + 2, heads=64, kv_heads=8, dim=128, dtype=dtype)
    check(q, k, v, g, q_ptr=ptr(nq, 1), k_ptr=ptr(nk, 1))


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("axes", [0, 1, 2])
def test_key_ranges_split_to_fill_rounds(axes, dtype):
    """Key ranges split for the forward pass and for the query gradient: pieces of uneven length, one without keys."""
    nq, nk = [11, 20, 0, 13, 9, 31, 8, 7, 1], [2100, 4000, 500, 0, 1, 3000, 33, 5000, 4001]
    q, k, v, g = make(sum(nq) + 4, sum(nk) + 9, heads=64, kv_heads=32, dim=16, dtype=dtype)
    gen = torch.Generator().manual_seed(8)
    mask = (torch.rand(k.shape[0], generator=gen) > 0.3).to(DEV)
    mask[5 + 2100:5 + 2100 + 1990] = False
    kw = bias_args(q.shape[0], k.shape[0], 64, axes, 200) if axes else {}
    check(q, k, v, g, q_ptr=ptr(nq, 2), k_ptr=ptr(nk, 5), key_mask=mask, **kw)


def test_rows_outside_a_split_forward_are_left_as_they_were():
    from gnn_amd import ops
    q, k, v, _ = make(3 * 40 + 20, 9 * 2048 + 5, heads=8)
    out = torch.full_like(q, 7.0)
    args = dict(q_ptr=ptr([40, 40, 40], 6), k_ptr=ptr([6000, 6000, 6000], 5))
    ops.cross_attention(q, k, v, out=out, **args)
    assert_close(out, reference(q, k, v, **args), "o", outside_kept=7.0)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("nq,nk,heads,dim", [(2, 300, 4, 32), (60, 90, 4, 32), (700, 1500, 8, 64), (1000, 700, 64, 32)])
@pytest.mark.parametrize("axes", [0, 2])
def test_nan_comes_out_where_it_went_in(nq, nk, heads, dim, dtype, axes):
    """A NaN in a query is its row's alone; in a key it reaches every query of the key's segment, in a value one column."""
    from gnn_amd import ops
    kw = bias_args(nq, 2 * nk, heads, axes, 30) if axes else {}
    kw.update(q_ptr=ptr([nq // 2, nq - nq // 2]), k_ptr=ptr([nk, nk]))
    q, k, v, _ = make(nq, 2 * nk, heads, heads, dim, dtype)
    want = ops.cross_attention(q, k, v, **kw)
    assert torch.isfinite(want).all()
    for which, at in ((0, (0, 1, 3)), (1, (nk + 5, 2, 7)), (2, (3, 1, 4))):
        ops_in = [q, k, v]
        ops_in[which] = ops_in[which].clone()
        ops_in[which][at] = math.nan
        o = ops.cross_attention(*ops_in, **kw)
        hit = torch.zeros_like(o, dtype=torch.bool)
        if which == 0:
            hit[0, 1] = True
        elif which == 1:
            hit[nq // 2:, 2] = True
        else:
            hit[:nq // 2, 1, 4] = True
        assert torch.isnan(o[hit]).all()
        assert torch.isfinite(o[~hit]).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("axes,dim", [(2, 32), (3, 64), (2, 128)])
def test_buckets_listed_for_the_backward_pass(axes, dim, dtype):
    """Ragged segments, all 64 buckets, masked keys; the lists are read by both backward kernels."""
    nq, nk = [700, 0, 33, 640, 200], [900, 64, 0, 300, 500]
    q, k, v, g = make(sum(nq) + 7, sum(nk) + 3, heads=4, kv_heads=2, dim=dim, dtype=dtype)
    gen = torch.Generator().manual_seed(8)
    mask = (torch.rand(k.shape[0], generator=gen) > 0.2).to(DEV)
    check(q, k, v, g, q_ptr=ptr(nq, 4), k_ptr=ptr(nk, 1), key_mask=mask, **bias_args(q.shape[0], k.shape[0], 4, axes, 300, 64))


@pytest.mark.parametrize("heads,nq,nk", [(1, [1300, 200], [1200, 300]), (2, [1, 2, 3, 0] * 256, [3, 2, 1, 1] * 256)])
def test_lattice_backward_without_lists(heads, nq, nk):
    """One head has nobody to share a list with; very many segments would take too large a one."""
    q, k, v, g = make(sum(nq), sum(nk), heads=heads, kv_heads=1)
    check(q, k, v, g, q_ptr=ptr(nq), k_ptr=ptr(nk), **bias_args(sum(nq), sum(nk), heads, 2, 50))


def test_two_threads_with_different_bucket_counts():
    """The backward pass asks for LDS by the number of buckets; threads that launch side by side do not set it under each other."""
    import threading
    from gnn_amd import ops
    jobs = []
    for n_buckets in (4, 64):
        q, k, v, g = make(140, 100, heads=2, kv_heads=2, dim=64)
        kw = bias_args(140, 100, 2, 1, 90, n_buckets)
        st = torch.empty(2, 2, 140, device=DEV)
        o = ops.cross_attention(q, k, v, stats=st, **kw)
        jobs.append(lambda q=q, k=k, v=v, g=g, o=o, st=st, kw=kw: ops.cross_attention_bwd(g, q, k, v, o, st, **kw))
    want = [job() for job in jobs]
    torch.cuda.synchronize()
    bad = []

    def loop(at):
        try:
            for _ in range(50):
                if not all(torch.equal(a, b) for a, b in zip(jobs[at](), want[at])):
                    bad.append(at)
        except Exception as e:  # noqa: BLE001
            bad.append(e)
    threads = [threading.Thread(target=loop, args=(at,)) for at in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.parametrize("nq,nk,heads", [(1, 300, 4), (40, 300, 4), (1200, 300, 64), (700, 2000, 4)])
@pytest.mark.parametrize("axes", [1, 2, 3])
def test_places_over_the_whole_range_of_int32(nq, nk, heads, axes, monkeypatch):
    """Differences of places that do not fit 32 bits are far, not near or on the other side."""
    import attention_reference

    def held(q_pos, k_pos, lut):
        # squares of such differences do not fit 64 bits: everything beyond +-4096 is beyond the reach of 50 on any axis
        reach = lut.shape[0] // 2 if axes == 1 else lut.shape[0] - 1
        d = (k_pos.long()[None] - q_pos.long()[:, None]).clamp(-4096, 4096)
        if axes == 1:
            return lut.long()[d[..., 0].clamp(-reach, reach) + reach]
        return lut.long()[(d * d).sum(-1).double().sqrt().long().clamp(max=reach)]
    monkeypatch.setattr(attention_reference, "buckets", held)
    kw = bias_args(nq, nk, heads, axes, 50)
    gen = torch.Generator().manual_seed(6)
    ends = torch.tensor([-2 ** 31, -2 ** 31 + 3, -2 ** 30 - 1, -7, 0, 5, 2 ** 30 + 1, 2 ** 31 - 40, 2 ** 31 - 1], dtype=torch.int32)
    for name, n in (("q_pos", nq), ("k_pos", nk)):
        kw[name] = ends[torch.randint(0, 9, (n, axes), generator=gen)].to(DEV)
    q, k, v, g = make(nq, nk, heads, heads)
    check(q, k, v, g, **kw)
