"""Host side of the attention over another set of states: the buckets, and what is refused before anything is launched."""
import ctypes

import pytest
import torch


def test_buckets_are_whole_number_exact():
    from gnn_amd.attention import RelativeBuckets
    b = RelativeBuckets(32, 128, 2).table.tolist()
    assert len(b) == 129 and b[:16] == list(range(16)) and b[128] == 31 and b == sorted(b)
    # bucket n of the second half starts at the first d with (d / 16)^16 >= (128 / 16)^(n - 16), i.e. d >= 16 * 2^(3 (n - 16) / 16)
    for n in range(17, 32):
        first = b.index(n) if n in b else None
        d = next(d for d in range(16, 129) if d ** 16 >= 16 ** 16 * 8 ** (n - 16))
        assert first == d or first is None
    line = RelativeBuckets(32, 128, 1).table.tolist()
    assert len(line) == 257 and line[128] == 0 and line[127] == 1 and line[129] == 17 and line[0] == 15 and line[256] == 31
    assert max(RelativeBuckets(64, 1024, 3).table.tolist()) == 63
    assert RelativeBuckets(2, 1, 2).table.tolist() == [0, 1]


@pytest.mark.parametrize("args", [(1, 10, 2), (65, 10, 2), (32, 0, 2), (32, 1025, 2), (32, 10, 4), (31, 10, 1), (2, 10, 1)])
def test_bucket_refusals(args):
    from gnn_amd.attention import RelativeBuckets
    with pytest.raises(ValueError):
        RelativeBuckets(*args)


def test_cpu_tensors_are_refused():
    from gnn_amd import attention
    x = torch.zeros(4, 2, 32)
    with pytest.raises(RuntimeError, match="CUDA/HIP"):
        attention.cross_attention(x, x, x)


def args(**kw):
    from gnn_amd import _lib
    a = _lib.MgnAttn()
    base = dict(q=4096, k=4096, v=4096, q_st=128, q_sh=32, k_st=128, k_sh=32, v_st=128, v_sh=32, n_q=10, n_k=20, n_seg=1, heads=4,
                kv_heads=4, dim=32, dtype=0, scale=0.1)
    for k, v in dict(base, **kw).items():
        setattr(a, k, v)
    return a


BAD = [dict(dtype=3), dict(dtype=-1), dict(dim=0), dict(dim=12), dict(dim=136), dict(heads=0), dict(kv_heads=3), dict(kv_heads=0),
       dict(heads=2048, kv_heads=1), dict(n_q=-1), dict(n_k=-1), dict(n_q=2 ** 31), dict(n_seg=0), dict(n_seg=2), dict(n_seg=2, q_ptr=64),
       dict(q_ptr=64), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(q=0), dict(k=0), dict(v=0),
       dict(q=4100), dict(q_st=129), dict(k_sh=33), dict(dtype=1, v_st=132), dict(bias_table=64), dict(bias_table=64, bucket_lut=64, q_pos=64),
       dict(bias_table=64, bucket_lut=64, q_pos=64, k_pos=64, axes=0, reach=5, n_bucket=4),
       dict(bias_table=64, bucket_lut=64, q_pos=64, k_pos=64, axes=2, reach=1025, n_bucket=4),
       dict(bias_table=64, bucket_lut=64, q_pos=64, k_pos=64, axes=2, reach=0, n_bucket=4),
       dict(bias_table=64, bucket_lut=64, q_pos=64, k_pos=64, axes=2, reach=5, n_bucket=65)]


@pytest.mark.parametrize("bad", BAD, ids=lambda d: ",".join(f"{k}={v}" for k, v in d.items()))
def test_the_library_refuses(bad):
    """Every check runs on the host before a pointer is used."""
    from gnn_amd import _lib
    lib, a = _lib.lib(), args(**bad)
    assert lib.mgn_attn_fwd_workspace_bytes(ctypes.byref(a)) == -1
    assert lib.mgn_attn_bwd_workspace_bytes(ctypes.byref(a), 1) == -1
    assert lib.mgn_attn_fwd(ctypes.byref(a), 4096, 128, 32, None, None, 4096, 1 << 40, None) == -1
    assert lib.mgn_attn_bwd(ctypes.byref(a), 4096, 128, 32, 4096, 128, 32, 4096, 4096, 4096, 4096, None, 4096, 1 << 40, None) == -1
    assert lib.mgn_last_error()


def test_null_arguments_and_small_workspaces_are_refused():
    from gnn_amd import _lib
    lib, a = _lib.lib(), args()
    need = lib.mgn_attn_fwd_workspace_bytes(ctypes.byref(args(n_q=100000)))
    assert need > 0
    assert lib.mgn_attn_fwd(None, 4096, 128, 32, None, None, 4096, 1 << 40, None) == -1
    assert lib.mgn_attn_fwd(ctypes.byref(args(n_q=100000)), 4096, 128, 32, None, None, 4096, need - 1, None) == -1
    assert lib.mgn_attn_fwd(ctypes.byref(args(n_q=100000)), 4096, 128, 32, None, None, None, need, None) == -1
    assert lib.mgn_attn_fwd(ctypes.byref(a), None, 128, 32, None, None, 4096, 1 << 40, None) == -1
    assert lib.mgn_attn_fwd(ctypes.byref(a), 4100, 128, 32, None, None, 4096, 1 << 40, None) == -1
    need = lib.mgn_attn_bwd_workspace_bytes(ctypes.byref(a), 0)
    ok = [4096, 128, 32, 4096, 128, 32, 4096, 4096, 4096, 4096, None, 4096, need, None]
    for i, v in ((0, None), (3, None), (6, None), (7, None), (8, None), (9, None), (10, 4096), (11, None), (12, need - 1), (7, 4100)):
        bad = list(ok)
        bad[i] = v
        assert lib.mgn_attn_bwd(ctypes.byref(a), *bad) == -1, i


def test_forward_mode_tangents_are_refused():
    """They would be dropped without a word where no operand requires a gradient."""
    from torch.autograd import forward_ad
    from gnn_amd import attention
    x = torch.zeros(4, 2, 32)
    with forward_ad.dual_level():
        for at in range(3):
            ops = [x, x, x]
            ops[at] = forward_ad.make_dual(x, torch.ones_like(x))
            with pytest.raises(RuntimeError, match="tangent"):
                attention.cross_attention(*ops)
            with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):
                attention.cross_attention(*ops)
        table = forward_ad.make_dual(torch.zeros(2, 4), torch.ones(2, 4))
        with pytest.raises(RuntimeError, match="tangent"):
            attention.cross_attention(x, x, x, bias_table=table)
        with pytest.raises(RuntimeError, match="CUDA/HIP"):                  # no tangent: the ordinary checks
            attention.cross_attention(x, x, x)


@pytest.mark.parametrize("fits,kw", [
    (True, dict(n_seg=1 << 20, q_ptr=64, k_ptr=64, n_q=1 << 20, n_k=1 << 20, heads=15, kv_heads=15)),
    (False, dict(n_seg=1 << 20, q_ptr=64, k_ptr=64, n_q=1 << 22, n_k=1 << 20, heads=16, kv_heads=16)),
    (False, dict(n_seg=1 << 20, q_ptr=64, k_ptr=64, n_q=1 << 22, n_k=1 << 20, heads=1024, kv_heads=1024)),
    (True, dict(n_seg=1 << 20, q_ptr=64, k_ptr=64, n_q=1 << 23, n_k=1 << 20, heads=8, kv_heads=8)),
    (False, dict(n_seg=1 << 20, q_ptr=64, k_ptr=64, n_q=1 << 23, n_k=1 << 20, heads=16, kv_heads=16)),
    (False, dict(n_q=1000, n_k=1 << 30, heads=4, kv_heads=4, n_seg=1)),
    (True, dict(n_q=4, n_k=1 << 30, heads=4, kv_heads=4, n_seg=1)),
    (True, dict(n_q=1 << 28, n_k=1000, heads=4, kv_heads=4, n_seg=1))])
def test_counts_that_no_launch_takes_are_refused(fits, kw):
    """A grid has fewer than 2^32 threads; what does not fit is an error of the host's checks, not of the launch."""
    from gnn_amd import _lib
    lib, a = _lib.lib(), args(**kw)
    assert (lib.mgn_attn_fwd_workspace_bytes(ctypes.byref(a)) >= 0) is fits
    if not fits:
        assert b"launch" in lib.mgn_last_error() or b"tokens x heads" in lib.mgn_last_error()
        assert lib.mgn_attn_fwd(ctypes.byref(a), 4096, 128, 32, None, None, 4096, 1 << 50, None) == -1
    many = args(n_seg=1 << 20, q_ptr=64, k_ptr=64, n_q=1 << 20, n_k=1 << 20, heads=17, kv_heads=17)
    assert lib.mgn_attn_bwd_workspace_bytes(ctypes.byref(many), 0) == -1
    assert lib.mgn_attn_bwd_workspace_bytes(ctypes.byref(args(n_q=1 << 20, n_k=1 << 20, heads=8, kv_heads=8)), 0) > 0


def test_operands_on_another_device_are_refused(monkeypatch):
    """Checked by the tensors' attributes alone: stand-ins for tensors of two cards."""
    from gnn_amd import ops
    from gnn_amd.attention import RelativeBuckets

    class Stub:
        is_cuda, dtype, shape = True, torch.float32, (2, 3)

        def __init__(self, at):
            self.device = torch.device("cuda", at)

        def is_contiguous(self):
            return True

        def data_ptr(self):
            return 4096
    assert ops._dev_on(Stub(0), torch.float32, (2, 3), torch.device("cuda", 0), "stats") == 4096
    with pytest.raises(RuntimeError, match="stats: on cuda:1"):
        ops._dev_on(Stub(1), torch.float32, (2, 3), torch.device("cuda", 0), "stats")
    # "cuda" is the current card of each call
    seen = []
    b = RelativeBuckets(4, 3, 2)
    b.table = type("T", (), {"to": lambda self, d: seen.append(d) or d})()
    for at in (0, 1, 0):
        monkeypatch.setattr(torch.cuda, "current_device", lambda at=at: at)
        assert b.lut("cuda") == torch.device("cuda", at)
    assert seen == [torch.device("cuda", 0), torch.device("cuda", 1)]


def test_capture_guard_looks_behind_operands_to_their_leaves(monkeypatch):
    """An operand is seldom a leaf: a projection's weights are, and an eager graph that holds them is found through it."""
    from gnn_amd import attention
    capturing = [False]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    w, other = torch.randn(8, 8, requires_grad=True), torch.randn(8, 8, requires_grad=True)
    x = torch.randn(4, 8)
    live = attention._guard_capture((x @ w, (x @ w).relu(), None, x))
    assert live is not None
    capturing[0] = True
    for t in (w, x @ w, (x @ w).view(2, 2, 8), (x @ other) * (x @ w)):
        with pytest.raises(RuntimeError, match="still alive"):
            attention._guard_capture((t,))
    assert attention._guard_capture((x @ other, x)) is None
    del live
    assert attention._guard_capture((x @ w,)) is None


def test_operands_that_are_no_rows_of_heads_are_refused():
    """Also where a gradient is wanted, in front of anything that looks at their shape."""
    from gnn_amd import attention
    x = torch.zeros(4, 2, 32)
    for bad in (None, 3.0, torch.zeros(4, 64), torch.zeros(4, 64, requires_grad=True), torch.zeros(1, 4, 2, 32, requires_grad=True)):
        for at in range(3):
            ops = [x, x, x]
            ops[at] = bad
            with pytest.raises(RuntimeError, match="cross_attention: q"):
                attention.cross_attention(*ops)


def test_readout_plan_follows_the_readouts_reach():
    """Kept with the coarse graph, but a readout of another reach or with other buckets gets its own."""
    from gnn_amd.meshgraphnet import EncodeProcessDecodeMultiScale
    model = EncodeProcessDecodeMultiScale(10, 7, node_out_dim=3, sample_ratio=0.5, coarse_readout="attention")
    pos = torch.rand(20, 2, generator=torch.Generator().manual_seed(1))
    cg = type("Coarse", (), {})()
    cg.first, cg.block_sizes = torch.arange(0, 20, 2), None
    first = model._readout_plan(cg, pos, None, {})
    assert model._readout_plan(cg, pos, None, {}) is first and int(first["q_pos"].max()) == 128
    from gnn_amd.attention import CrossScaleReadout
    model.readout = CrossScaleReadout(reach=16, num_buckets=8)
    second = model._readout_plan(cg, pos, None, {})
    assert int(second["q_pos"].max()) == 16 and second["bucket_lut"].shape[0] == 17
