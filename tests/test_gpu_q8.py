"""Activations in 8 bits on the GPU: codes and scales, the Linear and edge backward passes that read them, and the training
step that keeps them.

Bounds: codes and scales are exact by definition (one rounded division each, a product rounded once to a whole number), so
they are compared bit for bit.  Products run on three bf16 terms per operand (exact splits) with fp32 sums: an entry that adds
n products is off by at most (n / 32 + 8) 2^-23 of the sum of their magnitudes (32 rows, or 16 of the width, per matrix
instruction, 6 instructions of partial products each), plus 2^-24 for the last rounding."""
import math

import pytest
import torch

import oracle as O
from test_gpu_model import DEV, graph_to

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def exact_codes(x, keep=False):
    """From the definition, in 64 bits: the factor and the scale are 32-bit numbers, each rounded once."""
    x = x.double().cpu()
    m = x.abs().amax(1, keepdim=True)
    factor = torch.where(m >= 2.0 ** -119, 127.0 / m, torch.zeros_like(m)).float().double()
    codes = torch.round(x * factor).clamp(-127, 127)
    if keep:
        codes = torch.where((codes == 0) & (x != 0), torch.sign(x), codes)
    return codes.to(torch.int8), (m[:, 0] / 127.0).float()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 128), (33, 128), (1000, 128), (7, 3), (65, 130), (9, 64), (40, 256), (12, 300), (5, 1000), (3, 1024)])
def test_codes_scales_and_restored_rows(rows, width, dtype):
    from gnn_amd import ops
    gen = torch.Generator().manual_seed(rows + width)
    x = (torch.randn(rows, width, generator=gen) * torch.exp(2 * torch.randn(rows, 1, generator=gen))).to(DEV, dtype)
    x[::5, ::2] = 0
    for keep in (False, True):
        kept = ops.q8_rows(x, keep_nonzero=keep)
        codes, scale = exact_codes(x, keep)
        assert torch.equal(kept.codes.cpu(), codes) and torch.equal(kept.scale.cpu(), scale)
        back = ops.q8_restore(kept, dtype)
        assert torch.equal(back.cpu(), (codes.float() * scale[:, None]).to(dtype))
        if keep:
            assert torch.equal(back != 0, x != 0) or dtype is F16        # a scale may be below fp16's smallest number
        half = scale[:, None].double() * (1.0 if keep else 0.5) * (1 + 2.0 ** -20)
        if dtype is F32:
            assert ((back.cpu().double() - x.cpu().double()).abs() <= half).all()


def test_ties_and_ends():
    """Exact halves go to the even code; the largest magnitude has code 127 whatever its sign."""
    from gnn_amd import ops
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -126.5, 126.5], [-127.0, 3.5, 4.5, -3.5, -4.5, 0.25, 0.75, -0.75]], device=DEV)
    k = ops.q8_rows(x)
    assert k.codes.tolist() == [[127, 0, 2, 2, 0, -2, -126, 126], [-127, 4, 4, -4, -4, 0, 1, -1]]


def test_rows_of_zeros_tiny_rows_and_rows_that_are_not_finite():
    from gnn_amd import ops
    x = torch.ones(6, 128, device=DEV)
    x[0] = 0
    x[1] *= 2.0 ** -125
    x[2, 5], x[3, 100], x[4, 0] = math.inf, math.nan, -math.inf
    for keep in (False, True):
        back = ops.q8_restore(ops.q8_rows(x, keep_nonzero=keep))
        assert (back[0] == 0).all() and (back[1].abs() <= 2.0 ** -125).all()
        assert torch.isnan(back[2:5]).all() and (back[5] == 1).all()


def test_refusals():
    from gnn_amd import ops
    x = torch.zeros(4, 128, device=DEV)
    for bad in (torch.zeros(4, 128), torch.zeros(4, 1025, device=DEV), torch.zeros(4, 128, dtype=torch.float64, device=DEV),
                torch.zeros(128, 4, device=DEV).t(), torch.zeros(4, device=DEV)):
        with pytest.raises(RuntimeError):
            ops.q8_rows(bad)
    kept = ops.q8_rows(x)
    with pytest.raises(RuntimeError):
        ops.q8_restore(kept, torch.float64)
    with pytest.raises(RuntimeError):
        ops.q8_restore(ops.Q8Rows(kept.codes, kept.scale[:3]))
    scratch = torch.empty(ops.train_scratch_bytes(), dtype=torch.uint8, device=DEV)
    w, ga = torch.zeros(128, 128, device=DEV), torch.empty_like(x)
    with pytest.raises(RuntimeError):
        ops.train_linear_bwd(x, scratch, a=kept, w=w, ga=ga)                                  # codes without a weight gradient
    with pytest.raises(RuntimeError):
        ops.train_linear_bwd(x, scratch, a=kept, w=w, mask=ops.q8_rows(x), ga=ga, dw=w)       # a mask of another tensor
    with pytest.raises(RuntimeError):
        ops.train_linear_bwd(x, scratch, a=ops.q8_rows(x[:3].contiguous()), w=w, ga=ga, dw=w)
    assert ops.q8_rows(x[:0]).codes.shape == (0, 128)


@pytest.mark.parametrize("rows", [1, 31, 33, 561, 20001])
@pytest.mark.parametrize("masked", [False, True])
def test_linear_backward_reads_codes(rows, masked):
    from gnn_amd import ops
    gen = torch.Generator().manual_seed(rows)
    a = torch.randn(rows, 128, generator=gen).to(DEV)
    kept = ops.q8_rows(a.relu(), keep_nonzero=True) if masked else ops.q8_rows(a)
    g, res = (torch.randn(rows, 128, generator=gen).to(DEV) * 1e-3 for _ in range(2))
    w = torch.randn(128, 256, generator=gen).to(DEV)
    scratch = torch.empty(ops.train_scratch_bytes(), dtype=torch.uint8, device=DEV)
    ga, dw, db = torch.empty_like(g), torch.full((128, 384), 5.0, device=DEV), torch.empty(128, device=DEV)
    ops.train_linear_bwd(g, scratch, a=kept, w=w, koff=128, mask=kept if masked else None, res=res, ga=ga, dw=dw, dw_koff=128, db=db)
    x, g64, w64 = kept.codes.double().cpu() * kept.scale.double().cpu()[:, None], g.double().cpu(), w.double().cpu()[:, 128:]
    want = [g64 @ w64, g64.T @ x, g64.sum(0)]
    size = [g64.abs() @ w64.abs(), g64.abs().T @ x.abs(), g64.abs().sum(0)]
    if masked:
        want[0] = want[0] * (x > 0)
        assert torch.equal(x.to(DEV) > 0, a > 0)
    want[0] = want[0] + res.double().cpu()
    size[0] = size[0] + res.double().cpu().abs()
    for got, wn, sz, n in zip((ga, dw[:, 128:256], db), want, size, (128, rows, rows)):
        tol = (n / 32 + 8) * 6 * 2.0 ** -23 * sz + 2.0 ** -24 * wn.abs()
        assert ((got.double().cpu() - wn).abs() <= tol).all()
    assert (dw[:, :128] == 5).all() and (dw[:, 256:] == 5).all()
    only = torch.empty(128, 128, device=DEV)
    ops.train_linear_bwd(g, scratch, a=kept, dw=only)                     # the weight gradient alone
    assert ((only.double().cpu() - want[1]).abs() <= (rows / 32 + 8) * 6 * 2.0 ** -23 * size[1]).all()


def small_model(**kw):
    from gnn_amd.meshgraphnet import EncodeProcessDecodeMultiScale
    torch.manual_seed(11)
    return EncodeProcessDecodeMultiScale(10, 7, hidden_size=128, process_steps=3, coarse_process_steps=kw.pop("coarse", 0), node_out_dim=3,
                                         attention=False, with_mat_params=False, time_dim=1, device=DEV, **kw).to(DEV).train()


def restored(kept):
    from gnn_amd import ops
    return ops.q8_restore(kept) if isinstance(kept, ops.Q8Rows) else kept


@pytest.mark.parametrize("ratio", [0.0, 0.5])
def test_training_step_with_kept_activations_in_8_bits(ratio):
    """The gradients are those of the fp32 backward pass on the restored activations (the per-node projections formed from
    them): the same kernels and sums, except that a weight gradient's products with codes may be grouped differently, hence
    the bound of the products, relative per tensor."""
    from gnn_amd import ops, training
    model = small_model(sample_ratio=ratio, coarse=2 if ratio else 0)
    model.coarse_start = 0
    g = graph_to(O.synthetic_graph(20, 14, seed=3, with_target=True), DEV)
    tgt = model._normalized_target(g)
    for nr in (model.node_features_normalizer, model.edge_features_normalizer) + ((model.coarse_edge_features_normalizer,) if ratio else ()):
        nr._max_accumulations = nr._num_accumulations + 1
    loss32, _ = training.forward_saving(model, g, tgt)
    model.activation_bits = 8
    loss8, saved = training.forward_saving(model, g, tgt)
    assert torch.equal(loss32, loss8)                                     # the forward pass is the same
    one = torch.ones(3, device=DEV)
    got = training.backward(model, saved, one)

    def full(layers, blocks):
        out = []
        for blk, (x, el, _, _, aggr, h1n, vn, _, _, _) in zip(blocks, layers):
            x, el, aggr, h1n, vn = (restored(t) for t in (x, el, aggr, h1n, vn))
            ps, pr = torch.empty_like(x), torch.empty_like(x)
            w0 = blk.edge_mlp[0].weight.detach()
            ops.train_linear_fwd(x, w0, 0, ps)
            ops.train_linear_fwd(x, w0, 128, pr, bias=blk.edge_mlp[0].bias.detach())
            out.append((x, el, None, None, aggr, h1n, vn, ps, pr, None))
        return out
    plain = dict(saved, layers=full(saved["layers"], model.processors), enc_n=tuple(map(restored, saved["enc_n"])), enc_e=tuple(map(restored, saved["enc_e"])))
    if ratio:
        c = saved["coarse"]
        plain["coarse"] = dict(c, layers=full(c["layers"], model.coarse_processors), enc_c=tuple(map(restored, c["enc_c"])))
    model.activation_bits = 32
    want = training.backward(model, plain, one)
    assert list(got) == list(want)
    for k in got:
        off = float((got[k].double() - want[k].double()).norm() / want[k].double().norm().clamp_min(1e-30))
        assert off <= 2.0 ** -18, (k, off)


def test_kept_activations_take_a_quarter_of_the_memory():
    from gnn_amd import training
    model = small_model(sample_ratio=0.0)
    g = graph_to(O.synthetic_graph(200, 150, seed=3, with_target=True), DEV)
    tgt = model._normalized_target(g)
    held = {}
    for bits in (32, 8):
        model.activation_bits = bits
        training.forward_saving(model, g, tgt)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        saved = training.forward_saving(model, g, tgt)[1]["layers"]
        torch.cuda.synchronize()
        held[bits] = torch.cuda.memory_allocated() - before
        del saved
    # per block: 5 + 1 tensors of which the fp32 step also keeps two projections and the edge latents dominate; 132 of 512 bytes a row
    assert held[8] < 0.27 * held[32], held


def test_loss_backward_and_captured_step():
    """Through ``loss().backward()`` and through a captured training step; the same numbers both ways."""
    from gnn_amd.optim import FusedAdam
    from gnn_amd.training import CapturedTrainStep
    g = graph_to(O.synthetic_graph(20, 14, seed=3, with_target=True), DEV)
    losses = []
    for captured in (False, True):
        model = small_model(sample_ratio=0.0)
        model.activation_bits = 8
        opt = FusedAdam(model.parameters(), lr=1e-3, capturable=captured)
        step = CapturedTrainStep(model, opt) if captured else None
        seen = []
        for _ in range(5):
            if captured:
                seen.append(float(step(g)[0]))
            else:
                opt.zero_grad()
                total = model.loss(g)[0]
                total.backward()
                opt.step()
                seen.append(float(total.detach()))
        losses.append(seen)
    assert losses[0] == losses[1] and all(math.isfinite(v) for v in losses[0])


def test_combinations_that_are_refused():
    from gnn_amd import ops
    g = graph_to(O.synthetic_graph(8, 6, seed=3, with_target=True), DEV)
    model = small_model(sample_ratio=0.0)
    model.activation_bits = 16
    with pytest.raises(ValueError):
        model.loss(g)
    model.activation_bits = 8
    prev = ops.set_matmul_mode("f32")
    try:
        with pytest.raises(NotImplementedError):
            model.loss(g)
    finally:
        ops.set_matmul_mode(prev)


def test_more_rows_than_one_launch_takes():
    """Rows beyond 2^26 go into a second launch; widths that are not a multiple of four as well."""
    from gnn_amd import ops
    rows = (1 << 26) + 1000
    x = torch.arange(rows, dtype=torch.int32, device="cuda").remainder_(251).to(torch.float16).add_(1).unsqueeze(1)
    kept = ops.q8_rows(x)
    assert bool((kept.codes == 127).all())
    one = (torch.arange(1, 252, dtype=torch.float64, device="cuda") / 127).float()       # rounded once, from 64 bits
    scales = bool((kept.scale == one[x[:, 0].long() - 1]).all())
    assert scales
    back = bool((ops.q8_restore(kept, torch.float16) == x).all())            # 127 fl(m / 127) is within 2^-23 of m, a fp16 number
    assert back


@pytest.mark.parametrize("rows", [64, 777])
def test_input_gradient_keeps_its_digits_under_the_row_scales(rows):
    """GA does not depend on the layer input, but is formed with the rows' scales and freed of them again.  Bound: 8 steps of 16
    products, 6 partial products each, so 48 sums in fp32 that may each drop up to 2^-23 of what they hold; the terms left out of
    the three-term splits, less than 2^-23; m G, 1 / m and their product, 3 roundings of 2^-24; all of the sum of magnitudes."""
    from gnn_amd import ops
    gen = torch.Generator().manual_seed(rows)
    a = torch.randn(rows, 128, generator=gen) * torch.exp(4 * torch.randn(rows, 1, generator=gen))
    a[:, 0] = a.abs().amax(1) * (1 + torch.rand(rows, generator=gen))             # scales all over [1, 2) 2^e
    g, w = torch.randn(rows, 128, generator=gen).to(DEV), torch.randn(128, 128, generator=gen).to(DEV)
    scratch = torch.empty(ops.train_scratch_bytes(), dtype=torch.uint8, device=DEV)
    ga, dw = torch.empty_like(g), torch.empty_like(w)
    ops.train_linear_bwd(g, scratch, a=ops.q8_rows(a.to(DEV)), w=w, ga=ga, dw=dw)
    g64, w64 = g.double().cpu(), w.double().cpu()
    tol = (48 + 1 + 1.5) * 2.0 ** -23 * (g64.abs() @ w64.abs())
    assert ((ga.double().cpu() - g64 @ w64).abs() <= tol).all()
