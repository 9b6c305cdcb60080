"""The attention readout of the coarse branch inside the model: forward, predict, rollout, loss and gradients, against the
oracle's restatement in plain torch."""
import pytest
import torch

import oracle as O
from conftest import rel_l2
from test_gpu_model import DEV, TOL, graph_to
from test_gpu_options import _oracle_loss_and_grads, freeze_to, norm_pairs  # noqa: F401

pytestmark = pytest.mark.gpu


def build(cfg, sd, heads=4, seed=1):
    """(model, state dict with the readout's parameters): the bias table is given values, it starts at zero."""
    from gnn_amd.meshgraphnet import EncodeProcessDecodeMultiScale
    torch.manual_seed(seed)
    m = EncodeProcessDecodeMultiScale(cfg.node_in_dim, cfg.edge_in_dim, hidden_size=128, process_steps=cfg.process_steps,
                                      coarse_process_steps=cfg.coarse_process_steps, node_out_dim=cfg.node_out_dim, attention=cfg.attention,
                                      with_mat_params=cfg.with_mat_params, sample_ratio=cfg.sample_ratio, time_dim=cfg.time_dim, device=DEV,
                                      coarse_readout="attention", readout_heads=heads)
    assert not m.readout.bias_table.any()
    with torch.no_grad():
        m.readout.bias_table.normal_(0, 0.5)
    full = dict(m.state_dict())
    for k, v in sd.items():
        full[k] = v
    m.load_state_dict(full)
    m = m.to(DEV)
    return m, {k: v.cpu() for k, v in full.items()}


@pytest.mark.parametrize("heads", [1, 4, 16])
def test_forward_and_predict_vs_oracle(heads):
    """At equal statistics, fp32, the bar of every other model test (1e-5)."""
    cfg = O.OracleConfig(process_steps=2, sample_ratio=0.4, coarse_process_steps=1, coarse_readout="attention")
    model, sd = build(cfg, O.init_state_dict(cfg, 5), heads)
    model.eval()
    model.coarse_start = 3
    norms = O.make_norms(cfg)
    g = O.synthetic_graph(30, 21, seed=3)
    ref = O.forward(sd, cfg, norms, g, coarse_start=3)
    freeze_to(model, cfg, norms)
    assert rel_l2(model.forward(graph_to(g, DEV)), ref) <= TOL
    assert rel_l2(model.predict(graph_to(g, DEV)), O.predict(sd, cfg, norms, g, coarse_start=3)) <= TOL


def test_loss_and_gradients_vs_oracle():
    """Every parameter's gradient against the oracle's autograd in 32 and 64 bits, with the bounds of the copy readout's test
    (tests/test_gpu_options.py: single ReLUs on the other side of zero move tensors by 1e-3)."""
    from test_gpu_training import FixedStats
    cfg = O.OracleConfig(process_steps=2, sample_ratio=0.5, coarse_process_steps=2, coarse_readout="attention")
    model, sd = build(cfg, O.init_state_dict(cfg, 5))
    model.train()
    model.coarse_start = 3
    norms = O.make_norms(cfg)
    g = O.synthetic_graph(14, 9, seed=3, with_target=True)
    l32, g32 = _oracle_loss_and_grads(cfg, sd, norms, g, 3, torch.float32)
    freeze_to(model, cfg, norms)
    _, g64 = _oracle_loss_and_grads(cfg, sd, {k: FixedStats(v, torch.float64) for k, v in norms.items()}, g, 3, torch.float64)
    out = model.loss(graph_to(g, DEV))
    out[0].backward()
    for c in range(4):
        assert abs(float(out[c].detach()) - l32[c]) <= 1e-5 * abs(l32[c])
    seen = 0
    for k, p in model.named_parameters():
        if k == "readout.to_k.bias":
            # adding one vector to all keys shifts every score of a query alike: the gradient is zero up to rounding.
            # dK entries are rounded sums of dS q, so it is held against the size of the weight's gradient instead
            assert float(p.grad.norm()) <= 1e-4 * float(model.readout.to_k.weight.grad.norm())
            continue
        assert rel_l2(p.grad, g32[k]) < 5e-3 and rel_l2(p.grad.double(), g64[k]) < 1e-2, k
        seen += k.startswith("readout")
    assert seen == 8


def test_every_mesh_of_a_batch_reads_its_own_coarse_graph():
    from gnn_amd.graph import batch_graphs
    cfg = O.OracleConfig(process_steps=2, sample_ratio=0.4, coarse_process_steps=1, coarse_readout="attention")
    model, _ = build(cfg, O.init_state_dict(cfg, 5))
    model.eval()
    model.coarse_start = 0
    frames = [graph_to(O.synthetic_graph(nx, ny, seed=s), DEV) for nx, ny, s in ((14, 9, 1), (20, 12, 2), (5, 4, 3))]
    norms = O.make_norms(cfg)
    for s, (nx, ny) in ((1, (14, 9)), (2, (20, 12))):
        O.forward({k: v.cpu() for k, v in model.state_dict().items()}, cfg, norms, O.synthetic_graph(nx, ny, seed=s))
    freeze_to(model, cfg, norms)
    alone = [model.predict(f) for f in frames]
    both = batch_graphs(frames)
    both["batch_sizes"] = [f["mesh_pos"].shape[0] for f in frames]
    together = model.predict(both)
    at = 0
    for a in alone:
        n = a.shape[1]
        # one tile of queries may be cut differently, but rows do not depend on their neighbours
        assert rel_l2(together[:, at: at + n], a) <= 1e-6
        at += n


def test_rollout_replays_and_training_steps_agree_with_eager():
    from gnn_amd.optim import FusedAdam
    from gnn_amd.training import CapturedTrainStep
    cfg = O.OracleConfig(process_steps=2, sample_ratio=0.4, coarse_process_steps=1, coarse_readout="attention")
    g = graph_to(O.synthetic_graph(16, 10, seed=3, with_target=True), DEV)
    losses = []
    for captured in (False, True):
        model, _ = build(cfg, O.init_state_dict(cfg, 5))
        model.train()
        model.coarse_start = 0
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
    assert losses[0] == losses[1]


def test_checkpoint_keeps_the_readout(tmp_path):
    cfg = O.OracleConfig(process_steps=1, sample_ratio=0.4, coarse_process_steps=1, coarse_readout="attention")
    a, _ = build(cfg, O.init_state_dict(cfg, 5))
    b, _ = build(cfg, O.init_state_dict(cfg, 6), seed=9)
    a.save_model(str(tmp_path))
    b.load_model(str(tmp_path))
    for (k, x), (_, y) in zip(a.state_dict().items(), b.state_dict().items()):
        assert torch.equal(x, y), k


def test_refusals():
    from gnn_amd.attention import CrossScaleReadout
    from gnn_amd.meshgraphnet import EncodeProcessDecodeMultiScale
    with pytest.raises(ValueError):
        EncodeProcessDecodeMultiScale(10, 7, node_out_dim=3, sample_ratio=0.0, coarse_readout="attention")
    with pytest.raises(ValueError):
        EncodeProcessDecodeMultiScale(10, 7, node_out_dim=3, sample_ratio=0.5, coarse_readout="nearest")
    for heads in (0, 3, 32):
        with pytest.raises(ValueError):
            CrossScaleReadout(128, heads)
    with pytest.raises(NotImplementedError):
        CrossScaleReadout(64)


@pytest.mark.parametrize("cells", [(20, 14), (60, 48)])
def test_readout_bias_and_8_bit_activations_together(cells):
    """Training steps of a model that reads its coarse graph by attention and keeps its activations in 8 bits: the same numbers
    eagerly and from a captured step, whose replays alternate with rollouts of the model on the same mesh."""
    from gnn_amd.meshgraphnet import EncodeProcessDecodeMultiScale
    from gnn_amd.optim import FusedAdam
    from gnn_amd.training import CapturedTrainStep
    g = graph_to(O.synthetic_graph(*cells, seed=3, with_target=True), DEV)
    runs = []
    for captured in (False, True):
        torch.manual_seed(11)
        model = EncodeProcessDecodeMultiScale(10, 7, hidden_size=128, process_steps=2, coarse_process_steps=1, node_out_dim=3, attention=False,
                                              with_mat_params=False, time_dim=1, device=DEV, sample_ratio=0.5, coarse_readout="attention").to(DEV).train()
        model.coarse_start = 0
        model.activation_bits = 8
        opt = FusedAdam(model.parameters(), lr=1e-3, capturable=captured)
        step = CapturedTrainStep(model, opt) if captured else None
        seen = []
        for _ in range(5):
            if captured:
                total = step(g)[0]
            else:
                opt.zero_grad()
                total = model.loss(g)[0]
                total.backward()
                opt.step()
            seen.append(float(total.detach()))
            with torch.no_grad():
                seen.append(float(model.forward(g).double().norm()))
        seen.append(float(model.readout.bias_table.detach().double().norm()))
        runs.append(seen)
    assert runs[0] == runs[1] and all(v == v and abs(v) != float("inf") for v in runs[0])
    assert runs[0][-1] > 0                                                # the table, zeros at first, has moved


@pytest.mark.parametrize("readout", ["copy", "attention"])
def test_captured_step_owns_what_it_reads(readout):
    """Between the calls of a captured training step the model predicts and rolls out on other meshes and on another copy of the
    same coordinates, which replaces its coarse graph, workspaces and scratch, and freed memory is overwritten: the same losses
    as the eager sequence, bit for bit."""
    import gnn_amd
    from gnn_amd.meshgraphnet import EncodeProcessDecodeMultiScale
    from gnn_amd.optim import FusedAdam
    from gnn_amd.rollout import rollout
    from gnn_amd.training import CapturedTrainStep
    g = graph_to(O.synthetic_graph(16, 10, seed=3, with_target=True), DEV)
    others = [graph_to(O.synthetic_graph(nx, ny, seed=4), DEV) for nx, ny in ((9, 7), (40, 30))]
    clone = graph_to(O.synthetic_graph(16, 10, seed=3), DEV)
    traj = gnn_amd.synthetic_frames(12, 8, n_frames=4, seed=2)

    def disturb(model):
        with torch.no_grad():
            for other in others + [clone]:
                model.predict(other)
        seen = float(rollout(model, traj, use_graph=True)["pred"].double().norm())
        junk = [torch.full((n,), float("nan"), device=DEV) for n in (100, 1000, 5000, 20000, 100000) for _ in range(8)]
        torch.cuda.synchronize()
        del junk
        return seen
    runs = []
    for captured in (False, True):
        torch.manual_seed(11)
        model = EncodeProcessDecodeMultiScale(10, 7, hidden_size=128, process_steps=2, coarse_process_steps=1, node_out_dim=3, attention=False,
                                              with_mat_params=False, time_dim=1, device=DEV, sample_ratio=0.5, coarse_readout=readout).to(DEV).train()
        model.coarse_start = 0
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
            seen.append(disturb(model))
        if captured:
            assert step.graph is not None and step.held
            step.close()
            assert step.held is None
        runs.append(seen)
    assert runs[0] == runs[1] and all(v == v for v in runs[0])
