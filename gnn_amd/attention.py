"""Attention of one set of states over another, with gradients: the fine nodes of a mesh reading the states of its coarse
graph, a probe point reading the states of a mesh, ragged batches of both.

    buckets = RelativeBuckets(32, reach=128, axes=2)
    out = cross_attention(q, k, v, bias_table=table, bucket_lut=buckets.lut(q.device), q_pos=cells_q, k_pos=cells_k)

``out_i = sum_j softmax_j(scale * <q_i, k_j> + bias_table[head, bucket]) v_j`` over the keys of query i's own segment.  The
arithmetic runs in ``libmgn_hip.so`` (``ops.cross_attention``, ``ops.cross_attention_bwd``); torch.autograd carries the
gradients of q, k, v and the bias table.

The reference's coarse branch hands its states to the sampled nodes only (core/meshgraphnet.py:192-194: all other rows of
the mapped-back tensor are zero); :class:`CrossScaleReadout` lets every fine node read all of them."""
from __future__ import annotations

import weakref
from typing import Optional

import torch
import torch.nn as nn
from torch.autograd import forward_ad

from . import ops
from ._lib import H


class RelativeBuckets:
    """Buckets of relative places for the learned bias of :func:`cross_attention`.

    The first half of the buckets holds one distance each, the others are spaced evenly in the logarithm up to ``reach``;
    everything further shares the last one.  ``axes`` 1: signed distances k - q on a line, half of the buckets for either
    side; 2 or 3: the whole part of the Euclidean distance between lattice points.  Borders come from whole-number
    comparisons, so no bucket depends on a rounding."""

    def __init__(self, num_buckets: int, reach: int, axes: int = 1):
        if axes not in (1, 2, 3) or not 1 <= reach <= 1024 or not 2 <= num_buckets <= 64 or (axes == 1 and (num_buckets % 2 or num_buckets < 4)):
            raise ValueError("RelativeBuckets: axes 1 .. 3, reach 1 .. 1024, 2 .. 64 buckets (an even number of at least 4 on a line)")
        self.num_buckets, self.reach, self.axes = num_buckets, reach, axes
        n = num_buckets // 2 if axes == 1 else num_buckets
        exact = max(1, n // 2)
        line, b = [], exact
        for d in range(reach + 1):
            if d >= exact:
                # (d / exact)^(n - exact) >= (reach / exact)^(b + 1 - exact), in whole numbers
                while b + 1 < n and reach > exact and d ** (n - exact) * exact ** (b + 1 - exact) >= reach ** (b + 1 - exact) * exact ** (n - exact):
                    b += 1
            line.append(d if d < exact else b)
        if axes == 1:
            line = [line[-r] for r in range(-reach, 0)] + [line[0]] + [n + v for v in line[1:]]
        self.table = torch.tensor(line, dtype=torch.int32)
        self._by_dev = {}

    def lut(self, device) -> torch.Tensor:
        """Bucket of every place, int32 [2 * reach + 1] on a line, else [reach + 1]."""
        device = torch.device(device)
        if device.type == "cuda" and device.index is None:           # the current one, which may be another at the next call
            device = torch.device("cuda", torch.cuda.current_device())
        if device not in self._by_dev:
            self._by_dev[device] = self.table.to(device)
        return self._by_dev[device]


class _Live:
    """Stands for an eager autograd graph of this module that is still alive, with the roots that lead to the leaves it
    accumulates into: leaves themselves, or the nodes that made an operand (the graph holds them anyway)."""
    alive: "weakref.WeakSet" = weakref.WeakSet()

    def __init__(self, roots):
        self.roots = roots
        _Live.alive.add(self)


def _leaves(roots) -> set:
    """Identities of the leaves that gradients reach from ``roots``."""
    found, seen, todo = set(), set(), list(roots)
    while todo:
        at = todo.pop()
        if isinstance(at, torch.Tensor):
            found.add(id(at))
        elif at not in seen:
            seen.add(at)
            leaf = getattr(at, "variable", None)              # the node that accumulates into a leaf
            if leaf is not None:
                found.add(id(leaf))
            todo += [n for n, _ in at.next_functions if n is not None]
    return found


def _guard_capture(tensors):
    """Leaves of a graph that is recorded into a HIP graph must not be held by an eager graph: their gradients would be
    accumulated on the eager graph's stream, which is not being captured, and the process would end."""
    roots = tuple(t if t.grad_fn is None else t.grad_fn for t in tensors if t is not None and t.requires_grad)
    if not torch.cuda.is_current_stream_capturing():
        return _Live(roots)
    mine = _leaves(roots)
    for other in list(_Live.alive):
        if _leaves(other.roots) & mine:
            raise RuntimeError("cross_attention: an eager result of the same leaves is still alive while a HIP graph is being captured; "
                               "delete it first (its gradients would be accumulated outside the capture)")
    return None


class _CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, bias_table, q_ptr, k_ptr, key_mask, bucket_lut, q_pos, k_pos, scale):
        stats = torch.empty(2, q.shape[1], q.shape[0], dtype=torch.float32, device=q.device)
        out32 = None
        if ctx.needs_input_grad[3] and q.dtype is not torch.float32:          # the table's gradient needs unrounded outputs
            out32 = torch.empty(q.shape, dtype=torch.float32, device=q.device)
        out = ops.cross_attention(q, k, v, q_ptr, k_ptr, key_mask, bias_table, bucket_lut, q_pos, k_pos, scale, stats=stats, out32=out32)
        ctx.save_for_backward(q, k, v, bias_table, q_ptr, k_ptr, key_mask, bucket_lut, q_pos, k_pos, out if out32 is None else out32, stats)
        ctx.scale = scale
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        q, k, v, bias_table, q_ptr, k_ptr, key_mask, bucket_lut, q_pos, k_pos, out, stats = ctx.saved_tensors
        need = ctx.needs_input_grad
        dq, dk, dv, dt = ops.cross_attention_bwd(g, q, k, v, out, stats, q_ptr, k_ptr, key_mask, bias_table, bucket_lut, q_pos, k_pos,
                                                 ctx.scale, table_grad=need[3])
        return (dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, dt) + (None,) * 7


def cross_attention(q, k, v, q_ptr=None, k_ptr=None, key_mask=None, bias_table=None, bucket_lut=None, q_pos=None, k_pos=None,
                    scale: Optional[float] = None):
    """:func:`gnn_amd.ops.cross_attention` with gradients of ``q``, ``k``, ``v`` and ``bias_table`` where they are wanted."""
    if not all(isinstance(t, torch.Tensor) and t.dim() == 3 for t in (q, k, v)):
        raise RuntimeError("cross_attention: q [queries, heads, dim] and k, v [keys, kv_heads, dim] tensors")
    grads = (q, k, v, bias_table)
    if getattr(forward_ad, "_current_level", 0) >= 0 and any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in grads):
        raise RuntimeError("cross_attention: no forward-mode derivative; an operand carries a tangent, which would be dropped")
    if not torch.is_grad_enabled() or not (q.requires_grad or k.requires_grad or v.requires_grad or (bias_table is not None and bias_table.requires_grad)):
        return ops.cross_attention(q, k, v, q_ptr, k_ptr, key_mask, bias_table, bucket_lut, q_pos, k_pos, scale)
    live = _guard_capture(grads)
    out = _CrossAttention.apply(q, k, v, bias_table, q_ptr, k_ptr, key_mask, bucket_lut, q_pos, k_pos, scale)
    if live is not None:
        out.grad_fn.live = live
    return out


class CrossScaleReadout(nn.Module):
    """What the coarse branch's final states tell every fine node: ``to_out(attention(to_q(x), to_k(xc), to_v(xc)))`` with a
    learned bias by the distance between the two nodes, in lattice cells of the mesh (``reach`` cells along its longest side;
    its table starts at zero).  Takes the place of the copy onto the sampled nodes (core/meshgraphnet.py:192-193) in
    ``EncodeProcessDecodeMultiScale(coarse_readout="attention")``; every mesh of a batch reads its own coarse graph."""

    def __init__(self, hidden_dim: int = H, heads: int = 4, num_buckets: int = 32, reach: int = 128):
        super().__init__()
        if hidden_dim != H:
            raise NotImplementedError(f"CrossScaleReadout: hidden_dim must be {H} for the HIP kernels")
        if heads < 1 or H % heads or (H // heads) % 8:
            raise ValueError(f"CrossScaleReadout: {heads} heads do not divide {H} into widths that are multiples of 8")
        self.heads, self.reach, self.num_buckets = heads, reach, num_buckets
        self.to_q, self.to_k, self.to_v, self.to_out = (nn.Linear(H, H) for _ in range(4))
        self.bias_table = nn.Parameter(torch.zeros(heads, num_buckets))
        RelativeBuckets(num_buckets, reach, 2)                       # refuses sizes the kernels do not take
        self.__dict__["_buckets"] = {}

    def plan(self, mesh_pos: torch.Tensor, first: torch.Tensor, sizes=None, counts=None) -> dict:
        """Places and segments of one mesh, or of the blocks of a batch (``sizes`` fine and ``counts`` coarse nodes each);
        ``first``: the sampled nodes.  Depends on the mesh alone: kept with its coarse graph."""
        pos = mesh_pos.detach().to(torch.float32)
        axes = pos.shape[1]
        if axes not in (2, 3):
            raise RuntimeError(f"CrossScaleReadout: mesh coordinates have two or three axes, got {axes}")
        cells, at = [], 0
        for n in (sizes or (pos.shape[0],)):
            p = pos[at: at + n]
            low = p.amin(dim=0, keepdim=True)
            side = (p - low).amax().clamp_min(1e-30)
            cells.append(((p - low) * (self.reach / side)).to(torch.int32))
            at += n
        q_pos = torch.cat(cells).contiguous()
        by_axes = self.__dict__["_buckets"]
        if axes not in by_axes:
            by_axes[axes] = RelativeBuckets(self.num_buckets, self.reach, axes)
        many = sizes is not None and len(sizes) > 1
        return dict(q_pos=q_pos, k_pos=q_pos[first].contiguous(), bucket_lut=by_axes[axes].lut(pos.device),
                    q_ptr=ops._block_ptr(sizes, pos.device) if many else None, k_ptr=ops._block_ptr(counts, pos.device) if many else None)

    def run(self, x: torch.Tensor, xc: torch.Tensor, plan: dict, out: torch.Tensor, keep: bool = False):
        """``x`` [n, 128] fine and ``xc`` [m, 128] coarse states -> ``out`` [n, 128]; with ``keep`` returns what
        :meth:`backward` needs."""
        def linear(lin, rows, to=None):
            to = torch.empty_like(rows) if to is None else to
            ops.train_linear_fwd(rows, lin.weight.detach(), 0, to, bias=lin.bias.detach())
            return to
        q, k, v = linear(self.to_q, x), linear(self.to_k, xc), linear(self.to_v, xc)
        split = lambda t: t.view(t.shape[0], self.heads, H // self.heads)  # noqa: E731
        stats = torch.empty(2, self.heads, x.shape[0], dtype=torch.float32, device=x.device) if keep else None
        o = torch.empty_like(q)
        ops.cross_attention(split(q), split(k), split(v), bias_table=self.bias_table.detach(), out=split(o), stats=stats, **plan)
        linear(self.to_out, o, out)
        return (x, xc, q, k, v, o, stats, plan) if keep else None

    def backward(self, kept, g: torch.Tensor, gx: torch.Tensor, gxc: torch.Tensor, scratch) -> dict:
        """For the gradient ``g`` of the output: adds the fine states' gradient to ``gx``, writes the coarse states' to
        ``gxc`` and returns the parameters' (deterministic sums throughout)."""
        x, xc, q, k, v, o, stats, plan = kept
        grads = {}

        def linear_bwd(name, g_out, a, ga, res=None):
            lin = getattr(self, name)
            dw, db = torch.empty_like(lin.weight), torch.empty_like(lin.bias)
            ops.train_linear_bwd(g_out, scratch, a=a, w=lin.weight.detach(), res=res, ga=ga, dw=dw, db=db)
            grads[name + ".weight"], grads[name + ".bias"] = dw, db
        split = lambda t: t.view(t.shape[0], self.heads, H // self.heads)  # noqa: E731
        go = torch.empty_like(o)
        linear_bwd("to_out", g, o, go)
        dq, dk, dv, grads["bias_table"] = ops.cross_attention_bwd(split(go), split(q), split(k), split(v), split(o), stats,
                                                                  bias_table=self.bias_table.detach(), **plan)
        linear_bwd("to_q", dq.view_as(q), x, gx, res=gx)
        linear_bwd("to_k", dk.view_as(k), xc, gxc)
        linear_bwd("to_v", dv.view_as(v), xc, gxc, res=gxc)
        return grads
