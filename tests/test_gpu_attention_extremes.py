"""Attention on operands of very different sizes: blocks that are zero, tiny or masked beside ordinary ones, rows far larger or
smaller than their neighbours, NaN and infinities.  Values and gradients against tests/attention_reference.py, whose bounds are
relative to the sums of magnitudes of each result's own row."""
import math

import pytest
import torch

from attention_reference import assert_close, reference
from test_gpu_attention import BF16, DEV, F16, F32, bias_args, check, make, ptr

pytestmark = pytest.mark.gpu

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
    for size in (1e4, 1e6):
        q, k, v, g = make(nq, nk, heads, heads, dim, F32)
        g[5::32] *= size
        check(q, k, v, g, **bias(nq, nk, heads, axes))


@pytest.mark.parametrize("dim", [32, 64])
@pytest.mark.parametrize("apart", [10, 14])
def test_fp16_gradient_rows_beside_larger_ones(apart, dim):
    """Rows 2^apart smaller than a neighbour at thousands of keys: no gradient sinks into the smallest numbers of fp16."""
    q, k, v, g = make(96, 5000, 2, 2, dim, F16)
    g *= 2.0 ** (10 - apart)
    g[5::32] *= 2.0 ** apart
    check(q, k, v, g)


@pytest.mark.parametrize("nq,nk,heads,dim", SHAPES)
def test_fp16_large_values_that_weigh_nothing(nq, nk, heads, dim):
    q, k, v, g = make(nq, nk, heads, heads, dim, F16)
    q[..., 0] = 4.0
    k[..., 0] = 0.0
    k[64:96, :, 0] = -5.0 * dim ** 0.5
    v *= 2.0 ** -6
    v[64:96] = v[64:96] * 2.0 ** 18
    check(q, k, v, g)


def test_keys_of_little_weight_keep_their_gradients():
    """Keys that a bias of -20 holds down for every query: their own gradients keep their digits."""
    q, k, v, g = make(200, 300)
    kw = bias_args(200, 300, 4, 1, 1)
    kw["q_pos"], kw["k_pos"] = torch.zeros(200, 1, dtype=torch.int32, device=DEV), (torch.arange(300, device=DEV)[:, None] // 60 % 2).int()
    kw["bias_table"] = torch.where(torch.arange(16, device=DEV) == kw["bucket_lut"][2], -20.0, 0.0).expand(4, 16).contiguous()
    check(q, k, v, g, **kw)
