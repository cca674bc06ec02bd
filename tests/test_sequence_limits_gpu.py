"""The sequence operators' memory, limits and layouts on an MI355X, beside test_sequence_gpu.py's values."""
import math

import pytest
import torch

import seq_ref as R
from test_sequence_gpu import DTYPES, S, check_attention, near, randn
from taco_amd import _lib

pytestmark = pytest.mark.gpu


def test_short_grouped_sequences_need_no_sums_of_parts():
    """a rollout's update with shared heads takes memory for its gradients and statistics, not for sums that no launch makes"""
    lens, H, Hk, d = [32] * 512, 32, 4, 64
    T = sum(lens)
    x = [randn(T, h, d, dtype=torch.bfloat16, seed=h).requires_grad_() for h in (H, Hk, Hk)]
    seqs = S().Packed(lens, "cuda:0")
    o = S().attention(*x, seqs)
    g = torch.ones_like(o)
    torch.autograd.grad(o, x, g, retain_graph=True)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    grads = torch.autograd.grad(o, x, g)
    torch.cuda.synchronize()
    own = sum(t.numel() * t.element_size() for t in grads) + T * H * 4       # dq, dk, dv and delta
    assert torch.cuda.max_memory_allocated() - before <= own + (1 << 20)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [40, 128])
def test_attention_group_in_parts_beside_short_sequences(monkeypatch, dtype, d):
    """the sums lie tile by tile: short sequences before, between and behind the long ones, in launches of their own"""
    monkeypatch.setattr(S(), "_FEW_SHORT", 0)
    lens = [3, 700, 33, 64, 129, 1]
    seqs = S().Packed(lens, "cuda:0")
    assert seqs._parts(64, 32, True) > 1 and [t[0] for t in seqs._tiles(64)] == [128, 32]
    check_attention(64, 2, d, lens, dtype)
