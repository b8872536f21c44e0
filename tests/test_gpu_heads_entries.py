"""GPU: the C entries of the batched attention operators, called as a C host calls them."""
import struct

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_weights_of_a_call_without_queries_need_no_queries_and_no_keys(pkg):
    """q_tokens = 0: the weights pass through; q, k, v, out and lse may be null"""
    lib = pkg.load()
    B, H, T = 2, 3, 300
    w, out = torch.rand((B, H, T), device="cuda"), torch.empty((B, H, T), device="cuda")
    fmt = struct.Struct("=60q13if")
    null = [0] * 4
    args = fmt.pack(fmt.size, *(null * 10), 0, 0, 0, w.data_ptr(), out.data_ptr(), H * T, T, H * T, T, *(null * 2), 0, 0,
                    0, B, 0, T, H, H, 64, 64, 0, 0, 0, 0, 0, 0.125)
    assert lib.sdpa_dev_heads_workspace(3, args) == 0
    assert lib.sdpa_dev_attention_scored(args, None, 0, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert torch.equal(out, w)
