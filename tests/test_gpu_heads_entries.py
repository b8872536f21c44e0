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


def test_what_is_written_counts_as_modified(pkg):
    """a graph that saved a tensor notices that a call has written it since"""
    q, k, v = (torch.randn((2, 3, 2, 64), device="cuda") for _ in range(3))
    out, lse, w, wo = torch.empty_like(q), torch.empty((2, 2, 3), device="cuda"), torch.zeros((2, 2, 3), device="cuda"), torch.zeros((2, 2, 3), device="cuda")
    ko, vo, dq, dk, dv = (torch.empty_like(q) for _ in range(5))

    def versions(f, written, others):
        before = [x._version for x in written + others]
        f()
        after = [x._version for x in written + others]
        assert all(a > b for a, b in zip(after[:len(written)], before)) and after[len(written):] == before[len(written):]
    versions(lambda: pkg.attention_window(q, k, v, 4, out=out, lse=lse), [out, lse], [q, k, v])
    versions(lambda: pkg.attention_window_backward(q, q, k, v, out, lse, 4, dq=dq, dk=dk, dv=dv), [dq, dk, dv], [q, k, v, out, lse])
    versions(lambda: pkg.attention_prefix(q, k[0], v[0], k, v, out=out), [out], [q, k, v, lse])
    versions(lambda: pkg.attention_scored(q, k, v, w), [w], [q, k, v])
    versions(lambda: pkg.attention_scored(q, k, v, w, weights_out=wo, lse=lse), [wo, lse], [q, k, v, w])
    versions(lambda: pkg.evict_cache(k, v, w, None, 2, k_out=ko, v_out=vo, weights_out=wo), [ko, vo, wo], [k, v, w])
    x = torch.zeros((2, 2, 3), device="cuda", requires_grad=True)
    y = x.exp()                                           # exp saves its result for its backward pass
    pkg.attention_scored(q, k, v, y.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with torch.inference_mode():
        pkg.attention_scored(q, k, v, torch.zeros((2, 2, 3), device="cuda"))
