"""GPU: a row of the batched attention operators is a function of its own query and of the keys it sees -- bit for bit, whatever its neighbours
in the call hold."""
import pytest
import torch

from test_gpu_heads import lens, make

pytestmark = pytest.mark.gpu
DTYPES = ["bf16", "f32"]


def rising(k, top=3.0):
    """keys that grow along the cache: a row's softmax maximum rises a little in tile after tile"""
    T = k.shape[-3]
    return k * torch.linspace(0.3, top, T, device=k.device).view(-1, 1, 1).to(k.dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,Tq,Tk", [(2, 3, 200), (2, 5, 5000), (200, 3, 1000), (2, 300, 300), (2, 700, 900), (40, 100, 600)])
def test_a_large_key_that_a_row_does_not_see(B, Tq, Tk, dtype, pkg):
    """finite keys of a later token, large enough to move the softmax maximum of the rows that do see them"""
    q, k, v = make((B, Tq, 4, 64), dtype, 1), rising(make((B, Tk, 2, 64), dtype, 2)), make((B, Tk, 2, 64), dtype, 3)
    want, wl = pkg.attention_window(q, k, v, Tk)
    ws = pkg.attention_scored(q, k, v, torch.zeros((B, 2, Tk), device="cuda"))
    for hit in sorted({1, Tq // 3, Tq // 2, Tq - 1} - {0}):      # the first row that sees the changed key
        for factor in (8.0, 50.0):
            K = k.clone()
            K[:, Tk - Tq + hit] = k[:, Tk - Tq + hit] * factor
            out, lse = pkg.attention_window(q, K, v, Tk)
            assert torch.equal(out[:, :hit], want[:, :hit]) and torch.equal(lse[..., :hit], wl[..., :hit]), (hit, factor)
            assert not torch.equal(out[:, hit:], want[:, hit:])
            so, sl, _ = pkg.attention_scored(q, K, v, torch.zeros((B, 2, Tk), device="cuda"))
            assert torch.equal(so[:, :hit], ws[0][:, :hit]) and torch.equal(sl[..., :hit], ws[1][..., :hit]), (hit, factor)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,Tq,P", [(3, 1, 700), (3, 1, 9000), (20, 2, 700), (20, 2, 9000)])
def test_another_sequence_behind_the_same_prefix(B, Tq, P, dtype, pkg):
    """the queries of a batch share the prefix's tiles, and nothing else"""
    Tk = 40
    q, k, v = make((B, Tq, 4, 64), dtype, 1), make((B, Tk, 2, 64), dtype, 2), make((B, Tk, 2, 64), dtype, 3)
    kp, vp = rising(make((1, P, 2, 64), dtype, 4)[0]), make((1, P, 2, 64), dtype, 5)[0]
    want, wl = pkg.attention_prefix(q, kp, vp, k, v)
    for factor in (3.0, 10.0, 40.0):
        Q = q.clone()
        Q[1] = q[1] * factor
        out, lse = pkg.attention_prefix(Q, kp, vp, k, v)
        for b in [b for b in range(B) if b != 1]:
            assert torch.equal(out[b], want[b]) and torch.equal(lse[b], wl[b]), (b, factor)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Tq,nq", [(4, 2), (6, 5), (100, 40), (260, 131)])
def test_padded_rows_beside_values_that_are_no_numbers(Tq, nq, dtype, pkg):
    """a ragged call whose last live rows share a wave with rows that do not exist: a hidden cache row without numbers changes nothing"""
    Tk, nk, window, sinks = 1500, 1401, 1100, 3
    q, k, v = make((1, Tq, 4, 64), dtype, 1), make((1, Tk, 2, 64), dtype, 2), make((1, Tk, 2, 64), dtype, 3)
    q, k = q.abs(), -rising(k.abs().flip(1), 4.0).flip(1)        # scores below those of an empty query, and rising
    B = 130                                               # (so many that a workgroup walks many tiles)
    q, k, v = (x.expand(B, -1, -1, -1) for x in (q, k, v))
    kw = dict(sinks=sinks, q_lens=lens([nq] * B), kv_lens=lens([nk] * B))
    want = pkg.attention_window(q, k, v, window, **kw)
    V = v.clone()
    V[:, nk:] = V[:, sinks:nk - nq - window + 2] = float("nan")       # (the last of them is the first row's first key)
    got = pkg.attention_window(q, k, V, window, **kw)
    assert got[0][:, 0].isnan().all() and torch.equal(got[0][:, 1:], want[0][:, 1:]) and torch.equal(got[1], want[1])
    Q = q.clone()
    Q[:, nq:] = 1e4                                       # what rows behind the length hold
    got = pkg.attention_window(Q, k, v, window, **kw)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Tk", [60, 700, 6000])
@pytest.mark.parametrize("Tq", [5, 40])
def test_a_row_without_numbers_gives_its_weights_only_to_keys_it_sees(Tq, Tk, dtype, pkg):
    """attention_scored: the weights of the keys behind a row whose query holds NaN are those of the other rows"""
    q, k, v = make((2, Tq, 4, 64), dtype, 1), make((2, Tk, 2, 64), dtype, 2), make((2, Tk, 2, 64), dtype, 3)
    w = torch.rand((2, 2, Tk), generator=torch.Generator().manual_seed(4)).cuda()
    _, _, want = pkg.attention_scored(q, k, v, w, weights_out=torch.empty_like(w))
    Q = q.clone()
    Q[1, 1, 2] = float("nan")                             # one head of the second token, of the second key head's group
    out, lse, got = pkg.attention_scored(Q, k, v, w, weights_out=torch.empty_like(w))
    first = Tk - Tq + 2                                   # keys from here on are not seen by it
    assert torch.equal(got[0], want[0]) and torch.equal(got[1, 0], want[1, 0])
    assert torch.equal(got[1, 1, first:], want[1, 1, first:]) and got[1, 1, :first].isnan().all()
    assert out[1, 1, 2].isnan().all() and lse[1, 2, 1].isnan() and out.isnan().sum() == out.shape[-1]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("Tq,Tk,D", [(3, 70, 64), (2, 3000, 128), (4, 60, 256), (64, 64, 64), (90, 200, 128), (40, 60, 256), (70, 90, 33)])
def test_a_single_element_that_is_no_number(Tq, Tk, D, value, dtype, pkg):
    """one element of one hidden row, at every place inside a 16-byte piece: neither outputs nor gradients of rows that do not see it change"""
    q, k, v = make((1, Tq, 4, D), dtype, 1), make((1, Tk, 2, D), dtype, 2), make((1, Tk, 2, D), dtype, 3)
    dout = make((1, Tq, 4, D), dtype, 4)
    want = pkg.attention_window(q, k, v, Tk)
    grads = pkg.attention_window_backward(dout, q, k, v, *want, Tk)
    ws = pkg.attention_scored(q, k, v, torch.zeros((1, 2, Tk), device="cuda"))
    key = Tk - max(1, Tq // 2)                            # seen from this row on
    hit = key - (Tk - Tq)
    for col in list(range(8)) + [D // 2 + 3, D - 2, D - 1]:
        K, V = k.clone(), v.clone()
        K[0, key, 0, col] = V[0, key, 1, col] = value
        out, lse = pkg.attention_window(q, K, V, Tk)
        assert torch.equal(out[:, :hit], want[0][:, :hit]) and torch.equal(lse[..., :hit], want[1][..., :hit]), col
        so, sl, _ = pkg.attention_scored(q, K, V, torch.zeros((1, 2, Tk), device="cuda"))
        assert torch.equal(so[:, :hit], ws[0][:, :hit]) and torch.equal(sl[..., :hit], ws[1][..., :hit]), col
        # (values: dQ of the rows before; queries and output gradients: dK, dV of the keys behind them)
        dq, _, _ = pkg.attention_window_backward(dout, q, K, V, *want, Tk)
        assert torch.equal(dq[:, :hit], grads[0][:, :hit]), col
        Q, DO = q.clone(), dout.clone()
        Q[0, 0, 0, col] = DO[0, 0, 2, col] = value
        _, dk, dv = pkg.attention_window_backward(DO, Q, k, v, *want, Tk)
        first = Tk - Tq + 1                               # keys the first row does not see
        assert torch.equal(dk[:, first:], grads[1][:, first:]) and torch.equal(dv[:, first:], grads[2][:, first:]), col


@pytest.mark.parametrize("dtype", DTYPES)
def test_every_element_of_a_masked_tile_is_looked_at(dtype, pkg):
    T = 40
    for D in (64, 128):
        q, k, v = make((1, T, 1, D), dtype, 1), make((1, T, 1, D), dtype, 2), make((1, T, 1, D), dtype, 3)
        want, _ = pkg.attention_window(q, k, v, T)
        for col in range(D):
            V = v.clone()
            for row in (1, 17, 38):
                V[0, row:, 0, col] = float("inf")
                out, _ = pkg.attention_window(q, k, V, T)
                assert torch.equal(out[:, :row], want[:, :row]), (D, row, col)
                V[0, row:, 0, col] = v[0, row:, 0, col]
