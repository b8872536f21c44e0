"""GPU: bf16 results of the batched attention operators are off by the rounding of the results, and by little else.

Softmax weights and their slopes dS are operands of bf16 products in two terms, the value rounded (half a step: 2^-8 of it) and what is left
of it rounded: 2^-16 in all.  The rest is counted as in tests/_heads_reference.py, which allows for one term."""
import numpy as np
import pytest
import torch

import _heads_reference as ref
from test_gpu_heads import f64, lens, make, reference

pytestmark = pytest.mark.gpu
U, W = 2.0 ** -8, 2.0 ** -16


def check(got, want, off, what):
    """off: what the value is off by before it is rounded"""
    got = f64(got)
    tol = U * (np.abs(want) + off) + off + 1e-30
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), "%s: %d of %d off, worst %.3g times its bound" % (what, bad.sum(), bad.size, np.nanmax(np.abs(got - want) / tol))
    # half a step is 2^-8 of the smallest value of a binade, and a value's place in it is any: the roundings of many values have a norm of
    # 2^-8 times sqrt(1/3) (uniform errors) times at most 1
    n = np.linalg.norm(got - want) / max(np.linalg.norm(want), 1e-30)
    assert want.size < 4096 or n <= U * 0.58 + np.linalg.norm(off) / np.linalg.norm(want), "%s: %.3g of its norm off" % (what, n)


def forward_off(q, k, v, ql, kl, window, sinks, prefix=None):
    scale = q.shape[3] ** -0.5
    want, _, _, _, heads = reference(q, k, v, ql, kl, window, sinks, scale, "bf16", prefix=prefix)
    off, V, G = np.zeros(want.shape), f64(v), q.shape[2] // k.shape[2]
    for (b, h), (nq, nk, p, o, err) in heads.items():
        vv = np.abs(V[b, :nk, h // G])
        if prefix is not None:
            vv = np.concatenate([np.abs(f64(prefix[1])[:, h // G]), vv])
        off[b, :nq, h] = (p @ vv) * (W + err[:, None] + 2 * p.shape[1] * ref.F32)
    return want, off, heads


CASES = [
    # B, Tq, Tk, Hq, Hkv, Dk, Dv, window, sinks, q_lens, kv_lens
    (2, 1, 700, 8, 2, 128, 128, 300, 4, None, [700, 333]),
    (3, 2, 4000, 4, 4, 64, 64, 1 << 30, 0, None, [4000, 1999, 31]),
    (2, 5, 300, 2, 1, 256, 200, 100, 2, None, None),
    (1, 300, 300, 8, 2, 128, 128, 64, 4, None, None),
    (2, 257, 257, 6, 2, 80, 72, 100, 3, [257, 130], [257, 130]),
    (1, 200, 400, 2, 1, 64, 64, 1 << 30, 0, None, None),
    (1, 150, 150, 4, 1, 256, 256, 40, 2, None, None),
    (2, 70, 90, 3, 1, 33, 17, 40, 1, [70, 31], [90, 40]),
    (1, 60, 60, 40, 1, 64, 64, 20, 1, None, None),
]


@pytest.mark.parametrize("c", CASES, ids=str)
def test_outputs_and_gradients(c, pkg):
    B, Tq, Tk, Hq, Hkv, Dk, Dv, window, sinks, ql, kl = c
    q, k, v = make((B, Tq, Hq, Dk), "bf16", 1, 1.5), make((B, Tk, Hkv, Dk), "bf16", 2), make((B, Tk, Hkv, Dv), "bf16", 3)
    kw = dict(sinks=sinks, q_lens=lens(ql), kv_lens=lens(kl))
    out, lse = pkg.attention_window(q, k, v, window, **kw)
    want, off, heads = forward_off(q, k, v, ql, kl, window, sinks)
    check(out, want, off, "out")
    # every row of a workgroup sees at most 512 keys here but in the second case, where delta is the sum of dO times the rounded output
    U_delta = U if Tk > 512 and window > 512 else 0.0
    dout = make((B, Tq, Hq, Dv), "bf16", 4)
    grads = pkg.attention_window_backward(dout, q, k, v, out, lse, window, **kw)
    G, scale, a = Hq // Hkv, Dk ** -0.5, np.abs
    Q, K, V, D = f64(q), f64(k), f64(v), f64(dout)
    wants, offs = [np.zeros(x.shape) for x in (Q, K, V)], [np.zeros(x.shape) for x in (Q, K, V)]
    for (b, h), (nq, nk, p, o, err) in heads.items():
        g, n = h // G, max(nq, nk)
        qq, kk, vv, dd = Q[b, :nq, h], K[b, :nk, g], V[b, :nk, g], D[b, :nq, h]
        dp = dd @ vv.T
        ds = p * (dp - (dd * o).sum(1, keepdims=True))
        mag = (p * (a(dd) @ a(vv).T)).sum(1, keepdims=True)                            # of the sum that delta is
        e = a(ds) * (W + err[:, None]) + p * ((Dv + 4) * ref.F32 * (a(dd) @ a(vv).T) + (err[:, None] + (n + Dv + 4) * ref.F32) * mag +
                                              U_delta * (a(dd) * a(o)).sum(1, keepdims=True))
        wants[0][b, :nq, h] = scale * ds @ kk
        offs[0][b, :nq, h] = scale * (e + 2 * n * ref.F32 * a(ds)) @ a(kk)
        wants[1][b, :nk, g] += scale * ds.T @ qq
        offs[1][b, :nk, g] += scale * (e + 2 * G * n * ref.F32 * a(ds)).T @ a(qq)
        wants[2][b, :nk, g] += p.T @ dd
        offs[2][b, :nk, g] += (p * (W + err[:, None] + 2 * G * n * ref.F32)).T @ a(dd)
    for got, w, o, name in zip(grads, wants, offs, ("dq", "dk", "dv")):
        check(got, w, o, name)


@pytest.mark.parametrize("B,Tq,Tk,P,D", [(5, 1, 40, 1000, 128), (20, 3, 77, 700, 64), (3, 50, 60, 130, 64), (2, 2, 64, 65, 256)])
def test_behind_a_prefix(B, Tq, Tk, P, D, pkg):
    q, k, v = make((B, Tq, 4, D), "bf16", 1, 1.5), make((B, Tk, 2, D), "bf16", 2), make((B, Tk, 2, D), "bf16", 3)
    kp, vp = make((1, P, 2, D), "bf16", 4)[0], make((1, P, 2, D), "bf16", 5)[0]
    out, lse = pkg.attention_prefix(q, kp, vp, k, v)
    want, off, _ = forward_off(q, k, v, None, None, 1 << 40, 0, prefix=(kp, vp))
    check(out, want, off, "out")


@pytest.mark.parametrize("B,Tq,Tk", [(3, 1, 900), (2, 50, 150)])
def test_scored(B, Tq, Tk, pkg):
    q, k, v = make((B, Tq, 8, 128), "bf16", 1, 1.5), make((B, Tk, 2, 128), "bf16", 2), make((B, Tk, 2, 128), "bf16", 3)
    out, lse, w = pkg.attention_scored(q, k, v, torch.zeros((B, 2, Tk), device="cuda"))
    want, off, _ = forward_off(q, k, v, None, None, 1 << 40, 0)
    check(out, want, off, "out")


@pytest.mark.parametrize("Tq", [1, 3, 100])
@pytest.mark.parametrize("at", [10, 150])
def test_infinities_that_rows_see_come_out_as_they_are(at, Tq, pkg):
    """what is left of a weight may be 0 or negative, and an infinity times it no number: the value itself is what a row that sees it gets"""
    Tk = 300
    q, k, v = make((2, Tq, 4, 64), "bf16", 1), make((2, Tk, 2, 64), "bf16", 2), make((2, Tk, 2, 64), "bf16", 3)
    want, _ = pkg.attention_window(q, k, v, Tk)
    V = v.clone()
    V[0, at, 0, 5], V[0, at, 0, 6], V[0, at + 1, 0, 6], V[1, at, 1, 7] = float("inf"), float("inf"), -float("inf"), -float("inf")
    out, _ = pkg.attention_window(q, k, V, Tk)
    assert out[0, :, :2, 5].eq(float("inf")).all() and out[0, :, :2, 6].isnan().all() and out[1, :, 2:, 7].eq(-float("inf")).all()
    same = torch.ones_like(out, dtype=torch.bool)
    same[0, :, :2, 5:7] = same[1, :, 2:, 7] = False
    assert torch.equal(out[same], want[same])
