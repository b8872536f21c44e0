"""GPU: the batched attention operators against the formulas in 64 bits (tests/_heads_reference.py counts the tolerances)."""
import numpy as np
import pytest
import torch

import _heads_reference as ref

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def make(shape, dtype, seed, scale=1.0, layout="tokens"):
    """a [B, T, H, D] tensor on the device, stored token-major, head-major, or as a misaligned part of a larger one"""
    g = torch.Generator().manual_seed(seed)
    B, T, H, D = shape
    x = (torch.randn(shape, generator=g) * scale).to(DT[dtype])
    if layout == "heads":
        return x.transpose(1, 2).contiguous().cuda().transpose(1, 2)
    if layout == "odd":
        big = torch.full((B, T + 2, H + 1, D + 3), float("nan"), dtype=DT[dtype], device="cuda")
        big[:, 1:T + 1, 1:, 1:D + 1] = x.cuda()
        return big[:, 1:T + 1, 1:, 1:D + 1]
    return x.cuda()


def f64(x):
    return x.detach().double().cpu().numpy()


def lens(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")


def close(got, want, tol, what):
    got = f64(got) if torch.is_tensor(got) else got
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    off = np.where(same, 0.0, np.abs(np.where(same, 0.0, got) - np.where(same, 0.0, want)))
    bad = ~(off <= tol) & ~same
    assert not bad.any(), "%s: %d of %d off, worst %.3g times its bound" % (what, bad.sum(), bad.size, np.nanmax(off / tol))


def reference(q, k, v, ql, kl, window, sinks, scale, dtype, prefix=None):
    """out, lse and their bounds for the whole batch; per (b, head): (nq, nk, see, p, out, err)"""
    B, Tq, Hq, Dk = q.shape
    Tk, Hkv, Dv = k.shape[1], k.shape[2], v.shape[3]
    G = Hq // Hkv
    Q, K, V = f64(q), f64(k), f64(v)
    out, lse = np.zeros((B, Tq, Hq, Dv)), np.full((B, Hq, Tq), -np.inf)
    to, tl = np.zeros(out.shape), np.zeros(lse.shape)
    heads = {}
    for b in range(B):
        nq, nk = (ql[b] if ql else Tq), (kl[b] if kl else Tk)
        see = ref.visible(nq, nk, window, sinks)
        for h in range(Hq):
            kk, vv, s = K[b, :nk, h // G], V[b, :nk, h // G], see
            if prefix is not None:
                P = prefix[0].shape[0]
                kk = np.concatenate([f64(prefix[0])[:, h // G], kk])
                vv = np.concatenate([f64(prefix[1])[:, h // G], vv])
                s = np.concatenate([np.ones((nq, P), bool), see], 1)
            o, l, p, a, c, err = ref.attention(Q[b, :nq, h], kk, vv, s, scale, dtype)
            out[b, :nq, h], lse[b, h, :nq], to[b, :nq, h], tl[b, h, :nq] = o, l, a, c
            heads[b, h] = (nq, nk, p, o, err)
    return out, lse, to, tl, heads


WINDOW = [
    # dtype, B, Tq, Tk, Hq, Hkv, Dk, Dv, window, sinks, q_lens, kv_lens, layout
    ("bf16", 1, 1, 1, 1, 1, 64, 64, 1, 0, None, None, "tokens"),
    ("f32", 1, 1, 1, 1, 1, 64, 64, 1, 0, None, None, "tokens"),
    ("bf16", 2, 1, 700, 8, 2, 128, 128, 256, 4, None, [700, 333], "tokens"),
    ("f32", 2, 1, 700, 8, 2, 128, 128, 256, 4, None, [1, 0], "tokens"),
    ("bf16", 3, 1, 2000, 4, 4, 64, 64, 5000, 0, None, [2000, 1999, 31], "heads"),
    ("bf16", 1, 300, 300, 4, 1, 128, 128, 64, 4, None, None, "tokens"),
    ("f32", 1, 300, 300, 4, 2, 64, 64, 64, 4, None, None, "tokens"),
    ("bf16", 2, 257, 257, 6, 2, 80, 72, 100, 3, [257, 130], [257, 130], "tokens"),
    ("f32", 2, 129, 200, 3, 1, 33, 17, 40, 40, [129, 1], [200, 77], "odd"),
    ("bf16", 2, 129, 200, 3, 1, 33, 17, 40, 1, [100, 129], [200, 129], "odd"),
    ("bf16", 1, 40, 97, 2, 1, 256, 256, 33, 2, None, None, "heads"),
    ("f32", 1, 40, 97, 2, 1, 256, 200, 33, 2, None, None, "tokens"),
    ("f32", 1, 5, 97, 2, 1, 256, 200, 33, 2, None, None, "tokens"),
    ("bf16", 1, 5, 97, 2, 1, 200, 256, 33, 2, None, None, "tokens"),
    ("bf16", 2, 64, 64, 2, 1, 64, 64, 0, 3, None, None, "tokens"),          # sinks only
    ("f32", 2, 64, 64, 2, 1, 64, 64, 0, 0, None, None, "tokens"),           # nothing is seen
    ("bf16", 2, 70, 50, 2, 1, 64, 64, 9, 2, None, None, "tokens"),          # the first 20 queries lie before the cache
    ("f32", 3, 40, 50, 2, 2, 96, 96, 1000, 0, [40, 0, 17], [50, 50, 0], "tokens"),
    ("bf16", 1, 3, 1500, 16, 1, 128, 64, 1 << 40, 0, None, None, "tokens"),
    ("bf16", 1, 1, 64, 48, 1, 64, 64, 64, 0, None, None, "tokens"),         # more than 32 rows of one token
    ("f32", 1, 33, 33, 1, 1, 1, 1, 7, 1, None, None, "tokens"),
]


def window_case(c, seed=0):
    dtype, B, Tq, Tk, Hq, Hkv, Dk, Dv, window, sinks, ql, kl, layout = c
    q = make((B, Tq, Hq, Dk), dtype, seed + 1, 1.5, layout)
    k = make((B, Tk, Hkv, Dk), dtype, seed + 2, 1.0, layout)
    v = make((B, Tk, Hkv, Dv), dtype, seed + 3, 1.0, layout)
    return q, k, v


@pytest.mark.parametrize("c", WINDOW, ids=str)
def test_window(c, pkg):
    dtype, B, Tq, Tk, Hq, Hkv, Dk, Dv, window, sinks, ql, kl, layout = c
    q, k, v = window_case(c)
    out, lse = pkg.attention_window(q, k, v, window, sinks=sinks, q_lens=lens(ql), kv_lens=lens(kl))
    want, wl, to, tl, _ = reference(q, k, v, ql, kl, window, sinks, Dk ** -0.5, dtype)
    close(out, want, to, "out")
    close(lse, wl, tl, "lse")


@pytest.mark.parametrize("c", WINDOW, ids=str)
def test_window_backward(c, pkg):
    dtype, B, Tq, Tk, Hq, Hkv, Dk, Dv, window, sinks, ql, kl, layout = c
    q, k, v = window_case(c)
    dout = make((B, Tq, Hq, Dv), dtype, 9, 1.0, layout)
    kw = dict(sinks=sinks, q_lens=lens(ql), kv_lens=lens(kl))
    out, lse = pkg.attention_window(q, k, v, window, **kw)
    dq, dk, dv = pkg.attention_window_backward(dout, q, k, v, out, lse, window, **kw)
    again = pkg.attention_window_backward(dout, q, k, v, out, lse, window, **kw)
    for x, y in zip((dq, dk, dv), again):
        assert torch.equal(x, y)
    check_gradients(q, k, v, dout, dq, dk, dv, ql, kl, window, sinks, dtype)


def check_gradients(q, k, v, dout, dq, dk, dv, ql, kl, window, sinks, dtype, scale=None):
    B, Tq, Hq, Dk = q.shape
    Hkv = k.shape[2]
    G, u = Hq // Hkv, ref.half_step(dtype)
    scale = Dk ** -0.5 if scale is None else scale
    _, _, _, _, heads = reference(q, k, v, ql, kl, window, sinks, scale, dtype)
    Q, K, V, D = f64(q), f64(k), f64(v), f64(dout)
    wq, wk, wv = np.zeros(Q.shape), np.zeros(K.shape), np.zeros(V.shape)
    tq, tk, tv = np.full(Q.shape, 1e-30), np.full(K.shape, 1e-30), np.full(V.shape, 1e-30)
    for (b, h), (nq, nk, p, o, err) in heads.items():
        g = h // G
        a = ref.gradients(Q[b, :nq, h], K[b, :nk, g], V[b, :nk, g], D[b, :nq, h], p, o, err, scale, dtype)
        wq[b, :nq, h], tq[b, :nq, h] = a[0], a[3]
        wk[b, :nk, g] += a[1]
        wv[b, :nk, g] += a[2]
        tk[b, :nk, g] += a[4] + G * ref.F32 * np.abs(a[1])
        tv[b, :nk, g] += a[5] + G * ref.F32 * np.abs(a[2])
    close(dq, wq, tq, "dq")
    close(dk, wk, tk + u * np.abs(wk), "dk")
    close(dv, wv, tv + u * np.abs(wv), "dv")


PREFIX = [
    # dtype, B, Tq, Tk, P, Hq, Hkv, Dk, Dv, q_lens, kv_lens, layout
    ("bf16", 1, 1, 1, 1, 1, 1, 64, 64, None, None, "tokens"),
    ("bf16", 5, 1, 40, 1000, 8, 2, 128, 128, None, [40, 1, 0, 33, 7], "tokens"),
    ("f32", 5, 3, 77, 301, 8, 2, 96, 96, None, [77, 3, 40, 20, 1], "heads"),
    ("f32", 2, 2, 9, 50, 2, 1, 40, 24, [2, 1], [9, 0], "odd"),
    ("bf16", 3, 50, 60, 130, 4, 2, 64, 64, [50, 20, 0], [60, 20, 5], "tokens"),
    ("bf16", 40, 1, 33, 600, 4, 1, 64, 128, None, None, "tokens"),
    ("f32", 3, 2, 20, 0, 2, 1, 64, 64, None, [20, 3, 0], "tokens"),         # no prefix
    ("bf16", 3, 2, 0, 70, 2, 1, 64, 64, None, None, "tokens"),              # nothing but the prefix
    ("f32", 2, 3, 64, 65, 2, 1, 256, 256, None, None, "tokens"),
]


@pytest.mark.parametrize("c", PREFIX, ids=str)
def test_prefix(c, pkg):
    dtype, B, Tq, Tk, P, Hq, Hkv, Dk, Dv, ql, kl, layout = c
    q = make((B, Tq, Hq, Dk), dtype, 1, 1.5, layout)
    k, v = make((B, Tk, Hkv, Dk), dtype, 2, 1.0, layout), make((B, Tk, Hkv, Dv), dtype, 3, 1.0, layout)
    kp, vp = make((1, P, Hkv, Dk), dtype, 4, 1.0, layout)[0], make((1, P, Hkv, Dv), dtype, 5, 1.0, layout)[0]
    out, lse = pkg.attention_prefix(q, kp, vp, k, v, q_lens=lens(ql), kv_lens=lens(kl))
    want, wl, to, tl, _ = reference(q, k, v, ql, kl, 1 << 40, 0, Dk ** -0.5, dtype, prefix=(kp, vp))
    close(out, want, to, "out")
    close(lse, wl, tl, "lse")


SCORED = [
    # dtype, B, Tq, Tk, Hq, Hkv, Dk, Dv, q_lens, kv_lens, layout
    ("bf16", 1, 1, 1, 1, 1, 64, 64, None, None, "tokens"),
    ("bf16", 3, 1, 900, 8, 2, 128, 128, None, [900, 257, 0], "tokens"),
    ("f32", 3, 1, 900, 8, 2, 128, 128, None, [1, 899, 128], "heads"),
    ("f32", 2, 50, 150, 6, 2, 64, 48, [50, 20], [150, 20], "tokens"),
    ("bf16", 2, 50, 150, 3, 1, 33, 17, [50, 31], [150, 140], "odd"),
    ("bf16", 1, 70, 50, 2, 1, 64, 64, None, None, "tokens"),
    ("f32", 1, 2, 300, 2, 1, 256, 256, None, None, "tokens"),
    ("bf16", 2, 4, 260, 16, 2, 256, 64, None, None, "tokens"),
]


@pytest.mark.parametrize("c", SCORED, ids=str)
def test_scored(c, pkg):
    dtype, B, Tq, Tk, Hq, Hkv, Dk, Dv, ql, kl, layout = c
    q = make((B, Tq, Hq, Dk), dtype, 1, 1.5, layout)
    k, v = make((B, Tk, Hkv, Dk), dtype, 2, 1.0, layout), make((B, Tk, Hkv, Dv), dtype, 3, 1.0, layout)
    before = torch.rand((B, Hkv, Tk), generator=torch.Generator().manual_seed(4)).cuda()
    weights = before.clone()
    out, lse, same = pkg.attention_scored(q, k, v, weights, q_lens=lens(ql), kv_lens=lens(kl))
    assert same is weights
    other = torch.full((B, Hkv + 1, Tk + 5), 7.0, device="cuda")
    pkg.attention_scored(q, k, v, before, q_lens=lens(ql), kv_lens=lens(kl), weights_out=other[:, 1:, 2:Tk + 2])
    assert torch.equal(other[:, 1:, 2:Tk + 2], weights) and other[:, 0].eq(7).all() and other[:, :, Tk + 2:].eq(7).all()
    want, wl, to, tl, heads = reference(q, k, v, ql, kl, 1 << 40, 0, Dk ** -0.5, dtype)
    close(out, want, to, "out")
    close(lse, wl, tl, "lse")
    sums, tol = f64(before), np.zeros((B, Hkv, Tk))
    for (b, h), (nq, nk, p, o, err) in heads.items():
        sums[b, h // (Hq // Hkv), :nk] += p.sum(0)
        tol[b, h // (Hq // Hkv), :nk] += (p * (err[:, None] + 2 * nq * ref.F32)).sum(0)
    close(weights, sums, tol + 2 * Hq * ref.F32 * np.abs(sums) + 1e-30, "weights")


EVICT = [
    # dtype, B, T, H, Dk, Dv, budget, sinks, recent, lens, layout
    ("bf16", 1, 1, 1, 64, 64, 1, 0, 0, None, "tokens"),
    ("bf16", 2, 300, 2, 128, 128, 100, 4, 20, None, "tokens"),
    ("f32", 3, 1500, 2, 80, 72, 700, 0, 0, [1500, 701, 700], "heads"),
    ("f32", 3, 500, 1, 33, 17, 100, 3, 97, [500, 100, 0], "odd"),
    ("bf16", 2, 400, 3, 7, 5, 50, 50, 0, [400, 51], "odd"),
    ("bf16", 2, 4100, 2, 64, 64, 4099, 1, 1, None, "tokens"),
    ("f32", 2, 64, 2, 64, 64, 0, 0, 0, None, "tokens"),
    ("bf16", 2, 0, 2, 64, 64, 8, 2, 2, None, "tokens"),
    ("bf16", 2, 90, 2, 64, 64, 200, 2, 2, [90, 13], "tokens"),
]


@pytest.mark.parametrize("values", ["spread", "ties", "odd"])
@pytest.mark.parametrize("c", EVICT, ids=str)
def test_evict(c, values, pkg):
    dtype, B, T, H, Dk, Dv, budget, sinks, recent, ln, layout = c
    k, v = make((B, T, H, Dk), dtype, 2, 1.0, layout), make((B, T, H, Dv), dtype, 3, 1.0, layout)
    g = torch.Generator().manual_seed(6)
    w = torch.exp(3 * torch.randn((B, H, T), generator=g))
    if values == "ties":
        w = torch.randint(0, 3, (B, H, T), generator=g).float()
    if values == "odd" and T:
        pick = torch.randint(0, 8, (B, H, T), generator=g)
        for i, x in enumerate((float("nan"), float("inf"), -float("inf"), -0.0, 0.0, -1.5, 1e-42)):
            w = torch.where(pick == i, torch.tensor(x), w)
    wd = w.cuda()
    nk, nv, nw, nl, kept = pkg.evict_cache(k, v, wd, lens(ln), budget, sinks=sinks, recent=recent)
    K, V = k.cpu(), v.cpu()
    for b in range(B):
        n = ln[b] if ln else T
        assert nl[b].item() == min(n, budget)
        for h in range(H):
            want = ref.kept(w[b, h].tolist(), n, budget, sinks, recent)
            m = len(want)
            assert kept[b, h].tolist() == want + [-1] * (budget - m)
            assert torch.equal(nk[b, :m, h].cpu(), K[b, want, h]) and torch.equal(nv[b, :m, h].cpu(), V[b, want, h])
            assert torch.equal(nw[b, h, :m].cpu().view(torch.int32), w[b, h, want].view(torch.int32))
            assert not nk[b, m:, h].any() and not nv[b, m:, h].any() and not nw[b, h, m:].any()


def test_evict_leaves_what_lies_behind_the_budget(pkg):
    k, v = make((2, 90, 2, 64), "bf16", 1), make((2, 90, 2, 64), "bf16", 2)
    w = torch.rand((2, 2, 90), device="cuda")
    ko, vo = torch.full((2, 64, 2, 64), 5, dtype=torch.bfloat16, device="cuda"), torch.full((2, 70, 2, 64), 6, dtype=torch.bfloat16, device="cuda")
    wo = torch.full((2, 2, 80), 7.0, device="cuda")
    a = pkg.evict_cache(k, v, w, None, 40, sinks=2, recent=10, k_out=ko, v_out=vo, weights_out=wo)
    b = pkg.evict_cache(k, v, w, None, 40, sinks=2, recent=10)
    assert a[0] is ko and a[1] is vo and a[2] is wo
    assert torch.equal(ko[:, :40], b[0]) and torch.equal(vo[:, :40], b[1]) and torch.equal(wo[:, :, :40], b[2])
    assert ko[:, 40:].eq(5).all() and vo[:, 40:].eq(6).all() and wo[:, :, 40:].eq(7).all()


def poison(x, where, value):
    x = x.clone()
    x[where] = value
    return x


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("Tq", [1, 2, 100])
def test_a_key_that_a_row_does_not_see_has_no_influence(Tq, value, dtype, pkg):
    """cache rows outside the window, in the future or behind the length hold no numbers: rows that do not see them are bit for bit
    what they were, and so are gradients they do not reach"""
    Tk, window, sinks = 200, 30, 2
    q, k, v = make((2, Tq, 4, 64), dtype, 1), make((2, Tk, 2, 64), dtype, 2), make((2, Tk, 2, 64), dtype, 3)
    dout = make((2, Tq, 4, 64), dtype, 4)
    kl = [190, 150]
    kw = dict(sinks=sinks, kv_lens=lens(kl))
    clean, clse = pkg.attention_window(q, k, v, window, **kw)
    grads = pkg.attention_window_backward(dout, q, k, v, clean, clse, window, **kw)
    for at in (5, 60, 185, 195):
        where = (slice(None), at)
        for K, V in ((poison(k, where, value), v), (k, poison(v, where, value))):
            out, lse = pkg.attention_window(q, K, V, window, **kw)
            dq, dk, dv = pkg.attention_window_backward(dout, q, K, V, out, lse, window, **kw)
            for b in range(2):
                see = ref.visible(Tq, kl[b], window, sinks)
                hit = see[:, at] if at < kl[b] else np.zeros(Tq, bool)
                safe = torch.tensor(~hit).cuda()
                assert torch.equal(out[b, safe], clean[b, safe]) and torch.equal(lse[b][:, safe], clse[b][:, safe])
                assert torch.equal(dq[b, safe], grads[0][b, safe])
                for r in np.nonzero(hit)[0]:
                    if V is not v:            # 0 < weight: the value itself comes out
                        want = torch.full_like(out[b, r], value)
                        assert torch.equal(out[b, r].isnan(), want.isnan()) and (np.isnan(value) or torch.equal(out[b, r], want))
                # keys that share no row with the poisoned one keep their gradients
                touched = see[hit].any(0)
                far = torch.zeros(Tk, dtype=torch.bool)
                far[:kl[b]] = torch.tensor(~touched)
                far[at] = False
                far = far.cuda()
                assert torch.equal(dk[b, far], grads[1][b, far]) and torch.equal(dv[b, far], grads[2][b, far])


def test_gradients_against_differences(pkg):
    """the derivative of sum(out * dout) along random directions, by central differences of the 64-bit formula"""
    B, T, Hq, Hkv, D, window, sinks = 1, 50, 4, 2, 64, 17, 2
    q, k, v = make((B, T, Hq, D), "f32", 1), make((B, T, Hkv, D), "f32", 2), make((B, T, Hkv, D), "f32", 3)
    dout = make((B, T, Hq, D), "f32", 4)
    out, lse = pkg.attention_window(q, k, v, window, sinks=sinks)
    grads = pkg.attention_window_backward(dout, q, k, v, out, lse, window, sinks=sinks)
    see = ref.visible(T, T, window, sinks)
    X, Do = [f64(x) for x in (q, k, v)], f64(dout)

    def loss(Q, K, V):
        return sum((ref.attention(Q[0, :, h], K[0, :, h // 2], V[0, :, h // 2], see, D ** -0.5, "f32")[0] * Do[0, :, h]).sum() for h in range(Hq))
    rng = np.random.default_rng(5)
    for i in range(3):
        for _ in range(3):
            d = rng.standard_normal(X[i].shape)
            h = 1e-5
            up, down = list(X), list(X)
            up[i], down[i] = X[i] + h * d, X[i] - h * d
            want = (loss(*up) - loss(*down)) / (2 * h)
            got = (f64(grads[i]) * d).sum()
            # differences: h^2 of the third derivative (~1e-9 relative) and 2^-52 / h of the loss; the kernel: n 2^-24 of the magnitudes
            assert abs(got - want) <= 1e-6 * abs(f64(grads[i]) * d).sum() + 1e-6


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_generation_with_window_prefix_and_eviction(dtype, pkg):
    """as they would be used: a prompt, then single tokens over its cache; the same cache split into a shared prefix and own parts;
    a cache cut by what the weights say, and attention over what is left"""
    B, T, Hq, Hkv, D = 2, 300, 8, 2, 64
    q, k, v = make((B, T, Hq, D), dtype, 1, 1.5), make((B, T, Hkv, D), dtype, 2), make((B, T, Hkv, D), dtype, 3)
    u = ref.half_step(dtype)
    # a token attends as the prompt's row did: both are within their bounds of the same value
    out, lse = pkg.attention_window(q, k, v, 64, sinks=4)
    want, wl, to, tl, _ = reference(q, k, v, None, None, 64, 4, D ** -0.5, dtype)
    close(out, want, to, "prompt")
    for t in (0, 63, 64, 150, 299):
        one, l1 = pkg.attention_window(q[:, t:t + 1], k, v, 64, sinks=4, kv_lens=torch.full((B,), t + 1, dtype=torch.int32, device="cuda"))
        close(one, want[:, t:t + 1], to[:, t:t + 1], "token %d" % t)
    # the first 100 rows shared: the same as a cache that holds them for every sequence
    kp, vp = k[0, :100], v[0, :100]
    kk = torch.cat([kp.expand(B, -1, -1, -1), k[:, 100:]], 1)
    vv = torch.cat([vp.expand(B, -1, -1, -1), v[:, 100:]], 1)
    a, la = pkg.attention_prefix(q[:, -1:], kp, vp, k[:, 100:], v[:, 100:])
    want, wl, to, tl, _ = reference(q[:, -1:], kk, vv, None, None, 1 << 40, 0, D ** -0.5, dtype)
    close(a, want, to, "prefix")
    close(la, wl, tl, "prefix lse")
    # weights of the prompt and of one token more, then half of the keys leave
    w = torch.zeros((B, Hkv, T), device="cuda")
    n1 = torch.full((B,), T - 1, dtype=torch.int32, device="cuda")
    pkg.attention_scored(q[:, :T - 1], k, v, w, kv_lens=n1)
    assert torch.allclose(w.sum(-1), torch.full((B, Hkv), (T - 1) * 4.0, device="cuda"), rtol=2 * T * ref.F32 + ref.EXP * 4)
    full, fl, _ = pkg.attention_scored(q[:, T - 1:], k, v, w)
    assert torch.allclose(w.sum(-1), torch.full((B, Hkv), T * 4.0, device="cuda"), rtol=2 * T * ref.F32 + ref.EXP * 4)
    nk, nv, nw, nl, kept = pkg.evict_cache(k, v, w, None, 150, sinks=4, recent=32)
    left, ll = pkg.attention_window(q[:, T - 1:], nk, nv, 150, kv_lens=nl)
    for b in range(B):
        for h in range(Hkv):
            at = kept[b, h].long()
            assert torch.equal(nk[b, :, h], k[b, at, h]) and torch.equal(nw[b, h], w[b, h, at])
    want, wl, to, tl, _ = reference(q[:, T - 1:], nk, nv, None, None, 1 << 40, 0, D ** -0.5, dtype)
    close(left, want, to, "behind the eviction")
    # what left had the lower weights: the log sum can only have gone down
    assert (ll <= fl + 1e-5).all()


def test_calls_follow_their_stream_and_replay_in_graphs(pkg):
    """two captured calls side by side, replayed with eager work between; new values in the same tensors are picked up"""
    q, k, v = make((2, 1, 8, 128), "bf16", 1), make((2, 3000, 2, 128), "bf16", 2), make((2, 3000, 2, 128), "bf16", 3)
    q2, k2, v2 = make((1, 200, 4, 64), "f32", 4), make((1, 200, 2, 64), "f32", 5), make((1, 200, 2, 64), "f32", 6)
    w = torch.zeros((2, 2, 3000), device="cuda")
    wo = torch.empty_like(w)
    kl = torch.tensor([3000, 1777], dtype=torch.int32, device="cuda")
    dout = make((1, 200, 4, 64), "f32", 7)

    def a():
        o = pkg.attention_window(q, k, v, 2048, sinks=4, kv_lens=kl) + pkg.attention_scored(q, k, v, w, kv_lens=kl, weights_out=wo)
        return o + pkg.attention_prefix(q, k[0], v[0], k[:, :100], v[:, :100]) + pkg.evict_cache(k, v, wo, kl, 1000, sinks=4, recent=100)

    def b():
        o, l = pkg.attention_window(q2, k2, v2, 50, sinks=3)
        return (o, l) + pkg.attention_window_backward(dout, q2, k2, v2, o, l, 50, sinks=3)
    a(), b()
    graphs, outs = [], []
    for f in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = f()
        graphs.append(g)
        outs.append(o)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for turn in range(4):
        q.copy_(make(q.shape, "bf16", 20 + turn))
        q2.copy_(make(q2.shape, "f32", 30 + turn))
        kl.copy_(torch.tensor([3000 - 7 * turn, 1000 + 300 * turn], dtype=torch.int32))
        torch.cuda.synchronize()
        for s, g in ((s1, graphs[0]), (s2, graphs[1])):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, f in zip(outs, (a, b)):
            for x, y in zip(o, f()):
                assert torch.equal(x, y), turn
    # eager calls on a stream of their own
    with torch.cuda.stream(s1):
        x = a()
    s1.synchronize()
    for m, n in zip(x, a()):
        assert torch.equal(m, n)
