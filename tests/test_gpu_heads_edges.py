"""GPU: the batched attention operators where they can go wrong: scales, groups, long walks, offsets, lengths, outputs of the caller's."""
import numpy as np
import pytest
import torch

import _heads_reference as ref
from test_gpu_heads import check_gradients, close, f64, lens, make, poison, reference

pytestmark = pytest.mark.gpu


def run_both(pkg, q, k, v, window, sinks, ql, kl, scale, dtype, layout="tokens"):
    """forward and backward against the formulas"""
    Dv = v.shape[3]
    kw = dict(sinks=sinks, q_lens=lens(ql), kv_lens=lens(kl), scale=scale)
    out, lse = pkg.attention_window(q, k, v, window, **kw)
    scale = q.shape[3] ** -0.5 if scale is None else scale
    want, wl, to, tl, _ = reference(q, k, v, ql, kl, window, sinks, scale, dtype)
    close(out, want, to, "out")
    close(lse, wl, tl, "lse")
    dout = make(q.shape[:3] + (Dv,), dtype, 9, 1.0, layout)
    grads = pkg.attention_window_backward(dout, q, k, v, out, lse, window, **kw)
    check_gradients(q, k, v, dout, *grads, ql, kl, window, sinks, dtype, scale)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1.5, 1e-30])
@pytest.mark.parametrize("Tq", [1, 90])
def test_scales(Tq, scale, dtype, pkg):
    B, Tk, Hq, Hkv, D = 2, 150, 4, 2, 64
    q, k, v = make((B, Tq, Hq, D), dtype, 1), make((B, Tk, Hkv, D), dtype, 2), make((B, Tk, Hkv, D), dtype, 3)
    run_both(pkg, q, k, v, 40, 3, None, [150, 99], scale, dtype)
    kp, vp = make((1, 70, Hkv, D), dtype, 4)[0], make((1, 70, Hkv, D), dtype, 5)[0]
    out, lse = pkg.attention_prefix(q, kp, vp, k, v, scale=scale)
    want, wl, to, tl, _ = reference(q, k, v, None, None, 1 << 40, 0, scale, dtype, prefix=(kp, vp))
    close(out, want, to, "prefix out")
    close(lse, wl, tl, "prefix lse")
    w = torch.zeros((B, Hkv, Tk), device="cuda")
    out, lse, _ = pkg.attention_scored(q, k, v, w, scale=scale)
    want, wl, to, tl, heads = reference(q, k, v, None, None, 1 << 40, 0, scale, dtype)
    close(out, want, to, "scored out")
    sums, tol = np.zeros(w.shape), np.zeros(w.shape)
    for (b, h), (nq, nk, p, o, err) in heads.items():
        sums[b, h // 2] += p.sum(0)
        tol[b, h // 2] += (p * (err[:, None] + 2 * nq * ref.F32)).sum(0)
    close(w, sums, tol + 2 * Hq * ref.F32 * sums + 1e-30, "weights")


@pytest.mark.parametrize("c", [
    # dtype, B, Tq, Tk, Hq, Hkv, Dk, Dv, window, sinks, q_lens, kv_lens, layout
    ("bf16", 1, 70, 90, 48, 1, 64, 64, 30, 2, None, None, "tokens"),          # two row blocks to a token
    ("f32", 1, 20, 20, 33, 1, 64, 64, 9, 1, None, None, "tokens"),
    ("bf16", 1, 11, 40, 65, 1, 40, 64, 9, 1, None, None, "tokens"),
    ("bf16", 2, 75, 75, 7, 1, 128, 128, 20, 2, [75, 33], [75, 60], "tokens"),  # groups that leave rows of a block over
    ("f32", 1, 75, 80, 10, 2, 96, 96, 20, 2, None, None, "heads"),
    ("bf16", 1, 61, 61, 24, 1, 128, 64, 20, 5, None, None, "heads"),
    ("bf16", 1, 1300, 1300, 2, 1, 64, 64, 100, 130, None, None, "tokens"),     # tails behind several blocks of sinks
    ("f32", 1, 900, 1000, 2, 1, 64, 64, 70, 70, [900], [950], "tokens"),
    ("bf16", 1, 1100, 1100, 1, 1, 128, 128, 2000, 4, None, None, "tokens"),    # every key by every later row
    ("bf16", 2, 500, 900, 2, 2, 256, 256, 200, 4, [500, 333], [900, 340], "tokens"),
    ("f32", 1, 400, 400, 2, 1, 256, 256, 60, 4, None, None, "tokens"),
    ("bf16", 1, 700, 700, 2, 1, 50, 50, 100, 70, None, None, "odd"),
    ("bf16", 1, 1, 9000, 4, 1, 64, 64, 1 << 20, 0, None, None, "tokens"),       # one row over many slots
    ("f32", 1, 1, 5000, 2, 1, 128, 128, 1 << 20, 0, None, [4097], "tokens"),
    ("bf16", 1, 3000, 20, 1, 1, 64, 64, 8, 2, None, None, "tokens"),            # most queries lie before the cache
], ids=str)
def test_groups_and_walks(c, pkg):
    dtype, B, Tq, Tk, Hq, Hkv, Dk, Dv, window, sinks, ql, kl, layout = c
    q = make((B, Tq, Hq, Dk), dtype, 1, 1.5, layout)
    k, v = make((B, Tk, Hkv, Dk), dtype, 2, 1.0, layout), make((B, Tk, Hkv, Dv), dtype, 3, 1.0, layout)
    run_both(pkg, q, k, v, window, sinks, ql, kl, None, dtype, layout)


def test_lengths_out_of_range_are_clamped(pkg):
    q, k, v = make((3, 40, 4, 64), "bf16", 1), make((3, 70, 2, 64), "bf16", 2), make((3, 70, 2, 64), "bf16", 3)
    wild = dict(q_lens=lens([-5, 1000, 2147483647]), kv_lens=lens([1 << 30, -2147483648, 71]))
    tame = dict(q_lens=lens([0, 40, 40]), kv_lens=lens([70, 0, 70]))
    a, b = pkg.attention_window(q, k, v, 20, **wild), pkg.attention_window(q, k, v, 20, **tame)
    dout = make((3, 40, 4, 64), "bf16", 4)
    a += pkg.attention_window_backward(dout, q, k, v, *a, 20, **wild)
    b += pkg.attention_window_backward(dout, q, k, v, *b, 20, **tame)
    w = torch.zeros((3, 2, 70), device="cuda")
    a += pkg.attention_scored(q, k, v, w.clone(), **wild) + pkg.evict_cache(k, v, w, wild["kv_lens"], 30)
    b += pkg.attention_scored(q, k, v, w.clone(), **tame) + pkg.evict_cache(k, v, w, tame["kv_lens"], 30)
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    assert not a[0][0].any() and not a[0][1].any() and a[1][:2].eq(-float("inf")).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_outputs_of_the_callers(dtype, pkg):
    """packed gradients, strided results: the same values, and nothing beside them is touched"""
    B, T, Hq, Hkv, D = 2, 100, 4, 2, 64
    q, k, v = make((B, T, Hq, D), dtype, 1), make((B, T, Hkv, D), dtype, 2), make((B, T, Hkv, D), dtype, 3)
    dout = make((B, T, Hq, D), dtype, 4)
    want = pkg.attention_window(q, k, v, 30, sinks=2)
    wantg = pkg.attention_window_backward(dout, q, k, v, *want, 30, sinks=2)
    for pad in (0, 1):                                    # (1: rows off their 16-byte alignment)
        big = torch.full((B, T + 1, Hq + 1, D + pad), 7.0, dtype=q.dtype, device="cuda")
        lse = torch.empty((B, Hq, T), device="cuda")
        o, l = pkg.attention_window(q, k, v, 30, sinks=2, out=big[:, 1:, 1:, pad:], lse=lse)
        assert l is lse and torch.equal(o, want[0]) and torch.equal(l, want[1])
        assert big[:, 0].eq(7).all() and big[:, :, 0].eq(7).all() and (pad == 0 or big[..., 0].eq(7).all())
        g = torch.full((B, T, Hq + 2 * Hkv + 1, D + pad), 7.0, dtype=q.dtype, device="cuda")
        parts = g[:, :, :Hq, pad:], g[:, :, Hq:Hq + Hkv, pad:], g[:, :, Hq + Hkv:-1, pad:]
        for x, y in zip(pkg.attention_window_backward(dout, q, k, v, *want, 30, sinks=2, dq=parts[0], dk=parts[1], dv=parts[2]), wantg):
            assert torch.equal(x, y)
        assert g[:, :, -1].eq(7).all() and (pad == 0 or g[..., 0].eq(7).all())


@pytest.mark.parametrize("T,budget", [(20001, 9000), (32768, 32767), (40001, 20000), (70000, 100)])
def test_evict_long_caches(T, budget, pkg):
    k, v = make((2, T, 1, 8), "bf16", 1), make((2, T, 1, 8), "bf16", 2)
    g = torch.Generator().manual_seed(3)
    w = torch.randint(0, 500, (2, 1, T), generator=g).float()
    nk, nv, nw, nl, kept = pkg.evict_cache(k, v, w.cuda(), lens([T, T - 1]), budget, sinks=4, recent=50)
    for b, n in enumerate((T, T - 1)):
        want = ref.kept(w[b, 0].tolist(), n, budget, 4, 50)
        assert kept[b, 0].tolist() == want
        assert torch.equal(nk[b, :, 0].cpu(), k[b, want, 0].cpu()) and torch.equal(nv[b, :, 0].cpu(), v[b, want, 0].cpu())


def far(shape, strides, dtype, seed):
    """a tensor with given strides inside a large allocation"""
    x = make(shape, dtype, seed)
    room = torch.empty(sum((n - 1) * s for n, s in zip(shape, strides)) + shape[-1], dtype=x.dtype, device="cuda")
    y = room.as_strided(shape, strides)
    y.copy_(x)
    return y


@pytest.mark.parametrize("strides", ["batch", "token", "head"])
@pytest.mark.parametrize("Tq", [1, 60])
def test_offsets_beyond_32_bits(Tq, strides, pkg):
    """more than 2^32 bytes between the parts of a cache and of the queries"""
    B, T, H, D, off = 2, 70, 2, 64, (1 << 31) + 1024
    kv, qs = {"batch": ((off, H * D, D, 1), (off, 2 * H * D, D, 1)), "head": ((T * D, D, off, 1), (T * D, D, off, 1)),
              "token": ((D, 1 << 26, 1 << 24, 1), (D, 1 << 27, 1 << 24, 1))}[strides]
    k, v, q = far((B, T, H, D), kv, "bf16", 1), far((B, T, H, D), kv, "bf16", 2), far((B, Tq, 2 * H, D), qs, "bf16", 3)
    run_both(pkg, q, k, v, 30, 2, None, None, None, "bf16")
    w = torch.rand((B, H, T), generator=torch.Generator().manual_seed(4)).cuda()
    want, wl, to, tl, heads = reference(q, k, v, None, None, 1 << 40, 0, D ** -0.5, "bf16")
    out, lse, sums = pkg.attention_scored(q, k, v, w, weights_out=torch.empty_like(w))
    close(out, want, to, "scored out")
    more, tol = f64(w), np.zeros(w.shape)
    for (b, h), (nq, nk, p, o, err) in heads.items():
        more[b, h // 2] += p.sum(0)
        tol[b, h // 2] += (p * (err[:, None] + 2 * nq * ref.F32)).sum(0)
    close(sums, more, tol + 4 * H * ref.F32 * more, "weights")
    out, lse = pkg.attention_prefix(q, k[0], v[0], k, v)
    want, wl, to, tl, _ = reference(q, k, v, None, None, 1 << 40, 0, D ** -0.5, "bf16", prefix=(k[0], v[0]))
    close(out, want, to, "prefix out")
    ko, vo = far((B, 30, H, D), kv, "bf16", 5), far((B, 30, H, D), kv, "bf16", 6)
    pkg.evict_cache(k, v, w, None, 30, k_out=ko, v_out=vo)
    for x, y in zip((ko, vo), pkg.evict_cache(k.contiguous(), v.contiguous(), w, None, 30)):
        assert torch.equal(x, y)


def test_the_end_of_a_cache_of_many_gigabytes(pkg):
    """four million tokens of 2 KB: the window and the sinks lie more than 2^32 bytes apart"""
    T, H, D, Tq, window, sinks = (1 << 22) + 3, 8, 128, 3, 200, 3
    k, v = (torch.zeros((1, T, H, D), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ks, vs = make((1, window + Tq + sinks, H, D), "bf16", 1), make((1, window + Tq + sinks, H, D), "bf16", 2)
    for x, y in ((k, ks), (v, vs)):
        x[:, :sinks] = y[:, :sinks]
        x[:, -(window + Tq):] = y[:, sinks:]
    q, dout = make((1, Tq, H, D), "bf16", 3), make((1, Tq, H, D), "bf16", 4)
    out, lse = pkg.attention_window(q, k, v, window, sinks=sinks)
    want, wl, to, tl, _ = reference(q, ks, vs, None, None, window, sinks, D ** -0.5, "bf16")
    close(out, want, to, "out")
    close(lse, wl, tl, "lse")
    dq, dk, dv = pkg.attention_window_backward(dout, q, k, v, out, lse, window, sinks=sinks)
    ends = [torch.cat([x[:, :sinks], x[:, -(window + Tq):]], 1) for x in (dk, dv)]
    check_gradients(q, ks, vs, dout, dq, *ends, None, None, window, sinks, "bf16")
    assert not dk[:, sinks:-(window + Tq)].any() and not dv[:, sinks:-(window + Tq)].any()


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("f32", 64), ("bf16", 40)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_values_a_row_does_not_see_in_long_walks(value, dtype, D, pkg):
    """as in a cache whose unused rows hold no numbers: among the sinks' neighbours, in the middle, behind the length"""
    T, window, sinks = 700, 100, 70
    q, k, v = make((1, T, 2, D), dtype, 1), make((1, T, 1, D), dtype, 2), make((1, T, 1, D), dtype, 3)
    dout = make((1, T, 2, D), dtype, 4)
    kw = dict(sinks=sinks)
    clean = pkg.attention_window(q, k, v, window, **kw)
    grads = pkg.attention_window_backward(dout, q, k, v, *clean, window, **kw)
    for at in (71, 300, 699):
        hit = torch.tensor(ref.visible(T, T, window, sinks)[:, at]).cuda()
        for K, V in ((poison(k, (0, at), value), v), (k, poison(v, (0, at), value))):
            out, lse = pkg.attention_window(q, K, V, window, **kw)
            dq, dk, dv = pkg.attention_window_backward(dout, q, K, V, out, lse, window, **kw)
            assert torch.equal(out[:, ~hit], clean[0][:, ~hit]) and torch.equal(lse[:, :, ~hit], clean[1][:, :, ~hit])
            assert torch.equal(dq[:, ~hit], grads[0][:, ~hit])


def test_two_streams_at_once(pkg):
    """eager calls side by side have scratch of their own"""
    shapes = [(1, 1, 5000), (2, 300, 300)]
    x = [(make((B, Tq, 4, 64), "bf16", i), make((B, Tk, 2, 64), "bf16", 10 + i), make((B, Tk, 2, 64), "bf16", 20 + i),
          make((B, Tq, 4, 64), "bf16", 30 + i)) for i, (B, Tq, Tk) in enumerate(shapes)]

    def f(q, k, v, d):
        o = pkg.attention_window(q, k, v, 4000, sinks=2)
        return o + pkg.attention_window_backward(d, q, k, v, *o, 4000, sinks=2) + pkg.attention_prefix(q, k[0], v[0], k, v)
    want = [f(*a) for a in x]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in x]
    got = [[] for _ in x]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(f(*x[i]))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        for o in g:
            for m, n in zip(w, o):
                assert torch.equal(m, n)


def test_more_rows_than_a_launch_has_workgroups_for_a_row_each(pkg):
    """2^24 rows and more: the last sequence is as right as a call of its own"""
    B, T, Hq, Hkv, D = 1050, 500, 32, 2, 16
    q, k, v = make((1, T, Hq, D), "bf16", 1, 1.5), make((1, T, Hkv, D), "bf16", 2), make((1, T, Hkv, D), "bf16", 3)
    dout = make((1, T, Hq, D), "bf16", 4)
    all_q, all_k, all_v = (x.expand(B, -1, -1, -1) for x in (q, k, v))
    out, lse = pkg.attention_window(all_q, all_k, all_v, 40, sinks=2)
    grads = pkg.attention_window_backward(dout.expand(B, -1, -1, -1), all_q, all_k, all_v, out, lse, 40, sinks=2)
    for x in (out, lse, *grads):
        assert torch.equal(x[0], x[-1]) and torch.equal(x[0], x[B // 2])
    want, wl, to, tl, _ = reference(q, k, v, None, None, 40, 2, D ** -0.5, "bf16")
    close(out[-1:], want, to, "out")
    close(lse[-1:], wl, tl, "lse")
    check_gradients(q, k, v, dout, *(x[-1:] for x in grads), None, None, 40, 2, "bf16")


@pytest.mark.parametrize("B,Tq,Tk", [(0, 3, 5), (2, 0, 5), (2, 3, 0), (2, 90, 0), (2, 0, 0)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_nothing_to_do(dtype, B, Tq, Tk, pkg):
    """no sequences, no queries, no keys: zeros, log sums of -inf, weights and caches as they were"""
    q, k, v = make((B, Tq, 4, 64), dtype, 1), make((B, Tk, 2, 64), dtype, 2), make((B, Tk, 2, 64), dtype, 3)
    kp, vp = make((1, 6, 2, 64), dtype, 4)[0], make((1, 6, 2, 64), dtype, 5)[0]
    w = torch.rand((B, 2, Tk), device="cuda")
    out, lse = pkg.attention_window(q, k, v, 4, sinks=1)
    grads = pkg.attention_window_backward(q.clone(), q, k, v, out, lse, 4, sinks=1)
    o2, l2, w2 = pkg.attention_scored(q, k, v, w, weights_out=torch.empty_like(w))
    if Tq == 0 or Tk == 0:
        assert torch.equal(w2, w) and not any(x.any() for x in (out, o2, *grads)) and lse.eq(-float("inf")).all() and l2.eq(-float("inf")).all()
    assert [tuple(x.shape) for x in grads] == [tuple(x.shape) for x in (q, k, v)]
    assert pkg.attention_prefix(q, kp, vp, k, v)[0].shape == q.shape
    nk, nv, nw, nl, kept = pkg.evict_cache(k, v, w, None, 3, sinks=1)
    assert nk.shape == (B, 3, 2, 64) and nl.eq(min(Tk, 3)).all() and (Tk or kept.eq(-1).all())


@pytest.mark.parametrize("Tq", [1, 100])
def test_sinks_beyond_the_cache_are_plain_causal_attention(Tq, pkg):
    q, k, v = make((2, Tq, 4, 64), "bf16", 1), make((2, 150, 2, 64), "bf16", 2), make((2, 150, 2, 64), "bf16", 3)
    run_both(pkg, q, k, v, 0, 1 << 40, None, [150, 60], None, "bf16")
    run_both(pkg, q, k, v, 1, 151, None, [150, 60], None, "bf16")


def test_a_long_selection_in_a_graph(pkg):
    k, v = make((2, 20001, 1, 8), "bf16", 1), make((2, 20001, 1, 8), "bf16", 2)
    w = torch.zeros((2, 1, 20001), device="cuda")
    pkg.evict_cache(k, v, w, None, 900)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = pkg.evict_cache(k, v, w, None, 900, sinks=3, recent=20)
    for turn in range(3):
        w.copy_(torch.rand(w.shape, generator=torch.Generator().manual_seed(turn)))
        g.replay()
        torch.cuda.synchronize()
        for x, y in zip(got, pkg.evict_cache(k, v, w, None, 900, sinks=3, recent=20)):
            assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("D", [64, 100, 128, 256])
@pytest.mark.parametrize("Tk,window", [(200, 60), (6000, 5000)])
def test_a_token_does_not_see_what_holds_no_numbers(Tk, window, D, dtype, pkg):
    """single tokens, one of whose tiles is masked and holds NaN or Inf in rows they do not see (the form of one workgroup, and the split one)"""
    q, k, v = make((2, 3, 4, D), dtype, 1), make((2, Tk, 2, D), dtype, 2), make((2, Tk, 2, D), dtype, 3)
    n = [Tk - 3, Tk - 40]
    kw = dict(sinks=2, kv_lens=lens(n))
    want = pkg.attention_window(q, k, v, window, **kw)
    ws = pkg.attention_scored(q, k, v, torch.zeros((2, 2, Tk), device="cuda"), kv_lens=lens(n))
    for value in (float("nan"), float("inf"), -float("inf")):
        K, V = k.clone(), v.clone()
        for b in range(2):
            for x in (K, V):
                x[b, n[b]:] = value
        got = pkg.attention_scored(q, K, V, torch.zeros((2, 2, Tk), device="cuda"), kv_lens=lens(n))
        assert all(torch.equal(x, y) for x, y in zip(got, ws))
        for b in range(2):                                # right before the window, behind the sinks
            for x in (K, V):
                x[b, 2:n[b] - 2 - window] = value
        got = pkg.attention_window(q, K, V, window, **kw)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("c", [
    # dtype, B, T, Hq, Hkv, D, window, sinks: several blocks of sinks, and so many groups that their tails have few or no workgroups of their own
    ("bf16", 20, 450, 8, 4, 64, 40, 300),
    ("f32", 17, 500, 4, 4, 64, 70, 200),
    ("bf16", 3, 900, 2, 2, 64, 30, 700),
    ("bf16", 70, 330, 8, 8, 64, 9, 4),
], ids=str)
def test_many_sinks_of_many_sequences(c, pkg):
    dtype, B, T, Hq, Hkv, D, window, sinks = c
    q, k, v = make((B, T, Hq, D), dtype, 1, 1.5), make((B, T, Hkv, D), dtype, 2), make((B, T, Hkv, D), dtype, 3)
    n = [T - (37 * b) % (T // 2) for b in range(B)]
    run_both(pkg, q, k, v, window, sinks, n, n, None, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("D", [64, 100, 128, 256])
@pytest.mark.parametrize("B,Tq,Tk,G", [(8, 40, 1200, 2), (9, 130, 1000, 1)])
def test_weights_of_chunks_of_many_sequences(B, Tq, Tk, G, D, dtype, pkg):
    """so many key heads that a workgroup of the weights' kernel takes 128 keys; lengths that end inside its tiles, one of no tokens"""
    H = 8
    q, k, v = make((B, Tq, H * G, D), dtype, 1, 1.5), make((B, Tk, H, D), dtype, 2), make((B, Tk, H, D), dtype, 3)
    ql, kl = [Tq - (11 * b) % Tq for b in range(B)], [Tk - (157 * b) % Tk for b in range(B)]
    ql[2] = kl[3] = 0
    w = torch.rand((B, H, Tk), generator=torch.Generator().manual_seed(4)).cuda()
    out, lse, got = pkg.attention_scored(q, k, v, w, q_lens=lens(ql), kv_lens=lens(kl), weights_out=torch.empty_like(w))
    want, wl, to, tl, heads = reference(q, k, v, ql, kl, 1 << 40, 0, D ** -0.5, dtype)
    close(out, want, to, "out")
    close(lse, wl, tl, "lse")
    sums, tol = f64(w), np.zeros(w.shape)
    for (b, h), (nq, nk, p, o, err) in heads.items():
        sums[b, h // G, :nk] += p.sum(0)
        tol[b, h // G, :nk] += (p * (err[:, None] + 2 * nq * ref.F32)).sum(0)
    close(got, sums, tol + 2 * H * G * ref.F32 * np.abs(sums) + 1e-30, "weights")
    again = pkg.attention_scored(q, k, v, w, q_lens=lens(ql), kv_lens=lens(kl))[2]
    assert again is w and torch.equal(w, got)
