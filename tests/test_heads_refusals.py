"""CPU: the batched attention operators refuse what they cannot do, before anything is enqueued, and there is no CPU fallback."""
import ctypes
import struct

import numpy as np
import pytest
import torch

import _heads_reference as ref


def qkv(B=2, Tq=3, Tk=5, Hq=4, Hkv=2, Dk=8, Dv=6, dtype=torch.float32):
    return torch.zeros(B, Tq, Hq, Dk, dtype=dtype), torch.zeros(B, Tk, Hkv, Dk, dtype=dtype), torch.zeros(B, Tk, Hkv, Dv, dtype=dtype)


@pytest.mark.parametrize("kw", [
    dict(q=torch.zeros(2, 3, 4)), dict(q=torch.zeros(2, 3, 3, 8)), dict(q=torch.zeros(2, 3, 4, 7)), dict(q=torch.zeros(1, 3, 4, 8)),
    dict(q=torch.zeros(2, 3, 4, 8, dtype=torch.float64)), dict(q=torch.zeros(2, 3, 4, 8, dtype=torch.bfloat16)),
    dict(q=torch.zeros(2, 3, 4, 16)[..., ::2]), dict(k=torch.zeros(2, 5, 2, 9)), dict(v=torch.zeros(2, 4, 2, 6)),
    dict(v=torch.zeros(2, 5, 1, 6)), dict(q=torch.zeros(2, 3, 4, 8).requires_grad_()), dict(window=-1), dict(window=1.5),
    dict(sinks=-1), dict(window=True), dict(q_lens=torch.zeros(2)), dict(q_lens=torch.zeros(3, dtype=torch.int32)),
    dict(kv_lens=torch.zeros(2, dtype=torch.int64)), dict(kv_lens=[5, 5]), dict(kv_lens=torch.zeros(4, dtype=torch.int32)[::2]),
    dict(out=torch.zeros(2, 3, 4, 8)), dict(lse=torch.zeros(2, 3, 4)), dict(q=torch.zeros(2, 3, 4, 300), k=torch.zeros(2, 5, 2, 300)),
], ids=lambda kw: "-".join("%s" % k for k in kw))
def test_window_refuses(kw, pkg):
    q, k, v = qkv()
    args = dict(q=q, k=k, v=v, window=4)
    args.update(kw)
    with pytest.raises(ValueError):
        pkg.attention_window(**args)


def test_outputs_over_inputs_are_refused(pkg):
    q, k, v = qkv(Dv=8)
    with pytest.raises(ValueError, match="overlaps"):
        pkg.attention_window(q, k, v, 4, out=q)
    with pytest.raises(ValueError, match="overlaps"):
        pkg.attention_window_backward(q, q, k, v, q.clone(), torch.zeros(2, 4, 3), 4, dk=k)
    w = torch.zeros(2, 2, 5)
    with pytest.raises(ValueError, match="overlaps"):
        pkg.evict_cache(k, v, w, None, 4, k_out=k)
    with pytest.raises(ValueError, match="overlaps"):
        pkg.evict_cache(k, v, w, None, 4, weights_out=w)


def test_one_tensor_for_two_outputs_is_refused(pkg):
    q, kv = torch.zeros(2, 3, 2, 8), torch.zeros(2, 3, 2, 8)
    o, lse, g = torch.zeros(2, 3, 2, 8), torch.zeros(2, 2, 3), torch.zeros(2, 3, 2, 8)
    w = torch.zeros(2, 2, 3)
    for kw in (dict(dq=g, dk=g), dict(dk=g, dv=g), dict(dq=g, dv=g)):
        with pytest.raises(ValueError, match="two outputs"):
            pkg.attention_window_backward(g.clone(), q, kv, kv, o, lse, 4, **kw)
    flat = torch.zeros(200)
    with pytest.raises(ValueError, match="two outputs"):
        pkg.attention_window(q, kv, kv, 4, out=flat[:96].view(2, 3, 2, 8), lse=flat[:12].view(2, 2, 3))
    with pytest.raises(ValueError, match="overlap"):
        pkg.attention_scored(q, kv, kv, w, weights_out=flat[:12].view(2, 2, 3), lse=flat[:12].view(2, 2, 3))
    with pytest.raises(ValueError, match="two outputs"):
        pkg.evict_cache(kv, kv, w, None, 2, k_out=g, v_out=g)
    with pytest.raises(ValueError, match="two outputs"):
        pkg.evict_cache(kv, kv, w, None, 2, v_out=flat[:96].view(2, 3, 2, 8), weights_out=flat[:12].view(2, 2, 3))


@pytest.mark.parametrize("kw", [dict(dout=torch.zeros(2, 3, 4, 8)), dict(out=torch.zeros(2, 3, 4, 6, dtype=torch.bfloat16)),
                                dict(lse=torch.zeros(2, 3, 4)), dict(dq=torch.zeros(2, 3, 4, 6)), dict(dv=torch.zeros(2, 5, 2, 8))],
                         ids=lambda kw: "-".join(kw))
def test_backward_refuses(kw, pkg):
    q, k, v = qkv()
    args = dict(dout=torch.zeros(2, 3, 4, 6), q=q, k=k, v=v, out=torch.zeros(2, 3, 4, 6), lse=torch.zeros(2, 4, 3), window=4)
    args.update(kw)
    with pytest.raises(ValueError):
        pkg.attention_window_backward(**args)


@pytest.mark.parametrize("kw", [dict(k_prefix=torch.zeros(7, 2, 6)), dict(v_prefix=torch.zeros(6, 2, 6)), dict(k_prefix=torch.zeros(1, 7, 2, 8)),
                                dict(v_prefix=torch.zeros(7, 1, 6))], ids=str)
def test_prefix_refuses(kw, pkg):
    q, k, v = qkv()
    args = dict(q=q, k_prefix=torch.zeros(7, 2, 8), v_prefix=torch.zeros(7, 2, 6), k=k, v=v)
    args.update(kw)
    with pytest.raises(ValueError):
        pkg.attention_prefix(**args)


@pytest.mark.parametrize("kw", [dict(weights=torch.zeros(2, 2, 4)), dict(weights=torch.zeros(2, 2, 5, dtype=torch.bfloat16)),
                                dict(weights=torch.zeros(1, 2, 5).expand(2, 2, 5)), dict(weights_out=torch.zeros(2, 4, 5))], ids=str)
def test_scored_refuses(kw, pkg):
    q, k, v = qkv()
    args = dict(q=q, k=k, v=v, weights=torch.zeros(2, 2, 5))
    args.update(kw)
    with pytest.raises(ValueError):
        pkg.attention_scored(**args)


@pytest.mark.parametrize("kw", [dict(budget=-1), dict(budget=3, sinks=2, recent=2), dict(lens=torch.zeros(2)), dict(lens=[5, 5]),
                                dict(weights=torch.zeros(2, 5, 2)), dict(k_out=torch.zeros(2, 3, 2, 8)), dict(v_out=torch.zeros(2, 4, 2, 8)),
                                dict(weights_out=torch.zeros(2, 2, 3)), dict(sinks=-1), dict(recent=-1)], ids=str)
def test_evict_refuses(kw, pkg):
    _, k, v = qkv()
    args = dict(k=k, v=v, weights=torch.zeros(2, 2, 5), lens=None, budget=4)
    args.update(kw)
    with pytest.raises(ValueError):
        pkg.evict_cache(**args)


def test_no_cpu_fallback(pkg):
    q, k, v = qkv()
    w = torch.zeros(2, 2, 5)
    for f in (lambda: pkg.attention_window(q, k, v, 4), lambda: pkg.attention_scored(q, k, v, w),
              lambda: pkg.attention_prefix(q, k[0], v[0], k, v), lambda: pkg.evict_cache(k, v, w, None, 4),
              lambda: pkg.attention_window_backward(torch.zeros(2, 3, 4, 6), q, k, v, torch.zeros(2, 3, 4, 6), torch.zeros(2, 4, 3), 4)):
        with pytest.raises(pkg.SdpaError) as e:
            f()
        assert e.value.code == pkg._lib.SDPA_ENODEV


# ---- the C entries: nothing but the checks runs here -----------------------------------------------------------------------------
def pack(**kw):
    """struct sdpa_heads of a small valid problem (pointers that are never followed), with fields replaced"""
    f = dict(size=None, q=(4096, 96, 32, 8), k=(4096, 80, 16, 8), v=(4096, 60, 12, 6), out=(4096, 72, 24, 6), kp=(0, 0, 0, 0), vp=(0, 0, 0, 0),
             dout=(4096, 72, 24, 6), dq=(4096, 96, 32, 8), dk_out=(4096, 80, 16, 8), dv_out=(4096, 60, 12, 6), lse=4096, q_lens=0, kv_lens=0,
             weights=4096, weights_out=4096, ws=(10, 5, 10, 5), k_out=(8192, 64, 16, 8), v_out=(8192, 48, 12, 6), lens_out=4096, kept=4096,
             dtype=0, batch=2, q_tokens=3, kv_tokens=5, q_heads=4, kv_heads=2, dk=8, dv=6, window=4, sinks=1, prefix=0, budget=4, recent=1,
             scale=0.5)
    f.update(kw)
    fmt = struct.Struct("=60q13if")
    return fmt.pack(fmt.size if f["size"] is None else f["size"], *f["q"], *f["k"], *f["v"], *f["out"], *f["kp"], *f["vp"], *f["dout"], *f["dq"],
                    *f["dk_out"], *f["dv_out"], f["lse"], f["q_lens"], f["kv_lens"], f["weights"], f["weights_out"], *f["ws"], *f["k_out"],
                    *f["v_out"], f["lens_out"], f["kept"], f["dtype"], f["batch"], f["q_tokens"], f["kv_tokens"], f["q_heads"], f["kv_heads"],
                    f["dk"], f["dv"], f["window"], f["sinks"], f["prefix"], f["budget"], f["recent"], f["scale"])


ENTRIES = ["sdpa_dev_attention_window", "sdpa_dev_attention_window_backward", "sdpa_dev_attention_prefix", "sdpa_dev_attention_scored",
           "sdpa_dev_evict_cache"]


@pytest.mark.parametrize("op", range(5))
@pytest.mark.parametrize("kw,code", [
    (dict(size=8), -1), (dict(dtype=2), -1), (dict(batch=-1), -1), (dict(kv_tokens=-1), -1), (dict(kv_heads=0), -1), (dict(dk=0), -1),
    (dict(dv=257), -6), (dict(dk=1000), -6), (dict(kv_tokens=(1 << 30) + 1), -6), (dict(sinks=-1), -1), (dict(k=(0, 80, 16, 8)), -1),
    (dict(k=(4096, 80, -16, 8)), -1)], ids=str)
def test_c_entries_refuse(op, kw, code, pkg):
    lib = pkg.load()
    assert getattr(lib, ENTRIES[op])(pack(**kw), 4096, 1 << 20, None) == code
    if "k" not in kw:
        assert lib.sdpa_dev_heads_workspace(op, pack(**kw)) == code


@pytest.mark.parametrize("op,kw,code", [
    (0, dict(q_heads=3), -1), (0, dict(window=-1), -1), (0, dict(lse=0), -1), (0, dict(out=(4096, 0, 24, 6)), -1), (0, dict(scale=float("nan")), -1),
    (0, dict(scale=float("inf")), -1), (3, dict(scale=float("-inf")), -1), (2, dict(prefix=4, kp=(4096, 0, 8, 8), vp=(4096, 0, 8, 6), q_tokens=1 << 22), -6),
    (0, dict(q_tokens=1 << 24), -6), (1, dict(batch=1 << 20, kv_tokens=64, sinks=4, q_tokens=200), -6), (1, dict(dq=(0, 96, 32, 8)), -1), (1, dict(dv_out=(4096, 60, 0, 6)), -1), (1, dict(dout=(0, 1, 1, 1)), -1), (2, dict(prefix=4), -1),
    (2, dict(prefix=-1), -1), (3, dict(weights=0), -1), (3, dict(ws=(10, 5, -1, 5)), -1), (3, dict(ws=(10, 5, 0, 5)), -1), (4, dict(ws=(10, 5, 10, 0)), -1), (4, dict(budget=1), -1), (4, dict(kept=0), -1),
    (4, dict(lens_out=0), -1), (4, dict(k_out=(4096, 64, 0, 8)), -1), (0, dict(batch=1 << 20, q_tokens=1 << 20), -6)], ids=str)
def test_c_entries_refuse_their_own(op, kw, code, pkg):
    assert getattr(pkg.load(), ENTRIES[op])(pack(**kw), 4096, 1 << 20, None) == code


def test_c_entries_refuse_null_and_too_little_scratch(pkg):
    lib = pkg.load()
    for op, name in enumerate(ENTRIES):
        assert getattr(lib, name)(None, None, 0, None) == -1
        assert lib.sdpa_dev_heads_workspace(op, None) == -1
    need = lib.sdpa_dev_heads_workspace(1, pack())
    assert need > 0
    assert lib.sdpa_dev_attention_window_backward(pack(), None, need, None) == -1
    assert lib.sdpa_dev_attention_window_backward(pack(), 4096, need - 1, None) == -1
    assert lib.sdpa_dev_attention_window_backward(pack(), 4100, need, None) == -1
    assert lib.sdpa_dev_heads_workspace(9, pack()) == -1


def test_the_reference_gradient_is_the_derivative():
    """the 64-bit formulas the GPU tests go by, against central differences"""
    rng = np.random.default_rng(3)
    q, k, v, g = (rng.standard_normal(s) for s in ((9, 5), (11, 5), (11, 4), (9, 4)))
    see, scale = ref.visible(9, 11, 4, 2), 0.4
    out, _, p, _, _, err = ref.attention(q, k, v, see, scale, "f32")
    grads = ref.gradients(q, k, v, g, p, out, err, scale, "f32")[:3]

    def loss(q, k, v):
        return (ref.attention(q, k, v, see, scale, "f32")[0] * g).sum()
    for i, x in enumerate((q, k, v)):
        d, h = rng.standard_normal(x.shape), 1e-6
        up, down = [q, k, v], [q, k, v]
        up[i], down[i] = x + h * d, x - h * d
        assert abs((loss(*up) - loss(*down)) / (2 * h) - (grads[i] * d).sum()) < 1e-7


@pytest.mark.parametrize("batch,tokens,window,sinks,heads,dk", [
    (1, 8192, 0, 8192, (32, 8), 128), (4, 32768, 0, 1 << 30, (32, 8), 128), (2, 8192, 128, 1024, (32, 8), 128), (64, 4096, 128, 4, (32, 8), 128),
    (2, 4096, 1024, 4, (16, 4), 128), (1, 500, 20, 500, (4, 1), 64), (1, 1 << 20, 512, 100, (8, 8), 256), (512, 300, 10, 70, (2, 2), 64)])
def test_the_backward_scratch_is_bounded_by_the_chip_and_the_gradients(batch, tokens, window, sinks, heads, dk, pkg):
    """two row statistics for every row, and slots of 64 keys: at most 1024 of them and 3/16 of the key blocks, however many keys are sinks"""
    hq, hkv = heads
    args = pack(batch=batch, q_tokens=tokens, kv_tokens=tokens, q_heads=hq, kv_heads=hkv, dk=dk, dv=dk, window=window, sinks=sinks, dtype=1)
    need = pkg.load().sdpa_dev_heads_workspace(1, args)
    stats = 2 * 4 * batch * hkv * (tokens * (hq // hkv) + 64)
    blocks = batch * hkv * ((tokens + 63) // 64)
    assert 0 < need <= stats + (1024 + 3 * blocks / 16) * 64 * 2 * dk * 4 + 16


def test_the_question_of_the_scratch_is_refused_as_the_call_is(pkg):
    """sizes beyond a launch are refused before anybody allocates the scratch for them; so is a call that there is none of"""
    lib = pkg.load()
    for kw in (dict(batch=1 << 20, kv_tokens=64, sinks=4, q_tokens=200), dict(batch=1 << 21, kv_tokens=256, sinks=0, q_tokens=1)):
        assert lib.sdpa_dev_heads_workspace(1, pack(**kw)) == lib.sdpa_dev_attention_window_backward(pack(**kw), 4096, 1 << 20, None) == -6
    for op in (-1, 5, 9):
        assert lib.sdpa_dev_heads_workspace(op, pack(batch=0)) == -1


def calls(pkg):
    """every tensor of every operator, read or written: (call, name, shape)"""
    q, k, v = qkv()
    o, lse, w, kp, vp = torch.zeros(2, 3, 4, 6), torch.zeros(2, 4, 3), torch.zeros(2, 2, 5), torch.zeros(7, 2, 8), torch.zeros(7, 2, 6)
    out = dict(out=torch.zeros(2, 3, 4, 6), lse=torch.zeros(2, 4, 3))
    sets = [
        (pkg.attention_window, dict(q=q, k=k, v=v, **out), dict(window=4)),
        (pkg.attention_window_backward, dict(dout=o, q=q, k=k, v=v, out=o.clone(), lse=lse, dq=q.clone(), dk=k.clone(), dv=v.clone()), dict(window=4)),
        (pkg.attention_prefix, dict(q=q, k_prefix=kp, v_prefix=vp, k=k, v=v, **out), {}),
        (pkg.attention_scored, dict(q=q, k=k, v=v, weights=w, weights_out=w.clone(), **out), {}),
        (pkg.evict_cache, dict(k=k, v=v, weights=w, k_out=k.clone(), v_out=v.clone(), weights_out=w.clone()), dict(lens=None, budget=4)),
    ]
    return [(f, tensors, other, name) for f, tensors, other in sets for name in tensors]


def test_no_tensor_that_requires_a_gradient_is_read_or_written(pkg):
    for f, tensors, other, name in calls(pkg):
        args = dict(tensors, **{name: tensors[name].clone().requires_grad_()})
        with pytest.raises(ValueError, match="%s requires a gradient" % name):
            f(**args, **other)
        with torch.no_grad(), pytest.raises(pkg.SdpaError):      # (allowed here: the call gets as far as the device)
            f(**args, **other)
    q, k, v = qkv()
    with pytest.raises(ValueError, match="weights requires"):     # (written in place)
        pkg.attention_scored(q, k, v, torch.zeros(2, 2, 5).requires_grad_())


def test_no_tensor_with_a_forward_mode_tangent(pkg):
    with torch.autograd.forward_ad.dual_level():
        for f, tensors, other, name in calls(pkg):
            dual = torch.autograd.forward_ad.make_dual(tensors[name], torch.ones_like(tensors[name]))
            with pytest.raises(ValueError, match="%s requires a gradient" % name):
                f(**dict(tensors, **{name: dual}), **other)
        f, tensors, other, _ = calls(pkg)[0]
        with pytest.raises(pkg.SdpaError):                        # (others are not refused)
            f(**tensors, **other)


def test_outputs_that_overlap_in_part_are_refused(pkg):
    q, kv = torch.zeros(2, 3, 2, 8), torch.zeros(2, 3, 2, 8)
    o, lse, w = torch.zeros(2, 3, 2, 8), torch.zeros(2, 2, 3), torch.zeros(2, 2, 3)
    packed = torch.zeros(2, 3, 6, 8)
    back = lambda **kw: pkg.attention_window_backward(o, q, kv, kv, o.clone(), lse, 4, **kw)
    for dk, dv in ((packed[:, :, 0:2], packed[:, :, 1:3]), (packed[:, :, 2:4], packed[:, :, 0:6:2][:, :, 1:]), (packed[:, :, 4:], packed[:, :, 3:5])):
        with pytest.raises(ValueError, match="two outputs overlap"):
            back(dk=dk, dv=dv)
    with pytest.raises(pkg.SdpaError):                    # (side by side, and every second head: they lie between each other)
        back(dq=packed[:, :, 4:], dk=packed[:, :, 0:4:2], dv=packed[:, :, 1:4:2])
    flat = torch.zeros(400)
    with pytest.raises(ValueError, match="repeats elements"):
        back(dk=flat.as_strided((2, 3, 2, 8), (48, 16, 4, 1)))
    with pytest.raises(ValueError, match="repeats elements"):
        pkg.attention_window(q, kv, kv, 4, out=flat.as_strided((2, 3, 2, 8), (40, 16, 8, 1)))
    with pytest.raises(ValueError, match="repeats elements"):
        pkg.attention_scored(q, kv, kv, flat.as_strided((2, 2, 3), (5, 2, 1)))
    with pytest.raises(ValueError, match="two outputs overlap"):
        pkg.evict_cache(kv, kv, w, None, 2, k_out=packed[:, :, :2], v_out=packed[:, 1:, 0:2])
    with pytest.raises(pkg.SdpaError):                    # (what lies behind the budget is not written)
        pkg.evict_cache(kv, kv, w, None, 1, k_out=packed[:, :, :2], v_out=packed[:, 1:, 0:2])
    with pytest.raises(pkg.SdpaError):                    # (an output between the parts of an input)
        pkg.attention_window(packed[:, :, 0:6:3], packed[:, :, 1:6:3], kv, 4, out=packed[:, :, 2:6:3])
    with pytest.raises(ValueError, match="overlaps an input"):
        pkg.attention_window(packed[:, :, 0:2], kv, kv, 4, out=packed[:, :, 1:3])


def test_the_overlap_of_strided_tensors_is_what_their_elements_say(pkg):
    """against the sets of their bytes"""
    from importlib import import_module
    heads = import_module(pkg.__name__ + ".heads")
    rng = np.random.default_rng(7)
    met = repeated = 0
    for turn in range(3000):
        room = torch.zeros(4000, dtype=torch.float32)
        views, bytes_of = [], []
        for _ in range(2):
            dtype = (torch.float32, torch.bfloat16)[rng.integers(2)]
            flat = room.view(dtype)
            shape = tuple(int(n) for n in rng.integers(1, 5, 4))
            if rng.random() < 0.5:                        # as a user's: a part of something larger, in some order
                base = flat[int(rng.integers(0, 40)):][:6 ** 4].view(6, 6, 6, 6).permute(*rng.permutation(4).tolist())
                x = base[tuple(slice(int(o), int(o) + n, int(rng.integers(1, 3))) for o, n in zip(rng.integers(0, 3, 4), shape))]
            else:
                x = flat.as_strided(shape, tuple(int(s) for s in rng.integers(0, 30, 4)), int(rng.integers(0, 60)))
            views.append(x)
            at = sum(np.arange(n).reshape([-1 if i == d else 1 for i in range(4)]) * s for d, (n, s) in enumerate(zip(x.shape, x.stride())))
            at = np.asarray(x.storage_offset() + at).ravel()
            bytes_of.append((at[:, None] * x.element_size() + np.arange(x.element_size())).ravel())
        x, y = views
        want = len(np.intersect1d(*bytes_of)) > 0
        xs, ys = heads._span(x), heads._span(y)
        assert heads._overlap(x, y, xs, ys) == want == heads._overlap(y, x, ys, xs)
        for z, b in zip(views, bytes_of):
            assert heads._repeats(z) == (len(np.unique(b)) < len(b))
            repeated += heads._repeats(z)
        met += want
    assert 300 < met < 2700 and 300 < repeated < 5000


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 3e38, -3e38, 1e39])
def test_scales_beyond_32_bits_are_refused(scale, pkg):
    q, k, v = qkv()
    for f in (lambda **kw: pkg.attention_window(q, k, v, 4, **kw), lambda **kw: pkg.attention_scored(q, k, v, torch.zeros(2, 2, 5), **kw),
              lambda **kw: pkg.attention_prefix(q, k[0], v[0], k, v, **kw),
              lambda **kw: pkg.attention_window_backward(torch.zeros(2, 3, 4, 6), q, k, v, torch.zeros(2, 3, 4, 6), torch.zeros(2, 4, 3), 4, **kw)):
        with pytest.raises(ValueError, match="scale"):
            f(scale=scale)
        with pytest.raises(pkg.SdpaError):
            f(scale=2.0 ** 127)
    if abs(scale) < 1e39 or scale != scale or scale in (float("inf"), -float("inf")):
        for op in range(4):
            assert getattr(pkg.load(), ENTRIES[op])(pack(scale=scale), 4096, 1 << 20, None) == -1


@pytest.mark.parametrize("kw", [dict(kv_lens=1 << 20, lens_out=1 << 20), dict(kv_lens=1 << 20, lens_out=(1 << 20) + 4), dict(kv_lens=(1 << 20) + 4, lens_out=1 << 20),
                                dict(weights=1 << 20, weights_out=1 << 20)], ids=str)
def test_an_eviction_over_its_own_lengths_or_weights_is_refused(kw, pkg):
    lib = pkg.load()
    far = dict(weights=1 << 16, weights_out=1 << 17)
    assert lib.sdpa_dev_heads_workspace(4, pack(**far, kv_lens=1 << 20, lens_out=(1 << 20) + 8)) == 0
    assert lib.sdpa_dev_heads_workspace(4, pack(**dict(far, **kw))) == -1 == lib.sdpa_dev_evict_cache(pack(**dict(far, **kw)), None, 0, None)


def test_outputs_over_the_lengths_are_refused(pkg):
    q, k, v = qkv(Dv=8)
    room = torch.zeros(96)
    n = room.view(torch.int32)[94:]
    for f in (lambda: pkg.attention_window(q[:, :1], k, v, 4, kv_lens=n, out=room[32:].view(2, 1, 4, 8)),
              lambda: pkg.attention_window(q, k, v, 4, q_lens=n, lse=room[72:].view(2, 4, 3)),
              lambda: pkg.attention_prefix(q, k[0], v[0], k, v, kv_lens=n, lse=room[72:].view(2, 4, 3)),
              lambda: pkg.attention_scored(q, k, v, torch.zeros(2, 2, 5), kv_lens=n, weights_out=room[76:].view(2, 2, 5)),
              lambda: pkg.evict_cache(k, v, torch.zeros(2, 2, 5), n, 4, weights_out=room[80:].view(2, 2, 4))):
        with pytest.raises(ValueError, match="overlaps an input"):
            f()
