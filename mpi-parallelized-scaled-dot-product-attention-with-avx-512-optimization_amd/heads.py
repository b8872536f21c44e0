"""Batched attention of grouped heads over a cache: the device-level operators of include/sdpa_hip.h (struct sdpa_heads) on torch
CUDA tensors.

    attention_window            causal, a sliding window plus the first `sinks` tokens; a prompt, a chunk or one new token
    attention_window_backward   its gradients
    attention_prefix            a batch whose sequences share the first rows of their caches
    attention_scored            causal, and every key's weight added to a running sum
    evict_cache                 keeps the keys of greatest accumulated weight and moves them together

Tensors are [batch, tokens, heads, dim] of float32 or bfloat16, any strides with contiguous dims (a head-major tensor is passed
transposed); q has G times as many heads as k and v, dims are 1 to 256.  `q_lens`, `kv_lens`: int32 [batch] on the device (None = all
tokens), clamped there to the tensors' token counts.  Query i < q_lens[b] is at position kv_lens[b] - q_lens[b] + i of its cache.  Rows
that see no key (and rows behind q_lens) get out 0, lse -inf and gradient 0; keys behind kv_lens get gradient 0.

All work is enqueued on torch's current stream of the tensors' device; scratch comes from torch's allocator, a piece of its own for
every call.  Nothing waits for the device, so every call can be captured into a graph.  The operators are not
recorded by autograd: a tensor that requires a gradient is refused while gradients are enabled, read or written (use `detach()` and
`attention_window_backward`), and so is one that carries a forward-mode tangent.  Tensors of the caller's that are written count as
modified in place: a graph that saved one notices.
"""
import math
import struct

import torch
from torch.autograd import forward_ad, graph

from . import _lib
from ._lib import SdpaError, check

HEAD_DIM_MAX = 256
_OP_WINDOW, _OP_WINDOW_BACKWARD, _OP_PREFIX, _OP_SCORED, _OP_EVICT = range(5)
_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
_INT_MAX = (1 << 31) - 1
_SCALE_MAX = 2.0 ** 127                    # (times log2(e) it is a 32-bit number still)
# struct sdpa_heads as bytes, a packer for each call: size, q k v out (16 words), prefix (8), gradients (16), lse and lengths (3),
# weights (6), k_out v_out (8), lens_out kept (2), then dtype and the seven sizes, window, sinks, prefix_tokens, budget, recent, scale.
# What a call has no use for is padding, which packs as zeros.
_SIZE = 8 * 60 + 14 * 4
_PACK_WINDOW = struct.Struct("=17q64x128x3q48x64x16x10i12xf")
_PACK_BACKWARD = struct.Struct("=17q64x16q3q48x64x16x10i12xf")
_PACK_PREFIX = struct.Struct("=17q8q128x3q48x64x16x8i8xi8xf")
_PACK_SCORED = struct.Struct("=17q64x128x3q6q64x16x8i20xf")
_PACK_EVICT = struct.Struct("=q32x8q32x64x128x16xq6q8q2q8i4xi4x2if")
# (the stream's number without a Stream object around it: a microsecond and a half of a call that takes ten)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def _at(x):
    return (x.data_ptr(),) + x.stride()[:3]


def _ptr(x):
    return 0 if x is None else x.data_ptr()


def _call(fn, name, op, x, args):
    """take the scratch and enqueue, on the device and current stream of tensor x"""
    i = x.get_device()
    if i != torch.cuda.current_device():
        with torch.cuda.device(i):
            return _call(fn, name, op, x, args)
    need = _lib.load().sdpa_dev_heads_workspace(op, args)
    ws = x.new_empty((need,), dtype=torch.uint8) if need > 0 else None          # (held until the work is enqueued)
    code = fn(args, None if ws is None else ws.data_ptr(), need, _raw_stream(i)) if need >= 0 else need
    if code:
        check(code, name)


def _need(ok, text):
    if not ok:
        raise ValueError(text)


def _rows(x, name, shape, dtype, device=None):
    _need(isinstance(x, torch.Tensor), "%s: expected a tensor" % name)
    _need(tuple(x.shape) == tuple(shape), "%s: expected shape %s, got %s" % (name, tuple(shape), tuple(x.shape)))
    _need(x.dtype == dtype, "%s: expected %s, got %s" % (name, dtype, x.dtype))
    _need(x.shape[-1] == 1 or x.stride(-1) == 1, "%s: the elements of a row must be contiguous" % name)
    _need(device is None or x.device == device, "%s: expected a tensor on %s, got %s" % (name, device, x.device))
    return x


def _span(x):
    n = x.numel()
    if n == 0:
        return 0, 0
    a = x.data_ptr()
    if not x.is_contiguous():
        n = sum((n - 1) * s for n, s in zip(x.shape, x.stride())) + 1
    return a, a + n * x.element_size()


def _box(x):
    """a tensor's bytes: (stride, count) of its dims from the largest stride on, the bytes of an element the last of them"""
    e = x.element_size()
    dims = sorted(((s * e, n) for s, n in zip(x.stride(), x.shape) if n > 1 and s > 0), reverse=True)
    if dims and dims[-1][0] == e:
        dims[-1] = (1, dims[-1][1] * e)                   # (a contiguous row)
    else:
        dims.append((1, e))
    return dims


def _reach(dims):
    return sum(s * (n - 1) for s, n in dims)


def _meet(d, a, b, left):
    """do two boxes share a byte, the second one `d` bytes behind the first?  Stride by stride, from the largest on: of its steps only those matter
    that bring what remains of the two within each other's reach, which are one or two where strides nest.  `left`: steps until
    the answer is "perhaps"."""
    left[0] -= 1
    if left[0] < 0:
        return True
    ra, rb = _reach(a), _reach(b)
    if d > ra or -d > rb:
        return False
    if not a and not b:
        return True
    s = max(a[0][0] if a else 0, b[0][0] if b else 0)
    lo = hi = 0                                           # steps of the first box less those of the second
    if a and a[0][0] == s:
        hi = a[0][1] - 1
        a = a[1:]
    if b and b[0][0] == s:
        lo = 1 - b[0][1]
        b = b[1:]
    ra, rb = _reach(a), _reach(b)
    return any(_meet(d - s * m, a, b, left) for m in range(max(lo, -((ra - d) // s)), min(hi, (rb + d) // s) + 1))


def _overlap(x, y, xs, ys):
    """(xs, ys: their spans)"""
    return xs[0] < ys[1] and ys[0] < xs[1] and _meet(ys[0] - xs[0], _box(x), _box(y), [4096])


def _repeats(x):
    """does a tensor hold an element twice?"""
    if x.numel() == 0 or x.is_contiguous():
        return False
    if any(n > 1 and s == 0 for n, s in zip(x.shape, x.stride())):
        return True
    dims = _box(x)
    while len(dims) > 1:
        (s, n), dims = dims[0], dims[1:]
        if any(_meet(s * m, dims, dims, [4096]) for m in range(1, min(n - 1, _reach(dims) // s) + 1)):
            return True
    return False


def _clear(outs, ins, name):
    """a caller's own output tensors hold no element twice and lie over no input and no other output (parts of one packed tensor may lie
    between each other)"""
    outs = [(x, _span(x)) for x in outs if x is not None]
    if not outs:
        return
    ins = [(x, _span(x)) for x in ins if x is not None]
    for i, (x, xs) in enumerate(outs):
        _need(not _repeats(x), "%s: an output repeats elements" % name)
        for y, ys in ins:
            _need(not _overlap(x, y, xs, ys), "%s: an output overlaps an input" % name)
        for y, ys in outs[:i]:
            _need(not _overlap(x, y, xs, ys), "%s: two outputs overlap" % name)


def _lens(x, name, batch, like):
    """lengths (None = all); accepted at once where all is well, as in the other checks a small call meets"""
    if x is None or (type(x) is torch.Tensor and x.dtype is torch.int32 and x.shape == (batch,) and x.device == like.device and
                     x.is_contiguous()):
        return
    _rows(x, name, (batch,), torch.int32, like.device)
    _need(x.is_contiguous(), "%s: must be contiguous" % name)


def _count(x, name):
    if type(x) is not int or x < 0:
        _need(isinstance(x, int) and not isinstance(x, bool) and x >= 0, "%s: expected an integer >= 0" % name)
    return x if x < _INT_MAX else _INT_MAX


def _recorded(x):
    """would autograd record what is done with x?  (the level: no forward-mode derivative is being taken anywhere)"""
    return (x.requires_grad and torch.is_grad_enabled()) or (forward_ad._current_level >= 0 and forward_ad.unpack_dual(x).tangent is not None)


def _unrecorded(x, name, call):
    if x is not None and _recorded(x):
        raise ValueError("%s requires a gradient: %s is not recorded by autograd, pass %s.detach()" % (name, call, name))


def _written(*given):
    """the caller's own tensors that a call wrote"""
    given = [x for x in given if x is not None]
    if given:
        graph.increment_version(given)


def _fits(x, shape, like):
    """an operand as it should be: shape, type, device, contiguous rows"""
    return (type(x) is torch.Tensor and x.shape == shape and x.dtype is like.dtype and x.device == like.device and
            (x.stride(-1) == 1 or shape[-1] == 1))


def _operand(x, name, shape, like, call):
    if not _fits(x, shape, like):
        _rows(x, name, shape, like.dtype, like.device)
    _unrecorded(x, name, call)


def _qkv(q, k, v, name):
    """the shapes every attention shares -> (B, Tq, Tk, Hq, Hkv, Dk, Dv)"""
    for x, n in ((q, "q"), (k, "k"), (v, "v")):
        if not isinstance(x, torch.Tensor) or x.dim() != 4:
            raise ValueError("%s: expected [batch, tokens, heads, dim]" % n)
    B, Tq, Hq, Dk = q.shape
    Tk, Hkv, Dv = k.shape[1], k.shape[2], v.shape[3]
    if q.dtype not in _DTYPES:
        raise ValueError("q: expected float32 or bfloat16, got %s" % q.dtype)
    if not (1 <= Dk <= HEAD_DIM_MAX and 1 <= Dv <= HEAD_DIM_MAX):
        raise ValueError("head dims must be 1 to %d" % HEAD_DIM_MAX)
    if Hkv < 1 or Hq < 1 or Hq % Hkv:
        raise ValueError("q's heads (%d) must be a multiple of k's (%d)" % (Hq, Hkv))
    _operand(q, "q", (B, Tq, Hq, Dk), q, name)
    _operand(k, "k", (B, Tk, Hkv, Dk), q, name)
    _operand(v, "v", (B, Tk, Hkv, Dv), q, name)
    return B, Tq, Tk, Hq, Hkv, Dk, Dv


def _scale(scale, dk):
    if scale is None:
        return 1.0 / math.sqrt(dk)
    scale = float(scale)
    _need(abs(scale) <= _SCALE_MAX, "scale: expected a number of at most %.4g in size, got %r" % (_SCALE_MAX, scale))
    return scale


def _on_gpu(x, name):
    if not x.is_cuda:
        raise SdpaError(_lib.SDPA_ENODEV, name)


def _outputs(q, Dv, out, lse, ins, name):
    B, Tq, Hq = q.shape[:3]
    if out is not None:
        _rows(out, "out", (B, Tq, Hq, Dv), q.dtype, q.device)
        _unrecorded(out, "out", name)
    if lse is not None:
        _rows(lse, "lse", (B, Hq, Tq), torch.float32, q.device)
        _unrecorded(lse, "lse", name)
        _need(lse.is_contiguous(), "lse: must be contiguous")
    _clear((out, lse), ins, name)
    _on_gpu(q, name)
    if out is None:
        out = q.new_empty((B, Tq, Hq, Dv))
    if lse is None:
        lse = q.new_empty((B, Hq, Tq), dtype=torch.float32)
    return out, lse


def attention_window(q, k, v, window, sinks=0, q_lens=None, kv_lens=None, scale=None, out=None, lse=None):
    """Causal attention over the last `window` tokens (the query's own included) plus the first `sinks` tokens of the cache.
    -> (out [B, Tq, Hq, Dv], lse [B, Hq, Tq]); window >= Tk is plain causal attention.  `out`, `lse`: tensors to write into."""
    name = "attention_window"
    B, Tq, Tk, Hq, Hkv, Dk, Dv = _qkv(q, k, v, name)
    scale = _scale(scale, Dk)
    window, sinks = _count(window, "window"), _count(sinks, "sinks")
    _lens(q_lens, "q_lens", B, q)
    _lens(kv_lens, "kv_lens", B, q)
    given = out, lse
    out, lse = _outputs(q, Dv, out, lse, (q, k, v, q_lens, kv_lens), name)
    args = _PACK_WINDOW.pack(_SIZE, *_at(q), *_at(k), *_at(v), *_at(out), lse.data_ptr(), _ptr(q_lens), _ptr(kv_lens), _DTYPES[q.dtype], B, Tq, Tk,
                             Hq, Hkv, Dk, Dv, window, sinks, scale)
    _call(_lib.load().sdpa_dev_attention_window, name, _OP_WINDOW, q, args)
    _written(*given)
    return out, lse


def attention_window_backward(dout, q, k, v, out, lse, window, sinks=0, q_lens=None, kv_lens=None, scale=None, dq=None, dk=None,
                              dv=None):
    """The gradients of attention_window from what it was given, what it returned and the gradient of `out`.
    -> (dq, dk, dv), shaped and typed like q, k, v.  Deterministic.  `dq`, `dk`, `dv`: tensors to write into."""
    name = "attention_window_backward"
    B, Tq, Tk, Hq, Hkv, Dk, Dv = _qkv(q, k, v, name)
    scale = _scale(scale, Dk)
    window, sinks = _count(window, "window"), _count(sinks, "sinks")
    _lens(q_lens, "q_lens", B, q)
    _lens(kv_lens, "kv_lens", B, q)
    _operand(dout, "dout", (B, Tq, Hq, Dv), q, name)
    _operand(out, "out", (B, Tq, Hq, Dv), q, name)
    _rows(lse, "lse", (B, Hq, Tq), torch.float32, q.device)
    _need(lse.is_contiguous(), "lse: must be contiguous")
    _unrecorded(lse, "lse", name)
    ins = (dout, q, k, v, out, lse, q_lens, kv_lens)
    for x, n, like in ((dq, "dq", q), (dk, "dk", k), (dv, "dv", v)):
        if x is not None:
            _rows(x, n, like.shape, q.dtype, q.device)
            _unrecorded(x, n, name)
    given = dq, dk, dv
    _clear(given, ins, name)
    _on_gpu(q, name)
    dq = q.new_empty(q.shape) if dq is None else dq
    dk = q.new_empty(k.shape) if dk is None else dk
    dv = q.new_empty(v.shape) if dv is None else dv
    args = _PACK_BACKWARD.pack(_SIZE, *_at(q), *_at(k), *_at(v), *_at(out), *_at(dout), *_at(dq), *_at(dk), *_at(dv), lse.data_ptr(), _ptr(q_lens),
                               _ptr(kv_lens), _DTYPES[q.dtype], B, Tq, Tk, Hq, Hkv, Dk, Dv, window, sinks, scale)
    _call(_lib.load().sdpa_dev_attention_window_backward, name, _OP_WINDOW_BACKWARD, q, args)
    _written(*given)
    return dq, dk, dv


def attention_prefix(q, k_prefix, v_prefix, k, v, q_lens=None, kv_lens=None, scale=None, out=None, lse=None):
    """Attention of a batch whose sequences all begin with the cache rows k_prefix [P, Hkv, Dk], v_prefix [P, Hkv, Dv]: every query
    sees the whole prefix and, causally, its own sequence's k, v (lengths count that own part only).  The prefix is read once for
    the batch.  -> (out, lse) over both parts."""
    name = "attention_prefix"
    B, Tq, Tk, Hq, Hkv, Dk, Dv = _qkv(q, k, v, name)
    scale = _scale(scale, Dk)
    for x, n in ((k_prefix, "k_prefix"), (v_prefix, "v_prefix")):
        _need(isinstance(x, torch.Tensor) and x.dim() == 3, "%s: expected [tokens, heads, dim]" % n)
    P = k_prefix.shape[0]
    _operand(k_prefix, "k_prefix", (P, Hkv, Dk), q, name)
    _operand(v_prefix, "v_prefix", (P, Hkv, Dv), q, name)
    _lens(q_lens, "q_lens", B, q)
    _lens(kv_lens, "kv_lens", B, q)
    given = out, lse
    out, lse = _outputs(q, Dv, out, lse, (q, k, v, k_prefix, v_prefix, q_lens, kv_lens), name)
    args = _PACK_PREFIX.pack(_SIZE, *_at(q), *_at(k), *_at(v), *_at(out), k_prefix.data_ptr(), 0, *k_prefix.stride()[:2], v_prefix.data_ptr(), 0,
                             *v_prefix.stride()[:2], lse.data_ptr(), _ptr(q_lens), _ptr(kv_lens), _DTYPES[q.dtype], B, Tq, Tk, Hq, Hkv, Dk, Dv,
                             P, scale)
    _call(_lib.load().sdpa_dev_attention_prefix, name, _OP_PREFIX, q, args)
    _written(*given)
    return out, lse


def _weights(x, name, shape, like, call, written=False):
    """[batch, heads, tokens] float32; one that is written must not repeat elements"""
    if not (type(x) is torch.Tensor and x.shape == shape and x.dtype is torch.float32 and x.device == like.device and x.is_contiguous()):
        _rows(x, name, shape, torch.float32, like.device)
        _need(not written or not _repeats(x), "%s: repeats elements" % name)
    _unrecorded(x, name, call)


def _sums(weights, weights_out):
    return (weights.data_ptr(), weights_out.data_ptr()) + weights.stride()[:2] + weights_out.stride()[:2]


def attention_scored(q, k, v, weights, q_lens=None, kv_lens=None, scale=None, weights_out=None, out=None, lse=None):
    """Causal attention over the whole cache that keeps account of it: weights [B, Hkv, Tk] float32 is increased, in place or into
    `weights_out`, by the softmax weight every key was given, summed over its group's heads and the queries.
    -> (out, lse, the increased weights).  evict_cache() goes by these sums."""
    name = "attention_scored"
    B, Tq, Tk, Hq, Hkv, Dk, Dv = _qkv(q, k, v, name)
    scale = _scale(scale, Dk)
    _weights(weights, "weights", (B, Hkv, Tk), q, name, weights_out is None)
    _lens(q_lens, "q_lens", B, q)
    _lens(kv_lens, "kv_lens", B, q)
    if weights_out is None:
        weights_out = weights
    elif weights_out is not weights:
        _weights(weights_out, "weights_out", (B, Hkv, Tk), q, name, True)
        _clear((weights_out,), (q, k, v, weights, q_lens, kv_lens), name)
    given = out, lse, weights_out
    out, lse = _outputs(q, Dv, out, lse, (q, k, v, weights, weights_out, q_lens, kv_lens), name)
    args = _PACK_SCORED.pack(_SIZE, *_at(q), *_at(k), *_at(v), *_at(out), lse.data_ptr(), _ptr(q_lens), _ptr(kv_lens), *_sums(weights, weights_out),
                             _DTYPES[q.dtype], B, Tq, Tk, Hq, Hkv, Dk, Dv, scale)
    _call(_lib.load().sdpa_dev_attention_scored, name, _OP_SCORED, q, args)
    _written(*given)
    return out, lse, weights_out


def evict_cache(k, v, weights, lens, budget, sinks=0, recent=0, k_out=None, v_out=None, weights_out=None):
    """Cuts the cache of every sequence and key head to `budget` keys: those of the first `sinks`, of the last `recent` and, between
    them, of the greatest accumulated weight (ties: the lower index; NaN counts below everything), in their order.  A sequence of
    at most `budget` keys keeps all of them.
    -> (k, v [B, budget, Hkv, dim], weights [B, Hkv, budget], lens [B], kept [B, Hkv, budget] = the old indices, -1 behind the end).
    Slots behind the new length are zero.  `k_out`, `v_out`, `weights_out`: tensors of their own to write into, with at least
    `budget` tokens; what lies behind `budget` in them is left as it was."""
    name = "evict_cache"
    for x, n in ((k, "k"), (v, "v")):
        _need(isinstance(x, torch.Tensor) and x.dim() == 4, "%s: expected [batch, tokens, heads, dim]" % n)
    _need(k.dtype in _DTYPES, "k: expected float32 or bfloat16, got %s" % k.dtype)
    B, T, H, Dk = k.shape
    Dv = v.shape[3]
    _need(1 <= Dk <= HEAD_DIM_MAX and 1 <= Dv <= HEAD_DIM_MAX and H > 0, "head dims must be 1 to %d" % HEAD_DIM_MAX)
    _operand(k, "k", (B, T, H, Dk), k, name)
    _operand(v, "v", (B, T, H, Dv), k, name)
    _weights(weights, "weights", (B, H, T), k, name)
    _lens(lens, "lens", B, k)
    budget, sinks, recent = _count(budget, "budget"), _count(sinks, "sinks"), _count(recent, "recent")
    _need(sinks + recent <= budget, "sinks + recent must not exceed the budget")
    for x, n, dim in ((k_out, "k_out", Dk), (v_out, "v_out", Dv)):
        if x is not None:
            _need(isinstance(x, torch.Tensor) and x.dim() == 4 and x.shape[1] >= budget, "%s: needs %d tokens" % (n, budget))
            _rows(x, n, (B, x.shape[1], H, dim), k.dtype, k.device)
            _unrecorded(x, n, name)
    if weights_out is not None:
        _need(isinstance(weights_out, torch.Tensor) and weights_out.dim() == 3 and weights_out.shape[2] >= budget,
              "weights_out: needs %d tokens" % budget)
        _weights(weights_out, "weights_out", (B, H, weights_out.shape[2]), k, name, True)
    given = k_out, v_out, weights_out
    _clear([x if x is None else x.narrow(d, 0, budget) for x, d in zip(given, (1, 1, 2))], (k, v, weights, lens), name)     # (what is written of them)
    _on_gpu(k, name)
    k_out = k.new_empty((B, budget, H, Dk)) if k_out is None else k_out
    v_out = k.new_empty((B, budget, H, Dv)) if v_out is None else v_out
    weights_out = k.new_empty((B, H, budget), dtype=torch.float32) if weights_out is None else weights_out
    lens_out = k.new_empty((B,), dtype=torch.int32)
    kept = k.new_empty((B, H, budget), dtype=torch.int32)
    args = _PACK_EVICT.pack(_SIZE, *_at(k), *_at(v), _ptr(lens), *_sums(weights, weights_out), *_at(k_out), *_at(v_out), lens_out.data_ptr(),
                            kept.data_ptr(), _DTYPES[k.dtype], B, 0, T, H, H, Dk, Dv, sinks, budget, recent, 1.0)
    _call(_lib.load().sdpa_dev_evict_cache, name, _OP_EVICT, k, args)
    _written(*given)
    return k_out, v_out, weights_out, lens_out, kept
