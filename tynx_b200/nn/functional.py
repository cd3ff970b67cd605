"""Loss functions and layers on CUDA (``tynx.nn.functional``).

``cross_entropy`` keeps the reference's contract
(``crates/tynx-python/python/tynx/nn/functional.py:133-145``: rank-2 float32 logits,
rank-1 int64 targets, ``-mean(log_softmax(z)[y])``) but runs as one fused
softmax-cross-entropy kernel forward and one backward kernel instead of the five
taped operations.  ``mse_loss`` follows ``loss.rs:10-23`` / ``functional.py:126-130``.
"""

from __future__ import annotations

import ctypes as C
import math
from typing import Optional

from .. import _native as N
from .._core import Fn, Storage, Tensor, _needs_grad, full, maximum
from .._native import lib
from .rotary import Rotary


def cross_entropy(input: Tensor, target: Tensor, reduction: str = "mean") -> Tensor:
    """Cross entropy for rank-2 logits and rank-1 int64 class targets."""
    if input.dtype != "float32" or input.ndim != 2:
        raise ValueError(
            f"cross_entropy input must be rank-2 float32 logits, got {input.dtype} {input.shape}"
        )
    if target.dtype != "int64" or target.shape != (input.shape[0],):
        raise ValueError(
            "cross_entropy target must be a rank-1 int64 Tensor with one class index per row, "
            f"got {target.dtype} {target.shape}"
        )
    if reduction != "mean":
        selected = input.log_softmax(1).gather(1, target.unsqueeze(1)).squeeze(1)
        return -selected if reduction == "none" else (-selected).sum()
    rows, cols = input.shape
    ctx = input.ctx
    loss = Tensor._empty((1,), "float32", ctx)
    ctx.check(lib.tx_softmax_xent_fwd(ctx.handle, input.ptr, target.ptr, rows, cols, loss.ptr),
              "cross_entropy")
    if _needs_grad(input):
        logits, labels = input.detach(), target.detach()

        def backward(g):
            dz = Tensor._empty((rows, cols), "float32", ctx)
            ctx.check(lib.tx_softmax_xent_bwd(ctx.handle, logits.ptr, labels.ptr, rows, cols,
                                              g[0].ptr, dz.ptr, 0), "cross_entropy backward")
            return [dz]

        loss._attach(Fn("cross_entropy", [input], backward))
    return loss


def mse_loss(input: Tensor, target: Tensor, reduction: str = "mean") -> Tensor:
    """Elementwise, mean, or summed squared error for exactly matching shapes."""
    if input.shape != target.shape:
        raise ValueError(
            f"mse_loss requires exactly matching shapes, got {input.shape} and {target.shape}"
        )
    error = input - target
    squared = error * error
    if reduction == "none":
        return squared
    if reduction == "mean":
        return squared.mean()
    if reduction == "sum":
        return squared.sum()
    raise ValueError(f"reduction must be 'none', 'mean', or 'sum', got {reduction!r}")


def ppo_loss(logits: Tensor, values: Tensor, actions: Tensor, old_log_prob: Tensor, advantages: Tensor,
             returns: Tensor, *, clip: float = 0.2, value_coef: float = 0.5,
             entropy_coef: float = 0.01) -> Tensor:
    """The clipped-surrogate PPO objective as one fused kernel forward and one
    backward: ``-mean(min(r*A, clamp(r, 1-clip, 1+clip)*A)) + value_coef *
    mse(values, returns) - entropy_coef * mean(entropy)`` with ``r =
    exp(log_softmax(logits)[actions] - old_log_prob)``.  The same value, and
    the same gradients for ``logits`` and ``values``, as that objective
    composed from ``distributions.Categorical``, ``minimum``, ``clamp`` and
    ``mse_loss`` (the reference's ``crates/tynx-python/tests/test_ppo.py:53-64``),
    without its twenty intermediate tensors.  ``values`` is [rows] or
    [rows, 1]; the other per-row inputs are [rows]."""
    if logits.dtype != "float32" or logits.ndim != 2:
        raise ValueError(f"ppo_loss logits must be rank-2 float32, got {logits.dtype} {logits.shape}")
    rows, cols = logits.shape
    if values.shape not in ((rows,), (rows, 1)):
        raise ValueError(f"ppo_loss values must be [rows] or [rows, 1], got {values.shape}")
    if actions.dtype != "int64" or actions.shape != (rows,):
        raise ValueError(f"ppo_loss actions must be a rank-1 int64 Tensor of {rows} rows")
    for name, t in (("old_log_prob", old_log_prob), ("advantages", advantages), ("returns", returns)):
        if t.dtype != "float32" or t.shape != (rows,):
            raise ValueError(f"ppo_loss {name} must be a rank-1 float32 Tensor of {rows} rows")
    ctx = logits.ctx
    scalars = (C.c_float(clip), C.c_float(value_coef), C.c_float(entropy_coef))

    def inputs(z, v, a, o, adv, ret):
        return (z.ptr, rows, cols, v.ptr, a.ptr, o.ptr, adv.ptr, ret.ptr) + scalars

    loss = Tensor._empty((1,), "float32", ctx)
    ctx.check(lib.tx_ppo_loss_fwd(ctx.handle, *inputs(logits, values, actions, old_log_prob, advantages,
                                                      returns), loss.ptr), "ppo_loss")
    if _needs_grad(logits, values):
        # detached views keep the inputs' storage alive until this node is freed
        saved = tuple(t.detach() for t in (logits, values, actions, old_log_prob, advantages, returns))
        want_v = values.requires_grad

        def backward(g):
            dz = Tensor._empty((rows, cols), "float32", ctx)
            dv = Tensor._empty(values.shape, "float32", ctx) if want_v else None
            ctx.check(lib.tx_ppo_loss_bwd(ctx.handle, *inputs(*saved), g[0].ptr, dz.ptr,
                                          dv.ptr if dv is not None else None, 0, 0), "ppo_loss backward")
            return [dz, dv]

        loss._attach(Fn("ppo_loss", [logits, values], backward))
    return loss


def _heads(name: str, what: str, t: Tensor, ctx, heads: str = "heads") -> tuple:
    shape = t.shape
    if t.dtype != "float32" or len(shape) != 4:
        raise ValueError(f"{name} {what} must be rank-4 float32 [batch, tokens, {heads}, head_dim], got "
                         f"{t.dtype} {shape}")
    _same_device(name, what, t, ctx)
    return shape


def _same_device(name: str, what: str, t: Tensor, ctx) -> None:
    if t.ctx is not ctx:
        raise ValueError(f"{name} {what} is on cuda:{t.ctx.index}, the other tensors are on cuda:{ctx.index}")


def _rotary_positions(name: str, rotary: Rotary, positions, shape: tuple, ctx) -> tuple:
    """(pointer, sequence stride) of the positions of the tokens of a tensor of this shape."""
    batch, seq, _, dim = shape
    if not isinstance(rotary, Rotary):
        raise TypeError(f"{name} rotary must be a Rotary, got {type(rotary).__qualname__}")
    if not 1 <= dim <= 2 * N.ROTARY_PAIRS:
        raise NotImplementedError(f"{name} supports head dimensions 1..{2 * N.ROTARY_PAIRS}, got {dim}")
    if rotary.dim > dim:
        raise ValueError(f"{name}: the rotary dim {rotary.dim} exceeds the head dimension {dim}")
    if positions is None:
        return None, 0
    if positions.dtype != "int64" or positions.shape not in ((seq,), (batch, seq)):
        raise ValueError(f"{name} positions must be int64 [{seq}] or [{batch}, {seq}], got "
                         f"{positions.dtype} {positions.shape}")
    _same_device(name, "positions", positions, ctx)
    return positions.ptr, seq if len(positions.shape) == 2 else 0


def rotary_embedding(input: Tensor, rotary: Rotary, positions: Optional[Tensor] = None) -> Tensor:
    """Rotate the pairs of every head of ``input [batch, tokens, heads, head_dim]``
    by the tokens' positions (:class:`~tynx_b200.nn.Rotary`); elements behind
    ``rotary.dim`` pass through.  ``positions`` is int64 [tokens] or
    [batch, tokens]; None counts every sequence from 0."""
    name, ctx = "rotary_embedding", input.ctx
    shape = batch, seq, heads, dim = _heads(name, "input", input, ctx)
    pos, stride = _rotary_positions(name, rotary, positions, shape, ctx)
    desc = rotary._desc
    out = Tensor._new(shape, ctx)
    ctx.check(lib.tx_rotary_apply(ctx.handle, input.ptr, out.ptr, batch, seq, heads, dim, pos, stride, desc, 0), name)
    if _needs_grad(input):
        held = positions.detach() if positions is not None else None

        def backward(g):
            dx = Tensor._new(shape, ctx)
            ctx.check(lib.tx_rotary_apply(ctx.handle, g[0].ptr, dx.ptr, batch, seq, heads, dim,
                                          held.ptr if held is not None else None, stride, desc, 1),
                      "rotary_embedding backward")
            return [dx]

        out._attach(Fn(name, [input], backward))
    return out


def qk_norm_rotary(q: Tensor, k: Tensor, q_weight: Tensor, k_weight: Tensor, rotary: Rotary,
                   positions: Optional[Tensor] = None, eps: float = 1e-6) -> tuple:
    """Root-mean-square norms of every query and key head, ``x / sqrt(mean(x^2) +
    eps) * weight``, and the rotation of :func:`rotary_embedding`, as one kernel
    over ``q [batch, tokens, heads, head_dim]`` and ``k [batch, tokens, kv_heads,
    head_dim]``; the weights are [head_dim].  Returns both rotated tensors."""
    name, ctx = "qk_norm_rotary", q.ctx
    shape = batch, seq, heads, dim = _heads(name, "q", q, ctx)
    kv_heads = _heads(name, "k", k, ctx, "kv_heads")[2]
    if k.shape != (batch, seq, kv_heads, dim):
        raise ValueError(f"{name} k must be [{batch}, {seq}, kv_heads, {dim}], got {k.shape}")
    for what, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w.dtype != "float32" or w.shape != (dim,):
            raise ValueError(f"{name} {what} must be a float32 Tensor of shape ({dim},), got {w.dtype} {w.shape}")
        _same_device(name, what, w, ctx)
    if not eps >= 0.0:
        raise ValueError(f"{name} eps must not be negative, got {eps}")
    pos, stride = _rotary_positions(name, rotary, positions, shape, ctx)
    desc = rotary._desc
    yq, yk = Tensor._new(shape, ctx), Tensor._new(k.shape, ctx)
    ctx.check(lib.tx_qk_norm_rotary_fwd(ctx.handle, q.ptr, k.ptr, q_weight.ptr, k_weight.ptr, yq.ptr, yk.ptr, batch,
                                        seq, heads, kv_heads, dim, pos, stride, desc, eps), name)
    if _needs_grad(q, k, q_weight, k_weight):
        sq, sk, swq, swk = (t.detach() for t in (q, k, q_weight, k_weight))
        held = positions.detach() if positions is not None else None

        def backward(g):
            gq, gk = (t if t is not None else full(s.shape, 0.0, ctx=ctx) for t, s in zip(g, (sq, sk)))
            dq, dk, dwq, dwk = (Tensor._new(t.shape, ctx) for t in (sq, sk, swq, swk))
            ctx.check(lib.tx_qk_norm_rotary_bwd(ctx.handle, sq.ptr, sk.ptr, swq.ptr, swk.ptr, gq.ptr, gk.ptr, dq.ptr,
                                                dk.ptr, dwq.ptr, dwk.ptr, batch, seq, heads, kv_heads, dim,
                                                held.ptr if held is not None else None, stride, desc, eps),
                      "qk_norm_rotary backward")
            return [dq, dk, dwq, dwk]

        fn = Fn(name, [q, k, q_weight, k_weight], backward, n_out=2)
        yq._attach(fn, 0)
        yk._attach(fn, 1)
    return yq, yk


def differential_attention(q: Tensor, k: Tensor, v: Tensor, lam: Tensor, *, scale: Optional[float] = None,
                           causal: bool = False, query_start: Optional[int] = None,
                           key_lengths: Optional[Tensor] = None) -> Tensor:
    """The difference of two attention maps a head with a learned weight,
    ``softmax(scale q1 k1^T) v - lam softmax(scale q2 k2^T) v``.

    ``q [batch, queries, 2 * heads, d]`` and ``k [batch, keys, 2 * kv_heads, d]``
    hold the two maps of head h at 2h and 2h + 1 (the layout that
    :func:`qk_norm_rotary` returns for twice the heads), ``v [batch, keys,
    kv_heads, dv]``, ``lam [heads]``; ``heads`` is a multiple of ``kv_heads`` and
    consecutive query heads share a key head; d <= 64, dv <= 128.  ``scale``
    defaults to ``d ** -0.5``.

    Query i sees key j if ``j < key_lengths[batch]`` (int64 [batch]; None: every
    key) and, with ``causal``, ``j <= i + query_start`` (the position of the first
    query among the keys; None: ``keys - queries``, so that the last query sees
    every key).  Keys and values behind a sequence's length are never read, within
    it they must be finite; a query that sees no key returns zeros.  A length
    outside [0, keys] raises IndexError at the next synchronisation.

    When a gradient is wanted, the output's second term, a number a query and map,
    and the operands in the form the tensor cores read (as large as q, k and v)
    are kept until the backward."""
    name, ctx = "differential_attention", q.ctx
    batch, queries, maps, d = _heads(name, "q", q, ctx, "2 * heads")
    _, keys, kv_maps, _ = _heads(name, "k", k, ctx, "2 * kv_heads")
    _heads(name, "v", v, ctx, "kv_heads")
    heads, kv_heads = maps // 2, kv_maps // 2
    if maps % 2 or kv_maps % 2 or not heads or not kv_heads or heads % kv_heads:
        raise ValueError(f"{name} needs two maps a head and a number of query heads that is a multiple of the key "
                         f"heads', got {maps} and {kv_maps} maps")
    if k.shape != (batch, keys, kv_maps, d):
        raise ValueError(f"{name} k must be [{batch}, keys, 2 * kv_heads, {d}], got {k.shape}")
    dv = v.shape[3]
    if v.shape != (batch, keys, kv_heads, dv):
        raise ValueError(f"{name} v must be [{batch}, {keys}, {kv_heads}, dv], got {v.shape}")
    if not 1 <= d <= 64 or not 1 <= dv <= 128:
        raise NotImplementedError(f"{name} supports head dimensions up to 64 and value dimensions up to 128, got "
                                  f"{d} and {dv}")
    if lam.dtype != "float32" or lam.shape != (heads,):
        raise ValueError(f"{name} lam must be a float32 Tensor of shape ({heads},), got {lam.dtype} {lam.shape}")
    _same_device(name, "lam", lam, ctx)
    if key_lengths is not None:
        if key_lengths.dtype != "int64" or key_lengths.shape != (batch,):
            raise ValueError(f"{name} key_lengths must be int64 [{batch}], got {key_lengths.dtype} "
                             f"{key_lengths.shape}")
        _same_device(name, "key_lengths", key_lengths, ctx)
    scale = d ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"{name} scale must be finite, got {scale}")
    start = keys - queries if query_start is None else int(query_start)
    if abs(start) > 1 << 30:
        raise ValueError(f"{name} query_start must be within +-2^30, got {start}")
    out = Tensor._new((batch, queries, heads, dv), ctx)
    desc = N.DiffAttentionDesc(batch, queries, keys, heads, kv_heads, d, dv, q.ptr, k.ptr, v.ptr, lam.ptr,
                               key_lengths.ptr if key_lengths is not None else None, scale, int(bool(causal)), start,
                               out.ptr)
    grad = _needs_grad(q, k, v, lam)
    if grad:
        size = C.c_int64()
        ctx.check(lib.tx_diff_attention_saved_bytes(ctx.handle, desc, C.byref(size)), name)
        # one block: the operands, out2 and lse, each from a 16-byte boundary
        at = -(-size.value // 16) * 16
        end = at + -(-out.nbytes // 16) * 16
        kept = Storage(ctx, end + batch * maps * queries * 4)
        desc.saved = kept.ptr if size.value else None
        desc.out2, desc.lse = kept.ptr + at, kept.ptr + end
    ctx.check(lib.tx_diff_attention_fwd(ctx.handle, desc), name)
    if grad:
        # detached views keep what the description points to alive until this node is freed
        held = [t.detach() for t in (q, k, v, lam, out)] + [kept, key_lengths]
        want = [t.requires_grad for t in (q, k, v, lam)]

        def backward(g):
            dq = Tensor._new(held[0].shape, ctx) if want[0] else None
            dk = Tensor._new(held[1].shape, ctx) if want[1] or want[2] else None
            dv_ = Tensor._new(held[2].shape, ctx) if want[1] or want[2] else None
            dlam = Tensor._new((heads,), ctx) if want[3] else None
            desc.dout = g[0].ptr
            for field, t in (("dq", dq), ("dk", dk), ("dv", dv_), ("dlam", dlam)):
                setattr(desc, field, t.ptr if t is not None else None)
            ctx.check(lib.tx_diff_attention_bwd(ctx.handle, desc), f"{name} backward")
            return [dq, dk, dv_, dlam]

        out._attach(Fn(name, [q, k, v, lam], backward))
    return out


def relu(input: Tensor) -> Tensor:
    return input.relu()


def binary_cross_entropy_with_logits(input: Tensor, target: Tensor, reduction: str = "mean"):
    if input.shape != target.shape:
        raise ValueError("binary_cross_entropy_with_logits requires exactly matching shapes")
    absolute = maximum(input, -input)
    loss = maximum(input, 0.0) - input * target + ((-absolute).exp() + 1.0).log()
    return mse_reduce(loss, reduction)


def mse_reduce(t: Tensor, reduction: str) -> Tensor:
    if reduction == "none":
        return t
    if reduction == "mean":
        return t.mean()
    if reduction == "sum":
        return t.sum()
    raise ValueError(f"reduction must be 'none', 'mean', or 'sum', got {reduction!r}")


def _pair(v, name: str, positive: bool) -> tuple:
    pair = (v, v) if isinstance(v, int) else tuple(v)
    if len(pair) != 2 or any(not isinstance(x, int) for x in pair):
        raise TypeError(f"{name} must be an int or a pair of ints")
    if any(x <= 0 if positive else x < 0 for x in pair):
        raise ValueError(f"{name} must be {'positive' if positive else 'non-negative'}")
    return pair


def _pool_out(size: int, k: int, s: int, p: int, d: int, ceil: bool) -> int:
    eff = d * (k - 1) + 1
    if size + 2 * p < eff:
        raise ValueError("pooling window larger than its padded input")
    if ceil:
        out = -(-(size + 2 * p - eff) // s) + 1
        if (out - 1) * s >= size + p:
            out -= 1
        return out
    return (size + 2 * p - eff) // s + 1


def _pool_geom(input: Tensor, kernel, stride, padding, dilation, ceil: bool):
    if input.ndim != 4 or input.dtype != "float32":
        raise ValueError(f"pooling expects a float32 NCHW input, got {input.dtype} {input.shape}")
    _, _, h, w = input.shape
    oh = _pool_out(h, kernel[0], stride[0], padding[0], dilation[0], ceil)
    ow = _pool_out(w, kernel[1], stride[1], padding[1], dilation[1], ceil)
    geom = [kernel[0], kernel[1], stride[0], stride[1], padding[0], padding[1], dilation[0], dilation[1], oh, ow,
            padding[0], padding[1]]
    return geom, oh, ow


def max_pool2d(input: Tensor, kernel_size, stride=None, padding=0, dilation=1, ceil_mode: bool = False) -> Tensor:
    """Two-dimensional max pooling of an NCHW input over the -inf padded
    input; the gradient goes to the first maximal tap of each window."""
    kernel = _pair(kernel_size, "kernel_size", True)
    geom, oh, ow = _pool_geom(input, kernel, kernel if stride is None else _pair(stride, "stride", True),
                              _pair(padding, "padding", False), _pair(dilation, "dilation", True), bool(ceil_mode))
    n, c, h, w = input.shape
    out = Tensor._empty((n, c, oh, ow), "float32", input.ctx)
    arg = Tensor._empty((n, c, oh, ow), "int64", input.ctx)  # int32 indices in the first half
    g = N.i64_array(geom)
    input.ctx.check(lib.tx_maxpool2d_fwd(input.ctx.handle, input.ptr, out.ptr, arg.ptr, n * c, h, w, g))
    if _needs_grad(input):
        x_shape, ctx = input.shape, input.ctx

        def backward(grads):
            dx = Tensor._empty(x_shape, "float32", ctx)
            ctx.check(lib.tx_maxpool2d_bwd(ctx.handle, grads[0].ptr, arg.ptr, dx.ptr, n * c, h, w,
                                           N.i64_array(geom), 0))
            return [dx]

        out._attach(Fn("max_pool2d", [input], backward))
    return out


def avg_pool2d(input: Tensor, kernel_size, stride=None, padding=0, ceil_mode: bool = False,
               count_include_pad: bool = True, divisor_override=None) -> Tensor:
    """Two-dimensional average pooling of an NCHW input (torch semantics:
    count_include_pad counts the padding, not a ceil-mode overhang)."""
    if divisor_override is not None:
        raise NotImplementedError("avg_pool2d divisor_override is not supported")
    kernel = _pair(kernel_size, "kernel_size", True)
    geom, oh, ow = _pool_geom(input, kernel, kernel if stride is None else _pair(stride, "stride", True),
                              _pair(padding, "padding", False), (1, 1), bool(ceil_mode))
    n, c, h, w = input.shape
    out = Tensor._empty((n, c, oh, ow), "float32", input.ctx)
    inc = int(bool(count_include_pad))
    input.ctx.check(lib.tx_avgpool2d_fwd(input.ctx.handle, input.ptr, out.ptr, n * c, h, w, N.i64_array(geom), inc))
    if _needs_grad(input):
        x_shape, ctx = input.shape, input.ctx

        def backward(grads):
            dx = Tensor._empty(x_shape, "float32", ctx)
            ctx.check(lib.tx_avgpool2d_bwd(ctx.handle, grads[0].ptr, dx.ptr, n * c, h, w, N.i64_array(geom), inc, 0))
            return [dx]

        out._attach(Fn("avg_pool2d", [input], backward))
    return out


def adaptive_avg_pool2d(input: Tensor, output_size) -> Tensor:
    """Average pooling to an exact spatial size.  Windows are the uniform
    k = size / out ones when the sizes divide (the global pool included); other
    sizes need uneven windows and are not supported."""
    oh, ow = _pair(output_size, "output_size", True)
    _, _, h, w = input.shape
    if h % oh or w % ow:
        raise NotImplementedError("adaptive_avg_pool2d needs output sizes that divide the input's")
    return avg_pool2d(input, (h // oh, w // ow), (h // oh, w // ow))


def embedding(input: Tensor, weight: Tensor, padding_idx=None, max_norm=None, norm_type: float = 2.0,
              scale_grad_by_freq: bool = False, sparse: bool = False) -> Tensor:
    """Rows of a dense [rows, width] table for int64 indices; the gradient is
    a scatter-add into the table (the padding row's stays zero)."""
    if max_norm is not None or norm_type != 2.0 or scale_grad_by_freq or sparse:
        raise NotImplementedError("embedding supports the dense lookup only")
    if input.dtype != "int64":
        raise TypeError(f"embedding input must be int64, got {input.dtype}")
    if weight.dtype != "float32" or weight.ndim != 2:
        raise ValueError(f"embedding weight must be rank-2 float32, got {weight.dtype} {weight.shape}")
    rows, width = weight.shape
    if padding_idx is not None:
        if not -rows <= padding_idx < rows:
            raise ValueError("padding_idx must be within the table")
        padding_idx %= rows
    out = Tensor._empty(tuple(input.shape) + (width,), "float32", weight.ctx)
    weight.ctx.check(lib.tx_gather_rows(weight.ctx.handle, weight.ptr, rows, width, input.ptr, input.numel, out.ptr))
    if _needs_grad(weight):
        idx, ctx = input.detach(), weight.ctx

        def backward(grads):
            from .._core import full

            dw = full((rows, width), 0.0, ctx=ctx)
            ctx.check(lib.tx_scatter_add_rows(ctx.handle, dw.ptr, rows, width, idx.ptr, idx.numel, grads[0].ptr))
            if padding_idx is not None:
                ctx.check(lib.tx_fill_f32(ctx.handle, dw.ptr + padding_idx * width * 4, width, C.c_float(0.0)))
            return [None, dw]

        out._attach(Fn("embedding", [input, weight], backward))
    return out


def dropout(input: Tensor, p: float = 0.5, training: bool = True, inplace: bool = False, *,
            seed: int = 0) -> Tensor:
    """Training-mode dropout on a device random stream that advances with every
    call (a compiled step draws a new mask on every replay); the identity when
    not training or p == 0."""
    if not 0.0 <= p < 1.0:
        raise ValueError("dropout probability must be in [0, 1)")
    if not training or p == 0.0:
        return input
    mask = Tensor._empty(input.shape, "float32", input.ctx)
    out = Tensor._empty(input.shape, "float32", input.ctx)
    input.ctx.check(lib.tx_dropout_fwd(input.ctx.handle, input.ptr, out.ptr, mask.ptr, input.numel, C.c_float(p),
                                       C.c_uint64(seed & 0xFFFFFFFFFFFFFFFF), None))
    if _needs_grad(input):
        m = mask

        def backward(grads):
            return [grads[0] * m]

        out._attach(Fn("dropout", [input], backward))
    return out


__all__ = ["adaptive_avg_pool2d", "avg_pool2d", "binary_cross_entropy_with_logits", "cross_entropy",
           "differential_attention", "dropout", "embedding", "max_pool2d", "mse_loss", "ppo_loss", "qk_norm_rotary",
           "relu", "rotary_embedding"]
