"""What stands between a decoder block's packed products: rotary positions, the key / value cache and attention.

``rotary`` and ``attention`` are the training forms (both differentiable); ``rotary_cache`` and ``cached_attention`` the
serving forms, which append the new tokens to a cache and attend over it.  The reference evaluates the same steps as separate
tensor operations (``impl/tf/moondream/layers.py:244-268``, ``impl/tf/attention.py:87-105``).  Every call is one or a few
hand-written HIP kernels behind the C ABI of ``include/tvl.h``, asynchronous on the current stream of the tensors' device;
tensors must live on the GPU, there is no CPU path.

Layout: ``[batch, tokens, heads, dim]`` with any strides (the last dimension dense, else the tensor is copied), caches
``[batch, kv_heads, slots, dim]``; float32, float16 or bfloat16; head dims up to 128 for attention.  Sums, maxima and
softmax statistics are float32.  Nothing is read back to the host, so every call can be captured into a HIP graph.
"""
from __future__ import annotations

import math
import struct
from typing import Optional, Union

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import custom_ops_mod as ops

MAX_HEAD_DIM = 128

# the argument blocks of include/tvl.h, field for field
_ROTARY = struct.Struct("=5Q15q4i")
_ROTARY_CACHE = struct.Struct("=8Q19q2i")
_ATTENTION = struct.Struct("=11Q22q2f2i")
_GRADS = struct.Struct("=5Q3q")

_F32_MAX = torch.finfo(torch.float32).max
_FLOATS = {torch.float32: ops.F32, torch.float16: ops.F16, torch.bfloat16: ops.BF16}


def _heads(t: torch.Tensor, name: str) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        ops._gpu(t, name)
    if t.dim() != 4:
        raise ValueError(f"{name}: expected a 4-D tensor of heads, got shape {tuple(t.shape)}")
    if t.dtype not in _FLOATS:
        raise ValueError(f"{name}: unsupported dtype {t.dtype}")
    return t if t.stride(3) == 1 or t.shape[3] <= 1 else t.contiguous()


def _vector(t: torch.Tensor, n: int, dtype: torch.dtype, device: torch.device, name: str) -> torch.Tensor:
    ops._gpu(t, name)
    if t.dtype != dtype or t.device != device or t.shape != (n,):
        raise ValueError(f"{name}: expected a {dtype} tensor of {n} values on {device}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    if t.requires_grad:
        raise ValueError(f"{name} gets no gradient: pass a tensor that does not require one")
    return t if t.is_contiguous() else t.contiguous()


def _same(t: torch.Tensor, like: torch.Tensor, name: str) -> None:
    if t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"{name}: {t.dtype} on {t.device}, the other operands are {like.dtype} on {like.device}")


def _no_tangents(name: str, *tensors) -> None:
    """Forward-mode derivatives are not formed: refused, where they would vanish silently."""
    if forward_ad._current_level >= 0 and any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{name}: no forward-mode derivatives: pass tensors without tangents")


# the current stream's handle without a Stream object around it (3 us less a call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _run(fn, device: torch.device, *args) -> None:
    index = device.index
    if torch.cuda.current_device() == index:   # skip the device guard when it is a no-op
        status = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            status = fn(*args, _raw_stream(index))
    if status:
        ops._check(status)


def _held(leaf: torch.Tensor, stream: int) -> bool:
    """Whether a graph that is alive holds the leaf's gradient node, other than one that calls recorded on `stream` made.  A leaf knows its node
    weakly, so a mark on the node is there at the next look only if something else keeps the node alive."""
    mark = object()
    torch.autograd.graph.get_gradient_edge(leaf).node.metadata["tvl_mark"] = mark
    metadata = torch.autograd.graph.get_gradient_edge(leaf).node.metadata
    return metadata.pop("tvl_mark", None) is mark and metadata.get("tvl_stream") != stream


def _recorded_leaves(name: str, *tensors: torch.Tensor):
    """The leaves among the operands of a differentiable call that is being recorded into a HIP graph; refused where its backward pass would end the
    process: a gradient node belongs to the stream of the operation that made it, whichever that was, and a captured backward pass that reaches a
    node of another stream joins that stream into the capture.  Which stream a node belongs to cannot be asked, so only nodes that calls of this module
    recorded on the same stream pass."""
    if not torch.is_grad_enabled():
        return ()
    leaves = [x for x in tensors if isinstance(x, torch.Tensor) and x.requires_grad and x.is_leaf and x.is_cuda]
    if not leaves:
        return ()
    index = leaves[0].device.index
    if torch.cuda.current_device() == index:
        recording = torch.cuda.is_current_stream_capturing()
    else:
        with torch.cuda.device(index):
            recording = torch.cuda.is_current_stream_capturing()
    if not recording:
        return ()
    stream = _raw_stream(index)
    if any(_held(x, stream) for x in leaves):
        raise RuntimeError(f"{name}: another graph of one of these leaves is alive: an eager graph, whose gradient nodes belong to its own stream so that the backward pass "
                           "cannot be captured (delete or detach the eager results before the capture), or another operation of this capture that took the leaf first")
    return [(x, stream) for x in leaves]


def _apply(fn, leaves, *args) -> torch.Tensor:
    y = fn.apply(*args)
    for x, stream in leaves:
        torch.autograd.graph.get_gradient_edge(x).node.metadata["tvl_stream"] = stream
    return y


# --------------------------------------------------------------------------------------------
# rotary positions
# --------------------------------------------------------------------------------------------

def rotary_table(rotary_dim: int, max_len: int, theta: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                 original_len: Optional[int] = None, device: Union[str, torch.device] = "cuda") -> torch.Tensor:
    """Rotation table for positions ``0 .. max_len - 1``: float32 ``[max_len, rotary_dim]``, the cosines of the ``rotary_dim / 2``
    angles, then their sines.  Angles are evaluated in float64; pair ``i`` turns by ``f_i = theta ** (-2 i / rotary_dim)`` a token.

    ``scaling`` stretches a model to ``factor`` times its context:
      ``"linear"``  every frequency divided by ``factor`` (positions squeezed into the trained range);
      ``"ntk"``     ``theta * factor ** (rotary_dim / (rotary_dim - 2))``: the fastest pair keeps its frequency, the slowest is divided by ``factor``;
      ``"parts"``   by the turns ``r_i = original_len f_i / (2 pi)`` a pair makes over the trained context: pairs with ``r >= 32`` keep their
                    frequency, pairs with ``r <= 1`` are divided by ``factor``, linear in ``r`` between; cosines and sines times ``0.1 ln(factor) + 1``."""
    rotary_dim, max_len, factor = int(rotary_dim), int(max_len), float(factor)
    if rotary_dim < 0 or rotary_dim % 2 or max_len < 0:
        raise ValueError(f"rotary_table: rotary_dim={rotary_dim} must be even and not negative, max_len={max_len} not negative")
    if not (theta > 0 and math.isfinite(theta) and factor >= 1 and math.isfinite(factor)):
        raise ValueError(f"rotary_table: theta={theta} must be positive, factor={factor} at least 1")
    if scaling is None and factor != 1.0:
        raise ValueError("rotary_table: a factor needs a scaling: linear, ntk or parts")
    amplitude = 1.0
    if scaling == "ntk":
        if rotary_dim <= 2:
            raise ValueError("rotary_table: ntk scaling needs rotary_dim > 2")
        theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
    f = theta ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / max(rotary_dim, 1))
    if scaling == "linear":
        f = f / factor
    elif scaling == "parts":
        if original_len is None or original_len <= 0:
            raise ValueError("rotary_table: parts scaling needs original_len, the context the model was trained on")
        keep = ((original_len * f / (2 * math.pi) - 1.0) / 31.0).clip(0.0, 1.0)
        f = f * keep + f / factor * (1.0 - keep)
        amplitude = 0.1 * math.log(factor) + 1.0
    elif scaling not in (None, "ntk"):
        raise ValueError(f"Unknown rotary scaling: {scaling}")
    a = torch.outer(torch.arange(max_len, dtype=torch.float64), f)
    return (torch.cat([a.cos(), a.sin()], dim=1) * amplitude).float().to(device)


def _check_table(table: torch.Tensor, dim: int, device: torch.device, name: str) -> None:
    ops._gpu(table, f"{name}(table)")
    if table.dtype != torch.float32 or table.dim() != 2 or table.device != device or (table.shape[1] > 1 and table.stride(1) != 1):
        raise ValueError(f"{name}: the table must be a float32 [positions, rotary_dim] tensor with dense rows on {device}")
    if table.requires_grad:
        raise ValueError(f"{name}: the table gets no gradient: pass a tensor that does not require one")
    rd = table.shape[1]
    if rd % 2 or rd > dim:
        raise ValueError(f"{name}: the table turns {rd} elements of heads of {dim}: an even number up to the head dim is wanted")


def _ld_table(table: torch.Tensor) -> int:
    return max(table.stride(0), table.shape[1]) if table.shape[0] > 1 else table.shape[1]


def _rotary(x: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, interleaved: bool, inverse: bool) -> torch.Tensor:
    b, t, h, d = x.shape
    y = x.new_empty((b, t, h, d))
    pb, pt = (0, positions.stride(0)) if positions.dim() == 1 else positions.stride()
    xs, ys = x.stride(), y.stride()
    args = _ROTARY.pack(_ROTARY.size, x.data_ptr(), y.data_ptr(), positions.data_ptr(), table.data_ptr(), b, t, h, d, table.shape[1], table.shape[0],
                        _ld_table(table), xs[0], xs[1], xs[2], ys[0], ys[1], ys[2], pb, pt, _FLOATS[x.dtype], int(interleaved), int(inverse), 0)
    _run(ops._lib.tvl_rotary, x.device, args)
    return y


class _RotaryFn(torch.autograd.Function):
    """A rotation's gradient is the transposed rotation."""

    @staticmethod
    def forward(ctx, x, positions, table, interleaved):
        ctx.save_for_backward(positions, table)
        ctx.interleaved = interleaved
        return _rotary(x, positions, table, interleaved, False)

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        positions, table = ctx.saved_tensors
        return _rotary(_heads(gy, "rotary(grad)"), positions, table, ctx.interleaved, True), None, None, None


def rotary(x: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, interleaved: bool = False) -> torch.Tensor:
    """Rotary positions on ``x [batch, tokens, heads, dim]``: the first ``table.shape[1]`` elements of every head are turned by the
    angles of the token's position, the others copied.  Pairs are ``(i, i + half)``, or neighbours ``(2 i, 2 i + 1)`` when
    ``interleaved``.  ``positions``: int64 ``[tokens]`` or ``[batch, tokens]``; ``table``: :func:`rotary_table`.  A position outside the table gives
    a row of NaN.  The rotation is evaluated in float32 and rounded once.  Query and key heads that lie next to each other (a joint projection) go as
    one tensor.  Differentiable in ``x``."""
    _no_tangents("rotary", x, table)
    leaves = _recorded_leaves("rotary", x)
    x = _heads(x, "rotary(x)")
    b, t, h, d = x.shape
    ops._gpu(positions, "rotary(positions)")
    if positions.dtype != torch.int64 or positions.device != x.device or positions.shape not in ((t,), (b, t)):
        raise ValueError(f"rotary: positions must be int64 [{t}] or [{b}, {t}] on {x.device}, got {tuple(positions.shape)} {positions.dtype} on {positions.device}")
    _check_table(table, d, x.device, "rotary")
    if x.requires_grad and torch.is_grad_enabled():
        return _apply(_RotaryFn, leaves, x, positions, table, bool(interleaved))
    return _rotary(x, positions, table, interleaved, False)


def _lengths(cache_len, count, b: int, t: int, slots: int, device: torch.device, name: str):
    """(pointer, stride, value, pointer of count) of the cache fill levels."""
    if isinstance(cache_len, torch.Tensor):
        ops._gpu(cache_len, f"{name}(cache_len)")
        if cache_len.dtype != torch.int64 or cache_len.device != device or cache_len.shape not in ((), (b,)):
            raise ValueError(f"{name}: cache_len must be an int, or an int64 tensor of one value or {b} values on {device}, got {tuple(cache_len.shape)} {cache_len.dtype} on {cache_len.device}")
        at, stride, value = cache_len.data_ptr(), (cache_len.stride(0) if cache_len.dim() else 0), 0
    else:
        at, stride, value = 0, 0, int(cache_len)
        if value < 0 or value > slots or (count is None and value + t > slots):
            raise ValueError(f"{name}: {t} tokens behind cache_len={value} do not fit {slots} slots")
    n = 0
    if count is not None:
        count = _vector(count, b, torch.int64, device, f"{name}(count)")
        n = count.data_ptr()
    return at, stride, value, n, count


def _apart(t: torch.Tensor) -> bool:
    """No two elements of a written tensor share memory (strides sorted, each past the extent of the ones inside it)."""
    extent = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if stride < extent:
            return False
        extent += stride * (size - 1)
    return True


def _meet(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two views of one layout, each without elements that share memory, share some with each other: their distance is a sum of steps that both can take.
    Views of different layouts are not looked at."""
    if a.is_contiguous() or a.stride() != b.stride() or a.untyped_storage().data_ptr() != b.untyped_storage().data_ptr():
        return False
    away = {a.storage_offset() - b.storage_offset()}
    for stride, size in sorted(((s, n) for s, n in zip(a.stride(), a.shape) if n > 1), reverse=True):
        # what is left after this dimension is less than a step of it
        away = {d - stride * k for d in away for k in (d // stride, d // stride + 1) if abs(k) < size}
    return 0 in away


def _check_cache(k_cache: torch.Tensor, v_cache: torch.Tensor, like: torch.Tensor, b: int, d: int, name: str, written: bool):
    if (isinstance(k_cache, torch.Tensor) and isinstance(v_cache, torch.Tensor) and k_cache.dtype is like.dtype and v_cache.dtype is like.dtype
            and k_cache.device == like.device and v_cache.device == like.device and k_cache.dim() == 4 and k_cache.shape == v_cache.shape
            and k_cache.shape[0] == b and k_cache.shape[3] == d and k_cache.is_contiguous() and v_cache.is_contiguous()
            and not (k_cache.requires_grad or v_cache.requires_grad)):
        return      # the common case
    for c, what in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        ops._gpu(c, f"{name}({what})")
        if c.dim() != 4 or c.shape != k_cache.shape or c.shape[0] != b or c.shape[3] != d:
            raise ValueError(f"{name}: {what} must be [{b}, kv_heads, slots, {d}] like the other cache, got {tuple(c.shape)}")
        _same(c, like, f"{name}({what})")
        if d > 1 and c.stride(3) != 1:
            raise ValueError(f"{name}: {what} must be dense in its last dimension")
        if c.requires_grad:
            raise ValueError(f"{name}: caches get no gradient: pass tensors that do not require one")
        if written and not _apart(c):
            raise ValueError(f"{name}: rows of {what} share memory")


def rotary_cache(qkv: torch.Tensor, table: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, cache_len, heads: int,
                 interleaved: bool = False, count: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The joint projection's output into the cache, in one launch: returns the rotated queries ``[batch, tokens, heads, dim]`` and
    writes the rotated keys and the values of the new tokens to ``k_cache`` / ``v_cache`` ``[batch, kv_heads, slots, dim]``.

    ``qkv [batch, tokens, >= (heads + 2 kv_heads) dim]`` holds query heads, key heads, value heads (a longer row, as of a product
    with more channels behind, is fine).  ``cache_len``: tokens of each sequence that are in the cache already, so token ``t`` gets position and
    slot ``cache_len + t``: an int, or an int64 tensor of one value or ``[batch]``.  ``count`` (int64 ``[batch]``): how many of the ``tokens`` are real; the
    rows behind are zero in the result and nothing of them is written.  A position that is negative or beyond table or cache gives a
    row of NaN and writes nothing: a table shorter than the cache leaves slots unwritten.  Without ``count``, an int ``cache_len`` whose tokens do not fit the
    cache raises instead (the table's end is not looked at).  No gradients."""
    _no_tangents("rotary_cache", qkv, table, k_cache, v_cache)
    ops._gpu(qkv, "rotary_cache(qkv)")
    if qkv.dim() != 3 or qkv.dtype not in _FLOATS:
        raise ValueError(f"rotary_cache: qkv must be a float [batch, tokens, channels] tensor, got {tuple(qkv.shape)} {qkv.dtype}")
    if qkv.requires_grad and torch.is_grad_enabled():
        raise ValueError("rotary_cache is a serving form without gradients: call it under torch.no_grad(), or use rotary")
    if qkv.shape[2] > 1 and qkv.stride(2) != 1:
        qkv = qkv.contiguous()
    b, t, width = qkv.shape
    ops._gpu(k_cache, "rotary_cache(k_cache)")
    if k_cache.dim() != 4:
        raise ValueError(f"rotary_cache: k_cache must be [batch, kv_heads, slots, dim], got {tuple(k_cache.shape)}")
    hk, slots, d = k_cache.shape[1:]
    heads = int(heads)
    if heads < 0 or width < (heads + 2 * hk) * d:
        raise ValueError(f"rotary_cache: rows of {width} channels do not hold {heads} query and 2 x {hk} key / value heads of {d}")
    _check_cache(k_cache, v_cache, qkv, b, d, "rotary_cache", True)
    ka, va = k_cache.data_ptr(), v_cache.data_ptr()
    if k_cache.numel() and (ka == va or (abs(ka - va) < k_cache.nbytes and k_cache.is_contiguous() and v_cache.is_contiguous()) or _meet(k_cache, v_cache)):
        raise ValueError("rotary_cache: k_cache and v_cache share memory")
    _check_table(table, d, qkv.device, "rotary_cache")
    at, stride, value, n, count = _lengths(cache_len, count, b, t, slots, qkv.device, "rotary_cache")
    q = qkv.new_empty((b, t, heads, d))
    ks, vs = k_cache.stride(), v_cache.stride()
    args = _ROTARY_CACHE.pack(_ROTARY_CACHE.size, qkv.data_ptr(), q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), table.data_ptr(), at, n,
                              b, t, heads, hk, d, table.shape[1], slots, table.shape[0], _ld_table(table), qkv.stride(0), qkv.stride(1),
                              ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], stride, value, _FLOATS[qkv.dtype], int(bool(interleaved)))
    _run(ops._lib.tvl_rotary_cache, qkv.device, args)
    return q


# --------------------------------------------------------------------------------------------
# attention
# --------------------------------------------------------------------------------------------

def _prefix(prefix, b: int, device: torch.device, name: str):
    if prefix is None:
        return 0, 0, None
    if isinstance(prefix, torch.Tensor):
        prefix = _vector(prefix, b, torch.int64, device, f"{name}(prefix)")
        return prefix.data_ptr(), 0, prefix
    return 0, min(max(int(prefix), 0), 1 << 62), None


def _scale_cap(scale, softcap, d: int, name: str):
    if scale is None and softcap == 0.0:
        return d ** -0.5, 0.0
    scale = d ** -0.5 if scale is None else float(scale)
    softcap = 0.0 if softcap is None else float(softcap)
    if not (abs(scale) <= _F32_MAX and 0.0 <= softcap <= _F32_MAX):
        raise ValueError(f"{name}: scale={scale} must be finite, softcap={softcap} finite and not negative, in float32")
    return scale, softcap


def _workspace(need: int, device: torch.device):
    """Scratch memory of one call, from torch's allocator on the current stream (a captured call takes it from its graph's pool,
    so no two graphs share it)."""
    if need == 0:
        return None, 0
    ws = torch.empty((need,), dtype=torch.uint8, device=device)
    return ws, ws.data_ptr()


def _attention_args(q, k, v, out, lse, causal, scale, softcap, slopes, prefix_at, prefix_value, documents) -> bytes:
    b, tq, hq, d = q.shape
    qs, ks, vs, os_ = q.stride(), k.stride(), v.stride(), out.stride()
    return _ATTENTION.pack(_ATTENTION.size, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr() if lse is not None else 0,
                           slopes.data_ptr() if slopes is not None else 0, prefix_at, documents.data_ptr() if documents is not None else 0, 0, 0,
                           b, tq, k.shape[1], hq, k.shape[2], d, qs[0], qs[1], qs[2], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], os_[0], os_[1], os_[2],
                           prefix_value, documents.stride(0) if documents is not None and b > 1 else 0, 0, 0, scale, softcap, _FLOATS[q.dtype], int(causal))


def _attention(q, k, v, causal, scale, softcap, slopes, prefix_at, prefix_value, documents, want_lse):
    b, tq, hq, d = q.shape
    out = q.new_empty((b, tq, hq, d))
    lse = torch.empty((b, hq, tq), dtype=torch.float32, device=q.device) if want_lse else None
    args = _attention_args(q, k, v, out, lse, causal, scale, softcap, slopes, prefix_at, prefix_value, documents)
    need = ops._lib.tvl_attention_workspace_bytes(args)
    ws, at = _workspace(need, q.device)
    _run(ops._lib.tvl_attention, q.device, args, at, need)
    return out, lse


class _AttentionFn(torch.autograd.Function):
    """Saves the operands, the result and one float32 per query row (log of the softmax's sum); the backward kernels form the
    scores again."""

    @staticmethod
    def forward(ctx, q, k, v, causal, scale, softcap, slopes, prefix, documents):
        at, value = (prefix.data_ptr(), 0) if isinstance(prefix, torch.Tensor) else (0, prefix)
        out, lse = _attention(q, k, v, causal, scale, softcap, slopes, at, value, documents, True)
        ctx.save_for_backward(q, k, v, out, lse, slopes, prefix if isinstance(prefix, torch.Tensor) else None, documents)
        ctx.rest = (causal, scale, softcap, value)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, go):
        q, k, v, out, lse, slopes, prefix, documents = ctx.saved_tensors
        causal, scale, softcap, value = ctx.rest
        go = _heads(go, "attention(grad)")
        args = _attention_args(q, k, v, out, lse, causal, scale, softcap, slopes, prefix.data_ptr() if prefix is not None else 0, value, documents)
        want_q, want_kv = ctx.needs_input_grad[0], ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        dq = torch.empty(q.shape, dtype=q.dtype, device=q.device) if want_q else None
        dk, dv = (torch.empty(k.shape, dtype=q.dtype, device=q.device) if want_kv else None for _ in range(2))
        gs = go.stride()
        grads = _GRADS.pack(_GRADS.size, go.data_ptr(), dq.data_ptr() if want_q else 0, dk.data_ptr() if want_kv else 0, dv.data_ptr() if want_kv else 0,
                            gs[0], gs[1], gs[2])
        need = ops._lib.tvl_attention_backward_workspace_bytes(args)
        ws, at = _workspace(need, q.device)
        _run(ops._lib.tvl_attention_backward, q.device, args, grads, at, need)
        return dq, dk if ctx.needs_input_grad[1] else None, dv if ctx.needs_input_grad[2] else None, None, None, None, None, None, None


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool = False, scale: Optional[float] = None, softcap: float = 0.0,
              slopes: Optional[torch.Tensor] = None, prefix=None, documents: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``softmax(cap(scale q k^T) - slope |distance|) v`` per head, without a stored score matrix.  Differentiable in q, k and v.

    ``q [batch, queries, heads, dim]``, ``k`` and ``v [batch, keys, kv_heads, dim]`` with ``heads`` a multiple of ``kv_heads`` (head ``h`` reads
    key head ``h // (heads / kv_heads)``), ``dim <= 128``; ``scale`` defaults to ``dim ** -0.5``.
    ``softcap`` c > 0: scores become ``c tanh(s / c)``.  ``slopes`` (float32 ``[heads]``, no gradient): ``slopes[h] * |p - j|`` is taken off the score of key j,
    with ``p = i + keys - queries`` the place of query i.
    ``causal``: query i sees keys ``j <= p``; with ``prefix`` (an int, or int64 ``[batch]``) also every ``j < prefix`` (an image or prompt that sees itself
    whole).  ``documents`` (int64 ``[batch, tokens]``, queries == keys): only keys of the query's own document are seen; a negative document is padding.
    A query that sees nothing gives zeros and passes no gradient."""
    _no_tangents("attention", q, k, v, slopes)
    leaves = _recorded_leaves("attention", q, k, v)
    q, k, v = _heads(q, "attention(q)"), _heads(k, "attention(k)"), _heads(v, "attention(v)")
    b, tq, hq, d = q.shape
    _same(k, q, "attention(k)")
    _same(v, q, "attention(v)")
    if k.shape != v.shape or k.shape[0] != b or k.shape[3] != d:
        raise ValueError(f"attention: k and v must be [{b}, keys, kv_heads, {d}], got {tuple(k.shape)} and {tuple(v.shape)}")
    if k.shape[2] == 0 or hq == 0 or hq % k.shape[2]:
        raise ValueError(f"attention: {hq} query heads are not a multiple of {k.shape[2]} key heads")
    if not 1 <= d <= MAX_HEAD_DIM:
        raise ValueError(f"attention: head dim {d} outside [1, {MAX_HEAD_DIM}]")
    scale, softcap = _scale_cap(scale, softcap, d, "attention")
    if slopes is not None:
        slopes = _vector(slopes, hq, torch.float32, q.device, "attention(slopes)")
    if prefix is not None and not causal:
        raise ValueError("attention: a prefix goes with causal=True (without it every key is seen anyway)")
    at, value, prefix = _prefix(prefix, b, q.device, "attention")
    if documents is not None:
        ops._gpu(documents, "attention(documents)")
        if documents.dtype != torch.int64 or documents.device != q.device or documents.shape != (b, tq) or k.shape[1] != tq:
            raise ValueError(f"attention: documents must be int64 [{b}, {tq}] on {q.device} with as many queries as keys, got {tuple(documents.shape)} {documents.dtype} for {k.shape[1]} keys")
        if tq > 1 and documents.stride(1) != 1:
            documents = documents.contiguous()
    if (q.requires_grad or k.requires_grad or v.requires_grad) and torch.is_grad_enabled():
        return _apply(_AttentionFn, leaves, q, k, v, bool(causal), scale, softcap, slopes, prefix if prefix is not None else value, documents)
    return _attention(q, k, v, bool(causal), scale, softcap, slopes, at, value, documents, False)[0]


def cached_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, cache_len, scale: Optional[float] = None, softcap: float = 0.0,
                     slopes: Optional[torch.Tensor] = None, prefix=None, count: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of new tokens over a key / value cache that holds them already (:func:`rotary_cache` wrote them): single decode
    tokens, drafted tokens or whole prompts.

    ``q [batch, tokens, heads, dim]``; caches ``[batch, kv_heads, slots, dim]``; ``cache_len`` and ``count`` as for :func:`rotary_cache`: token i of a sequence sits
    at slot ``cache_len + i`` and sees the slots up to its own, and with ``prefix`` (an int, or int64 ``[batch]``) every slot below it that
    holds a token.  ``scale``, ``softcap`` and ``slopes`` as for :func:`attention`.  Rows behind ``count`` are zero; a token whose slot is negative or beyond
    the cache gives a row of NaN (without ``count``, an int ``cache_len`` whose tokens do not fit raises instead).  Only the filled part of the cache is read.  No gradients."""
    _no_tangents("cached_attention", q, k_cache, v_cache, slopes)
    q = _heads(q, "cached_attention(q)")
    b, t, hq, d = q.shape
    if q.requires_grad and torch.is_grad_enabled():
        raise ValueError("cached_attention is a serving form without gradients: call it under torch.no_grad(), or use attention")
    _check_cache(k_cache, v_cache, q, b, d, "cached_attention", False)
    hk, slots = k_cache.shape[1], k_cache.shape[2]
    if hk == 0 or hq == 0 or hq % hk:
        raise ValueError(f"cached_attention: {hq} query heads are not a multiple of {hk} key heads")
    if not 1 <= d <= MAX_HEAD_DIM:
        raise ValueError(f"cached_attention: head dim {d} outside [1, {MAX_HEAD_DIM}]")
    scale, softcap = _scale_cap(scale, softcap, d, "cached_attention")
    if slopes is not None:
        slopes = _vector(slopes, hq, torch.float32, q.device, "cached_attention(slopes)")
    prefix_at, prefix_value, prefix = _prefix(prefix, b, q.device, "cached_attention")
    at, stride, value, n, count = _lengths(cache_len, count, b, t, slots, q.device, "cached_attention")
    out = q.new_empty((b, t, hq, d))
    qs, ks, vs, os_ = q.stride(), k_cache.stride(), v_cache.stride(), out.stride()
    args = _ATTENTION.pack(_ATTENTION.size, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), 0,
                           slopes.data_ptr() if slopes is not None else 0, prefix_at, 0, at, n, b, t, slots, hq, hk, d, qs[0], qs[1], qs[2],
                           ks[0], ks[2], ks[1], vs[0], vs[2], vs[1], os_[0], os_[1], os_[2], prefix_value, 0, stride, value, scale, softcap,
                           _FLOATS[q.dtype], 1)
    need = ops._lib.tvl_cached_attention_workspace_bytes(args)
    ws, ws_at = _workspace(need, q.device)
    _run(ops._lib.tvl_cached_attention, q.device, args, ws_at, need)
    return out
