"""Attention over ordered tokens: norm and position rotation of queries and keys, attention with a sliding window and a few first tokens that
stay in view, and its form for one new token over a paged cache.

Next to the grouped self-attention over a whole cloud (``backbone.SALayer``, ``train_ops.sa_attention_train``), whose cost grows with the square of the
points: here a point in a serial order of its cloud (a space-filling curve, cells of a grid, ...; the caller brings it), or a submap in the stream of a drive,
sees its neighbours within a window and the first ``sinks`` tokens.

  qk_norm_rotary      norm of every head of q and k, then the rotation by positions or coordinates          with gradients
  window_attention    prompts, clouds, training                                                                  with gradients
  paged_append        new keys and values into a paged cache
  paged_attention     one new token of every sequence over that cache

Types: float32, float16, bfloat16.  Scores, maxima, sums and norms are held in 32 bits; the weights of the soft-max are rounded to the tensors' type for
their products (16-bit results are off by up to 1.5 times their own rounding).  How work is split, and with it the last bits, goes by the sizes of the
whole batch.  Heads: ``H`` query heads share ``Hk`` key heads, ``H % Hk == 0``; query head ``i`` reads key head ``i // (H // Hk)``.  Everything runs on the
current stream of the tensors' device through libpatchaugnet_hip.so; there is no CPU form.
"""
import contextlib
import functools
import math

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from . import _lib

__all__ = ["qk_norm_rotary", "window_attention", "paged_append", "paged_attention"]

_DTYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_FAR = 1 << 22             # elements between neighbouring tokens or heads: 32-bit offsets inside a tile (pa_attn.h)
_PTYPE = {torch.int32: 0, torch.int64: 1, torch.float32: 2}
_HERE = contextlib.nullcontext()
_MAXLEN = 1 << 28            # tokens of a sequence (pa_attn.h)


def _check(name, *tensors):
    """Device tensors of one device and one supported type."""
    first = tensors[0]
    for t in tensors:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name}: expected a tensor, got {type(t).__name__}")
        if not t.is_cuda:
            raise RuntimeError(f"{name} runs on the MI355X only: got a tensor on {t.device} (there is no CPU form)")
        if t.dtype != first.dtype:
            raise TypeError(f"{name}: tensors of one type; got {[x.dtype for x in tensors]}")
        if t.get_device() != first.get_device():
            raise RuntimeError(f"{name}: tensors on {first.device} and {t.device}")
    dt = _DTYPE.get(first.dtype)
    if dt is None:
        raise TypeError(f"{name}: float32, float16 or bfloat16; got {first.dtype}")
    return dt


def _on(device):
    """The device's context; nothing where it is current already (entering costs as much as a launch)."""
    return _HERE if _lib._cur_device is not None and device.index == _lib._cur_device() else torch.cuda.device(device)


def _ints(name, what, t, device, n):
    """A (n,) int32 device vector or None."""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.get_device() != device.index or t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{name}: {what} has to be an int32 tensor of shape ({n},) on {device}")
    return t.contiguous()


def _fits(t, align=16, far=1 << 62):
    """Is the last dimension contiguous, does every row start at a multiple of `align` bytes, and do those of neighbouring tokens and heads lie at most `far`
    elements apart?"""
    if t.is_contiguous():
        return t.data_ptr() % align == 0
    s = t.stride()
    outer, es = 0, t.element_size()
    for i, n in zip(s[:-1], t.shape):
        if n > 1:
            outer |= i
    return s[-1] == 1 and t.data_ptr() % align == 0 and outer * es % align == 0 and (far > _FAR or _near(t, s))


def _rows(t, align=16, far=1 << 62):
    """t itself if it fits, else a contiguous copy."""
    if t.is_contiguous():
        return t if t.data_ptr() % align == 0 else t.clone()
    return t if _fits(t, align, far) else t.contiguous()


def _near(t, s):
    return all(i <= _FAR for i, n in zip(s[1:-1], t.shape[1:-1]) if n > 1) and t.shape[-2] * s[-2] * 4 < 1 << 31


def _unit(t):
    """t itself if its last dimension is contiguous, else a contiguous copy."""
    return t if t.stride(-1) == 1 else t.contiguous()


def _strides(t):
    """Strides of the first three of four dimensions (of fewer where t is not contiguous).  A dimension with one entry may report any stride, in contiguous
    tensors too; the library would hold that against its limits, so it gets the stride of the shape, or 0."""
    if t.is_contiguous():
        _, n, h, d = t.shape
        row = h * d
        return n * row, row, d
    return [s if n > 1 else 0 for s, n in zip(t.stride()[:-1], t.shape)]


def _side(name, what, n):
    if n is None:
        return -1
    if isinstance(n, bool) or not isinstance(n, int) or n < 0:
        raise ValueError(f"{name}: {what} has to be None or an integer >= 0, got {n!r}")
    return min(n, _MAXLEN)


def _heads(name, H, Hk, D):
    if Hk < 1 or H < 1 or H % Hk:
        raise ValueError(f"{name}: {H} query heads do not share {Hk} key heads evenly")
    if D < 8 or D > 128 or D % 8:
        raise ValueError(f"{name}: head width {D} is not a multiple of 8 up to 128")


def _scale(name, scale, D):
    s = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 2.0 ** -126 <= s <= 2.0 ** 127:
        raise ValueError(f"{name}: the scale has to be positive, 2^127 at most and a normal number in 32 bits, got {scale!r}")
    return s


def ptr(t):
    return t.data_ptr() if t is not None else None


_entry = {}


def call(name, *args):
    """An entry point on the current stream of the current device; raises what the library says."""
    f = _entry.get(name)
    if f is None:
        f = _entry[name] = getattr(_lib.lib(), name)
    rc = f(*args, _lib.stream_ptr())
    if rc:
        raise RuntimeError(f"{name} failed ({rc}): {_lib.lib().pa_last_error().decode()}")


@functools.lru_cache(maxsize=256)
def _size(name, *sizes):
    """Floats of scratch that the library asks for at these sizes."""
    return getattr(_lib.lib(), name)(*sizes)


def _floats(n, device):
    return torch.empty(n, dtype=torch.float32, device=device) if n else None


# ------------------------------------------------------------------------------------------------------------------ norm and rotation
def _norm_args(q, k, qw, kw, pos, freq, rest):
    """rest: axes, frequencies of an axis, elements between two sequences' positions, eps, interleaved."""
    B, N, H, D = q.shape
    w = qw if qw is not None else kw
    axes, per, apart, eps, interleaved = rest
    return (_DTYPE[q.dtype], B, N, H, k.shape[2], D, ptr(q), *_strides(q), ptr(k), *_strides(k), ptr(qw), ptr(kw), int(w is not None and w.dtype == torch.float32),
            ptr(pos), _PTYPE[pos.dtype] if axes else 0, apart, ptr(freq), axes, per, eps, interleaved)


def _norm_forward(q, k, qw, kw, pos, freq, rest):
    out = q.new_empty(q.shape), k.new_empty(k.shape)
    with _on(q.device):
        call("pa_qk_norm_rotary", *_norm_args(q, k, qw, kw, pos, freq, rest), ptr(out[0]), ptr(out[1]))
    return out


class _NormRotary(Function):
    @staticmethod
    def forward(ctx, q, k, qw, kw, pos, freq, rest):
        out = _norm_forward(q, k, qw, kw, pos, freq, rest)
        ctx.save_for_backward(q, k, qw, kw, pos, freq)
        ctx.rest = rest
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        q, k, qw, kw, pos, freq = ctx.saved_tensors
        D = q.shape[3]
        gq, gk = _unit(gq), _unit(gk)
        dq, dk = q.new_empty(q.shape), k.new_empty(k.shape)
        with _on(q.device):
            empty = q.shape[0] * q.shape[1] == 0
            make = torch.zeros if empty else torch.empty
            dqw = make(D, dtype=torch.float32, device=q.device) if ctx.needs_input_grad[2] else None
            dkw = make(D, dtype=torch.float32, device=q.device) if ctx.needs_input_grad[3] else None
            scratch = None
            if dqw is not None or dkw is not None:
                scratch = _floats(_size("pa_qk_norm_rotary_backward_scratch_floats", q.shape[0], q.shape[1], D), q.device)
            call("pa_qk_norm_rotary_backward", *_norm_args(q, k, qw, kw, pos, freq, ctx.rest), ptr(gq), *_strides(gq), ptr(gk), *_strides(gk),
                 ptr(dq), ptr(dk), ptr(dqw), ptr(dkw), ptr(scratch))
        cast = [None if g is None else g.to(w.dtype) for g, w in ((dqw, qw), (dkw, kw))]
        return dq, dk, cast[0], cast[1], None, None, None


def qk_norm_rotary(q, k, q_weight=None, k_weight=None, *, positions=None, inv_freq=None, eps=1e-6, interleaved=False):
    """Norm of every head of q (B, N, H, D) and k (B, N, Hk, D), then the rotation by the token's position -- one pass, (q', k') contiguous.

      n = x / sqrt(mean(x^2) + eps) * weight                 weights (D,), float32 or of q's type; None: 1
      the first 2 A F elements of n turned in pairs by the angles positions[..., a] * inv_freq[a, f]

    inv_freq: float32 (F,) or (A, F): F frequencies for each of A axes; pair number a F + f.  positions: (N,) or (B, N) for one axis, (N, A) or
    (B, N, A) for several, int32, int64 or float32 -- token numbers or coordinates.  Angles are reduced in 64 bits: up to 2^27 radians they keep full 32-bit accuracy, beyond
    that they are off by 2^-52 of their size.
    Pairs are elements (i, i + A F), with interleaved=True (2 i, 2 i + 1).  positions=None: the norm alone.  D up to 512, any strides.
    Gradients for q, k and the weights; positions and frequencies get none (a tensor of theirs that asks for one is refused)."""
    name = "qk_norm_rotary"
    _check(name, q, k)
    if q.dim() != 4 or k.dim() != 4 or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise ValueError(f"{name}: q (B, N, H, D) and k (B, N, Hk, D); got {tuple(q.shape)} and {tuple(k.shape)}")
    B, N, H, D = q.shape
    if not 1 <= D <= 512 or H < 1 or k.shape[2] < 1:
        raise ValueError(f"{name}: head width {D} is not in 1..512, or no heads ({H}, {k.shape[2]})")
    ws = [w for w in (q_weight, k_weight) if w is not None]
    for w in ws:
        if w.get_device() != q.get_device() or w.dtype not in (torch.float32, q.dtype) or w.dim() != 1 or w.shape[0] != D or w.dtype != ws[0].dtype:
            raise ValueError(f"{name}: weights have to be ({D},) on {q.device}, both float32 or both {q.dtype}")
    if not 0.0 <= eps < math.inf:
        raise ValueError(f"{name}: eps has to be finite and not negative")
    if (positions is None) != (inv_freq is None):
        raise ValueError(f"{name}: positions and inv_freq come together")
    A, F, apart = 0, 0, 0
    if positions is not None:
        if inv_freq.dtype != torch.float32 or inv_freq.get_device() != q.get_device() or inv_freq.dim() not in (1, 2) or inv_freq.numel() == 0:
            raise ValueError(f"{name}: inv_freq has to be a float32 (F,) or (A, F) tensor on {q.device}")
        if positions.dtype not in _PTYPE or positions.get_device() != q.get_device():
            raise TypeError(f"{name}: positions have to be int32, int64 or float32 on {q.device}")
        if positions.requires_grad or inv_freq.requires_grad:
            raise RuntimeError(f"{name}: positions and inv_freq have no gradient here")
        A, F = inv_freq.shape if inv_freq.dim() == 2 else (1, inv_freq.shape[0])
        if 2 * A * F > D:
            raise ValueError(f"{name}: {A} x {F} frequencies rotate more than the {D} elements of a head")
        shape = tuple(positions.shape)
        if shape == (B, N, A) or (A == 1 and shape == (B, N)):
            apart = N * A
        elif shape != (N, A) and not (A == 1 and shape == (N,)):
            raise ValueError(f"{name}: positions of shape {shape} fit neither (N, A) = ({N}, {A}) nor (B, N, A) with B = {B}")
        positions, inv_freq = positions.contiguous(), inv_freq.contiguous()
    rest = A, F, apart, float(eps), int(bool(interleaved))
    q, k = _unit(q), _unit(k)
    qw, kw = (w.contiguous() if w is not None else None for w in (q_weight, k_weight))
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or any(w.requires_grad for w in ws)):
        return _NormRotary.apply(q, k, qw, kw, positions, inv_freq, rest)
    return _norm_forward(q, k, qw, kw, positions, inv_freq, rest)


# ------------------------------------------------------------------------------------------------------------------- window attention
def _window_sizes(q, k, view):
    return q.shape[0], q.shape[1], k.shape[1], q.shape[2], k.shape[2], q.shape[3], view[0], view[1], view[2]


def _window_forward(q, k, v, start, length, view, back):
    out = q.new_empty(q.shape)
    low = q.new_empty(q.shape) if back and q.dtype != torch.float32 else None
    B, N, H, D = q.shape
    lse = torch.empty((B, H, N), dtype=torch.float32, device=q.device) if back else None
    left, right, sinks, scale = view
    with _on(q.device):
        scratch = _floats(_size("pa_window_attention_scratch_floats", *_window_sizes(q, k, view)), q.device)
        call("pa_window_attention", _DTYPE[q.dtype], B, N, k.shape[1], H, k.shape[2], D, ptr(q), *_strides(q), ptr(k), *_strides(k), ptr(v), *_strides(v),
             left, right, sinks, scale, ptr(start), ptr(length), ptr(out), ptr(low), ptr(lse), ptr(scratch))
    return out, low, lse


class _WindowAttention(Function):
    @staticmethod
    def forward(ctx, q, k, v, start, length, view):
        out, low, lse = _window_forward(q, k, v, start, length, view, True)
        ctx.save_for_backward(q, k, v, start, length, out, low, lse)
        ctx.view = view
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        q, k, v, start, length, out, low, lse = ctx.saved_tensors
        g = _rows(g, far=_FAR)
        left, right, sinks, scale = ctx.view
        dq, dk, dv = (t.new_empty(t.shape) for t in (q, k, v))
        B, N, H, D = q.shape
        with _on(q.device):
            scratch = _floats(_size("pa_window_attention_backward_scratch_floats", *_window_sizes(q, k, ctx.view)), q.device)
            call("pa_window_attention_backward", _DTYPE[q.dtype], B, N, k.shape[1], H, k.shape[2], D, ptr(q), *_strides(q), ptr(k), *_strides(k), ptr(v),
                 *_strides(v), ptr(out), ptr(low), ptr(lse), ptr(g), *_strides(g), left, right, sinks, scale, ptr(start), ptr(length), ptr(dq), ptr(dk), ptr(dv),
                 ptr(scratch))
        return dq, dk, dv, None, None, None


def window_attention(q, k, v, *, left=None, right=0, sinks=0, scale=None, lengths=None, q_start=None):
    """softmax(scale q k^T) v over the keys in view, (B, N, H, D): q (B, N, H, D), k and v (B, M, Hk, D), D a multiple of 8 up to 128.

    Query i of sequence b stands at position p = q_start[b] + i.  Key j is in view if j < lengths[b], j <= p + right, and j >= p - left or j < sinks.
    left / right None: no limit on that side (the default is causal attention); the first `sinks` keys never slide out on the left.
      lengths   int32 (B,): keys of each sequence (None: M).  Queries at p >= lengths[b] are padding: output and gradients are 0, and what the padding of
                q, k, v holds has no influence, NaN included.  Within a sequence a NaN or an infinity reaches rows that do not see it.
      q_start   int32 (B,): position of the first query (None: 0) -- the next part of a prompt, whose earlier keys lie in front of it in k and v.
    Values outside 0..M are clamped.  scale None: 1 / sqrt(D).  Strides are free except that a row is contiguous and starts at a multiple of 16 bytes
    (other tensors are copied; so are those with 2^22 elements and more between two tokens or heads; H D up to 2^22).  Gradients for q, k, v, all three
    whichever are asked for, the same bits on every run; in the 16-bit types what the rounding of out left, a tensor of its size, is kept for them.  Weights and the gradients of scores are rounded to the tensors' type
    for the products; float16: brought into its range by powers of two first, so neither small gradients nor those that pass 65504 there are lost."""
    name = "window_attention"
    _check(name, q, k, v)
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise ValueError(f"{name}: q (B, N, H, D), k and v (B, M, Hk, D); got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    _heads(name, q.shape[2], k.shape[2], q.shape[3])
    left, right, sinks = _side(name, "left", left), _side(name, "right", right), max(_side(name, "sinks", sinks), 0)
    view = (left, right, sinks, _scale(name, scale, q.shape[3]))
    length, start = _ints(name, "lengths", lengths, q.device, q.shape[0]), _ints(name, "q_start", q_start, q.device, q.shape[0])
    q, k, v = (_rows(t, far=_FAR) for t in (q, k, v))
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _WindowAttention.apply(q, k, v, start, length, view)
    return _window_forward(q, k, v, start, length, view, False)[0]


# ----------------------------------------------------------------------------------------------------------------------- paged cache
def _cache(name, k_pages, v_pages, table, B):
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape:
        raise ValueError(f"{name}: k_pages and v_pages (pages, page, Hk, D); got {tuple(k_pages.shape)}, {tuple(v_pages.shape)}")
    if k_pages.shape[1] < 1 or k_pages.shape[2] < 1:
        raise ValueError(f"{name}: empty pages or no key heads: {tuple(k_pages.shape)}")
    for t in (k_pages, v_pages):
        if not _fits(t) and t.numel():
            raise ValueError(f"{name}: a row of a page has to be contiguous and to start at a multiple of 16 bytes")
    if not isinstance(table, torch.Tensor) or table.dtype != torch.int32 or table.device != k_pages.device or table.dim() != 2 or table.shape[0] != B:
        raise ValueError(f"{name}: page_table has to be an int32 tensor (B, pages of a sequence) on {k_pages.device}, B = {B}")
    if table.shape[1] * k_pages.shape[1] > _MAXLEN:
        raise ValueError(f"{name}: {table.shape[1]} pages of {k_pages.shape[1]} tokens exceed 2^28 tokens")
    return table.contiguous()


def _no_gradient(name, *tensors):
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError(f"{name} has no gradient: call it under torch.no_grad() or on detached tensors (window_attention trains)")


def paged_append(k, v, k_pages, v_pages, page_table, starts, *, counts=None):
    """New keys and values k, v (B, T, Hk, D) into the cache k_pages, v_pages (pages, page, Hk, D), in place.

    Token t < counts[b] (None: T) of sequence b goes to position starts[b] + t: row position % page of page page_table[b, position // page].  int32
    tables.  Positions outside the table and entries outside the pool (-1, ...) are skipped; everything else in the pool stays as it is.  Two
    tokens for one row of one page leave either of them, in parts; k and v must not lie in the pools."""
    name = "paged_append"
    dt = _check(name, k, v, k_pages, v_pages)
    _no_gradient(name, k, v, k_pages, v_pages)
    if k.dim() != 4 or k.shape != v.shape or k_pages.dim() != 4 or k.shape[2:] != k_pages.shape[2:]:
        raise ValueError(f"{name}: k and v (B, T, Hk, D) with the Hk and D of the pages; got {tuple(k.shape)}, {tuple(v.shape)}, {tuple(k_pages.shape)}")
    B, T, Hk, D = k.shape
    _heads(name, Hk, Hk, D)
    table = _cache(name, k_pages, v_pages, page_table, B)
    if starts is None:
        raise ValueError(f"{name}: starts are needed")
    starts, counts = _ints(name, "starts", starts, k.device, B), _ints(name, "counts", counts, k.device, B)
    k, v = _rows(k), _rows(v)
    with _on(k.device):
        call("pa_paged_append", dt, B, T, Hk, D, ptr(k), *_strides(k), ptr(v), *_strides(v), ptr(k_pages), *_strides(k_pages), ptr(v_pages), *_strides(v_pages),
             k_pages.shape[0], k_pages.shape[1], ptr(table), table.shape[1], ptr(starts), ptr(counts))
    increment_version((k_pages, v_pages))                      # a backward pass that saved rows of the pools refuses them


def paged_attention(q, k_pages, v_pages, page_table, lengths, *, left=None, sinks=0, scale=None):
    """Attention of one new token of every sequence, q (B, H, D) -> (B, H, D), over the cache k_pages, v_pages (pages, page, Hk, D).

    lengths: int32 (B,), keys of each sequence, the new token's own (paged_append) among them; it stands at position lengths[b] - 1 and sees what
    window_attention(left, right=0, sinks) shows a query there.  A sequence of length 0 gives zeros; lengths beyond the table are clamped.  A
    page_table entry outside the pool holds no keys: pages that the window has left behind may be given back and marked -1."""
    name = "paged_attention"
    dt = _check(name, q, k_pages, v_pages)
    _no_gradient(name, q, k_pages, v_pages)
    if q.dim() != 3 or k_pages.dim() != 4 or q.shape[2] != k_pages.shape[3]:
        raise ValueError(f"{name}: q (B, H, D) and pages (pages, page, Hk, D); got {tuple(q.shape)}, {tuple(k_pages.shape)}")
    B, H, D = q.shape
    table = _cache(name, k_pages, v_pages, page_table, B)
    P, page, Hk, _ = k_pages.shape
    _heads(name, H, Hk, D)
    if lengths is None:
        raise ValueError(f"{name}: lengths are needed")
    lengths = _ints(name, "lengths", lengths, q.device, B)
    left, sinks = _side(name, "left", left), max(_side(name, "sinks", sinks), 0)
    scale = _scale(name, scale, D)
    q = _rows(q)
    out = q.new_empty(q.shape)
    with _on(q.device):
        scratch = _floats(_size("pa_paged_attention_scratch_floats", B, H, Hk, D, page, table.shape[1], left, sinks), q.device)
        call("pa_paged_attention", dt, B, H, Hk, D, ptr(q), *((H * D, D) if q.is_contiguous() else _strides(q)), ptr(k_pages), *_strides(k_pages), ptr(v_pages), *_strides(v_pages), P, page, ptr(table),
             table.shape[1], ptr(lengths), left, sinks, scale, ptr(out), ptr(scratch))
    return out
