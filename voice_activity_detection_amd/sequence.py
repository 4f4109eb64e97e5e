"""Sequence operators on the kernels of libvad_amd.so: layer norm, linear attention with a decay per head, attention with
a sliding window and sinks.

They are what a frame-by-frame model is built from next to the recurrent layers of ``Net`` (core/models.py:19-25), in the
two ways this path works: a whole recording at once (``layer_norm``, ``linear_attention``, ``window_attention``, with
gradients through ``torch.autograd``), and one live frame at a time (``linear_attention_step`` on a recurrent state,
``window_attention_step`` on a rolling cache that ``window_cache_fill`` starts from a recording).

Tensors are float32 or bfloat16 CUDA tensors.  Heads come as ``(batch, length, heads, dim)``, or packed as ``(rows, heads,
dim)`` with ``starts``, an int64 CUDA tensor of the sequences' first rows and the last one's end (the table of
``mfcc_delta_ragged``; not validated, clamped); ``dim`` is 1 .. 128 and dense, the other strides are free.  Everything
runs on the current stream of the tensors' device, allocates only through torch, synchronises nothing, and can be
captured into a HIP graph after ``init()``.
"""
import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib

MAX_HEAD_DIM = 128
MAX_SINKS = 64
_DTYPES = {torch.float32: 0, torch.bfloat16: 1}


def _ptr(t):
    return None if t is None else t.data_ptr()


def _strides(*s):
    return (ctypes.c_int64 * len(s))(*s)


class _on:
    """The device of a tensor as the current one, where it is not; yields its current stream."""

    def __init__(self, t):
        self.device = t.device
        self.guard = None

    def __enter__(self):
        if torch.cuda.current_device() != self.device.index:
            self.guard = torch.cuda.device(self.device)
            self.guard.__enter__()
        return torch.cuda.current_stream(self.device).cuda_stream

    def __exit__(self, *e):
        if self.guard is not None:
            self.guard.__exit__(*e)


def _scratch(n, device):
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


def _check_tensor(name, t, dtype=None, device=None):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError('%s must be a CUDA tensor' % name)
    if dtype is None:
        if t.dtype not in _DTYPES:
            raise ValueError('%s must be float32 or bfloat16, got %s' % (name, t.dtype))
    elif t.dtype != dtype:
        raise ValueError('%s must be %s, got %s' % (name, dtype, t.dtype))
    if device is not None and t.device != device:
        raise ValueError('%s is on %s, expected %s' % (name, t.device, device))


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ---- layer norm ----

def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension of ``x``; a tensor of x's shape and type.

    ``weight`` / ``bias``  (x.size(-1),) float32 or of x's type, both of the same one; None: ones / zeros.
    Gradients reach x, weight and bias."""
    _check_tensor('x', x)
    if x.dim() < 1 or x.size(-1) < 1:
        raise ValueError('x needs a last dimension of at least one value, got %s' % (tuple(x.shape),))
    if not 0.0 <= eps < math.inf:
        raise ValueError('eps must be finite and not negative, got %r' % (eps,))
    for name, p in (('weight', weight), ('bias', bias)):
        if p is None:
            continue
        _check_tensor(name, p, device=x.device)
        if tuple(p.shape) != (x.size(-1),):
            raise ValueError('%s must have shape (%d,), got %s' % (name, x.size(-1), tuple(p.shape)))
        if p.dtype not in (torch.float32, x.dtype):
            raise ValueError('%s must be float32 or %s, got %s' % (name, x.dtype, p.dtype))
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError('weight and bias must have the same type')
    if _wants_grad(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, eps)
    return _norm_forward(x, weight, bias, eps, False)[0]


def _as_rows(x):
    """(rows, cols) with dense columns: a view of x where its strides allow, else a copy."""
    rows = x.reshape(-1, x.size(-1)) if x.numel() else x.new_empty((x.numel() // x.size(-1), x.size(-1)))
    return rows if rows.stride(1) == 1 or rows.size(1) == 1 else rows.contiguous()


def _norm_forward(x, weight, bias, eps, keep):
    rows = _as_rows(x)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stats = torch.empty((rows.size(0), 2), dtype=torch.float32, device=x.device) if keep else None
    weight = weight if weight is None else weight.contiguous()
    bias = bias if bias is None else bias.contiguous()
    wt = weight if weight is not None else bias
    with _on(x) as stream:
        _lib.check(_lib.lib().vad_layer_norm_forward(
            rows.data_ptr(), rows.size(0), rows.size(1), rows.stride(0), _ptr(weight), _ptr(bias), _DTYPES[x.dtype],
            0 if wt is None else _DTYPES[wt.dtype], eps, y.data_ptr(), _ptr(stats), stream))
    return y, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = _norm_forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, stats)
        ctx.param = None if weight is None and bias is None else (weight if weight is not None else bias).dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        rows, dyr = _as_rows(x), _as_rows(dy)
        n, cols = rows.shape
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need_x else None
        dw = torch.empty(cols, dtype=ctx.param, device=x.device) if need_w else None
        db = torch.empty(cols, dtype=ctx.param, device=x.device) if need_b else None
        L = _lib.lib()
        ws = _scratch(L.vad_layer_norm_workspace_bytes(n, cols) if need_w or need_b else 0, x.device)
        weight = weight if weight is None else weight.contiguous()
        with _on(x) as stream:
            _lib.check(L.vad_layer_norm_backward(
                rows.data_ptr(), dyr.data_ptr(), n, cols, rows.stride(0), dyr.stride(0), _ptr(weight), _DTYPES[x.dtype],
                0 if ctx.param is None else _DTYPES[ctx.param], stats.data_ptr(), _ptr(dx), _ptr(dw), _ptr(db),
                _ptr(ws), 0 if ws is None else ws.numel(), stream))
        return dx, dw, db, None


# ---- heads over sequences ----

class _Layout:
    """Shape of a call over whole sequences: checked once, kept for the backward pass."""

    def __init__(self, q, k, v, starts, max_len, shared):
        for name, t in (('q', q), ('k', k), ('v', v)):
            _check_tensor(name, t, None if name == 'q' else q.dtype, q.device)
            if t.dim() != (4 if starts is None else 3):
                raise ValueError('%s must be (batch, length, heads, dim), or (rows, heads, dim) with starts; got %s'
                                 % (name, tuple(t.shape)))
        if k.shape != v.shape or q.shape[:-2] != k.shape[:-2] or q.size(-1) != k.size(-1):
            raise ValueError('shapes of q %s, k %s and v %s do not go together' % (tuple(q.shape), tuple(k.shape), tuple(v.shape)))
        self.heads, self.dim = q.shape[-2:]
        self.kv_heads = k.size(-2)
        if self.heads < 1 or self.kv_heads < 1 or not 1 <= self.dim <= MAX_HEAD_DIM:
            raise ValueError('heads must be positive and dim 1 .. %d, got %s' % (MAX_HEAD_DIM, tuple(q.shape)))
        if self.heads % self.kv_heads or (not shared and self.heads != self.kv_heads):
            raise ValueError('%d query heads cannot use %d key heads' % (self.heads, self.kv_heads))
        self.rows_shape = q.shape[:-2]
        if starts is None:
            self.n_seq, self.max_len = q.shape[:2]
            self.n_rows = self.n_seq * self.max_len
        else:
            _check_tensor('starts', starts, torch.int64, q.device)
            if starts.dim() != 1 or starts.numel() < 1 or not starts.is_contiguous():
                raise ValueError('starts must be a contiguous 1-D tensor of at least one entry')
            self.n_seq, self.n_rows = starts.numel() - 1, q.size(0)
            if max_len is not None and max_len < 0:
                raise ValueError('max_len must not be negative, got %r' % (max_len,))
            self.max_len = self.n_rows if max_len is None else min(int(max_len), self.n_rows)
        self.n_tokens = self.n_rows if starts is not None else 0
        self.dtype = _DTYPES[q.dtype]
        self.packed = starts is not None

    def operand(self, t):
        """t with a dense head dimension, and its {sequence, row, head} strides."""
        if t.size(-1) > 1 and t.stride(-1) != 1:
            t = t.contiguous()
        return t, _strides(*((0,) + t.stride()[:2] if self.packed else t.stride()[:3]))

    def output(self, like, heads):
        # no sequence: nothing is launched that could set the rows to zero
        make = torch.zeros if self.n_seq == 0 else torch.empty
        return make(self.rows_shape + (heads, self.dim), dtype=like.dtype, device=like.device)

    def sequences(self, starts):
        return _ptr(starts), self.n_seq, self.n_tokens, self.max_len


def _scale(scale, dim):
    if scale is None:
        return dim ** -0.5
    if not math.isfinite(scale):
        raise ValueError('scale must be finite, got %r' % (scale,))
    return float(scale)


# ---- linear attention with a decay per head ----

def _check_decay(log_decay, heads, device):
    _check_tensor('log_decay', log_decay, torch.float32, device)
    if tuple(log_decay.shape) != (heads,) or not log_decay.is_contiguous():
        raise ValueError('log_decay must be a contiguous tensor of shape (%d,), got %s' % (heads, tuple(log_decay.shape)))
    if _wants_grad(log_decay):
        raise ValueError('log_decay is a constant of the operator and gets no gradient: pass log_decay.detach()')


def linear_attention(q, k, v, log_decay, scale=None, state=None, starts=None, max_len=None):
    """``S_t = exp(log_decay) S_{t-1} + k_t v_t^T``, ``o_t = scale q_t S_t`` over whole sequences; returns ``(o, state)``.

    ``log_decay``  (heads,) float32 CUDA tensor, <= 0 (values on the device are not validated: clamped into -87 .. 0).
    ``scale``      dim ** -0.5 unless given.
    ``state``      (sequences, heads, dim, dim) float32: S before the first row (None: zero).  The returned state is S behind
                   every sequence's last row, the one ``linear_attention_step`` goes on from.
    ``max_len``    longest sequence of a packed call, a hint that sizes the launch.
    Gradients reach q, k, v and state."""
    lay = _Layout(q, k, v, starts, max_len, False)
    _check_decay(log_decay, lay.heads, q.device)
    scale = _scale(scale, lay.dim)
    if state is not None:
        _check_tensor('state', state, torch.float32, q.device)
        if tuple(state.shape) != (lay.n_seq, lay.heads, lay.dim, lay.dim):
            raise ValueError('state must have shape %s, got %s' % ((lay.n_seq, lay.heads, lay.dim, lay.dim), tuple(state.shape)))
    if _wants_grad(q, k, v, state):
        return _LinearAttention.apply(q, k, v, state, log_decay, starts, scale, lay)
    return _decay_forward(q, k, v, state, log_decay, starts, scale, lay)


def _decay_forward(q, k, v, state, log_decay, starts, scale, lay):
    o = lay.output(q, lay.heads)
    out = torch.empty((lay.n_seq, lay.heads, lay.dim, lay.dim), dtype=torch.float32, device=q.device)
    (q, qs), (k, ks), (v, vs) = lay.operand(q), lay.operand(k), lay.operand(v)
    state = state if state is None else state.contiguous()
    L = _lib.lib()
    ws = _scratch(L.vad_linear_attention_workspace_bytes(lay.n_seq, lay.max_len, lay.heads, lay.dim, 0), q.device)
    with _on(q) as stream:
        _lib.check(L.vad_linear_attention_forward(
            q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, *lay.sequences(starts), lay.heads, lay.dim, lay.dtype,
            log_decay.data_ptr(), scale, _ptr(state), o.data_ptr(), out.data_ptr(), _ptr(ws),
            0 if ws is None else ws.numel(), stream))
    return o, out


class _LinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, state, log_decay, starts, scale, lay):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, v, state, log_decay, starts)
        ctx.scale, ctx.lay = scale, lay
        return _decay_forward(q, k, v, state, log_decay, starts, scale, lay)

    @staticmethod
    @once_differentiable
    def backward(ctx, do, dstate):
        q, k, v, state, log_decay, starts = ctx.saved_tensors
        lay = ctx.lay
        if do is None and dstate is None:
            return (None,) * 8
        do = torch.zeros_like(q) if do is None else do
        dstate = dstate if dstate is None else dstate.contiguous()
        dq, dk, dv = (lay.output(q, lay.heads) for _ in range(3))
        need_state = state is not None and ctx.needs_input_grad[3]
        dstate_in = torch.empty(state.shape, dtype=torch.float32, device=q.device) if need_state else None
        state = state if state is None else state.contiguous()
        (q, qs), (k, ks), (v, vs), (do, gs) = (lay.operand(t) for t in (q, k, v, do))
        L = _lib.lib()
        ws = _scratch(L.vad_linear_attention_workspace_bytes(lay.n_seq, lay.max_len, lay.heads, lay.dim, 1), q.device)
        with _on(q) as stream:
            _lib.check(L.vad_linear_attention_backward(
                q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, do.data_ptr(), gs, *lay.sequences(starts), lay.heads, lay.dim,
                lay.dtype, log_decay.data_ptr(), ctx.scale, _ptr(state), _ptr(dstate), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                _ptr(dstate_in), _ptr(ws), 0 if ws is None else ws.numel(), stream))
        return dq, dk, dv, dstate_in, None, None, None, None


def _step_operands(q, k, v, shared):
    for name, t in (('q', q), ('k', k), ('v', v)):
        _check_tensor(name, t, None if name == 'q' else q.dtype, q.device)
        if t.dim() != 3:
            raise ValueError('%s must be (batch, heads, dim), got %s' % (name, tuple(t.shape)))
    if k.shape != v.shape or q.size(0) != k.size(0) or q.size(2) != k.size(2):
        raise ValueError('shapes of q %s, k %s and v %s do not go together' % (tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    heads, dim, kv_heads = q.size(1), q.size(2), k.size(1)
    if heads < 1 or kv_heads < 1 or not 1 <= dim <= MAX_HEAD_DIM:
        raise ValueError('heads must be positive and dim 1 .. %d, got %s' % (MAX_HEAD_DIM, tuple(q.shape)))
    if heads % kv_heads or (not shared and heads != kv_heads):
        raise ValueError('%d query heads cannot use %d key heads' % (heads, kv_heads))
    out = []
    for t in (q, k, v):
        t = t if dim == 1 or t.stride(2) == 1 else t.contiguous()
        out.append((t, _strides(t.stride(0), t.stride(1))))
    return out


def linear_attention_step(q, k, v, log_decay, state, scale=None):
    """One row of ``linear_attention`` per sequence: q, k, v (batch, heads, dim); ``state`` (batch, heads, dim, dim) float32,
    contiguous, is updated in place.  Returns o (batch, heads, dim).  Inference only."""
    (q, qs), (k, ks), (v, vs) = _step_operands(q, k, v, False)
    batch, heads, dim = q.shape
    _check_decay(log_decay, heads, q.device)
    scale = _scale(scale, dim)
    _check_tensor('state', state, torch.float32, q.device)
    if tuple(state.shape) != (batch, heads, dim, dim) or not state.is_contiguous():
        raise ValueError('state must be a contiguous tensor of shape %s, got %s' % ((batch, heads, dim, dim), tuple(state.shape)))
    if _wants_grad(q, k, v, state):
        raise ValueError('linear_attention_step has no gradient: call it under torch.no_grad(), or use linear_attention')
    o = torch.empty((batch, heads, dim), dtype=q.dtype, device=q.device)
    with _on(q) as stream:
        _lib.check(_lib.lib().vad_linear_attention_step(
            q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, batch, heads, dim, _DTYPES[q.dtype], log_decay.data_ptr(), scale,
            state.data_ptr(), o.data_ptr(), stream))
    return o


# ---- attention with a sliding window and sinks ----

def _check_window(window, sinks, scale, dim):
    if not 1 <= window <= 1 << 30:
        raise ValueError('window must be 1 .. 2^30, got %r' % (window,))
    if not 0 <= sinks <= MAX_SINKS:
        raise ValueError('sinks must be 0 .. %d, got %r' % (MAX_SINKS, sinks))
    scale = _scale(scale, dim)
    if scale <= 0.0:
        raise ValueError('scale must be positive, got %r' % (scale,))
    return int(window), int(sinks), scale


def window_attention(q, k, v, window, sinks=0, scale=None, starts=None, max_len=None):
    """Softmax attention in which row i sees key j when ``j <= i`` and (``i - j < window`` or ``j < sinks``).

    ``window``  rows that a row sees, itself included; ``sinks`` 0 .. 64 first rows that stay visible.
    ``k``, ``v``  may have fewer heads than q: query head h reads key head ``h // (heads // kv_heads)``.
    ``scale``   positive, dim ** -0.5 unless given.  ``max_len`` as in ``linear_attention``.
    Returns a tensor of q's shape; gradients reach q, k and v."""
    lay = _Layout(q, k, v, starts, max_len, True)
    window, sinks, scale = _check_window(window, sinks, scale, lay.dim)
    if _wants_grad(q, k, v):
        return _WindowAttention.apply(q, k, v, starts, window, sinks, scale, lay)
    return _window_forward(q, k, v, starts, window, sinks, scale, lay, False)[0]


def _window_forward(q, k, v, starts, window, sinks, scale, lay, keep):
    o = lay.output(q, lay.heads)
    stats = torch.empty((lay.n_rows, lay.heads, 2), dtype=torch.float32, device=q.device) if keep else None
    (q, qs), (k, ks), (v, vs) = lay.operand(q), lay.operand(k), lay.operand(v)
    with _on(q) as stream:
        _lib.check(_lib.lib().vad_window_attention_forward(
            q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, *lay.sequences(starts), lay.heads, lay.kv_heads, lay.dim, lay.dtype,
            window, sinks, scale, o.data_ptr(), _ptr(stats), stream))
    return o, stats


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, starts, window, sinks, scale, lay):
        o, stats = _window_forward(q, k, v, starts, window, sinks, scale, lay, True)
        ctx.save_for_backward(q, k, v, o, stats, starts)
        ctx.call = window, sinks, scale
        ctx.lay = lay
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        q, k, v, o, stats, starts = ctx.saved_tensors
        lay = ctx.lay
        window, sinks, scale = ctx.call
        dq, dk, dv = lay.output(q, lay.heads), lay.output(q, lay.kv_heads), lay.output(q, lay.kv_heads)
        (q, qs), (k, ks), (v, vs), (do, gs) = (lay.operand(t) for t in (q, k, v, do))
        L = _lib.lib()
        ws = _scratch(L.vad_window_attention_workspace_bytes(lay.n_seq, lay.n_rows, lay.max_len, lay.heads, lay.kv_heads, lay.dim,
                                                             window, sinks), q.device)
        with _on(q) as stream:
            _lib.check(L.vad_window_attention_backward(
                q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, o.data_ptr(), do.data_ptr(), gs, stats.data_ptr(),
                *lay.sequences(starts), lay.heads, lay.kv_heads, lay.dim, lay.dtype, window, sinks, scale, dq.data_ptr(),
                dk.data_ptr(), dv.data_ptr(), _ptr(ws), 0 if ws is None else ws.numel(), stream))
        return dq, dk, dv, None, None, None, None, None


def _check_cache(name, c, batch, window, sinks, kv_heads, dim, dtype, device):
    _check_tensor(name, c, dtype, device)
    if tuple(c.shape) != (batch, sinks + window, kv_heads, dim):
        raise ValueError('%s must have shape %s, got %s' % (name, (batch, sinks + window, kv_heads, dim), tuple(c.shape)))
    if dim > 1 and c.stride(3) != 1 or any(n > 1 and s == 0 for n, s in zip(c.shape, c.stride())):
        raise ValueError('%s must have a dense last dimension and no broadcast one' % name)
    return _strides(*c.stride()[:3])


def window_attention_step(q, k, v, cache_k, cache_v, pos, window, sinks=0, scale=None):
    """One row of ``window_attention`` per sequence against its rolling cache.

    ``q`` (batch, heads, dim), ``k`` / ``v`` (batch, kv_heads, dim): the new row.
    ``cache_k`` / ``cache_v``  (batch, sinks + window, kv_heads, dim) of q's type, updated in place: row p goes to slot p
               while p < sinks, then to ``sinks + (p - sinks) % window``.
    ``pos``    (batch,) int64 CUDA tensor: rows the sequence has had before this one; not changed.  Where it is negative
               the output is zero and the cache stays as it is.
    Returns o (batch, heads, dim).  Inference only."""
    (q, qs), (k, ks), (v, vs) = _step_operands(q, k, v, True)
    batch, heads, dim = q.shape
    kv_heads = k.size(1)
    window, sinks, scale = _check_window(window, sinks, scale, dim)
    cks = _check_cache('cache_k', cache_k, batch, window, sinks, kv_heads, dim, q.dtype, q.device)
    cvs = _check_cache('cache_v', cache_v, batch, window, sinks, kv_heads, dim, q.dtype, q.device)
    _check_tensor('pos', pos, torch.int64, q.device)
    if tuple(pos.shape) != (batch,) or not pos.is_contiguous():
        raise ValueError('pos must be a contiguous tensor of shape (%d,), got %s' % (batch, tuple(pos.shape)))
    if _wants_grad(q, k, v, cache_k, cache_v):
        raise ValueError('window_attention_step has no gradient: call it under torch.no_grad(), or use window_attention')
    o = torch.empty((batch, heads, dim), dtype=q.dtype, device=q.device)
    L = _lib.lib()
    ws = _scratch(L.vad_window_step_workspace_bytes(batch, heads, kv_heads, dim, window, sinks), q.device)
    with _on(q) as stream:
        _lib.check(L.vad_window_attention_step(
            q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, cache_k.data_ptr(), cks, cache_v.data_ptr(), cvs, pos.data_ptr(), batch,
            heads, kv_heads, dim, _DTYPES[q.dtype], window, sinks, scale, o.data_ptr(), _ptr(ws), 0 if ws is None else ws.numel(), stream))
    return o


def window_cache_fill(k, v, cache_k, cache_v, window, sinks=0, starts=None):
    """Keys and values of whole sequences into rolling caches, as the steps after them expect it: (batch, length, kv_heads,
    dim), or packed with ``starts``.  Slots that no row belongs to stay as they are.  Returns ``pos`` (batch,) int64: the
    lengths."""
    lay = _Layout(k, k, v, starts, None, True)
    window, sinks, _ = _check_window(window, sinks, None, lay.dim)
    cks = _check_cache('cache_k', cache_k, lay.n_seq, window, sinks, lay.heads, lay.dim, k.dtype, k.device)
    cvs = _check_cache('cache_v', cache_v, lay.n_seq, window, sinks, lay.heads, lay.dim, k.dtype, k.device)
    pos = torch.empty(lay.n_seq, dtype=torch.int64, device=k.device)
    (k, ks), (v, vs) = lay.operand(k), lay.operand(v)
    with _on(k) as stream:
        _lib.check(_lib.lib().vad_window_cache_fill(
            k.data_ptr(), ks, v.data_ptr(), vs, *lay.sequences(starts), lay.heads, lay.dim, lay.dtype, window, sinks,
            cache_k.data_ptr(), cks, cache_v.data_ptr(), cvs, pos.data_ptr(), stream))
    return pos
