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
import functools
import math
import operator

import torch
from torch._C import _cuda_getCurrentRawStream, _cuda_getDevice
from torch._C import _len_torch_dispatch_stack as _dispatch_modes
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

MAX_HEAD_DIM = 128
MAX_SINKS = 64
MAX_ROW_STRIDE = 1 << 22
_DTYPES = {torch.float32: 0, torch.bfloat16: 1}

# A call's host time is a good part of a live frame's: what follows from shapes and strides alone (checks, stride tables,
# workspace sizes) is worked out once per shape and remembered by it; checks that touch the tensors are spelled out inline
# and explained only after they have failed.


def _ptr(t):
    return None if t is None else t.data_ptr()


def _strides(*s):
    return (ctypes.c_int64 * len(s))(*s)


def _call(fn, device, *args):
    """fn on the current stream of ``device`` (an index), with that device as the current one."""
    if _dispatch_modes() and torch._C._get_dispatch_mode(torch._C._TorchDispatchModeKey.PROXY) is not None:
        _refuse_tracing(None)
    if device == _cuda_getDevice():
        rc = fn(*args, _cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _cuda_getCurrentRawStream(device))
    if rc:
        _lib.check(rc)


def _written(*tensors):
    """Tensors that a call updates in place: a graph that saved one of them then refuses its backward pass."""
    torch._C._increment_version(tensors)


def _scratch(n, like):
    return like.new_empty(n, dtype=torch.uint8) if n else None


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


def _check_like(q, k, v):
    """q, k and v: CUDA tensors of one device and type."""
    if type(q) is type(k) is type(v) is torch.Tensor and q.is_cuda and q.dtype in _DTYPES and q.dtype is k.dtype is v.dtype \
            and q.get_device() == k.get_device() == v.get_device():
        return
    _check_tensor('q', q)
    _check_tensor('k', k, q.dtype, q.device)
    _check_tensor('v', v, q.dtype, q.device)


def _refuse_tangents(*tensors):
    """Derivatives in forward mode: a dual tensor does not ask for a gradient, and the kernels write plain tensors -- the result's
    tangent would read as zero.  (Called only inside a dual level.)"""
    for t in tensors:
        if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError('the sequence operators have no forward-mode derivatives')


def _refuse_tracing(size):
    """Calls under torch.jit.trace, where sizes are tensors, or make_fx (``_call``): a trace records torch's operators, and of these
    calls only the empty tensor that they write into."""
    if type(size) is not int:
        raise ValueError('calls of the sequence operators cannot be traced')


def _dense(t):
    return t if t.size(-1) <= 1 or t.stride(-1) == 1 else t.contiguous()


def _once(backward):
    """A backward pass that raises where its results are differentiated again, without once_differentiable's cost where the
    graph is not kept for that."""
    guarded = once_differentiable(backward)

    def run(ctx, *grads):
        if forward_ad._current_level >= 0:
            _refuse_tangents(*grads)
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return run


# ---- layer norm ----

def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension of ``x``; a tensor of x's shape and type.

    ``weight`` / ``bias``  (x.size(-1),) float32 or of x's type, both of the same one; None: ones / zeros.
    Gradients reach x, weight and bias."""
    if forward_ad._current_level >= 0:
        _refuse_tangents(x, weight, bias)
    _check_tensor('x', x)
    if x.dim() < 1 or x.size(-1) < 1:
        raise ValueError('x needs a last dimension of at least one value, got %s' % (tuple(x.shape),))
    _refuse_tracing(x.size(-1))
    if not 0.0 <= eps < math.inf:
        raise ValueError('eps must be finite and not negative, got %r' % (eps,))
    for name, p in (('weight', weight), ('bias', bias)):
        if p is None:
            continue
        _check_tensor(name, p, p.dtype if isinstance(p, torch.Tensor) else None)
        if p.get_device() != x.get_device():
            raise ValueError('%s is on %s, expected %s' % (name, p.device, x.device))
        if p.dim() != 1 or p.size(0) != x.size(-1):
            raise ValueError('%s must have shape (%d,), got %s' % (name, x.size(-1), tuple(p.shape)))
        if p.dtype is not torch.float32 and p.dtype is not x.dtype:
            raise ValueError('%s must be float32 or %s, got %s' % (name, x.dtype, p.dtype))
    if weight is not None and bias is not None and weight.dtype is not bias.dtype:
        raise ValueError('weight and bias must have the same type')
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or
                                    (bias is not None and bias.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, eps)
    return _norm_forward(x, weight, bias, eps, False)[0]


@functools.lru_cache(maxsize=1024)
def _norm_workspace(n, cols):
    return _lib.lib().vad_layer_norm_workspace_bytes(n, cols)


def _as_rows(x):
    """(rows, cols) with dense columns: a view of x where its strides allow, else a copy."""
    if x.dim() == 2 and x.stride(1) == 1:
        return x
    rows = x.reshape(-1, x.size(-1)) if x.numel() else x.new_empty((x.numel() // x.size(-1), x.size(-1)))
    return rows if rows.stride(1) == 1 or rows.size(1) == 1 else rows.contiguous()


def _norm_forward(x, weight, bias, eps, keep):
    rows = _as_rows(x)
    n, cols = rows.shape
    y = x.new_empty(x.shape)
    stats = x.new_empty((n, 2), dtype=torch.float32) if keep else None
    wt = 0
    if weight is not None:
        weight = weight if weight.is_contiguous() else weight.contiguous()
        wt = _DTYPES[weight.dtype]
    if bias is not None:
        bias = bias if bias.is_contiguous() else bias.contiguous()
        wt = _DTYPES[bias.dtype]
    _call(_lib.lib().vad_layer_norm_forward, x.get_device(), rows.data_ptr(), n, cols, rows.stride(0), _ptr(weight), _ptr(bias),
          _DTYPES[x.dtype], wt, eps, y.data_ptr(), _ptr(stats))
    return y, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = _norm_forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, stats)
        ctx.eps = eps
        ctx.param = None if weight is None and bias is None else (weight if weight is not None else bias).dtype
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        rows, dyr = _as_rows(x), _as_rows(dy)
        n, cols = rows.shape
        dx = x.new_empty(x.shape) if need_x else None
        dw = stats.new_empty(cols, dtype=ctx.param) if need_w else None
        db = stats.new_empty(cols, dtype=ctx.param) if need_b else None
        size = _norm_workspace(n, cols) if need_w or need_b else 0
        ws = _scratch(size, x)
        if weight is not None and not weight.is_contiguous():
            weight = weight.contiguous()
        _call(_lib.lib().vad_layer_norm_backward, x.get_device(), rows.data_ptr(), dyr.data_ptr(), n, cols, rows.stride(0), dyr.stride(0),
              _ptr(weight), _DTYPES[x.dtype], 0 if ctx.param is None else _DTYPES[ctx.param], ctx.eps, stats.data_ptr(), _ptr(dx), _ptr(dw),
              _ptr(db), _ptr(ws), size)
        return dx, dw, db, None


# ---- heads over sequences ----

class _Layout:
    """What the shapes of a call over whole sequences say; one object per combination, see ``_layout``."""

    def __init__(self, qs, ks, vs, n_starts, max_len, shared):
        if qs:
            _refuse_tracing(qs[-1])
        for name, s in (('q', qs), ('k', ks), ('v', vs)):
            if len(s) != (4 if n_starts is None else 3):
                raise ValueError('%s must be (batch, length, heads, dim), or (rows, heads, dim) with starts; got %s' % (name, tuple(s)))
        if ks != vs or qs[:-2] != ks[:-2] or qs[-1] != ks[-1]:
            raise ValueError('shapes of q %s, k %s and v %s do not go together' % (tuple(qs), tuple(ks), tuple(vs)))
        self.heads, self.dim = qs[-2:]
        self.kv_heads = ks[-2]
        if self.heads < 1 or self.kv_heads < 1 or not 1 <= self.dim <= MAX_HEAD_DIM:
            raise ValueError('heads must be positive and dim 1 .. %d, got %s' % (MAX_HEAD_DIM, tuple(qs)))
        if self.heads % self.kv_heads or (not shared and self.heads != self.kv_heads):
            raise ValueError('%d query heads cannot use %d key heads' % (self.heads, self.kv_heads))
        self.packed = n_starts is not None
        self.one_row = qs[-3] <= 1          # its stride says nothing, and a copy would not change it
        if self.packed:
            self.n_seq, self.n_rows = n_starts - 1, qs[0]
            if max_len is not None and max_len < 0:
                raise ValueError('max_len must not be negative, got %r' % (max_len,))
            self.max_len = self.n_rows if max_len is None else min(max_len, self.n_rows)
            self.sequences = self.n_seq, self.n_rows, self.max_len
        else:
            self.n_seq, self.max_len = qs[:2]
            self.n_rows = self.n_seq * self.max_len
            self.sequences = self.n_seq, 0, self.max_len
        self.state_shape = (self.n_seq, self.heads, self.dim, self.dim)
        self.table = functools.lru_cache(maxsize=64)(self._table)

    def _table(self, s):
        sequence, row, head = (0, *s[:2]) if self.packed else s[:3]
        return _strides(sequence, self.dim if self.one_row else row, head)

    def operand(self, t):
        """t with a dense head dimension, and its {sequence, row, head} strides.  Rows too far apart for the kernels are brought
        together; rows that overlap, which they would read value by value, are taken apart."""
        t = _dense(t)
        if not self.dim <= t.stride(-3) < MAX_ROW_STRIDE and not self.one_row:
            t = t.contiguous()
        return t, self.table(t.stride())

    def output(self, like):
        # no sequence: nothing is launched that could set the rows to zero
        return like.new_empty(like.shape) if self.n_seq else like.new_zeros(like.shape)

    @functools.cached_property
    def decay_workspace(self):
        size = _lib.lib().vad_linear_attention_workspace_bytes
        return [size(self.n_seq, self.max_len, self.heads, self.dim, back) for back in (0, 1)]

    @functools.lru_cache(maxsize=64)
    def window_workspace(self, window, sinks):
        return _lib.lib().vad_window_attention_workspace_bytes(self.n_seq, self.n_rows, self.max_len, self.heads, self.kv_heads,
                                                               self.dim, window, sinks)


_layout_of = functools.lru_cache(maxsize=256)(_Layout)


def _layout(q, k, v, starts, max_len, shared):
    _check_like(q, k, v)
    if starts is None:
        return _layout_of(q.shape, k.shape, v.shape, None, None, shared)
    _check_tensor('starts', starts, torch.int64, q.device)
    if starts.dim() != 1 or starts.numel() < 1 or not starts.is_contiguous():
        raise ValueError('starts must be a contiguous 1-D tensor of at least one entry')
    return _layout_of(q.shape, k.shape, v.shape, starts.numel(), None if max_len is None else operator.index(max_len), shared)


def _scale(scale, dim):
    if scale is None:
        return dim ** -0.5
    if not math.isfinite(scale):
        raise ValueError('scale must be finite, got %r' % (scale,))
    return float(scale)


# ---- linear attention with a decay per head ----

def _check_decay(log_decay, heads, like):
    if type(log_decay) is not torch.Tensor or log_decay.dtype is not torch.float32 or log_decay.get_device() != like.get_device():
        _check_tensor('log_decay', log_decay, torch.float32, like.device)
    if log_decay.dim() != 1 or log_decay.size(0) != heads or not log_decay.is_contiguous():
        raise ValueError('log_decay must be a contiguous tensor of shape (%d,), got %s' % (heads, tuple(log_decay.shape)))
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise ValueError('log_decay is a constant of the operator and gets no gradient: pass log_decay.detach()')


def linear_attention(q, k, v, log_decay, scale=None, state=None, starts=None, max_len=None):
    """``S_t = exp(log_decay) S_{t-1} + k_t v_t^T``, ``o_t = scale q_t S_t`` over whole sequences; returns ``(o, state)``.

    ``log_decay``  (heads,) float32 CUDA tensor, <= 0 (values on the device are not validated: clamped into -87 .. 0).
    ``scale``      dim ** -0.5 unless given.
    ``state``      (sequences, heads, dim, dim) float32: S before the first row (None: zero).  The returned state is S behind
                   every sequence's last row, the one ``linear_attention_step`` goes on from.
    ``max_len``    longest sequence of a packed call, a hint that sizes the launch.
    Gradients reach q, k, v and state."""
    if forward_ad._current_level >= 0:
        _refuse_tangents(q, k, v, log_decay, state)
    lay = _layout(q, k, v, starts, max_len, False)
    _check_decay(log_decay, lay.heads, q)
    scale = _scale(scale, lay.dim)
    if state is not None:
        _check_tensor('state', state, torch.float32, q.device)
        if state.shape != lay.state_shape:
            raise ValueError('state must have shape %s, got %s' % (lay.state_shape, tuple(state.shape)))
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or (state is not None and state.requires_grad)):
        return _LinearAttention.apply(q, k, v, state, log_decay, starts, scale, lay)
    return _decay_forward(q, k, v, state, log_decay, starts, scale, lay)


def _decay_forward(q, k, v, state, log_decay, starts, scale, lay):
    o = lay.output(q)
    out = q.new_empty(lay.state_shape, dtype=torch.float32)
    (q, qs), (k, ks), (v, vs) = lay.operand(q), lay.operand(k), lay.operand(v)
    state = state if state is None else state.contiguous()
    size = lay.decay_workspace[0]
    ws = _scratch(size, q)
    _call(_lib.lib().vad_linear_attention_forward, q.get_device(), q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, _ptr(starts),
          *lay.sequences, lay.heads, lay.dim, _DTYPES[q.dtype], log_decay.data_ptr(), scale, _ptr(state), o.data_ptr(), out.data_ptr(),
          _ptr(ws), size)
    return o, out


class _LinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, state, log_decay, starts, scale, lay):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, v, state, log_decay, starts)
        ctx.scale, ctx.lay = scale, lay
        return _decay_forward(q, k, v, state, log_decay, starts, scale, lay)

    @staticmethod
    @_once
    def backward(ctx, do, dstate):
        q, k, v, state, log_decay, starts = ctx.saved_tensors
        lay = ctx.lay
        if do is None and dstate is None:
            return (None,) * 8
        do = torch.zeros_like(q) if do is None else do
        dstate = dstate if dstate is None else dstate.contiguous()
        dq, dk, dv = lay.output(q), lay.output(k), lay.output(v)
        need_state = state is not None and ctx.needs_input_grad[3]
        dstate_in = torch.empty(lay.state_shape, dtype=torch.float32, device=q.device) if need_state else None
        state = state if state is None else state.contiguous()
        (q, qs), (k, ks), (v, vs), (do, gs) = lay.operand(q), lay.operand(k), lay.operand(v), lay.operand(do)
        size = lay.decay_workspace[1]
        ws = _scratch(size, q)
        _call(_lib.lib().vad_linear_attention_backward, q.get_device(), q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, do.data_ptr(),
              gs, _ptr(starts), *lay.sequences, lay.heads, lay.dim, _DTYPES[q.dtype], log_decay.data_ptr(), ctx.scale, _ptr(state),
              _ptr(dstate), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _ptr(dstate_in), _ptr(ws), size)
        return dq, dk, dv, dstate_in, None, None, None, None


@functools.lru_cache(maxsize=256)
def _step_shapes(qs, ks, vs, shared):
    if qs:
        _refuse_tracing(qs[-1])
    for name, s in (('q', qs), ('k', ks), ('v', vs)):
        if len(s) != 3:
            raise ValueError('%s must be (batch, heads, dim), got %s' % (name, tuple(s)))
    if ks != vs or qs[0] != ks[0] or qs[2] != ks[2]:
        raise ValueError('shapes of q %s, k %s and v %s do not go together' % (tuple(qs), tuple(ks), tuple(vs)))
    batch, heads, dim = qs
    kv_heads = ks[1]
    if heads < 1 or kv_heads < 1 or not 1 <= dim <= MAX_HEAD_DIM:
        raise ValueError('heads must be positive and dim 1 .. %d, got %s' % (MAX_HEAD_DIM, tuple(qs)))
    if heads % kv_heads or (not shared and heads != kv_heads):
        raise ValueError('%d query heads cannot use %d key heads' % (heads, kv_heads))
    return batch, heads, kv_heads, dim, (batch, heads, dim, dim)


@functools.lru_cache(maxsize=1024)
def _step_table(s):
    return _strides(*s[:-1])


def _step_operands(q, k, v):
    q, k, v = _dense(q), _dense(k), _dense(v)
    return q, _step_table(q.stride()), k, _step_table(k.stride()), v, _step_table(v.stride())


def linear_attention_step(q, k, v, log_decay, state, scale=None):
    """One row of ``linear_attention`` per sequence: q, k, v (batch, heads, dim); ``state`` (batch, heads, dim, dim) float32,
    contiguous, is updated in place.  Returns o (batch, heads, dim).  Inference only."""
    if forward_ad._current_level >= 0:
        _refuse_tangents(q, k, v, log_decay, state)
    _check_like(q, k, v)
    batch, heads, _, dim, state_shape = _step_shapes(q.shape, k.shape, v.shape, False)
    _check_decay(log_decay, heads, q)
    scale = _scale(scale, dim)
    if type(state) is not torch.Tensor or state.dtype is not torch.float32 or state.get_device() != q.get_device():
        _check_tensor('state', state, torch.float32, q.device)
    if state.shape != state_shape or not state.is_contiguous():
        raise ValueError('state must be a contiguous tensor of shape %s, got %s' % (state_shape, tuple(state.shape)))
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or state.requires_grad):
        raise ValueError('linear_attention_step has no gradient: call it under torch.no_grad(), or use linear_attention')
    o = q.new_empty(q.shape)
    q, qs, k, ks, v, vs = _step_operands(q, k, v)
    _call(_lib.lib().vad_linear_attention_step, q.get_device(), q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, batch, heads, dim,
          _DTYPES[q.dtype], log_decay.data_ptr(), scale, state.data_ptr(), o.data_ptr())
    _written(state)
    return o


# ---- attention with a sliding window and sinks ----

def _check_window(window, sinks, scale, dim):
    window, sinks = operator.index(window), operator.index(sinks)
    if not 1 <= window <= 1 << 30:
        raise ValueError('window must be 1 .. 2^30, got %r' % (window,))
    if not 0 <= sinks <= MAX_SINKS:
        raise ValueError('sinks must be 0 .. %d, got %r' % (MAX_SINKS, sinks))
    scale = _scale(scale, dim)
    if scale <= 0.0:
        raise ValueError('scale must be positive, got %r' % (scale,))
    return window, sinks, scale


def window_attention(q, k, v, window, sinks=0, scale=None, starts=None, max_len=None):
    """Softmax attention in which row i sees key j when ``j <= i`` and (``i - j < window`` or ``j < sinks``).

    ``window``  rows that a row sees, itself included; ``sinks`` 0 .. 64 first rows that stay visible.
    ``k``, ``v``  may have fewer heads than q: query head h reads key head ``h // (heads // kv_heads)``.
    ``scale``   positive, dim ** -0.5 unless given.  ``max_len`` as in ``linear_attention``.
    Returns a tensor of q's shape; gradients reach q, k and v."""
    if forward_ad._current_level >= 0:
        _refuse_tangents(q, k, v)
    lay = _layout(q, k, v, starts, max_len, True)
    window, sinks, scale = _check_window(window, sinks, scale, lay.dim)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _WindowAttention.apply(q, k, v, starts, window, sinks, scale, lay)
    return _window_forward(q, k, v, starts, window, sinks, scale, lay, False)[0]


def _window_forward(q, k, v, starts, window, sinks, scale, lay, keep):
    o = lay.output(q)
    stats = q.new_empty((lay.n_rows, lay.heads, 2), dtype=torch.float32) if keep else None
    (q, qs), (k, ks), (v, vs) = lay.operand(q), lay.operand(k), lay.operand(v)
    _call(_lib.lib().vad_window_attention_forward, q.get_device(), q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, _ptr(starts),
          *lay.sequences, lay.heads, lay.kv_heads, lay.dim, _DTYPES[q.dtype], window, sinks, scale, o.data_ptr(), _ptr(stats))
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
    @_once
    def backward(ctx, do):
        q, k, v, o, stats, starts = ctx.saved_tensors
        lay = ctx.lay
        window, sinks, scale = ctx.call
        dq, dk, dv = lay.output(q), lay.output(k), lay.output(v)
        (q, qs), (k, ks), (v, vs), (do, gs) = lay.operand(q), lay.operand(k), lay.operand(v), lay.operand(do)
        size = lay.window_workspace(window, sinks)
        ws = _scratch(size, q)
        _call(_lib.lib().vad_window_attention_backward, q.get_device(), q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, o.data_ptr(),
              do.data_ptr(), gs, stats.data_ptr(), _ptr(starts), *lay.sequences, lay.heads, lay.kv_heads, lay.dim, _DTYPES[q.dtype], window,
              sinks, scale, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _ptr(ws), size)
        return dq, dk, dv, None, None, None, None, None


@functools.lru_cache(maxsize=1024)
def _cache_table(name, shape, stride, batch, slots, kv_heads, dim):
    want = (batch, slots, kv_heads, dim)
    if shape != want:
        raise ValueError('%s must have shape %s, got %s' % (name, want, tuple(shape)))
    if dim > 1 and stride[3] != 1 or any(n > 1 and s == 0 for n, s in zip(shape, stride)):
        raise ValueError('%s must have a dense last dimension and no broadcast one' % name)
    return _strides(*stride[:3])


def _check_apart(k, v):
    if k.data_ptr() == v.data_ptr() and k.numel():
        raise ValueError('cache_k and cache_v are the same memory')


def _check_cache(name, c, like, batch, slots, kv_heads, dim):
    if type(c) is not torch.Tensor or c.dtype is not like.dtype or c.get_device() != like.get_device():
        _check_tensor(name, c, like.dtype, like.device)
    return _cache_table(name, c.shape, c.stride(), batch, slots, kv_heads, dim)


@functools.lru_cache(maxsize=1024)
def _step_workspace(batch, heads, kv_heads, dim, window, sinks):
    return _lib.lib().vad_window_step_workspace_bytes(batch, heads, kv_heads, dim, window, sinks)


def window_attention_step(q, k, v, cache_k, cache_v, pos, window, sinks=0, scale=None):
    """One row of ``window_attention`` per sequence against its rolling cache.

    ``q`` (batch, heads, dim), ``k`` / ``v`` (batch, kv_heads, dim): the new row.
    ``cache_k`` / ``cache_v``  (batch, sinks + window, kv_heads, dim) of q's type, updated in place: row p goes to slot p
               while p < sinks, then to ``sinks + (p - sinks) % window``.
    ``pos``    (batch,) int64 CUDA tensor: rows the sequence has had before this one; not changed.  Where it is negative
               the output is zero and the cache stays as it is.
    Returns o (batch, heads, dim).  Inference only."""
    if forward_ad._current_level >= 0:
        _refuse_tangents(q, k, v, cache_k, cache_v)
    _check_like(q, k, v)
    batch, heads, kv_heads, dim, _ = _step_shapes(q.shape, k.shape, v.shape, True)
    window, sinks, scale = _check_window(window, sinks, scale, dim)
    cks = _check_cache('cache_k', cache_k, q, batch, sinks + window, kv_heads, dim)
    cvs = _check_cache('cache_v', cache_v, q, batch, sinks + window, kv_heads, dim)
    _check_tensor('pos', pos, torch.int64, q.device)
    if pos.dim() != 1 or pos.size(0) != batch or not pos.is_contiguous():
        raise ValueError('pos must be a contiguous tensor of shape (%d,), got %s' % (batch, tuple(pos.shape)))
    _check_apart(cache_k, cache_v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or cache_k.requires_grad or cache_v.requires_grad):
        raise ValueError('window_attention_step has no gradient: call it under torch.no_grad(), or use window_attention')
    o = q.new_empty(q.shape)
    q, qs, k, ks, v, vs = _step_operands(q, k, v)
    size = _step_workspace(batch, heads, kv_heads, dim, window, sinks)
    ws = _scratch(size, q)
    _call(_lib.lib().vad_window_attention_step, q.get_device(), q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, cache_k.data_ptr(),
          cks, cache_v.data_ptr(), cvs, pos.data_ptr(), batch, heads, kv_heads, dim, _DTYPES[q.dtype], window, sinks, scale, o.data_ptr(),
          _ptr(ws), size)
    _written(cache_k, cache_v)
    return o


def window_cache_fill(k, v, cache_k, cache_v, window, sinks=0, starts=None):
    """Keys and values of whole sequences into rolling caches, as the steps after them expect it: (batch, length, kv_heads,
    dim), or packed with ``starts``.  Slots that no row belongs to stay as they are.  Returns ``pos`` (batch,) int64: the
    lengths.  Inference only."""
    if forward_ad._current_level >= 0:
        _refuse_tangents(k, v, cache_k, cache_v)
    lay = _layout(k, k, v, starts, None, True)
    window, sinks, _ = _check_window(window, sinks, None, lay.dim)
    cks = _check_cache('cache_k', cache_k, k, lay.n_seq, sinks + window, lay.heads, lay.dim)
    cvs = _check_cache('cache_v', cache_v, k, lay.n_seq, sinks + window, lay.heads, lay.dim)
    _check_apart(cache_k, cache_v)
    if torch.is_grad_enabled() and (k.requires_grad or v.requires_grad or cache_k.requires_grad or cache_v.requires_grad):
        raise ValueError('window_cache_fill has no gradient: call it under torch.no_grad()')
    pos = torch.empty(lay.n_seq, dtype=torch.int64, device=k.device)
    (k, ks), (v, vs) = lay.operand(k), lay.operand(v)
    _call(_lib.lib().vad_window_cache_fill, k.get_device(), k.data_ptr(), ks, v.data_ptr(), vs, _ptr(starts), *lay.sequences, lay.heads,
          lay.dim, _DTYPES[k.dtype], window, sinks, cache_k.data_ptr(), cks, cache_v.data_ptr(), cvs, pos.data_ptr())
    _written(cache_k, cache_v)
    return pos
