"""The sequence operators without a GPU: argument checks of the C entry points and of the Python host side, and the
float64 forms the GPU tests compare against, checked against the recurrence and torch's autograd."""
import ctypes
import math

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

import voice_activity_detection_amd as pkg
from oracle import sequence_ref as ref


@pytest.fixture(scope='module')
def L():
    pkg.build()
    return pkg.lib()


def _strides(*s):
    return (ctypes.c_int64 * len(s))(*s)


def test_c_entry_points_refuse_before_any_device_work(L):
    buf = np.zeros(256, np.float32)
    ok = buf.ctypes.data
    s3, s2 = _strides(1, 1, 1), _strides(1, 1)
    hd = (ok, s3) * 3

    def fwd(n_seq=1, n_tokens=0, max_len=4, heads=1, dim=4, dtype=0, ld=ok, o=ok, ws=(None, 0), s0=None, s1=None, t=hd, starts=None):
        return (*t, starts, n_seq, n_tokens, max_len, heads, dim, dtype, ld, 1.0, s0, o, s1, *ws, None)

    def win(n_seq=1, n_tokens=0, max_len=4, heads=2, kv=1, dim=4, dtype=0, window=3, sinks=0, scale=1.0, o=ok):
        return (*hd, None, n_seq, n_tokens, max_len, heads, kv, dim, dtype, window, sinks, scale, o, None, None)

    def step(batch=1, heads=2, kv=1, dim=4, dtype=0, window=3, sinks=0, scale=1.0, pos=ok, ws=(None, 0)):
        return (ok, s2, ok, s2, ok, s2, ok, s3, ok, s3, pos, batch, heads, kv, dim, dtype, window, sinks, scale, ok, *ws, None)

    cases = [
        ('vad_layer_norm_forward', (ok, 1, 4, 4, None, None, 2, 0, 1e-5, ok, None, None), b'dtype'),
        ('vad_layer_norm_forward', (ok, 1, 4, 4, None, None, 0, 1, 1e-5, ok, None, None), b'weight_dtype'),
        ('vad_layer_norm_forward', (ok, 1, 0, 4, None, None, 0, 0, 1e-5, ok, None, None), b'out of range'),
        ('vad_layer_norm_forward', (ok, -1, 4, 4, None, None, 0, 0, 1e-5, ok, None, None), b'out of range'),
        ('vad_layer_norm_forward', (ok, 1, 4, 4, None, None, 0, 0, math.nan, ok, None, None), b'eps'),
        ('vad_layer_norm_forward', (None, 1, 4, 4, None, None, 0, 0, 1e-5, ok, None, None), b'null pointer'),
        ('vad_layer_norm_backward', (ok, ok, 1, 4, 4, 4, None, 0, 0, 1e-5, ok, ok, ok, ok, ok, 8, None), b'too small'),
        ('vad_layer_norm_backward', (ok, ok, 1, 4, 4, 4, None, 0, 0, 1e-5, None, ok, ok, ok, ok, 32, None), b'null pointer'),
        ('vad_layer_norm_backward', (ok, ok, 1, 4, 4, 4, None, 0, 0, 1e-5, ok, ok, ok, ok, None, 32, None), b'workspace'),
        ('vad_layer_norm_backward', (ok, ok, 1, 4, 4, 4, None, 0, 0, -1.0, ok, ok, ok, ok, ok, 32, None), b'eps'),
        ('vad_linear_attention_forward', fwd(dtype=5), b'dtype'),
        ('vad_linear_attention_forward', fwd(dim=129), b'head dimension'),
        ('vad_linear_attention_forward', fwd(dim=0), b'head dimension'),
        ('vad_linear_attention_forward', fwd(heads=0), b'heads'),
        ('vad_linear_attention_forward', fwd(max_len=-1), b'negative'),
        ('vad_linear_attention_forward', fwd(n_seq=1 << 40), b'too many'),
        ('vad_linear_attention_forward', fwd(ld=None), b'null pointer'),
        ('vad_linear_attention_forward', fwd(o=None), b'null pointer'),
        ('vad_linear_attention_forward', fwd(s0=ok, s1=ok), b'state_out'),
        ('vad_linear_attention_forward', fwd(max_len=10000), b'too small'),
        ('vad_linear_attention_backward', (*hd, ok, s3, None, 1, 0, 4, 1, 4, 0, ok, 1.0, None, ok, ok, ok, ok, ok, None, 0, None), b'dstate_in'),
        ('vad_linear_attention_backward', (*hd, ok, None, None, 1, 0, 4, 1, 4, 0, ok, 1.0, None, None, ok, ok, ok, None, None, 0, None), b'null pointer'),
        ('vad_linear_attention_step', (ok, s2, ok, s2, ok, s2, 1, 1, 200, 0, ok, 1.0, ok, ok, None), b'head dimension'),
        ('vad_linear_attention_step', (ok, s2, ok, s2, ok, s2, 1, 1, 4, 0, ok, 1.0, None, ok, None), b'null pointer'),
        ('vad_window_attention_forward', win(heads=3, kv=2), b'cannot share'),
        ('vad_window_attention_forward', win(window=0), b'window'),
        ('vad_window_attention_forward', win(sinks=65), b'sinks'),
        ('vad_window_attention_forward', win(scale=0.0), b'scale'),
        ('vad_window_attention_forward', win(n_seq=70000), b'sequence count'),
        ('vad_window_attention_forward', win(max_len=1 << 31), b'length'),
        ('vad_window_attention_forward', win(o=None), b'null pointer'),
        ('vad_window_attention_backward', (*hd, ok, ok, s3, ok, None, 1, 0, 4, 2, 1, 4, 0, 3, 0, 1.0, ok, ok, ok, ok, 8, None), b'too small'),
        ('vad_window_attention_forward', win(n_seq=60000, heads=60000, kv=60000), b'too many'),
        ('vad_linear_attention_forward', fwd(t=(ok, s3, ok, _strides(1, 1 << 22, 1), ok, s3)), b'row stride'),
        ('vad_linear_attention_forward', fwd(heads=1 << 20, dim=8), b'rows of'),
        ('vad_linear_attention_forward', fwd(max_len=1 << 31), b'length'),
        ('vad_linear_attention_step', (ok, s2, ok, s2, ok, s2, 1 << 21, 2, 4, 0, ok, 1.0, ok, ok, None), b'too many'),
        ('vad_window_attention_step', step(dtype=-1), b'dtype'),
        ('vad_window_attention_step', step(pos=None), b'null pointer'),
        ('vad_window_attention_step', step(window=100000), b'too small'),
        ('vad_window_cache_fill', (ok, s3, ok, s3, None, 1, 0, 4, 1, 4, 0, 3, 0, None, s3, ok, s3, None, None), b'null pointer'),
    ]
    for name, args, needle in cases:
        rc = getattr(L, name)(*args)
        assert rc == -1, (name, args, rc)
        assert needle in L.vad_last_error(), (name, L.vad_last_error())
    # nothing to do is no error
    assert L.vad_layer_norm_forward(None, 0, 4, 4, None, None, 0, 0, 1e-5, None, None, None) == 0
    assert L.vad_linear_attention_forward(*fwd(n_seq=0)) == 0 and L.vad_window_attention_forward(*win(n_seq=0)) == 0
    assert L.vad_window_attention_step(*step(batch=0)) == 0


def test_cpu_tensors_are_refused():
    q = torch.zeros(1, 4, 2, 8)
    for call in (lambda: pkg.layer_norm(q), lambda: pkg.linear_attention(q, q, q, torch.zeros(2)), lambda: pkg.window_attention(q, q, q, 3),
                 lambda: pkg.linear_attention_step(q[0], q[0], q[0], torch.zeros(2), torch.zeros(4, 2, 8, 8)),
                 lambda: pkg.window_attention_step(q[0], q[0], q[0], q, q, torch.zeros(4, dtype=torch.int64), 3),
                 lambda: pkg.window_cache_fill(q, q, q, q, 3), lambda: pkg.layer_norm([1.0])):
        with pytest.raises(ValueError, match='CUDA tensor'):
            call()


def test_plain_linear_attention_is_the_recurrence():
    torch.manual_seed(0)
    n, d, a, scale = 37, 6, -0.2, 0.7
    q, k, v, do = (torch.randn(n, d, dtype=torch.float64, requires_grad=True) for _ in range(4))
    s0 = torch.randn(d, d, dtype=torch.float64, requires_grad=True)
    ds = torch.randn(d, d, dtype=torch.float64)
    s, out = s0, []
    for t in range(n):
        s = math.exp(a) * s + torch.outer(k[t], v[t])
        out.append(scale * q[t] @ s)
    grads = torch.autograd.grad((torch.stack(out), s), (q, k, v, s0), (do.detach(), ds))
    r = ref.decay_sequence(*(x.detach() for x in (q, k, v)), a, scale, s0.detach(), do.detach(), ds)
    for got, want in zip((r['o'], r['state'], r['dq'], r['dk'], r['dv'], r['dstate']), (torch.stack(out), s, *grads)):
        assert torch.allclose(got, want.detach(), rtol=1e-12, atol=1e-12)


def test_plain_window_attention_and_its_cache():
    torch.manual_seed(1)
    n, d, window, sinks = 40, 5, 7, 3
    q, k, v = (torch.randn(n, d, dtype=torch.float64, requires_grad=True) for _ in range(3))
    do = torch.randn(n, d, dtype=torch.float64)
    rows = []
    for i in range(n):
        sees = [j for j in range(i + 1) if i - j < window or j < sinks]
        # the slots that the rolling cache holds behind row i are exactly those rows
        slots = {}
        for j in range(i + 1):
            slots[ref.window_slot(j, window, sinks)] = j
        assert sorted(slots.values()) == sees and set(slots) == set(range(min(i + 1, sinks + window)))
        w = torch.softmax(0.4 * k[sees] @ q[i], 0)
        rows.append(w @ v[sees])
    o = torch.stack(rows)
    grads = torch.autograd.grad(o, (q, k, v), do)
    r = ref.window_sequence(*(x.detach() for x in (q, k, v)), window, sinks, 0.4, do)
    for got, want in zip((r['o'], r['dq'], r['dk'], r['dv']), (o, *grads)):
        assert torch.allclose(got, want.detach(), rtol=1e-11, atol=1e-12)


def test_plain_layer_norm():
    torch.manual_seed(2)
    x, w, b = torch.randn(5, 9, dtype=torch.float64), torch.randn(9, dtype=torch.float64), torch.randn(9, dtype=torch.float64)
    dy = torch.randn(5, 9, dtype=torch.float64)
    leaf = [t.clone().requires_grad_() for t in (x, w, b)]
    y = torch.nn.functional.layer_norm(leaf[0], (9,), leaf[1], leaf[2], 1e-5)
    for got, want in zip(ref.layer_norm(x, w, b, 1e-5, dy), (y, *torch.autograd.grad(y, leaf, dy))):
        assert torch.allclose(got, want.detach(), rtol=1e-11, atol=1e-12)


def test_forward_mode_derivatives_are_refused():
    """A dual tensor does not ask for a gradient, and a result without its tangent would read as a derivative of zero."""
    q = torch.zeros(1, 4, 2, 8)
    row, ld, state, cache = q[0], torch.zeros(2), torch.zeros(4, 2, 8, 8), torch.zeros(4, 4, 2, 8)
    pos, w = torch.zeros(4, dtype=torch.int64), torch.ones(8)
    calls = [(pkg.layer_norm, [q, w, w]), (pkg.linear_attention, [q, q, q, ld]), (pkg.linear_attention_step, [row, row, row, ld, state]),
             (lambda a, b, c: pkg.window_attention(a, b, c, 3), [q, q, q]), (lambda *t: pkg.linear_attention(q, q, q, ld, state=t[0]), [state]),
             (lambda a, b, c, d, e: pkg.window_attention_step(a, b, c, d, e, pos, 4), [row, row, row, cache, cache]),
             (lambda a, b, c, d: pkg.window_cache_fill(a, b, c, d, 4), [q, q, cache, cache])]
    with forward_ad.dual_level():
        for call, args in calls:
            for i, t in enumerate(args):
                with pytest.raises(ValueError, match='forward-mode'):
                    call(*args[:i], forward_ad.make_dual(t, torch.ones_like(t)), *args[i + 1:])
            with pytest.raises(ValueError, match='CUDA tensor'):        # others are as welcome as outside
                call(*args)


def test_scales_past_float32_are_refused(L):
    """A scale that a double holds and a float32 does not would come out as infinity."""
    buf = np.zeros(256, np.float32)
    ok = buf.ctypes.data
    s3, s2 = _strides(1, 1, 1), _strides(1, 1)
    hd = (ok, s3) * 3
    for scale in (1e39, -1e39, math.inf, math.nan):
        for name, args in (('vad_linear_attention_forward', (*hd, None, 1, 0, 4, 1, 4, 0, ok, scale, None, ok, None, None, 0, None)),
                           ('vad_linear_attention_backward', (*hd, ok, s3, None, 1, 0, 4, 1, 4, 0, ok, scale, None, None, ok, ok, ok, None, None, 0, None)),
                           ('vad_linear_attention_step', (ok, s2, ok, s2, ok, s2, 1, 1, 4, 0, ok, scale, ok, ok, None))):
            assert getattr(L, name)(*args) == -1 and b'scale' in L.vad_last_error(), (name, scale)
